"""
GPU parity tests of rotary positions against the float64 oracle, whose error bounds are the tolerances.
"""

import ctypes

import pytest
import torch

import attorch_amd
from oracle.attention import rotary
from .helpers import DTYPES, randn
from .test_gpu_attention import assert_within

pytestmark = pytest.mark.gpu


def tables(sections, base=10000.0):
    pairs = sum(sections)
    inv_freq = base ** (torch.arange(pairs, dtype=torch.float64) / -max(pairs, 1))
    return inv_freq, torch.cat([torch.full((n,), axis, dtype=torch.int32) for axis, n in enumerate(sections)])


def positions_of(shape, seed, high=5000, dtype=torch.int64):
    return torch.randint(-high // 10, high, shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def check(q, k, positions, inv_freq, pair_axis, adjacent):
    expected = [rotary(t, positions, inv_freq, pair_axis, adjacent) for t in (q, k)]
    qd, kd = q.cuda().requires_grad_(), k.cuda().requires_grad_()
    outs = attorch_amd.RotaryAutoGrad.apply(qd, kd, positions.cuda(), inv_freq.cuda(), pair_axis.cuda(), adjacent)
    grads = [randn(t.shape, 7 + n, t.dtype) for n, t in enumerate((q, k))]
    got = torch.autograd.grad(outs, (qd, kd), [g.cuda() for g in grads])
    for n, name in enumerate(('query', 'key')):
        assert outs[n].dtype is q.dtype and got[n].dtype is q.dtype
        assert_within(outs[n], expected[n], name)
        assert_within(got[n], rotary(grads[n], positions, inv_freq, pair_axis, adjacent, inverse=True), f'{name} gradient')
    return outs


# sizes with whole vectors and without, all features turned or some
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('adjacent', [False, True])
@pytest.mark.parametrize('dim, sections', [(64, (32,)), (128, (16, 24, 24)), (128, (32,)), (80, (20, 20)), (24, (3, 2)),
                                           (17, (1, 2, 3)), (2, (1,)), (96, (48,)), (40, (0, 4)), (8, ())])
def test_sizes(dim, sections, adjacent, dtype) -> None:
    sections = sections or (0,)
    axes = len(sections)
    inv_freq, pair_axis = tables(sections)
    q, k = randn((3, 5, 7, dim), 1, dtype), randn((3, 2, 7, dim), 2, dtype)
    check(q, k, positions_of((axes, 3, 7), 3), inv_freq, pair_axis, adjacent)


# numbers of pairs and of features behind them that no vector divides; more places than a workgroup has lanes
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('adjacent', [False, True])
@pytest.mark.parametrize('dim, pairs', [(80, 5), (80, 37), (72, 27), (24, 7), (31, 11), (3, 1), (1, 0), (127, 1), (129, 63),
                                        (2100, 512), (2100, 3), (4099, 0)])
def test_uneven_sizes(dim, pairs, adjacent, dtype) -> None:
    inv_freq, pair_axis = tables((pairs,))
    q, k = randn((2, 3, 5, dim), 1, dtype), randn((2, 2, 5, dim), 2, dtype)
    check(q, k, positions_of((1, 2, 5), 3), inv_freq, pair_axis, adjacent)


# at the C entry an output may be the input itself
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('adjacent', [False, True])
@pytest.mark.parametrize('dim, pairs', [(80, 5), (80, 37), (72, 27), (31, 11), (3, 1), (127, 1), (128, 64), (2100, 509)])
def test_in_place(dim, pairs, adjacent, dtype) -> None:
    inv_freq = tables((pairs,))[0].cuda()
    q, k = (randn((9, heads, 70, dim), heads, dtype).cuda() for heads in (3, 2))
    expected = attorch_amd.RotaryAutoGrad.apply(q, k, None, inv_freq, None, adjacent)
    layouts = [attorch_amd.rotary._layout(t) for t in (q, k)]
    shape = attorch_amd.rotary._plan(*layouts, None, attorch_amd.rotary._layout(inv_freq), None, adjacent, False)
    stream = attorch_amd._lib.stream_of(q)
    assert attorch_amd._lib.load().at_rotary(ctypes.byref(shape), q.data_ptr(), k.data_ptr(), q.data_ptr(), k.data_ptr(),
                                             None, inv_freq.data_ptr(), None, stream) == 0
    assert torch.equal(q, expected[0]) and torch.equal(k, expected[1])


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('batch, rows', [(1, 1), (64, 1), (1, 1000), (2, 333), (5, 3)])
def test_token_counts(batch, rows, dtype) -> None:
    inv_freq, pair_axis = tables((16,))
    q, k = randn((batch, 4, rows, 32), 1, dtype), randn((batch, 1, rows, 32), 2, dtype)
    check(q, k, positions_of((1, batch, rows), 3), inv_freq, pair_axis, False)


@pytest.mark.parametrize('position_type', [torch.int32, torch.int64, torch.float32])
def test_far_positions(position_type) -> None:
    """Angles of far tokens keep their precision; positions of float32 may be fractions."""
    inv_freq, pair_axis = tables((32, 32))
    q, k = randn((2, 2, 50, 128), 1), randn((2, 2, 50, 128), 2)
    positions = positions_of((2, 2, 50), 3, 1 << 24, position_type)
    if position_type is torch.float32:
        positions = positions / 4
    check(q, k, positions, inv_freq, pair_axis, False)


def test_layouts_and_absent_keys() -> None:
    inv_freq, pair_axis = (t.cuda() for t in tables((8, 8)))
    q, k = randn((2, 3, 9, 40), 1, torch.bfloat16).cuda(), randn((2, 1, 9, 40), 2, torch.bfloat16).cuda()
    positions = positions_of((2, 2, 9), 3).cuda()
    expected = attorch_amd.RotaryAutoGrad.apply(q, k, positions, inv_freq, pair_axis)
    packed = torch.cat([t.transpose(1, 2).flatten(2) for t in (q, k)], -1)
    views = [t.unflatten(2, (-1, 40)).transpose(1, 2) for t in packed.split([120, 40], -1)]
    odd = [torch.nn.functional.pad(t, (1, 2))[..., 1:-2] for t in (q, k)]
    apart = [torch.stack([t, t], -1)[..., 0] for t in (q, k)]
    dim_first = [t.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0) for t in (q, k)]
    for variant in (views, odd, apart, dim_first):
        for got, want in zip(attorch_amd.RotaryAutoGrad.apply(*variant, positions, inv_freq, pair_axis), expected):
            assert torch.equal(got, want)
    alone, none = attorch_amd.RotaryAutoGrad.apply(q, None, positions, inv_freq, pair_axis)
    assert none is None and torch.equal(alone, expected[0])
    # an expanded input and gradient
    wide = k.expand(2, 3, 9, 40).detach().requires_grad_()
    out, _ = attorch_amd.RotaryAutoGrad.apply(wide, None, positions, inv_freq, pair_axis)
    assert torch.equal(out, expected[1].expand(2, 3, 9, 40))
    (grad,) = torch.autograd.grad(out.sum(), wide)
    (same,) = torch.autograd.grad(attorch_amd.RotaryAutoGrad.apply(wide, None, positions, inv_freq, pair_axis)[0], wide,
                                  torch.ones_like(out))
    assert torch.equal(grad, same)


def test_module() -> None:
    """Tables, shapes of the positions, and dtype changes of the module."""
    q, k = randn((2, 3, 6, 32), 1).cuda(), randn((2, 1, 6, 32), 2).cuda()
    layer = attorch_amd.Rotary(32).to(torch.bfloat16)
    assert layer.inv_freq.dtype is torch.float64 and not layer.state_dict()
    running = layer(q, k)
    for positions in (torch.arange(6), torch.arange(6).expand(2, 6), torch.arange(6).expand(1, 2, 6),
                      torch.arange(6, dtype=torch.int32), torch.arange(6).float()):
        for got, want in zip(layer(q, k, positions.cuda()), running):
            assert torch.equal(got, want)
    inv_freq, pair_axis = tables((16,))
    assert_within(running[0], rotary(q.cpu(), torch.arange(6).expand(1, 2, 6), inv_freq, pair_axis), 'one axis')

    layer = attorch_amd.Rotary(32, sections=(4, 6, 2), axis_ladders=True, adjacent=True, base=100.0)
    positions = positions_of((3, 2, 6), 3, 50)
    inv_freq = torch.cat([100.0 ** (torch.arange(n, dtype=torch.float64) / -n) for n in (4, 6, 2)])
    _, pair_axis = tables((4, 6, 2))
    out, key = layer(q, k, positions.cuda())
    assert_within(out, rotary(q.cpu(), positions, inv_freq, pair_axis, True), 'three axes')
    assert_within(key, rotary(k.cpu(), positions, inv_freq, pair_axis, True), 'three axes, key')
    shared = layer(q, None, positions[:, 0].cuda())[0]
    assert torch.equal(shared, layer(q, None, positions[:, :1].expand(3, 2, 6).cuda())[0])


def test_partial_gradients_and_empty_calls() -> None:
    inv_freq, _ = (t.cuda() for t in tables((8,)))
    q, k = (randn((2, 3, 5, 16), n).cuda().requires_grad_() for n in (1, 2))
    outs = attorch_amd.RotaryAutoGrad.apply(q, k, None, inv_freq)
    both = torch.autograd.grad(outs, (q, k), [torch.ones_like(q), torch.ones_like(k)])
    outs = attorch_amd.RotaryAutoGrad.apply(q, k, None, inv_freq)
    (grad,) = torch.autograd.grad(outs[1].sum(), k)
    assert torch.equal(grad, both[1])
    outs = attorch_amd.RotaryAutoGrad.apply(q, k.detach(), None, inv_freq)
    (grad,) = torch.autograd.grad(outs[0].sum(), q)
    assert torch.equal(grad, both[0])
    for shape in ((0, 3, 5, 16), (2, 0, 5, 16), (2, 3, 0, 16)):
        empty = torch.empty(shape, device='cuda', requires_grad=True)
        out, _ = attorch_amd.RotaryAutoGrad.apply(empty, None, None, inv_freq)
        assert out.shape == shape and torch.autograd.grad(out.sum(), empty)[0].shape == shape


def test_stream_and_graph() -> None:
    inv_freq, pair_axis = (t.cuda() for t in tables((8, 8)))
    q, k = (randn((2, 3, 50, 32), n, torch.float16).cuda().requires_grad_() for n in (1, 2))
    positions = positions_of((2, 2, 50), 3).cuda()

    def step():
        outs = attorch_amd.RotaryAutoGrad.apply(q, k, positions, inv_freq, pair_axis)
        return [*outs, *torch.autograd.grad(outs, (q, k), [torch.ones_like(q), torch.ones_like(k)])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = [step(), step()][1]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(on_side, step()):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(3):
        positions.copy_(positions_of((2, 2, 50), seed))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()
