"""
GPU parity tests of attention over a sliding window with visible first tokens against the float64
oracle, whose error bounds (oracle/attention.py) are the tolerances.
"""

import pytest
import torch

import attorch_amd
from oracle.attention import attention
from .helpers import DTYPES, randn

pytestmark = pytest.mark.gpu


def heads_last(shape, seed, dtype, scale=1.0):
    """[batch, heads, tokens, dim] seen through a [batch, tokens, heads, dim] tensor."""
    batch, heads, tokens, dim = shape
    return randn((batch, tokens, heads, dim), seed, dtype, scale).transpose(1, 2)


def assert_within(actual, expected, what) -> None:
    value, bound = expected
    actual = actual.detach().double().cpu()
    assert actual.shape == value.shape, f'{what}: shape {tuple(actual.shape)} != {tuple(value.shape)}'
    excess = (actual - value).abs() - bound
    assert not torch.isnan(actual).any(), f'{what}: NaN'
    worst = excess.argmax() if excess.numel() else 0
    assert not excess.numel() or excess.max() <= 0, \
        f'{what}: {actual.reshape(-1)[worst]} is off {value.reshape(-1)[worst]} by more than {bound.reshape(-1)[worst]}'


def check(q, k, v, dout=None, lengths=None, query_lengths=None, causal=True, window=None, sinks=0, scale=None):
    """Forward, and backward where dout is given, on the GPU and in the oracle."""
    expected = attention(q, k, v, dout, lengths, query_lengths, causal, window, sinks, scale)
    qd, kd, vd = (t.cuda().requires_grad_(dout is not None) for t in (q, k, v))
    out = attorch_amd.WindowAttentionAutoGrad.apply(
        qd, kd, vd, None if lengths is None else lengths.cuda(), None if query_lengths is None else query_lengths.cuda(),
        causal, window, sinks, scale)
    assert out.dtype is q.dtype
    assert_within(out, expected['out'], 'output')
    if dout is not None:
        grads = torch.autograd.grad(out, (qd, kd, vd), dout.cuda())
        for grad, name in zip(grads, ('dq', 'dk', 'dv')):
            assert grad.dtype is q.dtype
            assert_within(grad, expected[name], name)
    return out


def inputs(batch, heads, kv_heads, rows, keys, dim, dtype, seed=0):
    return (heads_last((batch, heads, rows, dim), seed + 1, dtype), heads_last((batch, kv_heads, keys, dim), seed + 2, dtype),
            heads_last((batch, kv_heads, keys, dim), seed + 3, dtype), heads_last((batch, heads, rows, dim), seed + 4, dtype))


# lengths around the tiles of 32, 64 and 128 tokens, and from one token on
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('tokens', [1, 2, 31, 32, 33, 64, 65, 127, 128, 129, 200, 257])
def test_lengths(tokens, dtype) -> None:
    check(*inputs(2, 2, 1, tokens, tokens, 64, dtype))


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [1, 7, 8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 120, 128])
def test_head_dims(dim, dtype) -> None:
    check(*inputs(1, 4, 2, 150, 150, dim, dtype), window=70, sinks=3)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('heads, kv_heads', [(1, 1), (3, 3), (6, 2), (5, 1), (8, 1), (7, 7)])
def test_shared_heads(heads, kv_heads, dtype) -> None:
    check(*inputs(2, heads, kv_heads, 90, 90, 32, dtype), window=50, sinks=2)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('window, sinks', [(None, 0), (None, 5), (1, 0), (1, 1), (2, 64), (16, 4), (63, 0), (64, 1),
                                           (65, 130), (128, 7), (1000, 0), (1 << 60, 1 << 60)])
def test_windows(window, sinks, causal, dtype) -> None:
    check(*inputs(1, 2, 1, 300, 300, 64, dtype), causal=causal, window=window, sinks=sinks)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('heads, kv_heads, window, sinks', [(3, 1, 100, 0), (5, 1, 37, 3), (4, 4, 65, 0), (24, 3, 129, 1)])
def test_windows_over_many_tiles(heads, kv_heads, window, sinks, causal, dtype) -> None:
    """Tiles of keys whose rows are several windows away from the first one, in whole and padded batches."""
    check(*inputs(2, heads, kv_heads, 1100, 1100, 24, dtype), lengths=torch.tensor([1100, 777]), causal=causal, window=window,
          sinks=sinks)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('window, sinks', [(20, 1), (20, 33), (20, 64), (33, 65), (20, 129), (100, 140), (20, 300), (1, 700)])
def test_sinks_far_from_their_readers(window, sinks, causal, dtype) -> None:
    """
    Rows that see the sinks of a tile of keys and nothing else of it, in whole batches, padded ones and
    chunks over a cache.
    """
    check(*inputs(1, 4, 2, 700, 700, 32, dtype), causal=causal, window=window, sinks=sinks)
    check(*inputs(2, 3, 1, 650, 650, 16, dtype), lengths=torch.tensor([333, 650]), causal=causal, window=window, sinks=sinks)
    check(*inputs(1, 2, 2, 200, 900, 32, dtype), causal=causal, window=window, sinks=sinks)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('int_type', [torch.int32, torch.int64])
def test_ragged_batch(int_type, causal, dtype) -> None:
    lengths = torch.tensor([0, 1, 130, 77, 128, 64, -3, 999], dtype=int_type)
    check(*inputs(8, 4, 2, 130, 130, 40, dtype), lengths=lengths, causal=causal, window=40, sinks=3)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('causal', [True, False])
def test_padded_rows_beside_whole_tiles(causal, dtype) -> None:
    """Rows behind a sequence that share a wave with rows that see every key of a tile."""
    check(*inputs(3, 3, 1, 400, 400, 32, dtype), lengths=torch.tensor([301, 111, 397]), causal=causal)
    check(*inputs(3, 2, 2, 400, 400, 32, dtype), lengths=torch.tensor([301, 111, 397]), causal=causal, window=150, sinks=2)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('causal', [True, False])
def test_query_lengths(causal, dtype) -> None:
    lengths = torch.tensor([200, 5, 90, 0, 33, 200])
    query_lengths = torch.tensor([70, 70, 11, 8, 0, 500])
    check(*inputs(6, 4, 2, 70, 200, 64, dtype), lengths=lengths, query_lengths=query_lengths, causal=causal, window=50,
          sinks=2)
    check(*inputs(6, 4, 2, 70, 200, 64, dtype), query_lengths=query_lengths.int(), lengths=lengths, causal=causal)
    check(*inputs(6, 4, 2, 70, 200, 64, dtype), query_lengths=query_lengths, causal=causal, window=50)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows', [1, 2, 5, 17, 64, 100])
@pytest.mark.parametrize('heads, kv_heads', [(8, 2), (4, 4), (6, 1)])
def test_new_tokens_over_a_cache(heads, kv_heads, rows, dtype) -> None:
    """Single tokens and chunks; few rows and many keys are worked on in pieces that are joined."""
    q, k, v, dout = inputs(2, heads, kv_heads, rows, 1111, 64, dtype)
    lengths = torch.tensor([1111, 403])
    check(q, k, v, dout, lengths=lengths)
    check(q, k, v, dout, lengths=lengths, window=130, sinks=4)
    check(q, k, v, lengths=lengths)
    check(q, k, v, window=300, sinks=70)
    check(q, k, v, causal=False)


def test_scale_and_large_scores() -> None:
    for dtype in DTYPES:
        q, k, v, dout = inputs(1, 2, 2, 100, 100, 64, dtype)
        check(q, k, v, dout, scale=1.0)
        check((q.float() * 8).to(dtype), k, v, dout, scale=0.9)
        check(q, k, v, dout, scale=1e-3)
        # scores so negative or positive that exponentials without the maximum would vanish or overflow
        check(q, k + 10, v, dout, scale=2.0)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('garbage', [float('nan'), float('inf'), -float('inf'), 'lowest'])
def test_unseen_places_may_hold_anything(garbage, dtype) -> None:
    """
    Room behind the sequences, tokens that fell out of the window, padded query rows and their output
    gradients.
    """
    garbage = torch.finfo(dtype).min if garbage == 'lowest' else garbage
    q, k, v, dout = inputs(3, 4, 2, 90, 300, 64, dtype)
    lengths, query_lengths = torch.tensor([300, 150, 0]), torch.tensor([90, 20, 1])
    for t in (k, v):
        t[1, :, 150:] = garbage
        t[2] = garbage
        t[0, :, 4:300 - 90 - 29] = garbage     # between the sinks and the first row's window of 30
        t[1, :, 4:150 - 20 - 29] = garbage
    for t in (q, dout):
        t[1, :, 20:] = garbage
        t[2] = garbage
    check(q, k, v, dout, lengths=lengths, query_lengths=query_lengths, window=30, sinks=4)
    one = q[:, :, :1].clone()
    for t in (k, v):
        t[0, :, 4:300 - 30] = garbage
        t[1, :, 4:150 - 30] = garbage
    check(one, k, v, None, lengths=lengths, window=30, sinks=4)


@pytest.mark.parametrize('dtype', DTYPES)
def test_layouts(dtype) -> None:
    """Packed projections, head-major caches, expanded and misaligned tensors give the same results."""
    q, k, v, dout = inputs(2, 4, 2, 70, 70, 32, dtype)
    base = check(q, k, v, dout, window=20)

    def run(qd, kd, vd, dd):
        qd, kd, vd = (t.detach().requires_grad_() for t in (qd, kd, vd))
        out = attorch_amd.WindowAttention(window=20)(qd, kd, vd)
        return (out, *torch.autograd.grad(out, (qd, kd, vd), dd))

    expected = run(*(t.cuda() for t in (q, k, v, dout)))
    assert torch.equal(expected[0], base)
    packed = torch.cat([t.transpose(1, 2).flatten(2) for t in (q, k, v)], -1).cuda()
    views = [t.unflatten(2, (-1, 32)).transpose(1, 2) for t in packed.split([128, 64, 64], -1)]
    head_major = [t.contiguous().cuda() for t in (q, k, v)]
    odd = [torch.nn.functional.pad(t, (1, 2)).cuda()[..., 1:-2] for t in (q, k, v)]
    apart = [torch.stack([t, t], -1).cuda()[..., 0] for t in (q, k, v)]
    for variant in (views, head_major, odd, apart):
        for got, want in zip(run(*variant, dout.cuda()), expected):
            assert torch.equal(got, want)
    # an output gradient that is expanded, as sum() makes it
    ones = torch.ones((), dtype=dtype, device='cuda').expand(2, 4, 70, 32)
    for got, want in zip(run(*head_major, ones), run(*head_major, ones.contiguous())):
        assert torch.equal(got, want)
    # keys and values shared by the batch: their gradients are the sums over it
    kd, vd = (t[:1].cuda().requires_grad_() for t in (k, v))
    out = attorch_amd.WindowAttention(window=20)(q.cuda(), kd.expand(2, -1, -1, -1), vd.expand(2, -1, -1, -1))
    out.backward(dout.cuda())
    same = attention(q, k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1), dout, window=20)
    for grad, name in ((kd.grad, 'dk'), (vd.grad, 'dv')):
        value, bound = same[name]
        step = torch.finfo(dtype).eps / 2
        assert_within(grad, (value.sum(0, True), bound.sum(0, True) + step * value.sum(0, True).abs()), name)


def test_results_do_not_change_from_run_to_run() -> None:
    q, k, v, dout = (t.cuda() for t in inputs(2, 8, 2, 500, 500, 128, torch.bfloat16))
    first = None
    for _ in range(3):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = attorch_amd.WindowAttention(window=100, num_sinks=4)(*leaves)
        got = (out, *torch.autograd.grad(out, leaves, dout))
        first = got if first is None else first
        for a, b in zip(got, first):
            assert torch.equal(a, b)


def test_empty_calls() -> None:
    for batch, rows, keys in ((0, 4, 4), (2, 0, 5), (2, 0, 0)):
        q, k, v, _ = (t.cuda().requires_grad_() for t in inputs(batch, 4, 2, rows, keys, 16, torch.float32))
        out = attorch_amd.WindowAttention()(q, k, v)
        assert out.shape == q.shape
        grads = torch.autograd.grad(out, (q, k, v), torch.ones_like(out))
        for grad, leaf in zip(grads, (q, k, v)):
            assert grad.shape == leaf.shape and not grad.any()


@pytest.mark.parametrize('causal', [True, False])
def test_empty_batches_with_sinks_beyond_the_window(causal) -> None:
    q, k, v, dout = (t.cuda().requires_grad_() for t in inputs(0, 4, 2, 700, 700, 32, torch.bfloat16))
    out = attorch_amd.WindowAttention(causal=causal, window=20, num_sinks=4)(q, k, v)
    for grad, leaf in zip(torch.autograd.grad(out, (q, k, v), dout), (q, k, v)):
        assert grad.shape == leaf.shape


def test_autocast() -> None:
    q, k, v, dout = (t.cuda() for t in inputs(2, 4, 2, 60, 60, 64, torch.float32))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    with torch.autocast('cuda', dtype=torch.bfloat16):
        out = attorch_amd.WindowAttention(window=30)(*leaves)
    assert out.dtype is torch.bfloat16
    grads = torch.autograd.grad(out, leaves, dout.bfloat16())
    plain = [t.detach().bfloat16().requires_grad_() for t in leaves]
    same = attorch_amd.WindowAttention(window=30)(*plain)
    assert torch.equal(out, same)
    for grad, other in zip(grads, torch.autograd.grad(same, plain, dout.bfloat16())):
        assert grad.dtype is torch.float32 and torch.equal(grad, other.float())


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
@pytest.mark.parametrize('others', [(torch.float32, torch.float32), (torch.bfloat16, torch.float16),
                                    (torch.float16, torch.float32)])
def test_autocast_of_inputs_of_different_types(others, dtype) -> None:
    """Queries of a projection beside a cache in the weights' type: all are cast, and gradients cast back."""
    q, k, v, dout = (t.cuda() for t in inputs(2, 4, 2, 60, 60, 64, torch.float32))
    leaves = [t.to(d).requires_grad_() for t, d in zip((q, k, v), (dtype, *others))]
    with torch.autocast('cuda', dtype=dtype):
        out = attorch_amd.WindowAttention(window=30)(*leaves)
    assert out.dtype is dtype
    plain = [t.detach().to(dtype).requires_grad_() for t in leaves]
    same = attorch_amd.WindowAttention(window=30)(*plain)
    assert torch.equal(out, same)
    expected = torch.autograd.grad(same, plain, dout.to(dtype))
    for grad, leaf, other in zip(torch.autograd.grad(out, leaves, dout.to(dtype)), leaves, expected):
        assert grad.dtype is leaf.dtype and torch.equal(grad, other.to(leaf.dtype))


def laid_out_anew(tensor):
    """Equal values, contiguous and then in every second place."""
    return torch.stack([tensor, torch.zeros_like(tensor)], -1).contiguous()[..., 0]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [32, 20])
@pytest.mark.parametrize('hook', [
    lambda: torch.autograd.graph.save_on_cpu(), lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
    lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(memory_format=torch.contiguous_format),
                                                     lambda t: t),
    lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), laid_out_anew)])
def test_saved_tensors_in_another_layout(hook, dim, dtype) -> None:
    """Saved tensors that hooks return with other strides (as offloading them does) give the same gradients."""
    q, k, v, dout = inputs(2, 4, 2, 70, 70, dim, dtype)
    packed = torch.cat([t.transpose(1, 2).flatten(2) for t in (q, k, v)], -1).cuda()
    views = [t.unflatten(2, (-1, dim)).transpose(1, 2) for t in packed.split([4 * dim, 2 * dim, 2 * dim], -1)]
    lengths = torch.tensor([70, 33], device='cuda')
    layer = attorch_amd.WindowAttention(window=20, num_sinks=2)
    for variant in (views, [t.cuda() for t in (q, k, v)], [t.contiguous().cuda() for t in (q, k, v)]):
        leaves = [t.detach().requires_grad_() for t in variant]
        out = layer(*leaves, lengths)
        expected = torch.autograd.grad(out, leaves, dout.cuda())
        with hook():
            out = layer(*leaves, lengths)
        for got, want in zip(torch.autograd.grad(out, leaves, dout.cuda()), expected):
            assert torch.equal(got, want)


def test_frozen_inputs_and_no_grad() -> None:
    q, k, v, dout = (t.cuda() for t in inputs(1, 2, 2, 40, 40, 32, torch.float16))
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    full = torch.autograd.grad(attorch_amd.WindowAttention()(*leaves), leaves, dout)
    for n in range(3):
        some = [t.detach().requires_grad_(m == n) for m, t in enumerate((q, k, v))]
        (grad,) = torch.autograd.grad(attorch_amd.WindowAttention()(*some), some[n], dout)
        assert torch.equal(grad, full[n])
    with torch.no_grad():
        out = attorch_amd.WindowAttention()(*leaves)
    assert not out.requires_grad
    out = attorch_amd.WindowAttention()(*leaves)
    (grad,) = torch.autograd.grad(out, leaves[0], dout, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()          # no second derivatives


@pytest.mark.parametrize('dim', [32, 20])
def test_outputs_changed_in_place(dim) -> None:
    """Outputs are no views, so they may be changed in place where no backward pass needs them."""
    q, k, v, dout = (t.cuda() for t in inputs(1, 2, 2, 40, 40, dim, torch.float16))
    expected = attorch_amd.WindowAttention()(q, k, v)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attorch_amd.WindowAttention()(*leaves)
    assert torch.equal(out, expected) and out.stride() == expected.stride() and not out._is_view()
    out.mul_(2.0)
    assert torch.equal(out, 2.0 * expected)
    with torch.inference_mode():
        out = attorch_amd.WindowAttention()(*leaves)
        assert torch.equal(out.mul_(2.0), 2.0 * expected)
    if dim % 8:                        # a copy of what the backward pass needs
        out = attorch_amd.WindowAttention()(*leaves)
        got = torch.autograd.grad(out.mul_(2.0), leaves, dout)
        for a, b in zip(got, torch.autograd.grad(attorch_amd.WindowAttention()(*leaves), leaves, 2.0 * dout)):
            assert torch.equal(a, b)


def test_other_stream_and_graph() -> None:
    """A step on a side stream, then captured and replayed with eager work in between."""
    q, k, v, dout = (t.cuda() for t in inputs(2, 4, 2, 120, 120, 64, torch.bfloat16))
    one, cache_k, cache_v = (t.cuda() for t in inputs(2, 4, 2, 1, 3000, 64, torch.bfloat16, 9)[:3])
    lengths = torch.tensor([2000, 3000], device='cuda')
    leaves = [t.requires_grad_() for t in (q, k, v)]
    layer = attorch_amd.WindowAttention(window=50, num_sinks=4)

    def step():
        out = layer(*leaves)
        token = attorch_amd.WindowAttentionAutoGrad.apply(one, cache_k, cache_v, lengths)
        return [out, *torch.autograd.grad(out, leaves, dout), token]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(on_side, step()):
        assert torch.equal(a, b)
    graphs, outs = [], []
    for _ in range(2):                 # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for seed in range(3):
        with torch.no_grad():
            for n, t in enumerate((q, k, v, dout, one)):
                t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(10 * seed + n)))
            lengths.copy_(torch.tensor([100 + seed, 3000 - seed]))
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in out]
            for a, b in zip(got, step()):
                assert torch.equal(a, b)
            torch.cuda.synchronize()


def test_long_cache_offsets() -> None:
    """Keys beyond 4 GiB of one head's cache; a single row and a chunk see only the last ones and the sinks."""
    heads, tokens, dim = 2, (1 << 23) + 321, 128
    k = torch.zeros(1, heads, tokens, dim, dtype=torch.bfloat16, device='cuda')
    v = torch.zeros_like(k)
    assert k.stride(1) * 2 * 2 > 1 << 32
    tail_k, tail_v = randn((1, heads, 200, dim), 1, torch.bfloat16), randn((1, heads, 200, dim), 2, torch.bfloat16)
    k[:, :, -196:], v[:, :, -196:] = tail_k[:, :, 4:].cuda(), tail_v[:, :, 4:].cuda()
    k[:, :, :4], v[:, :, :4] = tail_k[:, :, :4].cuda(), tail_v[:, :, :4].cuda()
    for rows in (1, 40):
        q = randn((1, 4, rows, dim), 3, torch.bfloat16)
        out = attorch_amd.WindowAttention(window=100, num_sinks=4)(q.cuda(), k, v)
        assert_within(out, attention(q, tail_k, tail_v, window=100, sinks=4)['out'], f'{rows} rows')


# fp32 heads of more than 64 features, in workgroups of few keys: many rows, and many splits of single tokens
@pytest.mark.parametrize('batch, heads, kv_heads, rows, keys, dim, window, lengths', [
    (4, 32, 8, 1030, 1030, 72, 70, [1030, 0, 517, 1]), (4, 64, 64, 515, 515, 104, None, None),
    (64, 8, 8, 1, 1400, 128, None, list(range(1, 1400, 22))), (3, 4, 2, 5, 60000, 80, None, [60000, 33333, 7]),
    (2, 24, 8, 2, 20000, 120, 9000, None)])
def test_wide_heads_in_full_precision(batch, heads, kv_heads, rows, keys, dim, window, lengths) -> None:
    tensors = inputs(batch, heads, kv_heads, rows, keys, dim, torch.float32)
    check(*tensors, lengths=None if lengths is None else torch.tensor(lengths[:batch]), window=window, sinks=3)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('tokens, causal, window, lengths', [(1, True, None, None), (1, False, 3, None), (300, True, 1, None),
                                                             (300, False, 1, [300, 0, 77]), (70, False, None, [1, 0, 1])])
def test_single_keys(tokens, causal, window, lengths, dtype) -> None:
    """A token that sees one key has its value as output, whatever queries and keys are: their gradients are zeros."""
    batch = 3 if lengths else 2
    q, k, v, dout = (t.cuda() for t in inputs(batch, 6, 2, tokens, tokens, 40, dtype))
    counts = torch.tensor(lengths or [tokens] * batch, device='cuda')
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = attorch_amd.WindowAttention(causal=causal, window=window)(*leaves, counts)
    dq, dk, dv = torch.autograd.grad(out, leaves, dout)
    live = (torch.arange(tokens, device='cuda') < counts[:, None])[:, None, :, None]
    # the probability is within 2^-21 of 1, which is less than half a step of 16 bits and a few steps of 32
    same = v.detach().repeat_interleave(3, 1).float() * live
    steps = 0.5 if dtype is not torch.float32 else 8
    assert ((out.float() - same).abs() <= steps * torch.finfo(dtype).eps * same.abs()).all()
    assert not dq.any() and not dk.any()
    summed = (dout.double() * live).unflatten(1, (2, 3))
    error = (dv.double() - summed.sum(2)).abs()
    # probabilities and the result are rounded, and three terms added in fp32
    assert (error <= (torch.finfo(dtype).eps + 2.0 ** -20) * summed.abs().sum(2)).all()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('batch, tokens, window', [(40, 13, None), (100, 4, 3), (4, 256, None), (2, 512, None), (2, 700, 20)])
def test_gradients_of_rows_with_few_keys_keep_their_precision(batch, tokens, window, dtype) -> None:
    """
    Gradients of queries and keys are rounded twice, as ds and at the end: sqrt(2) times as far off as by
    the last rounding alone, and up to 1.5 times where few large terms make up a sum.  An output of rounded
    probabilities would add a third one through delta (1.5 to 2 times).
    """
    q, k, v, dout = inputs(batch, 4, 4, tokens, tokens, 64, dtype)
    leaves = [t.double().requires_grad_() for t in (q, k, v)]
    scores = leaves[0] @ leaves[1].transpose(2, 3) / 8.0
    distance = torch.arange(tokens)[:, None] - torch.arange(tokens)
    seen = (distance >= 0) & (distance < (window or tokens))
    expected = torch.autograd.grad(scores.masked_fill(~seen, float('-inf')).softmax(-1) @ leaves[2], leaves, dout.double())
    ours = [t.cuda().requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(attorch_amd.WindowAttention(window=window)(*ours), ours, dout.cuda())
    for name, a, b in zip(('query', 'key'), got, expected):
        once = (b.to(dtype).double() - b).norm()
        assert (a.cpu().double() - b).norm() <= 1.5 * once, name
