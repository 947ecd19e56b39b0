"""
CPU-only tests of what the attention and rotary layers pass to the C entry points when saved tensors
come back in another layout than they were saved in, as saved-tensor hooks may return them: the entry
points are replaced by ones that follow every stride on the host.
"""

import ctypes
import itertools

import pytest
import torch

import attorch_amd
from attorch_amd import _lib, attention

BATCH, HEADS, KV_HEADS, TOKENS, DIM = 2, 4, 2, 9, 16


class Recorder:
    """
    Stands in for the library, without launches; the output is filled with numbers.
    """
    def __init__(self) -> None:
        self.real = _lib.load()
        self.dtype = torch.float32

    def __getattr__(self, name):
        return getattr(self.real, name)

    def at_attention_fwd(self, shape, q, k, v, lengths, query_lengths, out, *_):
        values = torch.randn(BATCH * HEADS * TOKENS * DIM, generator=torch.Generator().manual_seed(2)).to(self.dtype)
        ctypes.memmove(out, values.data_ptr(), values.nbytes)
        return 0

    def at_rotary(self, *_):
        return 0


@pytest.fixture
def recorder(monkeypatch):
    record = Recorder()
    monkeypatch.setattr(_lib, 'load', lambda: record)
    monkeypatch.setattr(_lib, 'require_same_device', lambda *_: None)
    monkeypatch.setattr(_lib, 'device_guard', lambda _: _lib._NO_GUARD)
    monkeypatch.setattr(_lib, 'stream_of', lambda _: 0)
    return record


def values_at(address, strides, extents, features, dtype):
    """
    What a kernel reads: [batch, heads, tokens, features] from an address and the strides of the first three.
    """
    size = dtype.itemsize
    out = torch.empty(*extents, features, dtype=dtype)
    for at in itertools.product(*(range(n) for n in extents)):
        source = address + sum(i * s for i, s in zip(at, strides)) * size
        ctypes.memmove(out[at].data_ptr(), source, features * size)
    return out


def hooks(unpack):
    return torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().clone(), unpack)


def contiguous(tensor):
    return tensor.contiguous()


def reversed_order(tensor):
    """Equal values with the strides in the opposite order, where there are several."""
    order = tuple(reversed(range(tensor.ndim - 1))) + (tensor.ndim - 1,)
    return tensor.permute(order).contiguous().permute(order) if tensor.ndim > 1 else tensor


def misaligned(tensor):
    """Equal values that begin one element behind a boundary."""
    room = torch.empty(tensor.numel() + 1, dtype=tensor.dtype)
    return room[1:].view(tensor.shape).copy_(tensor)


def spread(tensor):
    """Equal values in every second place."""
    return torch.stack([tensor, torch.zeros_like(tensor)], -1)[..., 0]


class Kept(list):
    """
    Unpacked tensors, kept alive so that addresses can be followed after the call.
    """
    def unpack(self, relay):
        def hook(tensor):
            self.append(relay(tensor))
            return self[-1]
        return hook


def projections(dtype, packed):
    gen = torch.Generator().manual_seed(1)
    if packed:
        qkv = torch.randn(BATCH, TOKENS, HEADS + 2 * KV_HEADS, DIM, generator=gen).to(dtype).transpose(1, 2)
        parts = qkv.split((HEADS, KV_HEADS, KV_HEADS), 1)
    else:
        parts = [torch.randn(BATCH, TOKENS, n, DIM, generator=gen).to(dtype).transpose(1, 2)
                 for n in (HEADS, KV_HEADS, KV_HEADS)]
    return [t.detach().requires_grad_() for t in parts]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('packed', [True, False])
@pytest.mark.parametrize('relay', [contiguous, reversed_order, misaligned, spread])
def test_attention_follows_the_layouts_that_come_back(relay, packed, dtype, recorder, monkeypatch) -> None:
    leaves = projections(dtype, packed)
    recorder.dtype = dtype
    lengths = torch.tensor([TOKENS, 5])
    alive = Kept()
    # copies that the layer makes on the way are followed as well
    plain = attention._for_kernel
    monkeypatch.setattr(attention, '_for_kernel', lambda *args: alive.append(plain(*args)) or alive[-1])
    with hooks(alive.unpack(relay)):
        out = attorch_amd.WindowAttention()(*leaves, lengths)
    expected_out = out.detach().clone()
    dout = torch.randn(out.shape, generator=torch.Generator().manual_seed(3)).to(dtype)

    def bwd(shape, output_grad, q, k, v, counts, query_counts, stored, rest, lse, dq, dk, dv, *_):
        strides = [tuple(shape._obj.strides[3 * n:3 * n + 3]) for n in range(8)]
        for name, address, stride, tensor in (('query', q, strides[0], leaves[0]), ('key', k, strides[1], leaves[1]),
                                              ('value', v, strides[2], leaves[2]), ('grad', output_grad, strides[4], dout)):
            got = values_at(address, stride, tensor.shape[:3], DIM, dtype)
            assert torch.equal(got, tensor.detach()), name
        for address in (q, k, v, stored, rest, lse, dq, dk, dv, output_grad):
            assert address % 16 == 0
        assert torch.equal(values_at(stored, strides[3], out.shape[:3], DIM, dtype), expected_out), 'output'
        got = (ctypes.c_int64 * BATCH).from_address(counts)
        assert shape._obj.lengths_int64 and list(got) == lengths.tolist()
        # gradients: every place is written once, and within the tensor that was allocated for it
        for address, stride, tensor, value in ((dq, strides[5], leaves[0], 1.0), (dk, strides[6], leaves[1], 2.0),
                                               (dv, strides[7], leaves[2], 3.0)):
            for at in itertools.product(*(range(n) for n in tensor.shape[:3])):
                row = torch.full((DIM,), value, dtype=dtype)
                ctypes.memmove(address + sum(i * s for i, s in zip(at, stride)) * dtype.itemsize, row.data_ptr(),
                               DIM * dtype.itemsize)
        return 0

    recorder.at_attention_bwd = bwd
    grads = torch.autograd.grad(out, leaves, dout)
    for grad, leaf, value in zip(grads, leaves, (1.0, 2.0, 3.0)):
        assert grad.shape == leaf.shape and (grad == value).all()


@pytest.mark.parametrize('relay', [contiguous, spread])
def test_rotary_follows_the_layouts_that_come_back(relay, recorder) -> None:
    q, k, _ = projections(torch.float32, True)
    inv_freq = torch.rand(8, dtype=torch.float64)
    pair_axis = torch.arange(8, dtype=torch.int32) % 2
    positions = torch.arange(2 * BATCH * TOKENS).view(2, BATCH, TOKENS)
    alive = Kept()
    with hooks(alive.unpack(relay)):
        outs = attorch_amd.RotaryAutoGrad.apply(q, k, positions, inv_freq, pair_axis)
    seen = []

    def inverse(shape, *args):
        shape = shape._obj
        assert shape.inverse
        _, _, _, _, at, freq, axis, _ = args
        read = [[[ctypes.c_int64.from_address(at + 8 * sum(i * s for i, s in zip((x, b, t), shape.position_strides))).value
                  for t in range(TOKENS)] for b in range(BATCH)] for x in range(2)]
        assert read == positions.tolist()
        assert list((ctypes.c_double * 8).from_address(freq)) == inv_freq.tolist()
        assert list((ctypes.c_int32 * 8).from_address(axis)) == pair_axis.tolist()
        seen.append(True)
        return 0

    recorder.at_rotary = inverse
    torch.autograd.grad(outs, (q, k), [torch.ones_like(t) for t in outs])
    assert seen
