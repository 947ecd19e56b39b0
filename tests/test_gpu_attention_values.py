"""
GPU tests of attention on values at the edges of their types: padded rows and unseen keys beside numbers
that are not finite, and gradients of any size.
"""

import pytest
import torch

import attorch_amd
from oracle.attention import attention_visible
from .helpers import DTYPES
from .test_gpu_attention import check, inputs

pytestmark = pytest.mark.gpu
NAN, INF = float('nan'), float('inf')

# [rows, keys, lengths, query lengths]: rows behind a sequence beside rows that see every key of a tile, on
# their own, in halves of the keys and in splits that are joined
PADDED = [(400, 400, [301, 111, 397], None), (70, 400, [400, 290, 64], [33, 70, 10]), (100, 1111, [1111, 403, 700], [70, 1, 99])]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('heads, kv_heads', [(3, 1), (24, 24)])
@pytest.mark.parametrize('rows, keys, lengths, query_lengths', PADDED)
@pytest.mark.parametrize('bad', [NAN, INF, -INF])
def test_padded_rows_beside_keys_and_values_that_are_not_finite(bad, rows, keys, lengths, query_lengths, heads, kv_heads, causal,
                                                                dtype) -> None:
    counts = torch.tensor(lengths)
    query_counts = torch.tensor(query_lengths) if query_lengths else counts.clamp(max=rows)
    padded = torch.arange(rows) >= query_counts[:, None]
    for place in (1, 2):
        tensors = list(inputs(3, heads, kv_heads, rows, keys, 64, dtype))
        tensors[place][:, :, 3] = bad
        q, k, v, dout = (t.cuda() for t in tensors)
        leaves = [t.requires_grad_() for t in (q, k, v)]
        out = attorch_amd.WindowAttention(causal=causal)(*leaves, counts.cuda(), query_counts.cuda() if query_lengths else None)
        (dq,) = torch.autograd.grad(out, leaves[:1], dout)
        for name, x in (('output', out), ('query gradient', dq)):
            x = x.detach().cpu().transpose(1, 2)
            assert (x[padded] == 0).all(), (name, place)
            assert not torch.isfinite(x[~padded]).all()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('heads, kv_heads', [(3, 1), (24, 24)])
@pytest.mark.parametrize('rows, keys, lengths, query_lengths', PADDED)
@pytest.mark.parametrize('window, sinks', [(None, 0), (40, 3)])
@pytest.mark.parametrize('bad', [NAN, INF])
def test_unseen_keys_beside_rows_that_are_not_finite(bad, window, sinks, rows, keys, lengths, query_lengths, heads, kv_heads, causal,
                                                     dtype) -> None:
    counts = torch.tensor(lengths)
    query_counts = torch.tensor(query_lengths) if query_lengths else counts.clamp(max=rows)
    start = (counts - query_counts).clamp(min=0)
    key = torch.arange(keys)
    unseen = key >= counts[:, None]
    if window:
        unseen |= (key >= sinks) & (key <= (start - window)[:, None])
    for place in (0, 3):
        tensors = list(inputs(3, heads, kv_heads, rows, keys, 64, dtype))
        tensors[place][:, :, 0] = bad       # a row of every sequence that is a token
        q, k, v, dout = (t.cuda() for t in tensors)
        leaves = [t.requires_grad_() for t in (q, k, v)]
        out = attorch_amd.WindowAttention(causal=causal, window=window, num_sinks=sinks)(
            *leaves, counts.cuda(), query_counts.cuda() if query_lengths else None)
        _, dk, dv = torch.autograd.grad(out, leaves, dout)
        for name, x in (('key gradient', dk), ('value gradient', dv)):
            x = x.cpu().transpose(1, 2)
            assert (x[unseen] == 0).all(), (name, place)
        assert not torch.isfinite(x[~unseen]).all()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('heads, kv_heads, dim, causal, window, sinks', [
    (2, 1, 64, True, None, 0), (2, 2, 128, True, 700, 5), (6, 2, 24, False, 300, 70), (2, 1, 96, False, None, 0)])
@pytest.mark.parametrize('tokens, size', [(4096, 1e-4), (4096, 1e-3), (4096, 1.0), (8192, 1e-3), (3000, 8e3), (100, 8e3),
                                          (100, 1e-3)])
def test_gradients_of_any_size(tokens, size, heads, kv_heads, dim, causal, window, sinks, dtype) -> None:
    """
    Gradients keep their precision whatever the output gradient's size, whole and over the last rows and keys,
    whose gradients are the smallest.  A term is rounded once (ds, or a probability) and the sum once more: sqrt(2)
    times as far off as by the last rounding alone, and up to 1.5 times where few large terms make up a sum.

    Probabilities of flat rows are alike, and so are their roundings, which then do not average out: with a common
    relative error of up to u, half a step, the value gradients are off by up to u |dv| before the last rounding.
    That one is u 2^e / sqrt(3) on average for numbers m 2^e with m from 1 to 2, spread over their logarithm:
    mean m^2 = 3 / (2 log 2) = 2.16, so it is u |dv| / sqrt(3 * 2.16) = 0.39 u |dv|, and both
    together are sqrt(1 + 1 / 0.39^2) = 2.75 times as far off.
    """
    q, k, v, dout = (t.cuda() for t in inputs(1, heads, kv_heads, tokens, tokens, dim, dtype))
    dout *= size
    if size > 1.0:                     # ds beyond 65504, gradients within
        q, k, v = q * 0.25, k * 0.25, v * 4
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    got = torch.autograd.grad(attorch_amd.WindowAttention(causal, window, sinks)(*leaves), leaves, dout)
    expected = [torch.zeros(t.shape, dtype=torch.float64, device='cuda') for t in (q, k, v)]
    hidden = ~attention_visible(tokens, tokens, tokens, tokens, causal, window, sinks).cuda()
    for h in range(heads):
        shared = h * kv_heads // heads
        Q, K, V, D = (t.double() for t in (q[0, h], k[0, shared], v[0, shared], dout[0, h]))
        p = (Q @ K.T * dim ** -0.5).masked_fill(hidden, -INF).softmax(-1)
        ds = p * (D @ V.T - (D * (p @ V)).sum(-1, keepdim=True)) * dim ** -0.5
        expected[0][0, h] = ds @ K
        expected[1][0, shared] += ds.T @ Q
        expected[2][0, shared] += p.T @ D
    for name, a, b in zip(('query', 'key', 'value'), got, expected):
        assert torch.isfinite(b.to(dtype)).all()
        for part in (slice(None), slice(-(tokens // 8), None)):
            x, y = a[:, :, part].double(), b[:, :, part]
            once = (y.to(dtype).double() - y).norm()
            assert (x - y).norm() <= (2.75 if name == 'value' else 1.5) * once, name


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('batch, heads, kv_heads, rows, keys, dim, window, sinks', [
    (2, 4, 2, 300, 300, 64, None, 0), (1, 4, 2, 700, 700, 32, 20, 33), (1, 4, 2, 700, 700, 32, 20, 300), (2, 2, 1, 70, 1111, 128, None, 0),
    (3, 6, 2, 100, 100, 80, 30, 2), (8, 32, 32, 150, 150, 40, None, 0)])
def test_output_gradients_of_mixed_sizes(batch, heads, kv_heads, rows, keys, dim, window, sinks, causal, dtype) -> None:
    """Rows whose output gradients are eight orders of magnitude apart, large ones behind small ones and in front of them."""
    q, k, v, dout = inputs(batch, heads, kv_heads, rows, keys, dim, dtype)
    size = 10.0 ** ((torch.arange(rows) * 7 // 40) * 5 % 9 - 5.0)       # 1e-5 to 1e3, another one every six rows
    check(q, k, v, (dout * size[:, None]).to(dtype), causal=causal, window=window, sinks=sinks)
    check(q, k, v, (dout * size.flip(0)[:, None]).to(dtype), causal=causal, window=window, sinks=sinks)
