"""
GPU tests of attention on values at the edges of their types: padded rows and unseen keys beside numbers
that are not finite.
"""

import pytest
import torch

import attorch_amd
from .helpers import DTYPES
from .test_gpu_attention import inputs

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
