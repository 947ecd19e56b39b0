"""
Pins the attention and rotary oracles: against torch's attention with an explicit mask (values and
autograd gradients), central differences, and complex multiplication.
"""

import pytest
import torch

from oracle.attention import attention, attention_visible, rotary
from .helpers import randn


@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('window, sinks', [(None, 0), (4, 0), (4, 2), (1, 3), (30, 1)])
@pytest.mark.parametrize('rows, keys, heads, kv_heads', [(9, 9, 4, 2), (3, 11, 2, 2), (1, 7, 3, 1)])
def test_attention_matches_torch(rows, keys, heads, kv_heads, window, sinks, causal) -> None:
    q, k, v = (randn((2, n, t, 8), s).double().requires_grad_(True)
               for n, t, s in ((heads, rows, 1), (kv_heads, keys, 2), (kv_heads, keys, 3)))
    dout = randn((2, heads, rows, 8), 4).double()
    i = torch.arange(keys - rows, keys)[:, None]
    j = torch.arange(keys)[None]
    mask = torch.ones(rows, keys, dtype=torch.bool)
    if window is not None:
        mask &= ((i - j).abs() <= window - 1) | (j < sinks)
    if causal:
        mask &= j <= i
    assert torch.equal(mask, attention_visible(rows, keys, keys, rows, causal, window, sinks))
    group = heads // kv_heads
    ref = torch.nn.functional.scaled_dot_product_attention(
        q, k.repeat_interleave(group, 1), v.repeat_interleave(group, 1), attn_mask=mask)
    ref.backward(dout)
    got = attention(q.detach(), k.detach(), v.detach(), dout, causal=causal, window=window, sinks=sinks)
    for name, expected in (('out', ref.detach()), ('dq', q.grad), ('dk', k.grad), ('dv', v.grad)):
        torch.testing.assert_close(got[name][0], expected, rtol=1e-9, atol=1e-9)
        assert (got[name][1] > 0).all()


def test_attention_gradients_match_differences() -> None:
    q, k, v = (randn((1, 2, 5, 4), s).double() for s in (1, 2, 3))
    dout = randn((1, 2, 5, 4), 4).double()
    options = {'lengths': torch.tensor([4]), 'window': 2, 'sinks': 1}
    got = attention(q, k, v, dout, **options)
    step = 1e-5
    for name, x in (('dq', q), ('dk', k), ('dv', v)):
        grad = torch.zeros_like(x)
        for at in range(x.numel()):
            old = x.view(-1)[at].item()
            sums = []
            for delta in (step, -step):
                x.view(-1)[at] = old + delta
                sums.append((attention(q, k, v, **options)['out'][0] * dout).sum().item())
            x.view(-1)[at] = old
            grad.view(-1)[at] = (sums[0] - sums[1]) / (2 * step)
        torch.testing.assert_close(got[name][0], grad, rtol=1e-6, atol=1e-8)


def test_attention_padding_rows_and_lengths() -> None:
    q, k, v = (randn((3, 1, 4, 4), s) for s in (1, 2, 3))
    dout = randn((3, 1, 4, 4), 4)
    got = attention(q, k, v, dout, lengths=torch.tensor([0, 3, 9]), query_lengths=torch.tensor([4, 2, 4]))
    assert (got['out'][0][0] == 0).all() and (got['dk'][0][0] == 0).all()
    assert (got['out'][0][1, :, 2:] == 0).all() and (got['out'][0][1, :, :2] != 0).any()
    alone = attention(q[1:2, :, :2], k[1:2, :, :3], v[1:2, :, :3], dout[1:2, :, :2])
    for name, live in (('out', 2), ('dq', 2), ('dk', 3), ('dv', 3)):
        torch.testing.assert_close(got[name][0][1:2, :, :live], alone[name][0])
        assert (got[name][0][1:2, :, live:] == 0).all()


@pytest.mark.parametrize('adjacent', [False, True])
def test_rotary_matches_complex_multiplication(adjacent) -> None:
    x = randn((2, 3, 5, 12), 1)
    positions = torch.randint(-50, 5000, (2, 2, 5), generator=torch.Generator().manual_seed(2))
    inv_freq = 10000.0 ** (torch.arange(4, dtype=torch.float64) / -4)
    pair_axis = torch.tensor([0, 1, 1, 0], dtype=torch.int32)
    value, bound = rotary(x, positions, inv_freq, pair_axis, adjacent)
    first = torch.arange(4) * (2 if adjacent else 1)
    second = first + (1 if adjacent else 4)
    z = torch.complex(x[..., first].double(), x[..., second].double())
    z = z * torch.exp(1j * positions[pair_axis.long()].permute(1, 2, 0)[:, None] * inv_freq)
    torch.testing.assert_close(value[..., first], z.real)
    torch.testing.assert_close(value[..., second], z.imag)
    assert torch.equal(value[..., 8:], x[..., 8:].double()) and (bound[..., 8:] == 0).all()
    back, _ = rotary(value, positions, inv_freq, pair_axis, adjacent, inverse=True)
    torch.testing.assert_close(back, x.double())
