"""
Attention over a sliding window with visible first tokens, and rotary positions, in plain CPU
arithmetic in float64, each result with a bound of the error that a kernel may have.

The reference has neither (its attention layer cannot be constructed,
attorch/multi_head_attention_layer.py:77), so the formulas are the definition; the values are
pinned against torch's own attention and complex multiplication in tests/test_oracle_attention.py.

Error bounds.  u is half a step of the storage type (it rounds probabilities p, their
gradients ds, and results), e = 2^-24 the unit of the float32 arithmetic.  A float32 dot product of n
terms is off by at most (n + 1) e sum|x||y|.  Scores s (in units of log2, times 1.45) and the
row's log-sum both carry such an error, so a probability's relative error is at most
    eps = 4 ((D + 8) S + T + 16) e,
with S the row's largest scale sum|q||k| and T the number of summed keys' contribution to the
running sum (log2 of the tiles plus one tile: 64 bounds it).  Then
    out: (u + eps) P|V| + u|out|                 dv: (u + eps) P^T|dO| + u|dv|
    delta is a product of dO with the stored output: d = |dO| (bound of out) + (D + 2) e |dO||out|
    ds: x = (u + eps) |dS| + P (d + (D + 2) e |dO||V|)
    dq: scale x |K| + u|dq|                      dk: scale x^T |Q| + u|dk|
plus the accumulation errors of the second products, n e of the same sums, and half a step of the
storage type's smallest numbers.  The hardware's exponential returns zero where the result would be
below float32's smallest normal number: the row's largest exponential is 1, so a probability may lack up
to z = 2^-126, which adds z|V| to out, z|dO| to dv and z (|dp| + |delta|) to ds.
"""

from typing import Dict, Optional, Tuple

import torch
from torch import Tensor


def attention_visible(rows: int, keys: int, length: int, query_length: int, causal: bool, window: Optional[int],
                      sinks: int) -> Tensor:
    """
    [rows, keys] truth values: which key each query row of a sequence sees.
    """
    length = min(max(length, 0), keys)
    query_length = min(max(query_length, 0), rows)
    start = max(length - query_length, 0)
    row = torch.arange(rows)[:, None]
    token = start + row
    key = torch.arange(keys)[None]
    seen = (row < query_length) & (token < length) & (key < length)
    if causal:
        seen = seen & (key <= token)
    if window is not None:
        seen = seen & (((token - key).abs() < window) | (key < sinks))
    return seen


def _tiny(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def attention(q: Tensor, k: Tensor, v: Tensor, dout: Optional[Tensor] = None, lengths: Optional[Tensor] = None,
              query_lengths: Optional[Tensor] = None, causal: bool = True, window: Optional[int] = None, sinks: int = 0,
              scale: Optional[float] = None) -> Dict[str, Tuple[Tensor, Tensor]]:
    """
    {'out', 'dq', 'dk', 'dv'}: value and error bound, both float64.  What no row sees is set to
    zero before it is used, so that garbage there cannot spread.
    """
    dtype = q.dtype
    u, e = torch.finfo(dtype).eps / 2, 2.0 ** -24
    batch, heads, rows, dim = q.shape
    kv_heads, keys = k.shape[1], k.shape[2]
    group = heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    names = ('out',) if dout is None else ('out', 'dq', 'dk', 'dv')
    like = {'out': q, 'dq': q, 'dk': k, 'dv': v}
    result = {n: (torch.zeros(like[n].shape, dtype=torch.float64), torch.zeros(like[n].shape, dtype=torch.float64))
              for n in names}
    for b in range(batch):
        seen = attention_visible(rows, keys, keys if lengths is None else int(lengths[b]),
                                 rows if query_lengths is None else int(query_lengths[b]), causal, window, sinks)
        live, used = seen.any(1), seen.any(0)
        for h in range(heads):
            hk = h // group
            Q = torch.where(live[:, None], q[b, h].double(), 0.0)
            K = torch.where(used[:, None], k[b, hk].double(), 0.0)
            V = torch.where(used[:, None], v[b, hk].double(), 0.0)
            s = (Q @ K.T * scale).masked_fill(~seen, -torch.inf)
            top = s.amax(-1, keepdim=True) if keys else s
            p = torch.where(seen, torch.exp(s - torch.where(live[:, None], top, 0.0)), 0.0) if keys else s
            total = p.sum(-1, keepdim=True)
            p = torch.where(live[:, None], p / total, 0.0)
            out = p @ V
            big = torch.where(seen, Q.abs() @ K.abs().T * scale, 0.0)
            S = big.amax(-1, keepdim=True) if keys else torch.zeros(rows, 1, dtype=torch.float64)
            eps = 4 * ((dim + 8) * S + 64 + 16) * e
            n = seen.sum(-1, keepdim=True).double()
            z = seen * 2.0 ** -126
            out_err = ((u + eps + n * e) * p + z) @ V.abs() + u * out.abs() + _tiny(dtype)
            result['out'][0][b, h] = out
            result['out'][1][b, h] = out_err
            if dout is None:
                continue
            D = torch.where(live[:, None], dout[b, h].double(), 0.0)
            dp = D @ V.T
            delta = (D * out).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            d_err = (D.abs() * out_err).sum(-1, keepdim=True) + (dim + 2) * e * (D.abs() * out.abs()).sum(-1, keepdim=True)
            # a rounded ds is off by half a step, or less than the type's smallest number
            x = (u + eps) * ds.abs() + p * (d_err + (dim + 2) * e * (D.abs() @ V.abs().T)) + seen * _tiny(dtype) + \
                z * (dp.abs() + delta.abs())
            c = seen.sum(0).double()[:, None]
            dq, dk, dv = scale * (ds @ K), scale * (ds.T @ Q), p.T @ D
            result['dq'][0][b, h] = dq
            result['dq'][1][b, h] = scale * ((x + n * e * ds.abs()) @ K.abs()) + u * dq.abs() + _tiny(dtype)
            result['dk'][0][b, hk] += dk
            result['dk'][1][b, hk] += scale * ((x + group * c.T * e * ds.abs()).T @ Q.abs())
            result['dv'][0][b, hk] += dv
            result['dv'][1][b, hk] += ((u + eps + group * c.T * e) * p + z).T @ D.abs()
    for n in ('dk', 'dv'):
        if n in result:
            result[n] = (result[n][0], result[n][1] + u * result[n][0].abs() + _tiny(dtype))
    return result


def rotary(x: Tensor, positions: Tensor, inv_freq: Tensor, pair_axis: Tensor, adjacent: bool = False,
           inverse: bool = False) -> Tuple[Tensor, Tensor]:
    """
    x [batch, heads, rows, dim] with its pairs turned by positions [axes, batch, rows], and a bound of a
    kernel's error: cosine and sine are off by at most 2 units of float32 each (and the reduced angle,
    at most half a turn, by one rounding to float32), the products and their sum by one each.
    """
    pairs = inv_freq.shape[0]
    u, e = torch.finfo(x.dtype).eps / 2, 2.0 ** -24
    value = x.double().clone()
    error = torch.zeros_like(value)
    for n in range(pairs):
        first, second = (2 * n, 2 * n + 1) if adjacent else (n, n + pairs)
        angle = positions[int(pair_axis[n])].double() * inv_freq[n].double()
        cos, sin = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
        sin = -sin if inverse else sin
        a, b = x[..., first].double(), x[..., second].double()
        value[..., first], value[..., second] = a * cos - b * sin, a * sin + b * cos
        error[..., first] = error[..., second] = (2 + 3.15 + 2 + 2) * e * (a.abs() + b.abs())
    turned = error > 0
    return value, error + turned * (u * value.abs() + _tiny(x.dtype))
