"""
Rotary positions with one or several axes, with PyTorch autodiff support, running on a gfx950
kernel that turns queries and keys in one launch.

The reference has no counterpart: its example model adds learned absolute positions to the token
embeddings (examples/wikitext-2/gpt.py:95-110).
"""

import ctypes
import functools
from typing import Any, Optional, Sequence, Tuple

import torch
from torch import Tensor
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib

POSITION_TYPES = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
MAX_PAIRS = 512


class _Shape(ctypes.Structure):
    """
    at_rotary_t of include/attorch_hip.h.
    """
    _fields_ = ([(name, ctypes.c_int64) for name in ('batch', 'rows', 'q_heads', 'k_heads', 'dim', 'pairs', 'axes')] +
                [('strides', ctypes.c_int64 * 12), ('position_strides', ctypes.c_int64 * 3),
                 ('position_type', ctypes.c_int), ('adjacent', ctypes.c_int), ('inverse', ctypes.c_int),
                 ('dtype', ctypes.c_int)])


# A tensor's layout: (shape, stride, dtype)
Layout = Tuple[torch.Size, Tuple[int, ...], torch.dtype]


def _layout(tensor: Tensor) -> Layout:
    return tensor.shape, tensor.stride(), tensor.dtype


def _positions_of(positions: Optional[Tensor], axes: int, batch: int, rows: int) -> Optional[Tensor]:
    """
    Positions as [axes, batch, rows], without a copy.
    """
    if positions is None:
        if axes > 1:
            raise RuntimeError(f'Positions with {axes} axes must be given')
        return None
    if positions.dtype not in POSITION_TYPES:
        raise RuntimeError(f'Positions must be int32, int64 or float32, received {positions.dtype}')
    shape = tuple(positions.shape)
    if shape == (axes, batch, rows):
        return positions
    if axes == 1 and shape in ((rows,), (batch, rows)):   # (1, rows) means the same as one axis and as one sequence
        return positions.expand(1, batch, rows)
    assert shape == (axes, rows), \
        f'Positions must be of shape {(axes, batch, rows)} or {(axes, rows)}, received {shape}'
    return positions.unsqueeze(1).expand(axes, batch, rows)


def _check(query: Layout, key: Optional[Layout], positions: Optional[Layout], inv_freq: Layout,
           pair_axis: Optional[Layout]) -> int:
    """
    Refuses what the kernel does not compute, before anything is launched; returns the number of axes.
    """
    shape = tuple(query[0])
    assert len(shape) == 4, f'Queries must be [batch, heads, rows, head_dim], received {shape}'
    if key is not None:
        assert len(key[0]) == 4 and key[0][0] == shape[0] and tuple(key[0][2:]) == shape[2:], \
            f'Incompatible query ({shape}) and key ({tuple(key[0])}) shape'
        if key[2] is not query[2]:
            raise RuntimeError(f'Query and key must have the same dtype, received {query[2]} and {key[2]}')
    if inv_freq[2] is not torch.float64:
        raise RuntimeError(f'inv_freq must be float64, received {inv_freq[2]}')
    assert len(inv_freq[0]) == 1 and 2 * inv_freq[0][0] <= shape[3], \
        f'inv_freq ({tuple(inv_freq[0])}) must hold at most half the head dimension ({shape[3]})'
    if inv_freq[0][0] > MAX_PAIRS:
        raise RuntimeError(f'At most {MAX_PAIRS} pairs are supported, received {inv_freq[0][0]}')
    if pair_axis is None:
        return 1
    if pair_axis[2] is not torch.int32:
        raise RuntimeError(f'pair_axis must be int32, received {pair_axis[2]}')
    assert pair_axis[0] == inv_freq[0], \
        f'pair_axis ({tuple(pair_axis[0])}) must have the shape of inv_freq ({tuple(inv_freq[0])})'
    assert positions is not None and len(positions[0]) in (2, 3) and positions[0][0] > 0, \
        'Axes of pairs need positions of shape [axes, batch, rows] or [axes, rows]'
    return positions[0][0]


def _side_by_side(layout: Layout) -> bool:
    return layout[1][3] == 1 or layout[0][3] <= 1 or 0 in layout[0]


@functools.lru_cache(maxsize=4096)
def _plan(query: Optional[Layout], key: Optional[Layout], positions: Optional[Layout], inv_freq: Layout,
          pair_axis: Optional[Layout], adjacent: bool, inverse: bool) -> Optional[_Shape]:
    """
    Checks the arguments and describes the call for the kernel; None where the features of the queries or
    keys do not lie side by side.  Remembered by layouts and options: a program repeats few of them, and
    the description takes longer than a small call's kernel.
    """
    present = query if query is not None else key
    axes = _check(present, key if query is not None else None, positions, inv_freq, pair_axis)
    batch, _, rows, dim = present[0]
    position_type, position_strides = 0, (0, 0, 0)
    if positions is not None:
        expanded = _positions_of(torch.empty_strided(*positions[:2], dtype=positions[2], device='meta'), axes, batch, rows)
        position_type, position_strides = POSITION_TYPES[positions[2]], expanded.stride()
    strides = [0] * 12
    for n, layout in enumerate((query, key)):
        if layout is None:
            continue
        if not _side_by_side(layout):
            return None
        # the output takes the input's layout where that is dense; torch.empty_like keeps the order of the strides
        output = torch.empty_like(torch.empty_strided(*layout[:2], dtype=layout[2], device='meta'))
        strides[3 * n:3 * n + 3] = layout[1][:3]
        strides[6 + 3 * n:9 + 3 * n] = output.stride()[:3]
        if not _side_by_side((output.shape, output.stride(), output.dtype)):
            return None
    return _Shape(batch, rows, 0 if query is None else query[0][1], 0 if key is None else key[0][1], dim, inv_freq[0][0],
                  axes, (ctypes.c_int64 * 12)(*strides), (ctypes.c_int64 * 3)(*position_strides), position_type, adjacent,
                  inverse, _lib.dtype_id(present[2]))


def _rotate(query: Optional[Tensor], key: Optional[Tensor], positions: Optional[Tensor], inv_freq: Tensor,
            pair_axis: Optional[Tensor], adjacent: bool, inverse: bool) -> Tuple[Optional[Tensor], Optional[Tensor]]:
    """
    Turns the queries and keys (either may be absent) by their positions' angles, or back.
    """
    if not inv_freq.is_contiguous():
        inv_freq = inv_freq.contiguous()
    if pair_axis is not None and not pair_axis.is_contiguous():
        pair_axis = pair_axis.contiguous()
    tables = (None if positions is None else _layout(positions), _layout(inv_freq),
              None if pair_axis is None else _layout(pair_axis), adjacent, inverse)
    shape = _plan(None if query is None else _layout(query), None if key is None else _layout(key), *tables)
    if shape is None:
        query, key = (None if t is None else t.contiguous() for t in (query, key))
        shape = _plan(None if query is None else _layout(query), None if key is None else _layout(key), *tables)
    _lib.require_same_device('Rotary', inv_freq, query, key, positions, pair_axis)
    query_out = None if query is None else torch.empty_like(query)
    key_out = None if key is None else torch.empty_like(key)
    with _lib.device_guard(inv_freq):
        _lib.check(_lib.load().at_rotary(
            ctypes.byref(shape), None if query is None else query.data_ptr(), None if key is None else key.data_ptr(),
            None if query is None else query_out.data_ptr(), None if key is None else key_out.data_ptr(),
            None if positions is None else positions.data_ptr(), inv_freq.data_ptr(),
            None if pair_axis is None else pair_axis.data_ptr(), _lib.stream_of(inv_freq)), 'at_rotary')
    return query_out, key_out


class RotaryAutoGrad(torch.autograd.Function):
    """
    Autodiff for rotary positions.
    """
    @staticmethod
    def forward(
        ctx: Any,
        query: Tensor,
        key: Optional[Tensor],
        positions: Optional[Tensor],
        inv_freq: Tensor,
        pair_axis: Optional[Tensor] = None,
        adjacent: bool = False,
        ) -> Tuple[Tensor, Optional[Tensor]]:
        """
        Turns pair n of every head's features by the angle positions[pair_axis[n]] * inv_freq[n]:
        (x, y) becomes (x cos a - y sin a, x sin a + y cos a).  Features behind the pairs are kept.
        Angles are formed in 64 bits, so positions may be far.

        Args:
            query: Queries of shape [batch, heads, rows, head_dim].
            key: Optional keys of shape [batch, kv_heads, rows, head_dim].
            positions: Positions of the tokens, int32, int64 or float32: with pair_axis of shape
                [axes, batch, rows] or [axes, rows], without it [batch, rows], [rows] or
                [1, batch, rows]. None (without pair_axis): token t of every sequence is at t.
            inv_freq: Radians per position of each pair, float64, at most head_dim // 2 of them.
            pair_axis: Optional axis of each pair, int32 of inv_freq's shape (values are clamped to
                the axes there are). None: one axis.
            adjacent: Pairs are features (2 n, 2 n + 1) instead of (n, n + pairs).

        Returns:
            Turned queries and keys (None without keys), of the dtypes of the inputs.
        """
        if ctx.needs_input_grad[2] or ctx.needs_input_grad[3]:
            raise RuntimeError('Rotary has no gradients of positions and inv_freq; detach them')
        adjacent = bool(adjacent)
        outputs = _rotate(query, key, positions, inv_freq, pair_axis, adjacent, False)
        ctx.adjacent = adjacent
        ctx.save_for_backward(positions, inv_freq, pair_axis)
        ctx.set_materialize_grads(False)
        return outputs

    @staticmethod
    def backward(
        ctx: Any,
        query_grad: Optional[Tensor],
        key_grad: Optional[Tensor] = None,
        ) -> Tuple[Optional[Tensor], ...]:
        """
        Gradients of the queries and keys: the outputs' gradients, turned back.
        """
        # under create_graph the gradients are marked as not differentiable again
        backward = _backward_once if torch.is_grad_enabled() else _backward
        return backward(ctx, query_grad, key_grad)


def _backward(ctx: Any, query_grad: Optional[Tensor], key_grad: Optional[Tensor]) -> Tuple[Optional[Tensor], ...]:
    positions, inv_freq, pair_axis = ctx.saved_tensors
    if not ctx.needs_input_grad[0]:
        query_grad = None
    if not ctx.needs_input_grad[1]:
        key_grad = None
    if query_grad is not None or key_grad is not None:
        query_grad, key_grad = _rotate(query_grad, key_grad, positions, inv_freq, pair_axis, ctx.adjacent, True)

    # One gradient (or None) per forward argument.
    return query_grad, key_grad, None, None, None, None


_backward_once = once_differentiable(_backward)


class Rotary(nn.Module):
    """
    Rotary positions with one or several axes (time, height and width of a video's patches, say)
    for queries and keys; it has no parameters.  The tables of frequencies and axes are kept as
    buffers that follow the module from device to device; a change of the module's dtype leaves
    them as they are.

    Args:
        head_dim: Size of a head.
        sections: Number of pairs of each axis, in order; None selects one axis with all pairs.
        rotary_dim: Number of features to turn (an even one); None selects twice the sections'
            sum, or head_dim.
        base: Base of the frequencies: pair n of N turns by base ** (-n / N) radians per position.
        axis_ladders: Every axis has frequencies of its own (n counts within its section, and N is
            the section's size) instead of sharing one ladder over all pairs.
        adjacent: Pairs are features (2 n, 2 n + 1) instead of (n, n + rotary_dim / 2).
        device: Device to use.
    """
    def __init__(
        self,
        head_dim: int,
        sections: Optional[Sequence[int]] = None,
        rotary_dim: Optional[int] = None,
        base: float = 10000.0,
        axis_ladders: bool = False,
        adjacent: bool = False,
        device: Any = 'cuda',
        ) -> None:
        super().__init__()
        if rotary_dim is None:
            rotary_dim = 2 * sum(sections) if sections is not None else head_dim
        if rotary_dim % 2 != 0 or not 0 <= rotary_dim <= head_dim:
            raise RuntimeError(f'The rotary dimension must be even and at most {head_dim}, received {rotary_dim}')
        pairs = rotary_dim // 2
        sections = (pairs,) if sections is None else tuple(sections)
        if len(sections) == 0 or min(sections) < 0 or sum(sections) != pairs:
            raise RuntimeError(f'Sections {sections} must sum to half the rotary dimension ({pairs})')
        if not base > 0.0:
            raise RuntimeError(f'The base must be positive, received {base}')
        if pairs > MAX_PAIRS:
            raise RuntimeError(f'At most {MAX_PAIRS} pairs are supported, received {pairs}')

        self.head_dim = head_dim
        self.sections = sections
        self.base = base
        self.axis_ladders = axis_ladders
        self.adjacent = adjacent
        ladders = [[n / size for n in range(size)] for size in sections] if axis_ladders else \
            [[n / max(pairs, 1) for n in range(pairs)]]
        inv_freq = torch.tensor([base ** -step for ladder in ladders for step in ladder], dtype=torch.float64)
        pair_axis = torch.tensor([axis for axis, size in enumerate(sections) for _ in range(size)], dtype=torch.int32)
        # kept as the bits of the float64 values: module.to(torch.bfloat16) casts floating-point buffers
        self.register_buffer('inv_freq_bits', inv_freq.view(torch.int64).to(device), persistent=False)
        self.register_buffer('pair_axis', pair_axis.to(device), persistent=False)

    @property
    def inv_freq(self) -> Tensor:
        return self.inv_freq_bits.view(torch.float64)

    def forward(
        self,
        query: Tensor,
        key: Optional[Tensor] = None,
        positions: Optional[Tensor] = None,
        ) -> Tuple[Tensor, Optional[Tensor]]:
        if query.shape[-1] != self.head_dim:
            raise RuntimeError(f'Expected heads of size {self.head_dim}, received {query.shape[-1]}')
        axes = len(self.sections)
        if axes > 1 or positions is not None:
            assert query.ndim == 4, f'Queries must be [batch, heads, rows, head_dim], received {tuple(query.shape)}'
            positions = _positions_of(positions, axes, query.shape[0], query.shape[2])
        return RotaryAutoGrad.apply(query, key, positions, self.inv_freq, self.pair_axis if axes > 1 else None,
                                    self.adjacent)

    def extra_repr(self) -> str:
        return (f'{self.head_dim}, sections={self.sections}, base={self.base}, axis_ladders={self.axis_ladders}, '
                f'adjacent={self.adjacent}')
