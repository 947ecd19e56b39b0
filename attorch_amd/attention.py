"""
Attention over a sliding window with a few first tokens that stay visible, with PyTorch autodiff
support, running on the gfx950 matrix-core kernels.

The reference's attention layer cannot be constructed (attorch/multi_head_attention_layer.py:77),
so the interface is this package's own: tensors of shape [batch, heads, tokens, head_dim] in any
layout, fewer key heads than query heads, a padded batch or a key/value cache described by the
sequences' lengths, for training steps, prompts and single tokens alike.
"""

import ctypes
from typing import Any, Optional, Tuple

import torch
from torch import Tensor
from torch import nn
from torch.autograd.function import once_differentiable
from torch.nn import functional as F

from . import _lib
from .utils import get_output_dtype

MAX_HEAD_DIM = 128
_NO_STRIDES = (0, 0, 0)


class _Shape(ctypes.Structure):
    """
    at_attention_t of include/attorch_hip.h.
    """
    _fields_ = ([(name, ctypes.c_int64) for name in ('batch', 'heads', 'kv_heads', 'rows', 'keys', 'dim', 'window',
                                                     'sinks')] +
                [('strides', ctypes.c_int64 * 24), ('lengths', ctypes.c_void_p), ('query_lengths', ctypes.c_void_p),
                 ('scale', ctypes.c_float), ('causal', ctypes.c_int), ('dtype', ctypes.c_int),
                 ('lengths_int64', ctypes.c_int)])


def _readable(tensor: Tensor, group: int) -> bool:
    """
    Whether the kernels can read the tensor where it lies: whole features, everything on 16-byte
    boundaries, and a tile's tokens, of `group` heads, within the 31 bits of a buffer offset.
    """
    stride = tensor.stride()
    size = tensor.element_size()
    aligned = 16 // size
    return (stride[3] == 1 and tensor.data_ptr() % 16 == 0 and
            all(st % aligned == 0 or extent <= 1 for st, extent in zip(stride, tensor.shape[:3])) and
            (160 * stride[2] + (group - 1) * stride[1]) * size < (1 << 31) - 1024)


def _for_kernel(tensor: Tensor, dim: int, group: int) -> Tensor:
    """
    The tensor itself where the kernels can read it, otherwise a copy in [batch, tokens, heads, dim]
    order, its features padded with zeros to `dim`.
    """
    if tensor.shape[3] == dim and _readable(tensor, group):
        return tensor
    tensor = tensor.transpose(1, 2)
    if tensor.shape[3] != dim:
        tensor = F.pad(tensor, (0, dim - tensor.shape[3]))
    tensor = tensor.contiguous()
    return (tensor if tensor.data_ptr() % 16 == 0 else tensor.clone()).transpose(1, 2)


def _strides(tensor: Tensor) -> Tuple[int, int, int]:
    """
    Strides of batch, heads and tokens; 0 for an extent of one, whose stride is arbitrary.
    """
    shape, stride = tensor.shape, tensor.stride()
    return (stride[0] if shape[0] > 1 else 0, stride[1] if shape[1] > 1 else 0, stride[2] if shape[2] > 1 else 0)


def _like(tensor: Tensor) -> Tensor:
    """
    New tensor for a gradient of `tensor`: in its layout where that is dense.
    """
    grad = torch.empty_like(tensor)
    if _readable(grad, 1):
        return grad
    batch, heads, tokens, dim = tensor.shape
    return torch.empty((batch, tokens, heads, dim), device=tensor.device, dtype=tensor.dtype).transpose(1, 2)


def _check(query: Tensor, key: Tensor, value: Tensor, lengths: Optional[Tensor], query_lengths: Optional[Tensor],
           window: Optional[int], num_sinks: int, scale: Optional[float]) -> None:
    """
    Refuses what the kernels do not compute, before anything is launched.
    """
    assert query.ndim == 4 and key.ndim == 4 and value.ndim == 4, \
        f'Query, key and value must be [batch, heads, tokens, head_dim], received {tuple(query.shape)}, ' \
        f'{tuple(key.shape)} and {tuple(value.shape)}'
    assert key.shape == value.shape, \
        f'Key ({tuple(key.shape)}) and value ({tuple(value.shape)}) must have the same shape'
    assert query.shape[0] == key.shape[0] and query.shape[3] == key.shape[3], \
        f'Incompatible query ({tuple(query.shape)}) and key ({tuple(key.shape)}) shape'
    assert key.shape[1] > 0 and query.shape[1] > 0 and query.shape[1] % key.shape[1] == 0, \
        f'The number of query heads ({query.shape[1]}) must be a multiple of that of key heads ({key.shape[1]})'
    if query.shape[2] > key.shape[2]:
        raise RuntimeError(f'Queries are the last tokens of their sequences: expected at most {key.shape[2]} of them, '
                           f'as many as keys, received {query.shape[2]}')
    if not 1 <= query.shape[3] <= MAX_HEAD_DIM:
        raise RuntimeError(f'Head dimension {query.shape[3]} is not supported; it must be between 1 and {MAX_HEAD_DIM}')
    if key.dtype is not query.dtype or value.dtype is not query.dtype:
        raise RuntimeError(f'Query, key and value must have the same dtype, received {query.dtype}, {key.dtype} and '
                           f'{value.dtype}')
    if window is not None and window < 1:
        raise RuntimeError(f'The window must hold at least one token, received {window}')
    if num_sinks < 0:
        raise RuntimeError(f'The number of sinks must not be negative, received {num_sinks}')
    if scale is not None and not 0.0 < scale < 3e38:
        raise RuntimeError(f'The scale must be positive and finite, received {scale}')
    for name, counts in (('lengths', lengths), ('query_lengths', query_lengths)):
        if counts is None:
            continue
        if counts.dtype not in (torch.int32, torch.int64):
            raise RuntimeError(f'{name} must be int32 or int64, received {counts.dtype}')
        assert counts.shape == query.shape[:1], \
            f'{name} must have one entry per sequence ({query.shape[0]}), received shape {tuple(counts.shape)}'


def _shape_of(query: Tensor, key: Tensor, value: Tensor, others: Tuple[Tuple[int, int, int], ...],
              counts: Tuple[Optional[Tensor], Optional[Tensor]], options: Tuple[bool, int, int, float]) -> _Shape:
    batch, heads, rows, dim = query.shape
    causal, window, num_sinks, scale = options
    strides = [*_strides(query), *_strides(key), *_strides(value)]
    for other in others:
        strides += other
    some = counts[0] if counts[0] is not None else counts[1]
    return _Shape(batch, heads, key.shape[1], rows, key.shape[2], dim, window, num_sinks,
                  (ctypes.c_int64 * 24)(*strides), _lib.ptr(counts[0]), _lib.ptr(counts[1]), scale, causal,
                  _lib.dtype_id(query.dtype), int(some is not None and some.dtype is torch.int64))


class WindowAttentionAutoGrad(torch.autograd.Function):
    """
    Autodiff for attention over a sliding window with first tokens that stay visible.
    """
    @staticmethod
    def forward(
        ctx: Any,
        query: Tensor,
        key: Tensor,
        value: Tensor,
        lengths: Optional[Tensor] = None,
        query_lengths: Optional[Tensor] = None,
        causal: bool = True,
        window: Optional[int] = None,
        num_sinks: int = 0,
        scale: Optional[float] = None,
        ) -> Tensor:
        """
        Attends every query to the tokens of its sequence that it sees.

        With L and Q the sequence's entries of lengths and query_lengths, query row i is token
        p = max(L - Q, 0) + i of its sequence and sees token j < L if j <= p (or not causal) and
        |p - j| < window (or window is None, or j < num_sinks).  Rows with i >= Q or p >= L are
        padding: they come out as zeros and take no part in the gradients.  What keys and
        values hold where no query of their sequence sees them reaches no result, NaN included.

        Args:
            query: Queries of shape [batch, heads, rows, head_dim], the last tokens of their sequences.
            key: Keys of shape [batch, kv_heads, tokens, head_dim]; kv_heads divides heads, and
                query head n reads key head n // (heads // kv_heads).
            value: Values, shaped like the keys.
            lengths: Optional number of tokens of each sequence (int32 or int64, shape [batch],
                clamped to what the keys hold): the others are padding or unused room of a
                cache. None: all are tokens.
            query_lengths: Optional number of query rows of each sequence that are tokens. None:
                as many as the sequence has tokens for.
            causal: Tokens see no later ones.
            window: Optional number of tokens that a token sees, itself included, to its left (and
                as many to its right if not causal).
            num_sinks: Number of first tokens that are seen outside the window too.
            scale: Factor of the scores; None selects head_dim ** -0.5.

        Returns:
            Output of shape [batch, heads, rows, head_dim], laid out as [batch, rows, heads, head_dim].
        """
        _check(query, key, value, lengths, query_lengths, window, num_sinks, scale)
        _lib.require_same_device('WindowAttention', query, key, value, lengths, query_lengths)
        lib = _lib.load()
        batch, heads, rows, head_dim = query.shape
        if scale is None:
            scale = head_dim ** -0.5

        output_dtype = get_output_dtype(query.dtype, autocast='fp16')
        dim = (head_dim + 7) // 8 * 8
        query_k = _for_kernel(query.to(output_dtype), dim, heads // key.shape[1])
        key_k = _for_kernel(key.to(output_dtype), dim, 1)
        value_k = _for_kernel(value.to(output_dtype), dim, 1)
        counts = (lengths, query_lengths)
        if lengths is not None or query_lengths is not None:
            if lengths is not None and query_lengths is not None and lengths.dtype is not query_lengths.dtype:
                counts = (lengths.long(), query_lengths.long())
            counts = tuple(None if c is None else c.contiguous() for c in counts)

        output = torch.empty((batch, rows, heads, dim), device=query.device, dtype=output_dtype).transpose(1, 2)
        options = (bool(causal), min(window or 0, 1 << 40), min(num_sinks, 1 << 40), scale)
        shape = _shape_of(query_k, key_k, value_k, (_strides(output),) + (_NO_STRIDES,) * 4, counts, options)

        requires_grad = any(ctx.needs_input_grad[:3])
        lse = rest = None
        if requires_grad:
            if output_dtype is not torch.float32:
                rest = torch.empty((batch, rows, heads, dim), device=query.device, dtype=output_dtype)
            pitch = lib.at_attention_row_pitch(rows, heads, key.shape[1])
            lse = torch.empty(batch * key.shape[1] * pitch, device=query.device, dtype=torch.float32)
        workspace = None
        with _lib.device_guard(query):
            workspace_bytes = lib.at_attention_fwd_workspace_bytes(ctypes.byref(shape))
            if workspace_bytes:
                workspace = torch.empty(workspace_bytes, device=query.device, dtype=torch.uint8)
            _lib.check(lib.at_attention_fwd(
                ctypes.byref(shape), _lib.ptr(query_k), _lib.ptr(key_k), _lib.ptr(value_k), _lib.ptr(output), _lib.ptr(lse),
                _lib.ptr(rest), _lib.ptr(workspace), workspace_bytes, _lib.stream_of(query)), 'at_attention_fwd')

        if requires_grad:
            ctx.options = options
            ctx.head_dim = head_dim
            ctx.save_for_backward(query_k, key_k, value_k, output, rest, lse, *counts)
        return output if dim == head_dim else output[..., :head_dim]

    @staticmethod
    @once_differentiable
    def backward(
        ctx: Any,
        output_grad: Tensor,
        ) -> Tuple[Optional[Tensor], ...]:
        """
        Gradients of the queries, keys and values.
        """
        lib = _lib.load()
        query, key, value, output, rest, lse, *counts = ctx.saved_tensors
        _lib.require_same_device('WindowAttention backward', query, output_grad)
        head_dim = ctx.head_dim
        output_grad = _for_kernel(output_grad.to(query.dtype), query.shape[3], query.shape[1] // key.shape[1])
        grads = [_like(tensor) for tensor in (query, key, value)]
        shape = _shape_of(query, key, value,
                          (_strides(output), _strides(output_grad), *(_strides(grad) for grad in grads)), counts,
                          ctx.options)
        workspace_bytes = lib.at_attention_bwd_workspace_bytes(ctypes.byref(shape))
        workspace = torch.empty(workspace_bytes, device=query.device, dtype=torch.uint8)
        with _lib.device_guard(query):
            _lib.check(lib.at_attention_bwd(
                ctypes.byref(shape), _lib.ptr(output_grad), _lib.ptr(query), _lib.ptr(key), _lib.ptr(value), _lib.ptr(output),
                _lib.ptr(rest), _lib.ptr(lse), *(_lib.ptr(grad) for grad in grads), _lib.ptr(workspace), workspace_bytes,
                _lib.stream_of(query)), 'at_attention_bwd')
        if head_dim != query.shape[3]:
            grads = [grad[..., :head_dim] for grad in grads]

        # One gradient (or None) per forward argument.
        return (*grads, None, None, None, None, None, None)


class WindowAttention(nn.Module):
    """
    Attention over a sliding window with a few first tokens that stay visible (see
    WindowAttentionAutoGrad.forward); it has no parameters.

    Args:
        causal: Tokens see no later ones.
        window: Optional number of tokens that a token sees, itself included, to its left (and as
            many to its right if not causal); None for all.
        num_sinks: Number of first tokens that are seen outside the window too.
        scale: Factor of the scores; None selects head_dim ** -0.5.
    """
    def __init__(
        self,
        causal: bool = True,
        window: Optional[int] = None,
        num_sinks: int = 0,
        scale: Optional[float] = None,
        ) -> None:
        super().__init__()
        if window is not None and window < 1:
            raise RuntimeError(f'The window must hold at least one token, received {window}')
        if num_sinks < 0:
            raise RuntimeError(f'The number of sinks must not be negative, received {num_sinks}')
        self.causal = causal
        self.window = window
        self.num_sinks = num_sinks
        self.scale = scale

    def forward(
        self,
        query: Tensor,
        key: Tensor,
        value: Tensor,
        lengths: Optional[Tensor] = None,
        query_lengths: Optional[Tensor] = None,
        ) -> Tensor:
        return WindowAttentionAutoGrad.apply(query, key, value, lengths, query_lengths, self.causal, self.window,
                                             self.num_sinks, self.scale)

    def extra_repr(self) -> str:
        return f'causal={self.causal}, window={self.window}, num_sinks={self.num_sinks}, scale={self.scale}'
