"""
Attention over a sliding window with a few first tokens that stay visible, with PyTorch autodiff
support, running on the gfx950 matrix-core kernels.

The reference's attention layer cannot be constructed (attorch/multi_head_attention_layer.py:77),
so the interface is this package's own: tensors of shape [batch, heads, tokens, head_dim] in any
layout, fewer key heads than query heads, a padded batch or a key/value cache described by the
sequences' lengths, for training steps, prompts and single tokens alike.
"""

import ctypes
import functools
from typing import Any, Optional, Sequence, Tuple

import torch
from torch import Tensor
from torch import nn
from torch.autograd.function import once_differentiable
from torch.nn import functional as F

from . import _lib
from .utils import get_output_dtype

MAX_HEAD_DIM = 128


class _Shape(ctypes.Structure):
    """
    at_attention_t of include/attorch_hip.h.
    """
    _fields_ = ([(name, ctypes.c_int64) for name in ('batch', 'heads', 'kv_heads', 'rows', 'keys', 'dim', 'window',
                                                     'sinks')] +
                [('strides', ctypes.c_int64 * 24), ('scale', ctypes.c_float), ('causal', ctypes.c_int),
                 ('dtype', ctypes.c_int), ('lengths_int64', ctypes.c_int)])


# A tensor's layout: (shape, stride, dtype, whether its first byte lies on a 16-byte boundary)
Layout = Tuple[torch.Size, Tuple[int, ...], torch.dtype, bool]


def _layout(tensor: Tensor) -> Layout:
    return tensor.shape, tensor.stride(), tensor.dtype, tensor.data_ptr() % 16 == 0


def _readable(layout: Layout, group: int) -> bool:
    """
    Whether the kernels can read a tensor where it lies: whole vectors of features, everything on
    16-byte boundaries, and a tile's tokens, of `group` heads, within the 31 bits of a buffer offset.
    """
    shape, stride, dtype, aligned = layout
    size = dtype.itemsize
    return (aligned and stride[3] == 1 and shape[3] % 8 == 0 and
            all(st * size % 16 == 0 or extent <= 1 for st, extent in zip(stride, shape[:3])) and
            (160 * stride[2] + (group - 1) * stride[1]) * size < (1 << 31) - 1024)


def _for_kernel(tensor: Tensor, dtype: torch.dtype, group: int) -> Tensor:
    """
    The tensor itself where the kernels can read it, otherwise a copy in [batch, tokens, heads, dim]
    order, its features padded with zeros to whole vectors.
    """
    tensor = tensor.to(dtype)
    if _readable(_layout(tensor), group):
        return tensor
    return F.pad(tensor.transpose(1, 2), (0, -tensor.shape[3] % 8)).clone(
        memory_format=torch.contiguous_format).transpose(1, 2)


def _strides(shape: Sequence[int], stride: Sequence[int]) -> Tuple[int, int, int]:
    """
    Strides of batch, heads and tokens; 0 for an extent of one, whose stride is arbitrary.
    """
    return (stride[0] if shape[0] > 1 else 0, stride[1] if shape[1] > 1 else 0, stride[2] if shape[2] > 1 else 0)


def _check(query: Layout, key: Layout, value: Layout, lengths: Optional[Layout], query_lengths: Optional[Layout],
           causal: bool, window: Optional[int], num_sinks: int, scale: Optional[float]) -> None:
    """
    Refuses what the kernels do not compute, before anything is launched.
    """
    for name, option in (('causal', causal), ('window', window), ('num_sinks', num_sinks), ('scale', scale)):
        if isinstance(option, Tensor):      # its value could change behind the layers' back
            raise RuntimeError(f'{name} must be a plain value, received a tensor')
    (q, _, dtype, _), (k, _, k_dtype, _), (v, _, v_dtype, _) = query, key, value
    assert len(q) == 4 and len(k) == 4 and len(v) == 4, \
        f'Query, key and value must be [batch, heads, tokens, head_dim], received {tuple(q)}, {tuple(k)} and {tuple(v)}'
    assert k == v, f'Key ({tuple(k)}) and value ({tuple(v)}) must have the same shape'
    assert q[0] == k[0] and q[3] == k[3], f'Incompatible query ({tuple(q)}) and key ({tuple(k)}) shape'
    assert k[1] > 0 and q[1] > 0 and q[1] % k[1] == 0, \
        f'The number of query heads ({q[1]}) must be a multiple of that of key heads ({k[1]})'
    if q[2] > k[2]:
        raise RuntimeError(f'Queries are the last tokens of their sequences: expected at most {k[2]} of them, '
                           f'as many as keys, received {q[2]}')
    if not 1 <= q[3] <= MAX_HEAD_DIM:
        raise RuntimeError(f'Head dimension {q[3]} is not supported; it must be between 1 and {MAX_HEAD_DIM}')
    if k_dtype is not dtype or v_dtype is not dtype:
        raise RuntimeError(f'Query, key and value must have the same dtype, received {dtype}, {k_dtype} and {v_dtype}')
    if window is not None and window < 1:
        raise RuntimeError(f'The window must hold at least one token, received {window}')
    if num_sinks < 0:
        raise RuntimeError(f'The number of sinks must not be negative, received {num_sinks}')
    if scale is not None and not 0.0 < scale < 1e38:
        raise RuntimeError(f'The scale must be positive and finite, received {scale}')
    for name, counts in (('lengths', lengths), ('query_lengths', query_lengths)):
        if counts is None:
            continue
        if counts[2] not in (torch.int32, torch.int64):
            raise RuntimeError(f'{name} must be int32 or int64, received {counts[2]}')
        assert tuple(counts[0]) == (q[0],), \
            f'{name} must have one entry per sequence ({q[0]}), received shape {tuple(counts[0])}'


class _Plan:
    """
    What a forward call of given layouts and options passes on: nothing in it belongs to a tensor.
    """
    __slots__ = ('direct', 'options', 'dtype', 'shape', 'ref', 'group', 'scale', 'output_shape', 'output_stride', 'saved',
                 'counts_dtype', 'rest_bytes', 'kept_bytes', 'workspace_bytes', 'like_inputs', 'grad_strides')


@functools.lru_cache(maxsize=4096)
def _forward_plan(query: Layout, key: Layout, value: Layout, lengths: Optional[Layout], query_lengths: Optional[Layout],
                  causal: bool, window: Optional[int], num_sinks: int, scale: Optional[float],
                  dtype: torch.dtype, device: int) -> _Plan:
    """
    Checks the arguments and describes the call; `dtype` is the one to compute in, and the workspace
    depends on the device.  Remembered by layouts and options, since a program repeats few of them and
    the description takes longer than a small call's kernels.
    """
    _check(query, key, value, lengths, query_lengths, causal, window, num_sinks, scale)
    batch, heads, rows, dim = query[0]
    kv_heads, keys = key[0][1:3]
    plan = _Plan()
    plan.options, plan.dtype = (causal, window, num_sinks, scale), dtype
    plan.group = heads // kv_heads
    plan.scale = dim ** -0.5 if scale is None else scale
    counts = [c for c in (lengths, query_lengths) if c is not None]
    plan.direct = (query[2] is dtype and _readable(query, plan.group) and _readable(key, 1) and _readable(value, 1) and
                   all(c[1] == (1,) or batch <= 1 for c in counts) and len({c[2] for c in counts}) <= 1)
    if not plan.direct:
        return plan
    plan.output_shape, plan.output_stride = (batch, heads, rows, dim), (rows * heads * dim, dim, heads * dim, 1)
    strides = [*_strides(*query[:2]), *_strides(*key[:2]), *_strides(*value[:2]), *plan.output_stride[:3]]
    plan.shape = _Shape(batch, heads, kv_heads, rows, keys, dim, min(window or 0, 1 << 40), min(num_sinks, 1 << 40),
                        (ctypes.c_int64 * 24)(*strides), plan.scale, bool(causal), _lib.dtype_id(dtype),
                        int(bool(counts) and counts[0][2] is torch.int64))
    plan.ref = ctypes.byref(plan.shape)
    lib = _lib.load()
    plan.workspace_bytes = lib.at_attention_fwd_workspace_bytes(plan.ref)
    # what the backward pass needs, in one tensor: what the output's rounding leaves over, and the rows' sums
    plan.rest_bytes = 0 if dtype is torch.float32 else (batch * rows * heads * dim * dtype.itemsize + 255) // 256 * 256
    plan.kept_bytes = plan.rest_bytes + 4 * batch * kv_heads * lib.at_attention_row_pitch(rows, heads, kv_heads)
    plan.counts_dtype = counts[0][2] if counts else None
    plan.saved = ((query[0], key[0], value[0], plan.output_shape, (plan.kept_bytes,)),
                  (query[1], key[1], value[1], plan.output_stride, (1,)))
    # gradients take the inputs' layouts where these are dense and [batch, tokens, heads, dim] otherwise
    plan.like_inputs, plan.grad_strides = [], []
    for shape, stride, _, _ in (query, key, value):
        grad = torch.empty_like(torch.empty_strided(shape, stride, dtype=dtype, device='meta'))
        like = _readable((shape, grad.stride(), dtype, True), 1)
        plan.like_inputs.append(like)
        plan.grad_strides += _strides(shape, grad.stride() if like else
                                      (shape[2] * shape[1] * dim, dim, shape[1] * dim, 1))
    return plan


def _planned(what: str, query: Tensor, key: Tensor, value: Tensor, lengths: Optional[Tensor],
             query_lengths: Optional[Tensor], causal: bool, window: Optional[int], num_sinks: int, scale: Optional[float],
             dtype: torch.dtype) -> Tuple[_Plan, Tensor, Tensor, Tensor, Optional[Tensor], Optional[Tensor]]:
    """
    Description of a call and the tensors that it is of: copies of those that the kernels cannot read
    where they lie.
    """
    device = query.get_device()
    counts = (None if lengths is None else _layout(lengths), None if query_lengths is None else _layout(query_lengths))
    plan = _forward_plan(_layout(query), _layout(key), _layout(value), *counts, causal, window, num_sinks, scale, dtype, device)
    _lib.require_same_device(what, query, key, value, lengths, query_lengths)
    if not plan.direct:
        query, key, value = (_for_kernel(t, dtype, g) for t, g in ((query, plan.group), (key, 1), (value, 1)))
        lengths, query_lengths = (None if c is None else c.long().contiguous() for c in (lengths, query_lengths))
        counts = (None if lengths is None else _layout(lengths), None if query_lengths is None else _layout(query_lengths))
        plan = _forward_plan(_layout(query), _layout(key), _layout(value), *counts, causal, window, num_sinks, plan.scale, dtype,
                             device)
        if not plan.direct:
            raise RuntimeError(f'{what}: a tile of {query.shape[1]} heads is more than the kernels can address')
    return plan, query, key, value, lengths, query_lengths


@functools.lru_cache(maxsize=4096)
def _backward_plan(forward: _Plan, output_grad: Layout, dtype: torch.dtype, device: int) -> Optional[Tuple[_Shape, int]]:
    """
    Description of the backward call of a forward one, and its workspace in bytes; None where the
    kernels cannot read the output's gradient.
    """
    if output_grad[2] is not dtype or not _readable(output_grad, forward.group):
        return None
    shape = _Shape.from_buffer_copy(forward.shape)
    shape.strides = (ctypes.c_int64 * 24)(*shape.strides[:12], *_strides(*output_grad[:2]), *forward.grad_strides)
    return shape, _lib.load().at_attention_bwd_workspace_bytes(ctypes.byref(shape))


def _as_saved(plan: _Plan, query: Tensor, key: Tensor, value: Tensor, output: Tensor, kept: Tensor,
              lengths: Optional[Tensor], query_lengths: Optional[Tensor]) -> bool:
    """
    Whether saved tensors are laid out as the plan has them.
    """
    device = query.get_device()
    for counts in (lengths, query_lengths):
        if counts is not None and not (counts.is_contiguous() and counts.get_device() == device and
                                       counts.dtype is plan.counts_dtype):
            return False
    return (((query.shape, key.shape, value.shape, output.shape, kept.shape),
             (query.stride(), key.stride(), value.stride(), output.stride(), kept.stride())) == plan.saved and
            query.dtype is key.dtype is value.dtype is output.dtype is plan.dtype and
            device == key.get_device() == value.get_device() == output.get_device() == kept.get_device() and
            (query.data_ptr() | key.data_ptr() | value.data_ptr() | output.data_ptr() | kept.data_ptr()) % 16 == 0)


def _stored_output(plan: _Plan, query: Tensor, output: Tensor, kept: Tensor) -> Tuple[Tensor, Tensor]:
    """
    The output and what was kept beside it as the forward call stored them.
    """
    if (output.device != query.device or kept.device != query.device or output.shape != plan.output_shape or
            kept.shape != (plan.kept_bytes,) or kept.dtype is not torch.uint8):
        raise RuntimeError('WindowAttention backward: saved tensors came back on another device or in another shape')
    if output.stride() != plan.output_stride or output.dtype is not plan.dtype or output.data_ptr() % 16 != 0:
        output = torch.empty_strided(plan.output_shape, plan.output_stride, device=query.device, dtype=plan.dtype).copy_(output)
    if kept.stride() != (1,) or kept.data_ptr() % 16 != 0:
        kept = kept.clone(memory_format=torch.contiguous_format)
    return output, kept


def _gradient_of(tensor: Tensor, like: bool) -> Tensor:
    """
    New tensor for a gradient: in the layout of `tensor`, or as [batch, tokens, heads, dim].
    """
    if like:
        return torch.empty_like(tensor)
    batch, heads, tokens, dim = tensor.shape
    return torch.empty((batch, tokens, heads, dim), device=tensor.device, dtype=tensor.dtype).transpose(1, 2)


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
            query: Queries of shape [batch, heads, rows, head_dim], the last tokens of their sequences. They,
                the keys and the values must have one dtype; autocast casts them to its own.
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
        output_dtype = get_output_dtype(query.dtype, autocast='fp16')
        if not query.dtype is key.dtype is value.dtype is output_dtype and torch.is_autocast_enabled('cuda'):
            query, key, value = (t.to(output_dtype) for t in (query, key, value))
        given = query.shape
        plan, query, key, value, lengths, query_lengths = _planned(
            'WindowAttention', query, key, value, lengths, query_lengths, causal, window, num_sinks, scale, output_dtype)

        head_dim = given[3]

        # not as a view: autograd refuses to change those of a Function in place
        output = torch.empty_strided(plan.output_shape, plan.output_stride, device=query.device, dtype=output_dtype)
        kept = rest = lse = workspace = None
        needs_grad = ctx.needs_input_grad
        if needs_grad[0] or needs_grad[1] or needs_grad[2]:
            kept = torch.empty(plan.kept_bytes, device=query.device, dtype=torch.uint8)
            rest = kept.data_ptr()
            lse = rest + plan.rest_bytes
        if plan.workspace_bytes:
            workspace = torch.empty(plan.workspace_bytes, device=query.device, dtype=torch.uint8)
        with _lib.device_guard(query):
            _lib.check(_lib.load().at_attention_fwd(
                plan.ref, query.data_ptr(), key.data_ptr(), value.data_ptr(),
                None if lengths is None else lengths.data_ptr(),
                None if query_lengths is None else query_lengths.data_ptr(), output.data_ptr(), lse, rest,
                None if workspace is None else workspace.data_ptr(), plan.workspace_bytes, _lib.stream_of(query)),
                'at_attention_fwd')

        if kept is not None:
            ctx.plan = plan
            ctx.head_dim = head_dim
            ctx.save_for_backward(query, key, value, output, kept, lengths, query_lengths)
        if output.shape[3] == head_dim:
            return output
        batch, heads, rows, _ = plan.output_shape
        narrow = torch.empty_strided((batch, heads, rows, head_dim), (rows * heads * head_dim, head_dim, heads * head_dim, 1),
                                     device=query.device, dtype=output_dtype)
        return narrow.copy_(output[..., :head_dim])

    @staticmethod
    def backward(
        ctx: Any,
        output_grad: Tensor,
        ) -> Tuple[Optional[Tensor], ...]:
        """
        Gradients of the queries, keys and values.
        """
        # under create_graph the gradients are marked as not differentiable again
        return _backward_once(ctx, output_grad) if torch.is_grad_enabled() else _backward(ctx, output_grad)


def _backward(ctx: Any, output_grad: Tensor) -> Tuple[Optional[Tensor], ...]:
    query, key, value, output, kept, lengths, query_lengths = ctx.saved_tensors
    # hooks may return saved tensors in other layouts than they were saved in
    forward = ctx.plan
    if not _as_saved(forward, query, key, value, output, kept, lengths, query_lengths):
        forward, query, key, value, lengths, query_lengths = _planned(
            'WindowAttention backward', query, key, value, lengths, query_lengths, *forward.options, forward.dtype)
        output, kept = _stored_output(forward, query, output, kept)
    device = query.get_device()
    if output_grad.get_device() != device:
        _lib.require_same_device('WindowAttention backward', query, output_grad)
    plan = _backward_plan(forward, _layout(output_grad), query.dtype, device)
    if plan is None:
        output_grad = _for_kernel(output_grad, query.dtype, forward.group)
        plan = _backward_plan(forward, _layout(output_grad), query.dtype, device)
        if plan is None:
            raise RuntimeError(f'WindowAttention backward: a tile of {query.shape[1]} heads is more than the kernels can address')
    shape, workspace_bytes = plan
    like = forward.like_inputs
    query_grad, key_grad, value_grad = \
        _gradient_of(query, like[0]), _gradient_of(key, like[1]), _gradient_of(value, like[2])
    workspace = torch.empty(workspace_bytes, device=query.device, dtype=torch.uint8)
    rest = kept.data_ptr()
    with _lib.device_guard(query):
        _lib.check(_lib.load().at_attention_bwd(
            ctypes.byref(shape), output_grad.data_ptr(), query.data_ptr(), key.data_ptr(), value.data_ptr(),
            None if lengths is None else lengths.data_ptr(),
            None if query_lengths is None else query_lengths.data_ptr(), output.data_ptr(), rest,
            rest + forward.rest_bytes, query_grad.data_ptr(), key_grad.data_ptr(), value_grad.data_ptr(),
            workspace.data_ptr(), workspace_bytes, _lib.stream_of(query)), 'at_attention_bwd')
    head_dim = ctx.head_dim
    if head_dim != query.shape[3]:
        query_grad, key_grad, value_grad = (grad[..., :head_dim] for grad in (query_grad, key_grad, value_grad))

    # One gradient (or None) per forward argument.
    return query_grad, key_grad, value_grad, None, None, None, None, None, None


_backward_once = once_differentiable(_backward)


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
