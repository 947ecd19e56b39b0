"""
CPU-only tests of what attention and rotary positions refuse: by the Python layers before anything is
launched, and by the C entry points as negative codes.
"""

import ctypes

import pytest
import torch

import attorch_amd
from attorch_amd import _lib
from attorch_amd.attention import _Shape as AttentionShape
from attorch_amd.rotary import _Shape as RotaryShape
from examples.blocks import TinyGPT, new_tokens


def qkv(batch=2, heads=4, kv_heads=2, rows=5, keys=5, dim=16, dtype=torch.float32):
    return (torch.zeros(batch, heads, rows, dim, dtype=dtype), torch.zeros(batch, kv_heads, keys, dim, dtype=dtype),
            torch.zeros(batch, kv_heads, keys, dim, dtype=dtype))


@pytest.mark.parametrize('tensors', [
    (torch.zeros(2, 4, 16), torch.zeros(2, 2, 5, 16), torch.zeros(2, 2, 5, 16)),                # not 4D
    (torch.zeros(2, 4, 5, 16), torch.zeros(2, 2, 5, 16), torch.zeros(2, 2, 6, 16)),             # key and value differ
    (torch.zeros(2, 4, 5, 16), torch.zeros(1, 2, 5, 16), torch.zeros(1, 2, 5, 16)),             # batch
    (torch.zeros(2, 4, 5, 16), torch.zeros(2, 2, 5, 8), torch.zeros(2, 2, 5, 8)),               # head dimension
    (torch.zeros(2, 4, 5, 16), torch.zeros(2, 3, 5, 16), torch.zeros(2, 3, 5, 16)),             # heads
    (torch.zeros(2, 0, 5, 16), torch.zeros(2, 0, 5, 16), torch.zeros(2, 0, 5, 16)),
])
def test_attention_shapes(tensors) -> None:
    with pytest.raises(AssertionError):
        attorch_amd.WindowAttention()(*tensors)


def test_attention_arguments() -> None:
    apply = attorch_amd.WindowAttentionAutoGrad.apply
    with pytest.raises(RuntimeError, match='last tokens'):
        apply(*qkv(rows=6, keys=5))
    with pytest.raises(RuntimeError, match='Head dimension 136'):
        apply(*qkv(dim=136))
    with pytest.raises(RuntimeError, match='same dtype'):
        q, k, v = qkv()
        apply(q.half(), k, v)
    for options, match in (((True, 0), 'window'), ((True, -1), 'window'), ((True, 4, -1), 'sinks'),
                           ((True, 4, 0, 0.0), 'scale'), ((True, 4, 0, -1.0), 'scale'),
                           ((True, 4, 0, float('inf')), 'scale'), ((True, 4, 0, float('nan')), 'scale')):
        with pytest.raises(RuntimeError, match=match):
            apply(*qkv(), None, None, *options)
    for options, match in (((torch.tensor(True),), 'causal'), ((True, torch.tensor(3)), 'window'),
                           ((True, 3, torch.tensor(1)), 'num_sinks'), ((True, 3, 1, torch.tensor(0.5)), 'scale')):
        with pytest.raises(RuntimeError, match=f'{match} must be a plain value'):
            apply(*qkv(), None, None, *options)
    with pytest.raises(RuntimeError, match='int32 or int64'):
        apply(*qkv(), torch.zeros(2))
    with pytest.raises(AssertionError):
        apply(*qkv(), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(AssertionError):
        apply(*qkv(), None, torch.zeros(2, 1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match='no CPU path'):
        apply(*qkv())
    with pytest.raises(RuntimeError, match='window'):
        attorch_amd.WindowAttention(window=0)
    with pytest.raises(RuntimeError, match='sinks'):
        attorch_amd.WindowAttention(num_sinks=-1)


def test_continued_sequences_of_other_models() -> None:
    tokens, lengths = torch.zeros(1, 3, dtype=torch.int64), torch.tensor([3])
    for options in ({'rotary': True}, {}, {'window': 4}):
        model = TinyGPT(torch.nn, 20, 1, 32, 2, 8, **options)
        with pytest.raises(RuntimeError, match='continued'):
            model.extend(tokens, model.new_cache(1, 8), lengths)


@pytest.mark.parametrize('int_type', [torch.int32, torch.int64])
def test_places_of_new_tokens(int_type) -> None:
    """
    Tokens of continued sequences are counted from their starts and stored where the cache has room; the slots of
    padding are places of the cache too, and a sequence's are all different.
    """
    room, chunk = 12, 5
    lengths = torch.tensor([0, 3, 5, 9, 12, 13, 14, 17, 18, 40, -2], dtype=int_type)
    for given in (None, 0, 2, 5, 9):
        counts = None if given is None else torch.full_like(lengths, given)
        new = new_tokens(lengths, counts, chunk, room)
        wanted = chunk if given is None else min(given, chunk)
        for b, length in enumerate(lengths.tolist()):
            start = max(length - wanted, 0)
            live = [start + i for i in range(wanted) if start + i < min(length, room)]
            assert new.positions[b].tolist() == list(range(start, start + chunk))
            assert new.live[b].tolist() == [i < len(live) for i in range(chunk)]
            assert new.slots[b][new.live[b]].tolist() == live
            assert len(set(new.slots[b].tolist())) == chunk and all(0 <= s < room for s in new.slots[b].tolist())
            assert new.query_lengths[b] == len(live)
            # as attention places its rows
            assert not live or (new.lengths[b] - new.query_lengths[b] == start and new.lengths[b] <= room)


def test_rotary_arguments() -> None:
    q, k = torch.zeros(2, 4, 5, 16), torch.zeros(2, 2, 5, 16)
    freq, axis = torch.ones(8, dtype=torch.float64), torch.zeros(8, dtype=torch.int32)
    positions = torch.zeros(2, 2, 5, dtype=torch.int64)
    apply = attorch_amd.RotaryAutoGrad.apply
    for args in ((q[0], None, None, freq), (q, k[:1], None, freq), (q, k[:, :, :4], None, freq),
                 (q, k, None, torch.ones(9, dtype=torch.float64)), (q, k, None, freq[None]),
                 (q, k, positions, freq, axis[:4]), (q, k, None, freq, axis), (q, k, positions[0, 0], freq, axis),
                 (q, k, positions[:, :, :4], freq, axis), (q, k, positions[:, :1], freq), (q, k, positions[0, 0, :4], freq)):
        with pytest.raises(AssertionError):
            apply(*args)
    for args in ((q, k, torch.zeros(5, requires_grad=True), freq), (q, k, None, freq.clone().requires_grad_())):
        with pytest.raises(RuntimeError, match='no gradients of positions and inv_freq'):
            apply(*args)
    for args, match in (((q.half(), k, None, freq), 'same dtype'), ((q, k, None, freq.float()), 'float64'),
                        ((q, k, positions, freq, axis.long()), 'int32')):
        with pytest.raises(RuntimeError, match=match):
            apply(*args)
    with pytest.raises(RuntimeError, match='no CPU path'):
        apply(q, k, None, freq)
    with pytest.raises(RuntimeError, match='no CPU path'):
        attorch_amd.Rotary(16, device='cpu')(q, k)
    for options, match in (({'rotary_dim': 7}, 'even'), ({'rotary_dim': 18}, 'at most'), ({'sections': (4, 5)}, 'at most'),
                           ({'sections': (4, 2), 'rotary_dim': 16}, 'sum'), ({'sections': (-1, 9)}, 'sum'),
                           ({'base': 0.0}, 'base')):
        with pytest.raises(RuntimeError, match=match):
            attorch_amd.Rotary(16, device='cpu', **options)
    with pytest.raises(RuntimeError, match='heads of size 16'):
        attorch_amd.Rotary(16, device='cpu')(torch.zeros(1, 1, 1, 8))
    with pytest.raises(RuntimeError, match='must be given'):
        attorch_amd.Rotary(16, sections=(4, 4), device='cpu')(q, k)
    with pytest.raises(RuntimeError, match='int32, int64 or float32'):
        attorch_amd.Rotary(16, device='cpu')(q, k, torch.zeros(5, dtype=torch.float64))



def attention_shape(**changes):
    fields = {'batch': 1, 'heads': 4, 'kv_heads': 2, 'rows': 8, 'keys': 8, 'dim': 16, 'window': 0, 'sinks': 0,
              'scale': 0.25, 'causal': 1, 'dtype': 2, 'lengths_int64': 0, **changes}
    strides = fields.pop('strides', [512, 128, 16] * 8)
    return AttentionShape(strides=(ctypes.c_int64 * 24)(*strides), **fields)


def test_attention_codes() -> None:
    lib = _lib.load()
    p = (ctypes.addressof(ctypes.create_string_buffer(4096)) + 63) // 64 * 64
    fwd = lambda s, *a: lib.at_attention_fwd(ctypes.byref(s), *(a or (p, p, p, None, None, p, None, None, None, 0)), None)  # noqa: E731
    for changes, code in (({'batch': -1}, -2), ({'heads': 3}, -2), ({'kv_heads': 0}, -2), ({'rows': 9}, -2),
                          ({'keys': (1 << 29) + 1}, -2), ({'dim': 136}, -2), ({'dim': 0}, -2), ({'dim': 12}, -6),
                          ({'window': -1}, -2), ({'sinks': -1}, -2), ({'scale': 0.0}, -2), ({'scale': float('nan')}, -2),
                          ({'scale': float('inf')}, -2), ({'dtype': 3}, -3), ({'strides': [512, 128, 12] * 8}, -6),
                          ({'strides': [512, -128, 16] * 8}, -2), ({'strides': [1 << 40, 1 << 40, 1 << 40] * 8}, -2),
                          ({'batch': 65536}, -2), ({'rows': 1 << 29, 'keys': 1 << 29}, -2)):
        assert fwd(attention_shape(**changes)) == code, changes
        assert lib.at_attention_bwd(ctypes.byref(attention_shape(**changes)), *[p] * 13, 1 << 20, None) == code, changes
        assert lib.at_attention_fwd_workspace_bytes(ctypes.byref(attention_shape(**changes))) == 0
        assert lib.at_attention_bwd_workspace_bytes(ctypes.byref(attention_shape(**changes))) == 0
    assert lib.at_attention_fwd(None, p, p, p, None, None, p, None, None, None, 0, None) == -1
    assert fwd(attention_shape(), None, p, p, None, None, p, None, None, None, 0) == -1
    assert fwd(attention_shape(), p, p, p, None, None, p + 4, None, None, None, 0) == -6
    assert fwd(attention_shape(batch=0), *[None] * 9, 0) == 0
    # few rows and many keys: pieces in a workspace
    cache = attention_shape(rows=1, keys=100000)
    assert lib.at_attention_fwd_workspace_bytes(ctypes.byref(cache)) > 0
    assert fwd(cache) == -5
    bwd = lambda *a: lib.at_attention_bwd(ctypes.byref(attention_shape()), *a, None)  # noqa: E731
    assert bwd(*[p] * 12, None, 0) == -5 and bwd(*[p] * 13, 64) == -5
    assert bwd(None, *[p] * 12, 1 << 20) == -1 and bwd(p, p, p, p + 8, *[p] * 9, 1 << 20) == -6
    assert lib.at_attention_row_pitch(5, 4, 2) == 64 and lib.at_attention_row_pitch(33, 4, 2) == 128
    assert lib.at_attention_row_pitch(33, 4, 3) == 0


def test_attention_codes_of_misaligned_workspaces() -> None:
    lib = _lib.load()
    p = (ctypes.addressof(ctypes.create_string_buffer(4096)) + 63) // 64 * 64
    cache = ctypes.byref(attention_shape(rows=1, keys=100000))
    size = lib.at_attention_fwd_workspace_bytes(cache)
    assert lib.at_attention_fwd(cache, p, p, p, None, None, p, None, None, p + 8, size, None) == -6
    assert lib.at_attention_bwd(ctypes.byref(attention_shape()), *[p] * 12, p + 8, 1 << 20, None) == -6


@pytest.mark.parametrize('causal', [0, 1])
@pytest.mark.parametrize('window, sinks', [(0, 0), (20, 0), (20, 4), (20, 300), (0, 4)])
def test_attention_codes_of_empty_batches(window, sinks, causal) -> None:
    """No sequence, but rows that reach beyond the window: nothing to do, and no workspace to do it in."""
    lib = _lib.load()
    shape = ctypes.byref(attention_shape(batch=0, rows=700, keys=700, window=window, sinks=sinks, causal=causal,
                                         strides=[11200, 11200, 16] * 8))
    assert lib.at_attention_fwd_workspace_bytes(shape) == 0 and lib.at_attention_bwd_workspace_bytes(shape) == 0
    assert lib.at_attention_fwd(shape, *[None] * 9, 0, None) == 0
    assert lib.at_attention_bwd(shape, *[None] * 13, 0, None) == 0


def test_rotary_codes() -> None:
    lib = _lib.load()
    p = ctypes.addressof(ctypes.create_string_buffer(4096))
    base = {'batch': 1, 'rows': 2, 'q_heads': 2, 'k_heads': 1, 'dim': 8, 'pairs': 4, 'axes': 1, 'position_type': 0}

    def call(changes, *args):
        shape = RotaryShape(**{**base, **changes})
        return lib.at_rotary(ctypes.byref(shape), *(args or (p, p, p, p, p, p, p)), None)

    for changes, code in (({'batch': -1}, -2), ({'pairs': 5}, -2), ({'dim': 0}, -2), ({'axes': 0}, -2),
                          ({'position_type': 3}, -2), ({'dtype': 5}, -3), ({'q_heads': 1 << 17}, -2),
                          ({'dim': 2048, 'pairs': 513}, -2), ({'rows': (1 << 30) + 1}, -2)):
        assert call(changes) == code, changes
    assert call({}, None, p, p, p, p, p, p) == -1 and call({}, p, None, p, p, p, p, p) == -1
    assert call({}, p, p, p, p, p, None, p) == -1 and call({'axes': 2}, p, p, p, p, None, p, p) == -1
    assert call({'axes': 2}, p, p, p, p, p, p, None) == -1
    assert call({'batch': 0}, None, None, None, None, None, None, None) == 0
    assert lib.at_rotary(None, p, p, p, p, p, p, p, None) == -1
