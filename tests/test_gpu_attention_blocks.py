"""
Rotary positions and window attention together, as a language model uses them: the GPT block with
them against the same arithmetic on torch (loss and every parameter gradient), and sequences
continued from a cache of keys and values against whole ones.
"""

import pytest
import torch

import attorch_amd
import attorch_amd.nn as fused_nn
from examples.blocks import TinyGPT
from oracle.attention import attention, rotary
from .helpers import randn
from .test_gpu_attention import assert_within
from .test_gpu_examples import AMP_CASES, _assert_fp32_grads, _compare_grads, _pair

pytestmark = pytest.mark.gpu

OPTIONS = {'rotary': True, 'kv_heads': 2, 'window': 20, 'num_sinks': 3}


@pytest.mark.parametrize('dtype, rtol, atol', [(torch.float32, 2e-3, 2e-3), (torch.bfloat16, 6e-2, 6e-2)])
@pytest.mark.parametrize('options', [OPTIONS, {'window': 20}, {'rotary': True}, {'kv_heads': 1}])
def test_tiny_gpt(options, dtype, rtol, atol) -> None:
    ours, theirs = _pair(TinyGPT, dtype, 1000, 2, 128, 4, 64, **options)
    tokens = torch.randint(0, 1000, (4, 64), device='cuda')
    torch.testing.assert_close(ours(tokens).float(), theirs(tokens).float(), rtol=rtol, atol=atol)
    loss, ref = ours(tokens, return_loss=True), theirs(tokens, return_loss=True)
    torch.testing.assert_close(loss.float(), ref.float(), rtol=rtol, atol=atol)
    loss.backward()
    ref.backward()
    _compare_grads(ours, theirs, rtol, atol)


@pytest.mark.parametrize('amp_dtype, rtol, atol', AMP_CASES)
def test_tiny_gpt_under_autocast(amp_dtype, rtol, atol) -> None:
    ours, theirs = _pair(TinyGPT, torch.float32, 1000, 2, 128, 4, 64, **OPTIONS)
    tokens = torch.randint(0, 1000, (4, 64), device='cuda')
    with torch.autocast('cuda', dtype=amp_dtype):
        loss, ref = ours(tokens, return_loss=True), theirs(tokens, return_loss=True)
    torch.testing.assert_close(loss, ref.float(), rtol=rtol, atol=atol)
    loss.backward()
    ref.backward()
    _assert_fp32_grads(ours)
    _compare_grads(ours, theirs, rtol, atol, low_precision=True)


def test_continued_sequences() -> None:
    """
    Prompts of different lengths, then chunks and single tokens, give the logits of the whole sequences:
    fp32, so that the two differ by rounding only.  The cache starts out as garbage.
    """
    torch.manual_seed(3)
    model = TinyGPT(fused_nn, 500, 2, 128, 4, **OPTIONS).to('cuda')
    tokens = torch.randint(0, 500, (3, 60), device='cuda')
    with torch.no_grad():
        whole = model(tokens)
        cache = model.new_cache(3, 100)
        for pair in cache:
            for t in pair:
                t.fill_(float('nan'))
        done = 0
        for step in (33, 9, 1, 1, 7, 1, 1, 1, 6):
            lengths = torch.full((3,), done + step, device='cuda')
            logits = model.extend(tokens[:, done:done + step], cache, lengths)
            # sums of up to 128 products of rounded values differ in order only: 1e-4 of logits of order 1
            torch.testing.assert_close(logits, whole[:, done:done + step], rtol=1e-4, atol=1e-4)
            done += step
        assert done == 60
    # sequences of different lengths, one token each
    lengths = torch.tensor([41, 60, 50], device='cuda')
    with torch.no_grad():
        last = tokens.gather(1, lengths[:, None] - 1)
        logits = model.extend(last, cache, lengths)
        torch.testing.assert_close(logits[:, 0], whole[torch.arange(3), lengths - 1], rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
def test_rotary_and_attention_layers(dtype) -> None:
    """
    Both layers in a row against the float64 oracles, the second fed with what the first returned;
    the gradient goes back through both.  Two axes (height and width of patches), not causal.
    """
    q, k, v, dout = (randn((2, n, 150, 48), s, dtype) for n, s in ((4, 1), (2, 2), (2, 3), (4, 4)))
    step = torch.arange(150)
    positions = torch.stack([step // 12, step % 12])
    turn, core = attorch_amd.Rotary(48, sections=(12, 12), axis_ladders=True), attorch_amd.WindowAttention(causal=False, window=70)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    turned = turn(leaves[0], leaves[1], positions.cuda())
    out = core(*turned, leaves[2])
    grads = torch.autograd.grad(out, [*turned, *leaves], dout.cuda())
    ladder = 10000.0 ** (torch.arange(12, dtype=torch.float64) / -12)
    tables = (positions[:, None].expand(2, 2, 150), torch.cat([ladder, ladder]), torch.arange(24) // 12)
    for x, y in zip(turned, (q, k)):
        assert_within(x, rotary(y, *tables), 'turned')
    expected = attention(turned[0].detach().cpu(), turned[1].detach().cpu(), v, dout, causal=False, window=70)
    assert_within(out, expected['out'], 'output')
    for grad, name in zip((grads[0], grads[1], grads[4]), ('dq', 'dk', 'dv')):
        assert_within(grad, expected[name], name)
    for grad, inner, name in zip(grads[2:4], grads[:2], ('query', 'key')):
        assert_within(grad, rotary(inner.cpu(), *tables, inverse=True), f'{name} gradient')


@pytest.mark.parametrize('int_type', [torch.int32, torch.int64])
def test_prompts_of_different_lengths(int_type) -> None:
    """
    Padded prompts, chunks and single tokens of sequences that all grow at a pace of their own, one of them
    empty at first, give the logits of the whole sequences, and padding leaves the cache as it is: what was
    not written is still NaN, and the rest does not change.
    """
    torch.manual_seed(3)
    model = TinyGPT(fused_nn, 500, 2, 128, 4, **OPTIONS).to('cuda')
    room = 50
    tokens = torch.randint(0, 500, (4, room), device='cuda')
    done = [0, 0, 0, 0]
    with torch.no_grad():
        whole = model(tokens)
        cache = model.new_cache(4, room)
        for pair in cache:
            for t in pair:
                t.fill_(float('nan'))
        # new tokens of each sequence, and whether their numbers are given (otherwise a sequence's length says)
        for step, counted in (((33, 5, 0, 20), False), ((2, 0, 7, 9), True), ((1, 0, 1, 0), True), ((1, 1, 1, 1), False),
                              ((0, 40, 3, 12), True), ((13, 4, 1, 8), True)):
            before = [[t.clone() for t in pair] for pair in cache]
            chunk = torch.full((4, max(step)), 499, device='cuda')
            for b, n in enumerate(step):
                chunk[b, :n] = tokens[b, done[b]:done[b] + n]
            done = [d + n for d, n in zip(done, step)]
            lengths = torch.tensor(done, device='cuda', dtype=int_type)
            logits = model.extend(chunk, cache, lengths,
                                  torch.tensor(step, device='cuda', dtype=int_type) if counted else None)
            for b, n in enumerate(step):
                torch.testing.assert_close(logits[b, :n], whole[b, done[b] - n:done[b]], rtol=1e-4, atol=1e-4)
            for pair, old in zip(cache, before):
                for t, o in zip(pair, old):
                    for b, n in enumerate(step):
                        assert torch.isfinite(t[b, :, :done[b]]).all() and torch.isnan(t[b, :, done[b]:]).all()
                        assert torch.equal(t[b, :, :done[b] - n], o[b, :, :done[b] - n])
    assert done == [50, 50, 13, 50]


def test_sequences_that_fill_the_cache() -> None:
    """Tokens that find no room change nothing: neither what is stored nor the logits of those that do."""
    torch.manual_seed(3)
    model = TinyGPT(fused_nn, 500, 2, 128, 4, **OPTIONS).to('cuda')
    tokens = torch.randint(0, 500, (3, 40), device='cuda')
    with torch.no_grad():
        whole = model(tokens)
        cache = model.new_cache(3, 32)
        model.extend(tokens[:, :28], cache, torch.full((3,), 28, device='cuda'))
        logits = model.extend(tokens[:, 28:36], cache, torch.tensor([36, 32, 30], device='cuda'),
                              torch.tensor([8, 4, 2], device='cuda'))
        for b, n in enumerate((4, 4, 2)):
            torch.testing.assert_close(logits[b, :n], whole[b, 28:28 + n], rtol=1e-4, atol=1e-4)
        before = [[t.clone() for t in pair] for pair in cache]
        model.extend(tokens[:, 36:37], cache, torch.tensor([37, 33, 40], device='cuda'))
        for pair, old in zip(cache, before):
            for t, o in zip(pair, old):
                assert torch.equal(t[:2], o[:2]) and torch.equal(t[2, :, :30], o[2, :, :30])


@pytest.mark.parametrize('amp_dtype, rtol, atol', AMP_CASES)
@pytest.mark.parametrize('cache_dtype', [torch.float32, torch.float16, torch.bfloat16])
def test_continued_sequences_under_autocast(cache_dtype, amp_dtype, rtol, atol) -> None:
    """The cache may be of the weights' type or of a smaller one."""
    torch.manual_seed(3)
    model = TinyGPT(fused_nn, 500, 2, 128, 4, **OPTIONS).to('cuda')
    tokens = torch.randint(0, 500, (2, 40), device='cuda')
    with torch.no_grad(), torch.autocast('cuda', dtype=amp_dtype):
        whole = model(tokens)
        cache = [tuple(t.to(cache_dtype) for t in pair) for pair in model.new_cache(2, 40)]
        done = 0
        for step in (33, 1, 6):
            logits = model.extend(tokens[:, done:done + step], cache, torch.full((2,), done + step, device='cuda'))
            torch.testing.assert_close(logits.float(), whole[:, done:done + step].float(), rtol=rtol, atol=atol)
            done += step
