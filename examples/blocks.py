"""
The callers on either side of the layer-kernel hot path, as small models with synthetic inputs:
an MLP classifier (Linear+ReLU -> Linear -> CrossEntropy), a ResNet basic block
(conv -> BN+ReLU -> conv -> BN + residual + ReLU) and a GPT-style transformer block with a
language-model head (LayerNorm -> attention -> Linear+GELU -> Linear -> CrossEntropy).  They
follow the structure of attorch's examples (examples/mnist/mlp.py:14-50,
examples/imagenette/resnet.py:14-104, examples/wikitext-2/gpt.py:15-135), with the datasets
replaced by random tensors.

Each model takes `backend`: the module namespace its layers come from, either `attorch_amd.nn`
or `torch.nn`.  Fused options that only the former has (act_func of Linear / BatchNorm2d,
pre_act_add of BatchNorm2d) are spelled out as separate torch layers for the latter, and
`load_from` copies the parameters of one variant into the other so the two can be compared.
"""

from typing import List, NamedTuple, Optional, Tuple

import torch
from torch import Tensor
from torch import nn
from torch.nn import functional as F


def _is_fused(backend) -> bool:
    return getattr(backend, '__name__', '') == 'attorch_amd.nn'


class FusedLinear(nn.Module):
    """Linear followed by an activation: one fused layer on attorch_amd, two layers on torch."""
    def __init__(self, backend, in_dim: int, out_dim: int, act: Optional[str]) -> None:
        super().__init__()
        self.fused = _is_fused(backend)
        torch_act = {'relu': nn.ReLU, 'gelu': nn.GELU, None: nn.Identity}[act]
        if self.fused:
            self.linear = backend.Linear(in_dim, out_dim, act_func=act)
            self.act = nn.Identity()
        else:
            self.linear = backend.Linear(in_dim, out_dim)
            self.act = torch_act()

    def forward(self, input: Tensor) -> Tensor:
        return self.act(self.linear(input))

    def load_from(self, other: 'FusedLinear') -> None:
        weight = other.linear.weight.detach()
        if self.fused != other.fused:       # [in, out] on one side, [out, in] on the other
            weight = weight.T
        with torch.no_grad():
            self.linear.weight.copy_(weight)
            self.linear.bias.copy_(other.linear.bias)


class MLPClassifier(nn.Module):
    """Linear+ReLU hidden layers, a Linear head and the mean cross-entropy loss."""
    def __init__(self, backend, in_dim: int = 784, hidden_dim: int = 128, depth: int = 1,
                 num_classes: int = 10) -> None:
        super().__init__()
        dims = [in_dim] + [hidden_dim] * depth
        self.hidden = nn.ModuleList(FusedLinear(backend, a, b, 'relu') for a, b in zip(dims, dims[1:]))
        self.head = FusedLinear(backend, hidden_dim, num_classes, None)
        self.loss_func = backend.CrossEntropyLoss()

    def forward(self, input: Tensor, target: Optional[Tensor] = None) -> Tensor:
        output = input.flatten(start_dim=1)
        for layer in self.hidden:
            output = layer(output)
        output = self.head(output)
        return output if target is None else self.loss_func(output, target)

    def load_from(self, other: 'MLPClassifier') -> None:
        for mine, theirs in zip(list(self.hidden) + [self.head], list(other.hidden) + [other.head]):
            mine.load_from(theirs)


class ConvBNAct(nn.Module):
    """3x3 (or 1x1) convolution, batch normalization, optional residual and ReLU."""
    def __init__(self, backend, in_dim: int, out_dim: int, kernel_size: int = 3, stride: int = 1,
                 relu: bool = True) -> None:
        super().__init__()
        self.fused = _is_fused(backend)
        self.relu = relu
        self.conv = backend.Conv2d(in_dim, out_dim, kernel_size, stride=stride, padding=kernel_size // 2,
                                   bias=False)
        if self.fused:
            self.bn = backend.BatchNorm2d(out_dim, act_func='relu' if relu else None)
        else:
            self.bn = backend.BatchNorm2d(out_dim)

    def forward(self, input: Tensor, residual: Optional[Tensor] = None) -> Tensor:
        output = self.conv(input)
        if self.fused:
            return self.bn(output, residual)
        output = self.bn(output)
        if residual is not None:
            output = output + residual
        return F.relu(output) if self.relu else output

    def load_from(self, other: 'ConvBNAct') -> None:
        with torch.no_grad():
            self.conv.weight.copy_(other.conv.weight)
            self.bn.weight.copy_(other.bn.weight)
            self.bn.bias.copy_(other.bn.bias)


class BasicBlock(nn.Module):
    """ResNet basic block: conv-BN-ReLU, conv-BN, + identity (1x1 conv-BN when shapes change), ReLU."""
    def __init__(self, backend, in_dim: int, out_dim: int, stride: int = 1) -> None:
        super().__init__()
        self.first = ConvBNAct(backend, in_dim, out_dim, 3, stride)
        self.second = ConvBNAct(backend, out_dim, out_dim, 3)
        self.downsample = None
        if in_dim != out_dim or stride != 1:
            self.downsample = ConvBNAct(backend, in_dim, out_dim, 1, stride, relu=False)

    def forward(self, input: Tensor) -> Tensor:
        identity = input if self.downsample is None else self.downsample(input)
        return self.second(self.first(input), identity)

    def load_from(self, other: 'BasicBlock') -> None:
        self.first.load_from(other.first)
        self.second.load_from(other.second)
        if self.downsample is not None:
            self.downsample.load_from(other.downsample)


class NewTokens(NamedTuple):
    """
    Where the tokens of a call that continues sequences belong.
    """
    positions: Tensor       # [batch, chunk]
    slots: Tensor           # [batch, chunk] places in the cache, no two of a sequence the same
    live: Tensor            # [batch, chunk] the others are padding
    lengths: Tensor
    query_lengths: Tensor


def new_tokens(lengths: Tensor, query_lengths: Optional[Tensor], chunk: int, room: int) -> NewTokens:
    """
    The first `query_lengths` of a sequence's `chunk` tokens (None: as many as it has tokens for) are its last
    ones, the others are padding, and so are tokens that find no room.  Nothing here waits for the device.
    """
    lengths = lengths.long()
    new = chunk if query_lengths is None else query_lengths.long().clamp(0, chunk)
    start = (lengths - new).clamp(min=0)
    new = (lengths.clamp(max=room) - start).clamp(min=0)
    step = torch.arange(chunk, device=lengths.device)
    positions = start[:, None] + step
    return NewTokens(positions, positions % room, step < new[:, None], start + new, new)


class TransformerBlock(nn.Module):
    """
    Pre-norm block: x + attention(LN(x)), then + MLP(LN(.)) with a fused Linear+GELU.

    The attention core is torch's on both backends unless one of the options is given: rotary turns
    queries and keys by the tokens' positions, window and num_sinks limit what a token sees to the
    window's last tokens and the sequence's first ones, and kv_heads < num_heads shares key heads
    among query heads.  With any of them the fused backend runs on its Rotary and WindowAttention,
    and torch on the same arithmetic spelled out; only the former can continue sequences from a
    cache of keys and values.
    """
    def __init__(self, backend, dim: int, num_heads: int, kv_heads: Optional[int] = None, window: Optional[int] = None,
                 num_sinks: int = 0, rotary: bool = False) -> None:
        super().__init__()
        self.num_heads = num_heads
        self.kv_heads = num_heads if kv_heads is None else kv_heads
        self.head_dim = dim // num_heads
        self.window, self.num_sinks, self.rotary = window, num_sinks, rotary
        self.plain = window is None and not rotary and self.kv_heads == num_heads
        self.fused = _is_fused(backend) and not self.plain
        if self.fused:
            self.turn = backend.Rotary(self.head_dim) if rotary else None
            self.core = backend.WindowAttention(window=window, num_sinks=num_sinks)
        self.ln1 = backend.LayerNorm(dim)
        self.qkv = FusedLinear(backend, dim, dim + 2 * self.kv_heads * self.head_dim, None)
        self.proj = FusedLinear(backend, dim, dim, None)
        self.ln2 = backend.LayerNorm(dim)
        self.fc1 = FusedLinear(backend, dim, 4 * dim, 'gelu')
        self.fc2 = FusedLinear(backend, 4 * dim, dim, None)

    def _spelled_out(self, q: Tensor, k: Tensor, v: Tensor) -> Tensor:
        position = torch.arange(q.shape[2], device=q.device)
        if self.rotary:
            half = self.head_dim // 2
            angle = position[:, None] * 10000.0 ** (torch.arange(half, device=q.device, dtype=torch.float64) / -half)
            cos, sin = angle.cos().float(), angle.sin().float()

            def turned(x: Tensor) -> Tensor:
                a, b = x.float().chunk(2, -1)
                return torch.cat((a * cos - b * sin, a * sin + b * cos), -1).to(x.dtype)

            q, k = turned(q), turned(k)
        ahead = position - position[:, None]
        seen = ahead <= 0
        if self.window is not None:
            seen = seen & ((ahead > -self.window) | (position < self.num_sinks))
        group = self.num_heads // self.kv_heads
        return F.scaled_dot_product_attention(q, k.repeat_interleave(group, 1), v.repeat_interleave(group, 1),
                                              attn_mask=seen)

    def attention(self, input: Tensor, cache: Optional[Tuple[Tensor, Tensor]] = None,
                  lengths: Optional[Tensor] = None, query_lengths: Optional[Tensor] = None,
                  new: Optional[NewTokens] = None) -> Tensor:
        batch, seq, dim = input.shape
        if self.plain and cache is None:
            qkv = self.qkv(input).view(batch, seq, 3, self.num_heads, dim // self.num_heads)
            q, k, v = qkv.permute(2, 0, 3, 1, 4)
            out = F.scaled_dot_product_attention(q, k, v, is_causal=True)
            return self.proj(out.transpose(1, 2).reshape(batch, seq, dim))
        heads = self.qkv(input).view(batch, seq, self.num_heads + 2 * self.kv_heads, self.head_dim).transpose(1, 2)
        q, k, v = heads.split((self.num_heads, self.kv_heads, self.kv_heads), 1)
        if not self.fused:
            out = self._spelled_out(q, k, v)
        else:
            if cache is not None and new is None:
                new = new_tokens(lengths, query_lengths, seq, cache[0].shape[2])
            if self.turn is not None:
                q, k = self.turn(q, k, None if cache is None else new.positions)
            if cache is not None:
                live, slots = new.live[:, None, :, None], new.slots[:, None, :, None].expand(k.shape)
                for stored, fresh in zip(cache, (k, v)):     # padding rewrites what is there
                    stored.scatter_(2, slots, torch.where(live, fresh.to(stored.dtype), stored.gather(2, slots)))
                k, v = cache
                lengths, query_lengths = new.lengths, new.query_lengths
            out = self.core(q, k, v, lengths, query_lengths)
        return self.proj(out.transpose(1, 2).reshape(batch, seq, dim))

    def forward(self, input: Tensor, cache: Optional[Tuple[Tensor, Tensor]] = None, lengths: Optional[Tensor] = None,
                query_lengths: Optional[Tensor] = None, new: Optional[NewTokens] = None) -> Tensor:
        output = input + self.attention(self.ln1(input), cache, lengths, query_lengths, new)
        return output + self.fc2(self.fc1(self.ln2(output)))

    def load_from(self, other: 'TransformerBlock') -> None:
        for name in ('qkv', 'proj', 'fc1', 'fc2'):
            getattr(self, name).load_from(getattr(other, name))
        with torch.no_grad():
            for name in ('ln1', 'ln2'):
                getattr(self, name).weight.copy_(getattr(other, name).weight)
                getattr(self, name).bias.copy_(getattr(other, name).bias)


class TinyGPT(nn.Module):
    """
    Embeddings, transformer blocks, final LayerNorm, vocabulary head, next-token loss.  Further
    arguments go to the blocks; with rotary there are no position embeddings.
    """
    def __init__(self, backend, vocab_size: int, depth: int, dim: int, num_heads: int,
                 max_seq_len: int = 512, rotary: bool = False, **block_options) -> None:
        super().__init__()
        self.tok_embed = nn.Embedding(vocab_size, dim)
        self.pos_embed = None if rotary else nn.Embedding(max_seq_len, dim)
        self.blocks = nn.ModuleList(TransformerBlock(backend, dim, num_heads, rotary=rotary, **block_options)
                                    for _ in range(depth))
        self.norm = backend.LayerNorm(dim)
        self.head = FusedLinear(backend, dim, vocab_size, None)
        self.loss_func = backend.CrossEntropyLoss()

    def forward(self, tokens: Tensor, return_loss: bool = False) -> Tensor:
        output = self.tok_embed(tokens)
        if self.pos_embed is not None:
            output = output + self.pos_embed(torch.arange(tokens.shape[1], device=tokens.device))
        for block in self.blocks:
            output = block(output)
        logits = self.head(self.norm(output))
        if not return_loss:
            return logits
        return self.loss_func(logits[:, :-1].reshape(-1, logits.shape[-1]), tokens[:, 1:].reshape(-1))

    def new_cache(self, batch: int, max_tokens: int) -> List[Tuple[Tensor, Tensor]]:
        """
        Room for the keys and values of max_tokens tokens of each sequence, for every block.
        """
        weight = self.tok_embed.weight
        return [tuple(torch.empty(batch, block.kv_heads, max_tokens, block.head_dim, device=weight.device, dtype=weight.dtype)
                      for _ in range(2)) for block in self.blocks]

    def extend(self, tokens: Tensor, cache: List[Tuple[Tensor, Tensor]], lengths: Tensor,
               query_lengths: Optional[Tensor] = None) -> Tensor:
        """
        Logits of new tokens (prompts, parts of them or single tokens), which are the last ones of
        sequences that have `lengths` tokens with them; their keys and values go into the cache.
        Of a sequence's row of tokens the first `query_lengths` are new (None: all, or as many as it
        has tokens in all), the others are padding: they leave the cache as it is, and their logits
        mean nothing.  So do tokens for which the cache has no room left.  For the fused
        backend with rotary.
        """
        if self.pos_embed is not None or not all(block.fused for block in self.blocks):
            raise RuntimeError('Sequences are continued on attorch_amd.nn and with rotary positions only')
        if tokens.shape[1] > cache[0][0].shape[2]:
            raise RuntimeError(f'The cache has room for {cache[0][0].shape[2]} tokens, received {tokens.shape[1]} new ones')
        new = new_tokens(lengths, query_lengths, tokens.shape[1], cache[0][0].shape[2])
        output = self.tok_embed(tokens)
        for block, stored in zip(self.blocks, cache):
            output = block(output, stored, lengths, query_lengths, new)
        return self.head(self.norm(output))

    def load_from(self, other: 'TinyGPT') -> None:
        with torch.no_grad():
            self.tok_embed.weight.copy_(other.tok_embed.weight)
            if self.pos_embed is not None:
                self.pos_embed.weight.copy_(other.pos_embed.weight)
            self.norm.weight.copy_(other.norm.weight)
            self.norm.bias.copy_(other.norm.bias)
        for mine, theirs in zip(self.blocks, other.blocks):
            mine.load_from(theirs)
        self.head.load_from(other.head)
