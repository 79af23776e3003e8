"""Attention of prompts, a KV cache in 8 bits, attention over it and eviction from it.

The reference leaves attention and the cache to transformers' Qwen2; here they are HIP kernels
(``hxq_attn.hip``, ``hxq_kv8.hip``) that ``HelixDecoder`` calls and that a serving loop can call by
itself:

    cache = HelixKV8Cache.empty(batch, n_kv_heads, head_dim, max_tokens)
    q, k, v = cache.append(q, k, v, cached, cu_rows, theta=1e6)      # prompts: rotate, store
    o = attn_prompt(q, k, v, cu_rows)                                # their attention
    cached += lengths
    o, _ = cache.attend(q1, k1, v1, cached, theta=1e6, weight=w, weight_out=w)   # one token each
    cached += 1
    cached = cache.evict(w, cached, keep=64, sink=1, recent=4)       # fewer blocks from here on

Tensors of rows are [rows, heads, head_dim] views (row and head strides are free); offsets, counts
and positions are int32 on the device, so that nothing waits for the host.
"""
from __future__ import annotations

import math

import torch

from . import _hxq

BLOCK = _hxq.KV8_BLOCK


def attn_prompt(q, k, v, cu_q, cu_k=None, scale=None, causal=True, out=None):
    """Attention of packed prompts: sequence s owns q rows cu_q[s]..cu_q[s+1] and key rows
    cu_k[s]..cu_k[s+1] (None: cu_q).  Keys beyond the queries are earlier ones (a prompt that
    continues cached tokens).  bf16 or fp16, head_dim 64 or 128; scale None = head_dim^-1/2.
    Returns out, [rows, heads, head_dim]; rows that belong to no sequence stay as they were in a
    given out, and are undefined in a new one."""
    return _hxq.attn_prompt(q, k, v, cu_q, cu_k, q.shape[-1] ** -0.5 if scale is None else scale,
                            bool(causal), out)


def rope_rows(q, k, v, cu_rows, pos, theta, dtype=torch.bfloat16, outs=None):
    """Rows of packed prompts rotated to positions pos[s], pos[s] + 1, ... (q and k; v is only
    rounded), in a 16-bit dtype: what ``HelixKV8Cache.append`` does, without a cache.  outs: three
    tensors (or None) to write to, rows of a 16-bit cache for instance.  Returns (q, k, v); rows of
    no sequence, or of one with a negative pos, are not written."""
    desc = _hxq.HxqKv8(None, None, None, None, None, None, None, _hxq.dtype_code(dtype),
                       cu_rows.numel() - 1, k.shape[1], k.shape[2], 0)
    return _hxq.kv8_append(q, k, v, cu_rows, pos, None, theta, desc, outs)


def kv8_evict(weight, blocks, cached, keep, sink=0, recent=0):
    """The blocks that stay when every sequence and kv head keeps at most `keep` full blocks: the
    first `sink`, the last `recent`, and the greatest weight between them.  Returns new (blocks,
    weight, cached) tensors; see ``HelixKV8Cache.evict`` for a cache that is cut in place."""
    return _hxq.kv8_evict(weight, blocks, cached, keep, sink, recent)


class HelixKV8Cache:
    """Keys and values of `batch` sequences in blocks of 64 tokens, e4m3 with a power-of-two scale
    per block and kv head; the unfinished block of each in 16 bits.  Per kv head: 2 D bytes a token
    (4 D in a bf16 cache), 12 a block and 256 D a sequence.

    k, v: float8_e4m3fn [batch, n_kv, n_blocks, 64, D] and [batch, n_kv, n_blocks, D, 64];
    k_scale, v_scale: fp32 [batch, n_kv, n_blocks]; k_tail, v_tail: bf16 or fp16 [batch, n_kv, 64, D]
    and [batch, n_kv, D, 64]; blocks: int32 [batch, n_kv, n_blocks], the place of each block in
    order (None: in place; a permutation in every row otherwise).

    How many tokens a sequence holds is the caller's: `cached`, int32 [batch], is passed to every
    call and advanced by the caller (a captured graph advances it on the device)."""

    def __init__(self, k, v, k_scale, v_scale, k_tail, v_tail, blocks=None):
        self._tensors = (k, v, k_scale, v_scale, k_tail, v_tail, blocks)
        self._desc = _hxq.kv8_desc(*self._tensors)   # their addresses: the tensors are fixed

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scale = property(lambda self: self._tensors[2])
    v_scale = property(lambda self: self._tensors[3])
    k_tail = property(lambda self: self._tensors[4])
    v_tail = property(lambda self: self._tensors[5])
    blocks = property(lambda self: self._tensors[6])

    def clone(self):
        """A copy with tensors of its own."""
        return HelixKV8Cache(*(None if t is None else t.clone() for t in self._tensors))

    def __deepcopy__(self, memo):
        return self.clone()

    @classmethod
    def empty(cls, batch, n_kv_heads, head_dim, max_tokens, dtype=torch.bfloat16, device="cuda",
              table=True):
        """An empty cache of at least max_tokens per sequence.  table False: without a block table,
        which eviction needs."""
        if max_tokens < 1:
            raise ValueError("max_tokens must be positive")
        n = (max_tokens + BLOCK - 1) // BLOCK
        each = (batch, n_kv_heads, n)
        f8 = dict(dtype=torch.float8_e4m3fn, device=device)
        blocks = None
        if table:
            blocks = torch.arange(n, dtype=torch.int32, device=device).expand(each).contiguous()
        return cls(torch.zeros(*each, BLOCK, head_dim, **f8), torch.zeros(*each, head_dim, BLOCK, **f8),
                   torch.ones(each, device=device), torch.ones(each, device=device),
                   torch.zeros(batch, n_kv_heads, BLOCK, head_dim, dtype=dtype, device=device),
                   torch.zeros(batch, n_kv_heads, head_dim, BLOCK, dtype=dtype, device=device), blocks)

    @property
    def max_tokens(self):
        return self.k.shape[2] * BLOCK

    @property
    def dtype(self):
        return self.k_tail.dtype

    def new_weight(self):
        """Zeros for the accumulated attention weight of every block."""
        return torch.zeros_like(self.k_scale)

    def append(self, q, k, v, cached, cu_rows, pos=None, theta=0.0, outs=None):
        """Rows of packed prompts behind the cached tokens: q and k are rotated to positions pos,
        pos + 1, ... (None: cached; theta 0: not rotated), k and v stored.  Returns the rows in the
        cache's 16-bit dtype (q, k, v), which `attn_prompt` takes; q None gives None.  outs: three
        tensors (or None) to write them to; rows of no sequence, or of one with a negative cached,
        are not written.  Tokens past max_tokens are not stored."""
        return _hxq.kv8_append(q, k, v, cu_rows, cached, pos, theta, self._desc, outs)

    def attend(self, q, k, v, cached, pos=None, theta=0.0, scale=None, weight=None, weight_out=None,
               out=None, out_dtype=None):
        """One token of each sequence: rotate q and k to pos (None: cached), store k and v behind
        the cached tokens, and attend over them and the token itself.  weight_out gets weight
        (None: zeros) plus each block's share of the softmax summed over the query heads of its kv
        head; it may be weight.  Returns (out [batch, heads, D], weight_out); a sequence with a
        negative cached is skipped, its part of both not written.  One with no room left gives NaN."""
        return _hxq.kv8_attn_decode(q, k, v, cached, pos, theta,
                                    q.shape[-1] ** -0.5 if scale is None else scale, self._desc,
                                    weight, weight_out, out, out_dtype), weight_out

    def evict(self, weight, cached, keep, sink=0, recent=0):
        """Cut every sequence and head to `keep` full blocks (``kv8_evict``); the block table and
        weight are changed in place.  Returns the new cached counts.  Positions do not follow: pass
        the tokens' own as pos from here on."""
        if self.blocks is None:
            raise ValueError("eviction needs a cache with a block table")
        blocks, new_weight, cached = kv8_evict(weight, self.blocks, cached, keep, sink, recent)
        self.blocks.copy_(blocks)
        weight.copy_(new_weight)
        return cached

    def read(self, seq, cached):
        """Keys and values of one sequence's first `cached` tokens (a host number) in 16 bits,
        [cached, n_kv, D] each: what a prompt that continues them passes to `attn_prompt` before its
        own rows.  Exact in bf16; in fp16 up to its greatest value.  A block that the table places
        outside the cache reads as NaN."""
        n, held = divmod(int(cached), BLOCK)
        n_kv, n_blocks, _, D = self.k.shape[1:]
        if not 0 <= int(cached) <= self.max_tokens:
            raise ValueError("cached must lie within the cache")
        at = torch.arange(n, device=self.k.device).expand(n_kv, n)
        if self.blocks is not None:
            at = self.blocks[seq, :, :n].long()
        known = (at >= 0) & (at < n_blocks)
        at = at.where(known, 0)
        h = torch.arange(n_kv, device=self.k.device)[:, None]
        out = []
        for x8, scale, tail, turn in ((self.k, self.k_scale, self.k_tail, False),
                                      (self.v, self.v_scale, self.v_tail, True)):
            x = x8[seq].view(torch.uint8)[h, at].view(torch.float8_e4m3fn).float()
            x = x * scale[seq][h, at].where(known, math.nan)[..., None, None]
            if self.dtype == torch.float16:   # 63488 to 65504 were stored as 65536
                x = x.clamp(-65504, 65504)
            x = x.to(self.dtype)
            last = tail[seq]
            if turn:
                x, last = x.transpose(-1, -2), last.transpose(-1, -2)
            out.append(torch.cat([x.reshape(n_kv, n * BLOCK, D), last[:, :held]], 1)
                       .transpose(0, 1).contiguous())
        return tuple(out)
