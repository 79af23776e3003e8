"""Attention over prompts, the 8-bit KV cache, attention over that cache and eviction from it, as
cases that can be timed and compared.

``own`` false: elementary torch operations in fp32.  ``own`` true: the framework's kernels.

Cache layout (``HelixKV8Cache``): blocks of 64 tokens per sequence and kv head, keys e4m3
[batch, n_kv, n_blocks, 64, D], values e4m3 transposed in their block [batch, n_kv, n_blocks, D, 64],
a power-of-two scale per block for each, the unfinished block in 16 bits (k_tail [batch, n_kv, 64, D],
v_tail [batch, n_kv, D, 64]) and a table of each sequence's and head's blocks in order.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

DEV = "cuda"
BLOCK = 64
THETA = 1e6
E4M3_MAX = 448.0
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# query heads, kv heads, head dim: the attention of the framework's Qwen2.5-3B and -7B shapes, of
# its OLMoE shape, and of a model with 64-wide heads
HEADS = [(16, 2, 128), (28, 4, 128), (16, 16, 128), (16, 4, 64)]


def listed():
    return [
        # a chat turn of one user: a short prompt whose length fits no tile
        {"name": "prompt_short_bf16", "op": "prompt", "hq": 16, "hkv": 2, "d": 128, "n": 1,
         "new": 211, "past": 0, "spread": 1.0, "dtype": "bf16"},
        # a batch of prompts of different lengths, packed without padding
        {"name": "prompt_packed_bf16", "op": "prompt", "hq": 28, "hkv": 4, "d": 128, "n": 12,
         "new": 2048, "past": 0, "spread": 0.1, "dtype": "bf16"},
        # one long document
        {"name": "prompt_long_bf16", "op": "prompt", "hq": 16, "hkv": 2, "d": 128, "n": 1,
         "new": 16384, "past": 0, "spread": 1.0, "dtype": "bf16"},
        # the next piece of several prompts that are taken in pieces, 64-wide heads
        {"name": "prompt_piece_f16", "op": "prompt", "hq": 16, "hkv": 4, "d": 64, "n": 6,
         "new": 512, "past": 7000, "spread": 0.5, "dtype": "f16"},
        # a prompt's rows between the projections and the attention: rotation and the cache
        {"name": "append_prompt_bf16", "op": "append", "hq": 16, "hkv": 2, "d": 128, "n": 1,
         "new": 1000, "past": 0, "spread": 1.0, "dtype": "bf16", "cache": "bf16"},
        # a large batch of pieces that go on in the middle of a block
        {"name": "append_pieces_f32", "op": "append", "hq": 28, "hkv": 4, "d": 128, "n": 48,
         "new": 700, "past": 1000, "spread": 0.2, "dtype": "f32", "cache": "f16"},
        # one user's token in a short chat: what a step costs at least
        {"name": "decode_chat", "op": "decode", "hq": 16, "hkv": 2, "d": 128, "n": 1, "past": 500,
         "spread": 1.0, "dtype": "f32", "cache": "bf16", "weights": False, "table": False},
        # one user's token after a very long document
        {"name": "decode_document", "op": "decode", "hq": 16, "hkv": 2, "d": 128, "n": 1,
         "past": 131000, "spread": 1.0, "dtype": "f32", "cache": "bf16", "weights": True,
         "table": True},
        # a serving batch with evicted caches, sequences of very different lengths
        {"name": "decode_batch", "op": "decode", "hq": 28, "hkv": 4, "d": 128, "n": 64,
         "past": 16000, "spread": 0.05, "dtype": "bf16", "cache": "bf16", "weights": True,
         "table": True},
        # heads that share no keys, 64 wide, fp16
        {"name": "decode_heads_f16", "op": "decode", "hq": 16, "hkv": 4, "d": 64, "n": 24,
         "past": 4095, "spread": 1.0, "dtype": "f16", "cache": "f16", "weights": False,
         "table": False},
        # one sequence's cache cut to half
        {"name": "evict_chat", "op": "evict", "hkv": 2, "n": 1, "past": 10000, "keep": 78,
         "sink": 1, "recent": 4, "spread": 1.0},
        # a batch of long caches cut to what fits
        {"name": "evict_batch", "op": "evict", "hkv": 4, "n": 64, "past": 131000, "keep": 500,
         "sink": 2, "recent": 16, "spread": 0.1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["prompt", "append", "decode", "decode", "evict"])
    hq, hkv, d = rng.choice(HEADS)
    spread = rng.choice([1.0, 0.5, 0.1])
    if op == "prompt":
        n = _log(rng, 1, 16)
        new = _log(rng, 1, max(2, 8192 // n))
        past = _log(rng, 1, 8192 // n) if rng.random() < 0.4 else 0
        return {"op": op, "hq": hq, "hkv": hkv, "d": d, "n": n, "new": new, "past": past,
                "spread": spread, "dtype": rng.choice(["bf16", "f16"])}
    if op == "append":
        n = _log(rng, 1, 48)
        return {"op": op, "hq": hq, "hkv": hkv, "d": d, "n": n,
                "new": _log(rng, 1, max(2, 8000 // n)), "past": rng.choice([0, _log(rng, 1, 4000)]),
                "spread": spread, "dtype": rng.choice(["bf16", "f16", "f32"]),
                "cache": rng.choice(["bf16", "f16"])}
    if op == "decode":
        n = _log(rng, 1, 64)
        return {"op": op, "hq": hq, "hkv": hkv, "d": d, "n": n,
                "past": _log(rng, 1, min(131000, 2_000_000 // (n * hkv))), "spread": spread,
                "dtype": rng.choice(["bf16", "f16", "f32"]), "cache": rng.choice(["bf16", "f16"]),
                "weights": rng.random() < 0.5, "table": rng.random() < 0.5}
    past = _log(rng, 200, 131000)
    keep = max(2, int(past // BLOCK * rng.uniform(0.1, 1.2)))
    sink = rng.randint(0, min(4, keep))
    return {"op": op, "hkv": hkv, "n": _log(rng, 1, 64), "past": past, "keep": keep, "sink": sink,
            "recent": rng.randint(0, min(32, keep - sink)), "spread": spread}


def _lens(top, n, spread, salt):
    """n lengths between spread * top and top, the first of them top."""
    if top == 0:
        return [0] * n
    golden = 0.6180339887498949
    return [top if i == 0 else
            max(1, round(top * (spread + (1.0 - spread) * ((golden * (i + salt)) % 1.0))))
            for i in range(n)]


def _new_past(case):
    """New tokens and cached tokens of each sequence."""
    new = _lens(case.get("new", 1), case["n"], case["spread"], 1)
    past = _lens(case["past"], case["n"], case["spread"], 5)
    return new, past


def _ends(lens):
    out = [0]
    for x in lens:
        out.append(out[-1] + x)
    return out


def work(case):
    n = case["n"]
    new, past = _new_past(case)
    if case["op"] == "evict":
        blocks = case["hkv"] * sum(p // BLOCK for p in past)
        return {"bytes": 16 * blocks, "flops": blocks}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "prompt":
        seen = sum(a * p + a * (a + 1) // 2 for a, p in zip(new, past))
        rows = sum(new)
        return {"bytes": 2 * d * (2 * hq * rows + 2 * hkv * (rows + sum(past))),
                "flops": 4 * d * hq * seen}
    size = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "append":
        rows, kept = sum(new), sum((p + a) // BLOCK - p // BLOCK for a, p in zip(new, past))
        return {"bytes": d * rows * (hq + 2 * hkv) * (size + 2) + 2 * d * hkv * BLOCK * kept,
                "flops": 6 * d * rows * (hq + 2 * hkv)}
    full, tail = sum(p // BLOCK for p in past), sum(p % BLOCK for p in past)
    nbytes = (2 * d * hkv * (BLOCK * full + 2 * tail) + 8 * hkv * full
              + d * n * ((hq + 2 * hkv) * size + 2 * hkv * 2 + 2 * hq))
    if case["weights"]:
        nbytes += 8 * hkv * full
    return {"bytes": nbytes, "flops": 4 * d * hq * (sum(past) + n)}


# --- inputs -------------------------------------------------------------------------------------
def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _rows(case, rows, hq, hkv, d, dt, g):
    """Query, key and value rows as views of one buffer, as a fused projection leaves them.  Some
    key channels are far larger than the others, as the key bias of real models makes them."""
    qkv = torch.randn(rows, hq + 2 * hkv, d, generator=g, device=DEV)
    loud = torch.rand(hkv, d, generator=g, device=DEV) < 0.02
    qkv[:, hq:hq + hkv] += loud * 12.0
    qkv = qkv.to(dt)
    return qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]


def _cache(n, hkv, d, n_blocks, dt, table, g):
    shape = (n, hkv, n_blocks)
    k = torch.empty(*shape, BLOCK, d, dtype=torch.float8_e4m3fn, device=DEV)
    v = torch.empty(*shape, d, BLOCK, dtype=torch.float8_e4m3fn, device=DEV)
    for i in range(n):
        k[i] = (torch.randn(shape[1:] + (BLOCK, d), generator=g, device=DEV) * 90).clamp_(
            -E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        v[i] = (torch.randn(shape[1:] + (d, BLOCK), generator=g, device=DEV) * 90).clamp_(
            -E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)

    def scale():
        e = torch.randint(-7, -5, shape, generator=g, device=DEV)
        return torch.exp2(e.float())

    blocks = None
    if table:
        blocks = torch.rand(shape, generator=g, device=DEV).argsort(-1).to(torch.int32)
    return {"k": k, "v": v, "k_scale": scale(), "v_scale": scale(),
            "k_tail": torch.randn(n, hkv, BLOCK, d, generator=g, device=DEV).to(dt),
            "v_tail": torch.randn(n, hkv, d, BLOCK, generator=g, device=DEV).to(dt),
            "blocks": blocks}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op, n = case["op"], case["n"]
    new, past = _new_past(case)
    s = {"op": op}
    if op == "evict":
        n_blocks = max(past) // BLOCK + 1
        heat = torch.randn(n, case["hkv"], n_blocks, generator=g, device=DEV).exp_()
        heat *= torch.arange(n_blocks, device=DEV) <= (_i32(past) // BLOCK)[:, None, None]
        s.update(weight=heat, cached=_i32(past), keep=case["keep"], sink=case["sink"],
                 recent=case["recent"],
                 blocks=torch.rand(heat.shape, generator=g, device=DEV).argsort(-1).to(torch.int32))
        return s
    hq, hkv, d, dt = case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]]
    if op == "prompt":
        both = [a + p for a, p in zip(new, past)]
        q = _rows(case, sum(new), hq, hkv, d, dt, g)[0]
        _, k, v = _rows(case, sum(both), hq, hkv, d, dt, g)
        s.update(q=q, k=k, v=v, cu_q=_i32(_ends(new)), cu_k=_i32(_ends(both)), max_q=max(new),
                 max_k=max(both))
        return s
    rows = sum(new) if op == "append" else n
    s["q"], s["k"], s["v"] = _rows(case, rows, hq, hkv, d, dt, g)
    s["cached"] = _i32(past)
    cdt = DTYPES[case["cache"]]
    if op == "append":
        s["cu"], s["max_new"] = _i32(_ends(new)), max(new)
        s["pos"] = s["cached"] + 3 * BLOCK
        # room for the rows, and for the padded form's last block
        n_blocks = max(past) // BLOCK + (max(new) + 2 * BLOCK - 2) // BLOCK
        s["cache"] = _cache(n, hkv, d, n_blocks, cdt, True, g)
        s["fork"] = max(past) > 0
        return s
    s["cache"] = _cache(n, hkv, d, max(past) // BLOCK + 1, cdt, case["table"], g)
    s["pos"] = s["cached"] + (5 * BLOCK if case["table"] else 0)
    s["weight"] = None
    if case["weights"]:
        s["weight"] = torch.rand(s["cache"]["k_scale"].shape, generator=g, device=DEV)
    return s


# --- the framework's calls ------------------------------------------------------------------------
def _kernels():
    pkg = str(Path(__file__).resolve().parents[1] / "helix-substrate_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from helix_substrate import attention

    return attention


def _run_own(s):
    K = _kernels()
    if s["op"] == "prompt":
        return K.attn_prompt(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"])
    if s["op"] == "evict":
        return list(K.kv8_evict(s["weight"], s["blocks"], s["cached"], s["keep"], s["sink"],
                                s["recent"]))
    c = s["cache"]
    cache = K.HelixKV8Cache(c["k"], c["v"], c["k_scale"], c["v_scale"], c["k_tail"], c["v_tail"],
                            c["blocks"])
    if s["op"] == "append":
        rows = cache.append(s["q"], s["k"], s["v"], s["cached"], s["cu"], pos=s["pos"],
                            theta=THETA)
        return {**dict(zip("qkv", rows)), **_held(c)}
    out, weight = cache.attend(s["q"], s["k"], s["v"], s["cached"], pos=s["pos"], theta=THETA,
                               weight=s["weight"], out_dtype=c["k_tail"].dtype,
                               weight_out=None if s["weight"] is None
                               else torch.empty_like(s["weight"]))
    return {"out": out, **({} if weight is None else {"weight": weight}), **_held(c)}


def _held(c):
    return {"cache_" + name: c[name] for name in ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail")}


# --- the plain form -------------------------------------------------------------------------------
def _rotate(x, pos, ft):
    """x [rows, heads, D] turned to positions pos [rows], halves paired; angles in 64 bits."""
    half = x.shape[-1] // 2
    freq = THETA ** (torch.arange(half, dtype=torch.float64, device=DEV) / -half)
    ang = (pos.double()[:, None] * freq)[:, None, :]
    c, sn = ang.cos().to(ft), ang.sin().to(ft)
    a, b = x[..., :half].to(ft), x[..., half:].to(ft)
    return torch.cat([a * c - b * sn, b * c + a * sn], -1)


def _attention(q, k, v, seen, scale):
    """q [.., Lq, D], k, v [.., Lk, D], seen [.., Lq, Lk]; rows that see nothing give zeros."""
    s = (q @ k.transpose(-1, -2)) * scale
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    return p @ v, p


def _run_prompt(s):
    q, k, v, cu_q, cu_k = s["q"], s["k"], s["v"], s["cu_q"].long(), s["cu_k"].long()
    (rows, hq, d), hkv, n = q.shape, k.shape[1], cu_q.numel() - 1
    lq, lk = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]
    i, j = torch.arange(s["max_q"], device=DEV), torch.arange(s["max_k"], device=DEV)
    at_q = (cu_q[:-1, None] + i).clamp_(max=rows - 1)
    at_k = (cu_k[:-1, None] + j).clamp_(max=k.shape[0] - 1)
    # [n, hkv, hq / hkv * max_q, d]: the heads of a group one after the other
    qq = q.float()[at_q].view(n, len(i), hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)
    qq = qq.reshape(n, hkv, -1, d)
    kk, vv = k.float()[at_k].transpose(1, 2), v.float()[at_k].transpose(1, 2)
    seen = (j <= i[:, None] + (lk - lq)[:, None, None]) & (j < lk[:, None, None])
    seen = seen[:, None].repeat(1, 1, hq // hkv, 1)
    o, _ = _attention(qq, kk, vv, seen, d ** -0.5)
    o = o.view(n, hkv, hq // hkv, len(i), d).permute(0, 3, 1, 2, 4).reshape(n, len(i), hq, d)
    seq = torch.searchsorted(cu_q[1:], torch.arange(rows, device=DEV), right=True)
    return o[seq, torch.arange(rows, device=DEV) - cu_q[seq]].to(q.dtype)


def _to8(x, dims):
    """e4m3 values and power-of-two scales of blocks: the smallest scale that holds the block."""
    top = x.abs().amax(dims, keepdim=True)
    m, e = torch.frexp(top / E4M3_MAX)                  # top / 448 = m 2^e, m in [0.5, 1)
    e = torch.where(m == 0.5, e - 1, e).clamp_(-110, 120)
    e = torch.where(top == 0, torch.full_like(e, -110), e)
    scale = torch.exp2(e.to(x.dtype))
    return (x / scale).to(torch.float8_e4m3fn), scale


def _run_append(s):
    c, cu, cached = s["cache"], s["cu"].long(), s["cached"].long()
    dt = c["k_tail"].dtype
    (n, hkv, n_blocks), d = c["k_scale"].shape, s["k"].shape[-1]
    r = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(cu[1:], r, right=True)
    off = r - cu[seq]
    pos = s["pos"].long()[seq] + off
    q, k = (_rotate(x.float(), pos, torch.float32).to(dt) for x in (s["q"], s["k"]))
    v = s["v"].to(dt)
    # the touched part of each cache, from the start of its unfinished block on
    width = (s["max_new"] + 2 * BLOCK - 2) // BLOCK
    held = cached % BLOCK
    k_all = torch.zeros(n, hkv, width * BLOCK, d, dtype=dt, device=DEV)
    v_all = torch.zeros(n, hkv, width * BLOCK, d, dtype=dt, device=DEV)
    k_all[:, :, :BLOCK], v_all[:, :, :BLOCK] = c["k_tail"], c["v_tail"].transpose(-1, -2)
    k_all[seq, :, held[seq] + off], v_all[seq, :, held[seq] + off] = k, v
    k_all, v_all = (x.view(n, hkv, width, BLOCK, d) for x in (k_all, v_all))
    k8, ks = _to8(k_all.float(), (-1, -2))
    v8, vs = _to8(v_all.float(), (-1, -2))
    total = held + cu[1:] - cu[:-1]
    j = torch.arange(width, device=DEV)
    done = (j < (total // BLOCK)[:, None])[:, None]                      # [n, 1, width]
    at = c["blocks"].long().gather(2, ((cached // BLOCK)[:, None, None] + j).expand(n, hkv, width))
    b, h = torch.arange(n, device=DEV)[:, None, None], torch.arange(hkv, device=DEV)[:, None]

    def put(into, x):
        into, x = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (into, x))
        keep = done.view(n, 1, width, *[1] * (x.dim() - 3))
        into[b, h, at] = torch.where(keep, x, into[b, h, at])

    put(c["k"], k8)
    put(c["v"], v8.view(torch.uint8).transpose(-1, -2).contiguous())
    put(c["k_scale"], ks[..., 0, 0])
    put(c["v_scale"], vs[..., 0, 0])
    # the unfinished block; rows behind its end stay as they were
    last = (total // BLOCK).clamp(max=width - 1)
    t = torch.arange(BLOCK, device=DEV)
    fresh = (t < (total % BLOCK)[:, None])[:, None, :, None]
    one = torch.arange(n, device=DEV)
    c["k_tail"].copy_(torch.where(fresh, k_all[one, :, last], c["k_tail"]))
    c["v_tail"].copy_(torch.where(fresh.transpose(-1, -2), v_all[one, :, last].transpose(-1, -2),
                                  c["v_tail"]))
    return {"q": q, "k": k, "v": v, **_held(c)}


def _run_decode(s, ft=torch.float32):
    c, cached = s["cache"], s["cached"].long()
    dt = c["k_tail"].dtype
    (n, hkv, n_blocks), (hq, d) = c["k_scale"].shape, s["q"].shape[1:]
    q = _rotate(s["q"], s["pos"], ft)
    k, v = _rotate(s["k"], s["pos"], ft).to(dt), s["v"].to(dt)
    one, held, full = torch.arange(n, device=DEV), cached % BLOCK, cached // BLOCK
    c["k_tail"][one, :, held] = k
    c["v_tail"][one, :, :, held] = v
    b, h = one[:, None, None], torch.arange(hkv, device=DEV)[:, None]
    at = torch.arange(n_blocks, device=DEV).expand(n, hkv, -1)
    if c["blocks"] is not None:
        at = c["blocks"].long()
    k8, v8 = (c[x].view(torch.uint8)[b, h, at].view(torch.float8_e4m3fn) for x in "kv")
    kk = k8.to(ft) * c["k_scale"][b, h, at][..., None, None]
    vv = (v8.to(ft) * c["v_scale"][b, h, at][..., None, None]).transpose(-1, -2)
    kk = torch.cat([kk.reshape(n, hkv, -1, d), c["k_tail"].to(ft)], 2)
    vv = torch.cat([vv.reshape(n, hkv, -1, d), c["v_tail"].transpose(-1, -2).to(ft)], 2)
    t = torch.arange(n_blocks * BLOCK, device=DEV)
    seen = torch.cat([t < (full * BLOCK)[:, None],
                      torch.arange(BLOCK, device=DEV) <= held[:, None]], 1)[:, None, None]
    vv = vv * seen.transpose(-1, -2)
    o, p = _attention(q.view(n, hkv, hq // hkv, d), kk, vv, seen, d ** -0.5)
    got = {"out": o.reshape(n, hq, d).to(dt)}
    if s["weight"] is not None:
        share = p.view(n, hkv, hq // hkv, n_blocks + 1, BLOCK).sum((2, 4))
        weight = s["weight"] + share[..., :n_blocks]
        weight.scatter_add_(2, full[:, None, None].expand(n, hkv, 1), share[..., n_blocks:])
        got["weight"] = weight
    # the token that ends a block sends it to the cache
    ends = (held == BLOCK - 1)[:, None, None, None]
    i = at.gather(2, full[:, None, None].expand(n, hkv, 1))[..., 0]
    b, h = one[:, None], torch.arange(hkv, device=DEV)
    for name in "kv":
        x8, sc = _to8(c[name + "_tail"].float(), (-1, -2))
        c[name].view(torch.uint8)[b, h, i] = torch.where(
            ends, x8.view(torch.uint8), c[name].view(torch.uint8)[b, h, i])
        c[name + "_scale"][b, h, i] = torch.where(ends[..., 0, 0], sc[..., 0, 0],
                                                  c[name + "_scale"][b, h, i])
    return {**got, **_held(c)}


def _run_evict(s):
    w, blocks, full = s["weight"], s["blocks"], (s["cached"] // BLOCK)[:, None, None]
    j = torch.arange(w.shape[-1], device=DEV)
    key = torch.where((j < s["sink"]) | (j >= full - s["recent"]), math.inf, w)
    key = torch.where(j >= full, -math.inf, key)
    rank = key.argsort(dim=-1, descending=True, stable=True).argsort(-1)
    kept = (rank < s["keep"]) & (j < full)
    left = full.clamp(max=s["keep"])                                      # blocks that stay
    to = torch.where(kept, kept.cumsum(-1) - 1, left + (~kept).cumsum(-1) - 1)
    out = torch.empty_like(blocks).scatter_(2, to, blocks)
    # the unfinished block's weight stays with it, behind the full ones
    stays = torch.where(kept, w, 0.0)
    weight = torch.zeros_like(w).scatter_(2, to, stays)
    inside = (full < w.shape[-1]) & (left < w.shape[-1])
    last = w.gather(2, full.long().clamp(max=w.shape[-1] - 1).expand(*w.shape[:2], 1))
    weight = torch.where((j == left) & inside, last, weight)
    cached = left[:, 0, 0] * BLOCK + s["cached"] % BLOCK
    return [out, weight, cached.to(torch.int32)]


def run(state):
    if state["op"] == "append" and state["fork"]:
        # a continuation of a cache that others continue too: its unfinished block is its own copy
        c = state["cache"]
        state = {**state, "cache": {**c, "k_tail": c["k_tail"].clone(), "v_tail": c["v_tail"].clone()}}
    if own:
        return _run_own(state)
    return {"prompt": _run_prompt, "append": _run_append, "decode": _run_decode,
            "evict": _run_evict}[state["op"]](state)


# --- 64 bits --------------------------------------------------------------------------------------
def _turn64(x, pos):
    """One row's heads [heads, D] at one position, as complex numbers."""
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half].double(), x[..., half:].double())
    ang = pos * torch.exp(torch.arange(half, dtype=torch.float64, device=x.device)
                          * (-math.log(THETA) / half))
    z = z * torch.polar(torch.ones_like(ang), ang)
    return torch.cat([z.real, z.imag], -1)


def _exact_prompt(s):
    q, k, v = s["q"], s["k"], s["v"]
    cu_q, cu_k = s["cu_q"].tolist(), s["cu_k"].tolist()
    group, out = q.shape[1] // k.shape[1], torch.zeros(q.shape, dtype=torch.float64, device=DEV)
    for b in range(len(cu_q) - 1):
        past = (cu_k[b + 1] - cu_k[b]) - (cu_q[b + 1] - cu_q[b])
        for h in range(q.shape[1]):
            kk = k[cu_k[b]:cu_k[b + 1], h // group].double()
            vv = v[cu_k[b]:cu_k[b + 1], h // group].double()
            for r in range(cu_q[b], cu_q[b + 1], 4096):
                qq = q[r:min(r + 4096, cu_q[b + 1]), h].double()
                s64 = qq @ kk.t() / math.sqrt(q.shape[2])
                last = torch.arange(len(qq), device=DEV)[:, None] + (r - cu_q[b] + past)
                s64[torch.arange(len(kk), device=DEV) > last] = -math.inf
                out[r:r + len(qq), h] = torch.softmax(s64, -1) @ vv
    return out


def _exact_append(s):
    """The values before they are rounded to 16 and to 8 bits; the scales of the 16-bit rows."""
    c, cu, cached, pos = s["cache"], s["cu"].tolist(), s["cached"].tolist(), s["pos"].tolist()
    dt = c["k_tail"].dtype
    got = {"q": torch.empty(s["q"].shape, dtype=torch.float64, device=DEV),
           "k": torch.empty(s["k"].shape, dtype=torch.float64, device=DEV), "v": s["v"].double()}
    held = {name: x.double() for name, x in _held(c).items()}
    for b in range(len(cached)):
        lo, hi = cu[b], cu[b + 1]
        at = torch.arange(hi - lo, dtype=torch.float64, device=DEV)[:, None, None] + pos[b]
        got["q"][lo:hi] = _turn64(s["q"][lo:hi], at)
        got["k"][lo:hi] = _turn64(s["k"][lo:hi], at)
        old, full, first = cached[b] % BLOCK, cached[b] // BLOCK, c["blocks"][b]
        for name in "kv":
            tail = c[name + "_tail"][b].double()
            rows = torch.cat([(tail if name == "k" else tail.transpose(-1, -2))[:, :old],
                              got[name][lo:hi].transpose(0, 1)], 1)
            count = rows.shape[1] // BLOCK
            x = rows[:, :count * BLOCK].unflatten(1, (count, BLOCK))
            top = x.to(dt).double().abs().amax((-1, -2))
            scale = torch.exp2(torch.ceil(torch.log2(top / E4M3_MAX)))
            x = x / scale[..., None, None]
            for h in range(rows.shape[0]):
                at8 = first[h, full:full + count].long()
                held["cache_" + name][b, h, at8] = x[h] if name == "k" else x[h].transpose(-1, -2)
                held["cache_" + name + "_scale"][b, h, at8] = scale[h]
            rest = rows[:, count * BLOCK:]
            if name == "k":
                held["cache_k_tail"][b, :, :rest.shape[1]] = rest
            else:
                held["cache_v_tail"][b, :, :, :rest.shape[1]] = rest.transpose(-1, -2)
    return {**got, **held}


def _exact_decode(s):
    c, cached, pos = s["cache"], s["cached"].tolist(), s["pos"].tolist()
    dt, (hq, d), hkv = c["k_tail"].dtype, s["q"].shape[1:], s["k"].shape[1]
    out = torch.empty(len(cached), hq, d, dtype=torch.float64, device=DEV)
    weight = None if s["weight"] is None else s["weight"].double()
    k_tail, v_tail = c["k_tail"].double(), c["v_tail"].double()
    for b, t in enumerate(cached):
        full, old = t // BLOCK, t % BLOCK
        q, k = _turn64(s["q"][b], pos[b]), _turn64(s["k"][b], pos[b])
        k_tail[b, :, old], v_tail[b, :, :, old] = k, s["v"][b].double()
        for h in range(hkv):
            at = (torch.arange(full, device=DEV) if c["blocks"] is None
                  else c["blocks"][b, h, :full].long())
            kk = c["k"][b, h].view(torch.uint8)[at].view(torch.float8_e4m3fn).double()
            vv = c["v"][b, h].view(torch.uint8)[at].view(torch.float8_e4m3fn).double()
            kk, vv = (x * sc[b, h, at].double()[:, None, None]
                      for x, sc in ((kk, c["k_scale"]), (vv, c["v_scale"])))
            kk = torch.cat([kk.reshape(-1, d), c["k_tail"][b, h, :old].double(),
                            k[h:h + 1].to(dt).double()])
            vv = torch.cat([vv.transpose(1, 2).reshape(-1, d),
                            c["v_tail"][b, h, :, :old].t().double(),
                            s["v"][b, h:h + 1].to(dt).double()])
            group = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            p = torch.softmax(q[group] @ kk.t() / math.sqrt(d), -1)
            out[b, group] = p @ vv
            if weight is not None:
                p = torch.nn.functional.pad(p.sum(0), (0, BLOCK - 1 - old))
                weight[b, h, :full + 1] += p.view(-1, BLOCK).sum(-1)
    got = {"out": out, **({} if weight is None else {"weight": weight})}
    return {**got, **dict.fromkeys(_held(c)), "cache_k_tail": k_tail, "cache_v_tail": v_tail}


def _exact_evict(s):
    weight = torch.zeros(s["weight"].shape, dtype=torch.float64)
    for b, t in enumerate(s["cached"].tolist()):
        full = t // BLOCK
        for h, row in enumerate(s["weight"][b].double().tolist()):
            kept = list(range(full))
            if full > s["keep"]:
                middle = range(s["sink"], full - s["recent"])
                best = sorted(middle, key=lambda j: (-row[j], j))
                kept = sorted([*range(s["sink"]), *best[:s["keep"] - s["sink"] - s["recent"]],
                               *range(full - s["recent"], full)])
            weight[b, h, :len(kept) + 1] = torch.tensor([row[j] for j in [*kept, full]],
                                                        dtype=torch.float64)
    return [None, weight.to(DEV), None]


def exact(case, seed):
    return {"prompt": _exact_prompt, "append": _exact_append, "decode": _exact_decode,
            "evict": _exact_evict}[case["op"]](prepare(case, seed))
