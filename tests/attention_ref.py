"""Plain forms of the attention operators in 64 bits, on the CPU, with the sums that the tests'
tolerances are made of."""
import math

import torch

BLOCK = 64


def half_step(dt):
    """Largest relative error of a rounding to dt."""
    return torch.finfo(dt).eps / 2


def attention(q, k, v, scale, seen):
    """q [Lq, H, D], k, v [Lk, Hkv, D] in fp64, seen [Lq, Lk].  Returns out [Lq, H, D], the softmax
    p [H, Lq, Lk], sum_j p |v| and the error that fp32 scores may have: (D + 8) 2^-24 of the largest
    sum |q| |k| among the visible keys (D products and sums, the scale, log2(e), the shift by the
    maximum)."""
    group, D = q.shape[1] // k.shape[1], q.shape[2]
    kk, vv = (x.repeat_interleave(group, 1).transpose(0, 1) for x in (k, v))
    qq = q.transpose(0, 1)
    # what is not seen has no influence, whatever it holds
    used = seen.any(0)
    kk, vv = (torch.where(used[None, :, None], x, torch.zeros_like(x)) for x in (kk, vv))
    s = torch.where(seen, qq @ kk.transpose(1, 2) * scale, torch.tensor(-math.inf, dtype=q.dtype))
    top = s.amax(-1, keepdim=True) if s.shape[-1] else torch.zeros(*s.shape[:2], 1, dtype=q.dtype)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total == 0, torch.zeros_like(p), p / total)
    size = torch.where(seen, qq.abs() @ kk.abs().transpose(1, 2) * scale, torch.tensor(0.0, dtype=q.dtype))
    err = (D + 8) * 2.0 ** -24 * (size.amax(-1) if s.shape[-1] else torch.zeros(s.shape[:2], dtype=q.dtype))
    # rows of v that a query does not see must not meet its zeros
    safe = torch.nan_to_num(vv, 0.0, 0.0, 0.0)
    out, spread = p @ safe, p @ safe.abs()
    bad = (p > 0).to(q.dtype) @ (~torch.isfinite(vv)).to(q.dtype) > 0
    out = torch.where(bad, torch.tensor(math.nan, dtype=q.dtype), out)
    return out.transpose(0, 1), p, spread.transpose(0, 1), err.transpose(0, 1)[..., None]


def causal(lq, lk):
    return torch.arange(lk) <= torch.arange(lq)[:, None] + (lk - lq)


def rotate(x, pos, theta):
    """x [rows, heads, D] at positions pos [rows], in fp64 (halves paired); and a bound of what fp32
    arithmetic may be off by, relative to |a| + |b|: cos and sin 2^-22, products and sum 2^-23."""
    x = x.double()
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    if theta == 0:
        return x, torch.zeros_like(x)
    ang = pos.double()[:, None] * torch.tensor(float(theta), dtype=torch.float64) ** (
        -torch.arange(half, dtype=torch.float64) / half)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    off = (a.abs() + b.abs()) * 2.0 ** -21
    return torch.cat([a * c - b * s, b * c + a * s], -1), torch.cat([off, off], -1)


def scale_of(x):
    """Power-of-two scale of blocks [..., n] of finite values."""
    top = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(-1).double()
    e = torch.where(top > 0, torch.ceil(torch.log2(top.clamp(min=1e-300) / 448)),
                    torch.tensor(-110.0, dtype=torch.float64)).clamp(min=-110)
    return torch.exp2(e)


def to8(x):
    """x [..., n] of 16-bit values -> bytes of e4m3, scale (fp32)."""
    sc = scale_of(x)
    y = (x.double() / sc[..., None]).float()
    y = torch.where(torch.isfinite(y), y, torch.tensor(math.nan))
    return y.to(torch.float8_e4m3fn), sc.float()


def cached_rows(c, b, cached):
    """Keys and values [cached, n_kv, D] (fp64) that a cache's tensors (on the CPU) hold for
    sequence b."""
    n, held = divmod(cached, BLOCK)
    n_kv, n_blocks = c.k.shape[1:3]
    out = []
    for x8, sc, tail, turn in ((c.k, c.k_scale, c.k_tail, False), (c.v, c.v_scale, c.v_tail, True)):
        heads = []
        for h in range(n_kv):
            at = list(range(n)) if c.blocks is None else c.blocks[b, h, :n].tolist()
            full = [x8[b, h, i].double() * sc[b, h, i].double() for i in at]
            full = [x.t() if turn else x for x in full]
            last = tail[b, h].double()
            heads.append(torch.cat([*full, (last.t() if turn else last)[:held]]))
        out.append(torch.stack(heads, 1))
    return out


def evict(weight, blocks, cached, keep, sink, recent):
    """Plain selection, block by block."""
    batch, n_kv, n_blocks = weight.shape
    w_out, b_out, c_out = torch.zeros_like(weight), torch.empty_like(blocks), cached.clone()
    for b in range(batch):
        full = int(cached[b]) // BLOCK
        for h in range(n_kv):
            w = weight[b, h].tolist()
            kept = list(range(full))
            if full > keep:
                rank = lambda j: (0 if math.isnan(w[j]) else 1, -w[j] if w[j] == w[j] else 0, j)
                mid = sorted(range(sink, full - recent), key=rank)[:keep - sink - recent]
                kept = sorted([*range(sink), *mid, *range(full - recent, full)])
            rest = [j for j in range(n_blocks) if j not in set(kept)]
            order = torch.tensor(kept + rest)
            b_out[b, h] = blocks[b, h][order]
            w_out[b, h, :len(kept)] = weight[b, h][order[:len(kept)]]
            if full < n_blocks:
                w_out[b, h, len(kept)] = weight[b, h, full]
        c_out[b] = min(full, keep) * BLOCK + int(cached[b]) % BLOCK
    return b_out, w_out, c_out
