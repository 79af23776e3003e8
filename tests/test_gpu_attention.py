"""Prompt attention, the 8-bit KV cache, attention over it and eviction on the GPU, against plain
forms in 64 bits.  Tolerances are sums of the roundings that the operators are documented to make:
half a step of the output's type, half a step of the softmax weights (prompt: 16 bits; decode: bf16
hi + lo, 2^-16), fp32 scores (``attention_ref.attention``) and fp32 sums of n terms (n 2^-24)."""
import math
import types

import pytest
import torch

import attention_ref as ref
from helix_substrate.attention import BLOCK, HelixKV8Cache, attn_prompt, kv8_evict

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _ends(lens):
    return torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32)


def _i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


# --- prompts ---------------------------------------------------------------------------------------
def _prompt_case(lens, heads, kv, D, dt, seed, past=None, spike=3.0):
    g = _gen(seed)
    past = past or [0] * len(lens)
    q = torch.randn(sum(lens), heads, D, generator=g)
    k = torch.randn(sum(lens) + sum(past), kv, D, generator=g)
    v = torch.randn(sum(lens) + sum(past), kv, D, generator=g)
    k[::7] *= spike
    return q.to(dt), k.to(dt), v.to(dt), _ends(lens), _ends([a + b for a, b in zip(lens, past)])


def _check_prompt(got, q, k, v, cu_q, cu_k, scale=None, causal=True):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    h = ref.half_step(q.dtype)
    got = got.cpu().double()
    for s in range(len(cu_q) - 1):
        rq, rk = slice(int(cu_q[s]), int(cu_q[s + 1])), slice(int(cu_k[s]), int(cu_k[s + 1]))
        lq, lk = rq.stop - rq.start, rk.stop - rk.start
        seen = ref.causal(lq, lk) if causal else torch.ones(lq, lk, dtype=torch.bool)
        out, _, spread, err = ref.attention(q[rq].double(), k[rk].double(), v[rk].double(), scale, seen)
        tol = h * out.abs() + (h + 2 * err + lk * 2.0 ** -24) * spread * (1 + h) + 1e-30
        if q.dtype == FP:   # weights below 2^-14 are subnormal: half of 2^-24 each, times sum |v|
            tol = tol + 2.0 ** -25 * torch.nan_to_num(v[rk].double()).abs().sum(0).repeat_interleave(
                q.shape[1] // k.shape[1], 0) + 2.0 ** -25
        bad = ~(((got[rq] - out).abs() <= tol) | (out.isnan() & got[rq].isnan()))
        assert not bad.any(), (s, int(bad.sum()), float((got[rq] - out).abs().nan_to_num().max()))


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("heads,kv,D", [(16, 2, 128), (7, 1, 128), (4, 4, 64), (3, 1, 64)])
@pytest.mark.parametrize("lens", [[1], [2, 63, 64, 65], [0, 33, 0, 129, 1, 0], [300, 5]])
def test_prompt(dev, dt, heads, kv, D, lens):
    q, k, v, cu, _ = _prompt_case(lens, heads, kv, D, dt, 1)
    got = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev))
    _check_prompt(got, q, k, v, cu, cu)


def _behind(x, rows):
    """x with rows of no sequence behind it.  2100 rows of q and 5200 of k and v a sequence make a large
    call, which the 8-wave blocks take (from 64 heads on)."""
    more = torch.full((max(rows - x.shape[0], 0), *x.shape[1:]), math.nan, dtype=x.dtype)
    return torch.cat([x, more])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("large", [True, False])
@pytest.mark.parametrize("dt,D", [(BF, 128), (FP, 128), (BF, 64)])
@pytest.mark.parametrize("lens,past", [([257], [0]), ([300, 1, 130, 0, 64], [0, 90, 63, 0, 640]),
                                       ([512, 20], [-100, 1]), ([260, 60], [-270, -5]), ([700], [333])])
def test_prompt_with_many_heads(dev, dt, D, lens, past, causal, large):
    """Many heads over ragged sequences, keys before and fewer keys than queries; both block sizes."""
    q, k, v, cu, cu_k = _prompt_case(lens, 64, 8, D, dt, 10, [max(p, -n) for p, n in zip(past, lens)])
    qq, kk, vv = q, k, v
    if large:
        n = len(lens)
        qq, kk, vv = _behind(q, 2100 * n), _behind(k, 5200 * n), _behind(v, 5200 * n)
    got = attn_prompt(qq.to(dev), kk.to(dev), vv.to(dev), cu.to(dev), cu_k.to(dev),
                      causal=causal)[:q.shape[0]]
    _check_prompt(got, q, k, v, cu, cu_k, causal=causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,past", [([1, 1, 5], [0, 700, 64]), ([130, 64, 1], [31, 0, 128]),
                                       ([40, 0, 3], [-40, 17, -2]), ([257], [-200])])
def test_prompt_continues(dev, lens, past, causal):
    """Keys before the queries; fewer keys than queries (rows that see nothing give zeros)."""
    q, k, v, cu, cu_k = _prompt_case(lens, 8, 2, 128, BF, 2, past)
    got = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev), cu_k.to(dev), causal=causal)
    _check_prompt(got, q, k, v, cu, cu_k, causal=causal)
    if past == [-200] and causal:
        assert (got[:200] == 0).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dt,heads,kv,D", [(BF, 16, 2, 128), (FP, 4, 4, 64)])
@pytest.mark.parametrize("lens,past", [([1], [5000]), ([3, 130], [2000, 1500]), ([5, 0, 60, 70], [9, 6000, -30, 8190]),
                                       ([200], [1900])])
def test_prompt_of_few_queries_over_many_keys(dev, dt, heads, kv, D, lens, past, causal):
    """The keys split among blocks and joined; sequences shorter than the splits among them."""
    q, k, v, cu, cu_k = _prompt_case(lens, heads, kv, D, dt, 12, past)
    from helix_substrate import _hxq
    assert _hxq._prompt_workspace(sum(lens), k.shape[0], len(lens), heads, D, 0) > 0
    out = torch.full((sum(lens) + 4, heads, D), 3.0, dtype=dt, device=dev)
    pad = torch.cat([q, torch.full((4, heads, D), math.nan, dtype=dt)])
    got = attn_prompt(pad.to(dev), k.to(dev), v.to(dev), cu.to(dev), cu_k.to(dev), causal=causal, out=out)
    assert (got[sum(lens):] == 3).all()
    _check_prompt(got[:sum(lens)], q, k, v, cu, cu_k, causal=causal)
    bad = v.clone()
    bad[int(cu_k[1]) - 1, 0, 7] = math.nan       # the first sequence's last key: its last query only
    got2 = attn_prompt(pad.to(dev), k.to(dev), bad.to(dev), cu.to(dev), cu_k.to(dev), causal=causal, out=out.clone())
    group, last = heads // kv, lens[0] - 1
    if causal:
        assert torch.equal(got2[:last], got[:last])
    assert got2[last, :group, 7].isnan().all()
    assert torch.equal(got2[lens[0]:], got[lens[0]:])


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dt,heads,kv,D,lens,past", [
    (BF, 16, 2, 128, [2304], [1000]),                          # three splits, two rounds of blocks
    (FP, 16, 4, 64, [300, 0, 512, 256], [2000, 1500, 900, 0]),   # two to three, of uneven tiles
    (BF, 16, 2, 128, [1000], [0]), (BF, 16, 4, 64, [130, 7], [1000, 0])])
def test_prompt_splits_of_larger_calls(dev, dt, heads, kv, D, lens, past, causal):
    q, k, v, cu, cu_k = _prompt_case(lens, heads, kv, D, dt, 31, past)
    got = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev), cu_k.to(dev), causal=causal)
    _check_prompt(got, q, k, v, cu, cu_k, causal=causal)


@pytest.mark.parametrize("heads,kv,D", [(16, 2, 128), (4, 4, 64)])
def test_prompt_splits_leave_other_rows(dev, heads, kv, D):
    """Rows of no sequence before and behind, a sequence without keys and one without queries."""
    q, k, v, _, _ = _prompt_case([40], heads, kv, D, BF, 37, [6000])
    cu, cu_k = torch.tensor([5, 9, 9, 14, 33]), torch.tensor([100, 2500, 3000, 3000, 6040])
    out = torch.full_like(q, 7.0).to(dev)
    got = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.int().to(dev), cu_k.int().to(dev), out=out)
    assert got.data_ptr() == out.data_ptr()
    assert (got[:5] == 7).all() and (got[33:] == 7).all() and (got[9:14] == 0).all()
    _check_prompt(got, q, k, v, cu, cu_k)


def test_prompt_long(dev):
    q, k, v, cu, _ = _prompt_case([2500, 700], 4, 1, 128, BF, 3)
    got = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev), scale=0.11)
    _check_prompt(got, q, k, v, cu, cu, scale=0.11)


def test_prompt_many_sequences(dev):
    lens = [(7 * i) % 11 for i in range(200)]
    q, k, v, cu, _ = _prompt_case(lens, 2, 1, 64, FP, 4)
    got = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev))
    _check_prompt(got, q, k, v, cu, cu)


def test_prompt_scores_that_grow(dev):
    """The running maximum rises through the whole row, by steps of 2^-4 up to 2^9 powers of two."""
    q, k, v, cu, _ = _prompt_case([640], 2, 1, 128, BF, 5, spike=1.0)
    k = (k.float() * torch.linspace(0, 12, 640)[:, None, None]).to(BF)
    got = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev))
    _check_prompt(got, q, k, v, cu, cu)
    k = k.flip(0).contiguous()
    got = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev))
    _check_prompt(got, q, k, v, cu, cu)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lens", [[200], [70, 130]])
@pytest.mark.parametrize("heads,large", [(4, False), (64, False), (64, True)])
def test_prompt_unseen_values_have_no_influence(dev, bad, lens, heads, large):
    q, k, v, cu, _ = _prompt_case(lens, heads, 2, 128, BF, 6)
    if large:
        n = len(lens)
        q, k, v = _behind(q, 2100 * n), _behind(k, 5200 * n), _behind(v, 5200 * n)
    for t in (3, 40, 64, 101, 127, 199):
        v[t, 0, 5] = bad
        k[t, 1, 9] = math.nan
    got = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev), cu.to(dev))[:, :2]
    # kv head 0 (heads 0, 1): NaN or infinities in v reach exactly the queries that see them
    h0 = got.cpu().double()
    for s in range(len(lens)):
        r = slice(int(cu[s]), int(cu[s + 1]))
        first = next((t for t in (3, 40, 64, 101, 127, 199) if r.start <= t < r.stop), r.stop)
        assert torch.isfinite(h0[r.start:first]).all()
        assert torch.isfinite(h0[r, :, 6:]).all() and torch.isfinite(h0[r, :, :5]).all()
        assert not torch.isfinite(h0[first:r.stop, :, 5]).any()
    q, k, v = q[:200, :2], k[:, :1], v[:, :1].clone()
    v[:, 0, 5] = 0
    got = got[:200].clone()
    got[..., 5] = 0
    _check_prompt(got, q, k, v, cu, cu)


@pytest.mark.parametrize("lens,past,heads,bad", [
    ([70, 200], [0, 0], 4, [0, 1, 5, 64, 70, 71, 130]),          # rows that see only -inf at the start
    ([3], [2500], 4, list(range(1500))),                         # whole splits of -inf
    ([3, 2], [2500, 0], 4, list(range(2503)))])                  # a sequence of nothing else
@pytest.mark.parametrize("dt", [BF, FP])
def test_prompt_scores_of_minus_infinity(dev, dt, lens, past, heads, bad):
    """A key whose score is -inf has weight 0; where every score is -inf, the softmax is 0 / 0."""
    q, k, v, cu, cu_k = _prompt_case(lens, heads, 2, 64, dt, 23, past)
    q[..., 3] = q[..., 3].abs() + 0.5
    k[bad, :, 3] = -math.inf
    got = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev), cu_k.to(dev)).cpu().double()
    usable = torch.ones(len(k), dtype=torch.bool)
    usable[bad] = False
    h = ref.half_step(dt)
    for s in range(len(lens)):
        rq, rk = slice(int(cu[s]), int(cu[s + 1])), slice(int(cu_k[s]), int(cu_k[s + 1]))
        seen = ref.causal(lens[s], lens[s] + past[s])
        fine = seen & usable[rk]
        kk, vv = k[rk].double().nan_to_num(neginf=0.0), v[rk].double()
        out, _, spread, err = ref.attention(q[rq].double(), kk, vv, 64 ** -0.5, fine)
        tol = h * out.abs() + (h + 2 * err + len(kk) * 2.0 ** -24) * spread * (1 + h) + 1e-30
        if dt == FP:   # as above: subnormal weights
            tol = tol + 2.0 ** -25 * vv.abs().sum(0).repeat_interleave(heads // 2, 0) + 2.0 ** -25
        none = ~fine.any(1)
        assert got[rq][none].isnan().all()
        assert ((got[rq] - out).abs() <= tol)[~none].all()


@pytest.mark.parametrize("dt,heads,D,lens,past", [
    (BF, 4, 128, [5], [2000]), (FP, 4, 64, [40], [900]),       # waves with keys of their own, split or not
    (BF, 64, 128, [100], [6000]), (FP, 64, 64, [100], [9000])])  # blocks of 128 queries, split
def test_prompt_split_unseen_values(dev, dt, heads, D, lens, past):
    """Values that are not finite in the last rows, which the first queries do not see, and keys too."""
    q, k, v, cu, cu_k = _prompt_case(lens, heads, 2, D, dt, 41, past)
    n = len(k)
    v[n - 1, 0, 1], v[n - 3, 0, 7], v[n - 4, 1, 2] = math.nan, math.inf, -math.inf
    k[n - 2, 1, 5] = math.nan
    got = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev), cu_k.to(dev)).cpu()
    h = heads // 2
    assert got[-1, :h, 1].isnan().all() and got[:-1, :h, 1].isfinite().all()
    assert not got[-3:, :h, 7].isfinite().any() and got[:-3, :h, 7].isfinite().all()
    assert got[-2:, h:].isnan().all() and got[:-4, h:].isfinite().all()
    assert not got[-4:, h:, 2].isfinite().any()
    v[n - 1, 0, 1] = v[n - 3, 0, 7] = v[n - 4, 1, 2] = 0
    k[n - 2, 1, 5] = 0
    got[-1, :h, 1] = got[-3:, :h, 7] = got[-4:, h:] = 0
    want = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev), cu_k.to(dev)).cpu()
    _check_prompt(want, q, k, v, cu, cu_k)
    want[-1, :h, 1] = want[-3:, :h, 7] = want[-4:, h:] = 0
    assert torch.equal(got, want)


def test_prompt_neighbours_and_rows_behind(dev):
    """NaN in rows of no sequence reach nobody; their rows of out stay as they were."""
    q, k, v, cu, _ = _prompt_case([70, 60], 4, 2, 64, BF, 7)
    pad = lambda x: torch.cat([torch.full((9, *x.shape[1:]), math.nan, dtype=x.dtype), x,
                               torch.full((40, *x.shape[1:]), math.nan, dtype=x.dtype)])
    out = torch.full((179, 4, 64), 7.0, dtype=BF, device=dev)
    got = attn_prompt(pad(q).to(dev), pad(k).to(dev), pad(v).to(dev), (cu + 9).to(dev), out=out)
    assert (got[:9] == 7).all() and (got[139:] == 7).all()
    _check_prompt(got[9:139], q, k, v, cu, cu)


def test_prompt_strides(dev):
    """Views of a fused projection, and heads before rows; out likewise."""
    q, k, v, cu, _ = _prompt_case([100, 31], 8, 2, 128, FP, 8)
    want = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev))
    fused = torch.cat([q, k, v], 1).to(dev)
    out = torch.empty(131, 12, 128, dtype=FP, device=dev)
    got = attn_prompt(fused[:, :8], fused[:, 8:10], fused[:, 10:], cu.to(dev), out=out[:, 2:10])
    assert torch.equal(got, want)
    flip = [x.transpose(0, 1).contiguous().to(dev).transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(attn_prompt(*flip, cu.to(dev)), want)


def test_prompt_offsets_past_32_bits(dev):
    """One sequence's rows start 2^32 bytes behind the pointer (strides of 2^24 elements)."""
    rows, D = 300, 64
    q, k, v, cu, _ = _prompt_case([rows], 1, 1, D, BF, 9)
    step = 1 << 23
    big = torch.zeros(rows * step, dtype=BF, device=dev)
    assert big.numel() * 2 > 1 << 32
    kb = big.as_strided((rows, 1, D), (step, D, 1))
    vb = big[D:].as_strided((rows, 1, D), (step, D, 1))
    ob = big[2 * D:].as_strided((rows, 1, D), (step, D, 1))
    qb = big[3 * D:].as_strided((rows, 1, D), (step, D, 1))
    kb.copy_(k), vb.copy_(v), qb.copy_(q)
    got = attn_prompt(qb, kb, vb, cu.to(dev), out=ob)
    assert torch.equal(got, attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev)))


# --- rows into the cache ---------------------------------------------------------------------------
def _cpu(cache):
    """The cache's tensors as they are now, on the CPU."""
    c = types.SimpleNamespace()
    for n in ("k", "v", "k_scale", "v_scale", "k_tail", "v_tail", "blocks"):
        t = getattr(cache, n)
        setattr(c, n, None if t is None else t.cpu().clone())
    return c


def _same_bits(a, b, cached):
    """Both caches hold the same, in the blocks and in the tails' `cached` % 64 tokens."""
    for n in ("k", "v", "k_scale", "v_scale"):
        x, y = getattr(a, n), getattr(b, n)
        x, y = (t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t for t in (x, y))
        assert torch.equal(x, y), n
    for i, c in enumerate(cached):
        assert torch.equal(a.k_tail[i][:, :c % BLOCK], b.k_tail[i][:, :c % BLOCK])
        assert torch.equal(a.v_tail[i][..., :c % BLOCK], b.v_tail[i][..., :c % BLOCK])


def _rows(n, heads, kv, D, dt, seed):
    g = _gen(seed)
    x = torch.randn(n, heads + 2 * kv, D, generator=g)
    x[:, heads:heads + kv, 3::17] *= 40
    return x.to(dt)


def _shuffled(cache, seed):
    n = cache.k.shape[2]
    g = _gen(seed)
    for row in cache.blocks.view(-1, n):
        row.copy_(torch.randperm(n, generator=g).to(torch.int32))
    return cache


@pytest.mark.parametrize("dt,cdt", [(BF, BF), (F32, FP), (F32, BF), (FP, FP)])
@pytest.mark.parametrize("heads,kv,D", [(16, 2, 128), (5, 5, 64)])
@pytest.mark.parametrize("past,lens", [([0, 0, 0], [1, 64, 200]), ([3, 63, 64], [61, 1, 65]),
                                       ([100, 5, 0], [28, 300, 0]), ([1, 127, 60], [10, 130, 3])])
def test_append(dev, dt, cdt, heads, kv, D, past, lens):
    theta, batch = 1e4, 3
    cache = _shuffled(HelixKV8Cache.empty(batch, kv, D, 520, dtype=cdt, device=dev), 3)
    first = _rows(sum(past), heads, kv, D, dt, 4).to(dev)
    cut = lambda x: (x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:])
    cache.append(None, *cut(first)[1:], _i32([0] * batch, dev), _ends(past).to(dev), theta=theta)
    before = _cpu(cache)
    x = _rows(sum(lens), heads, kv, D, dt, 5)
    shift = [1000, 70000, 0]
    cached, cu = _i32(past, dev), _ends(lens)
    q, k, v = cache.append(*cut(x.to(dev)), cached, cu.to(dev),
                           pos=_i32([p + s for p, s in zip(past, shift)], dev), theta=theta)
    h = ref.half_step(cdt)
    tiny = torch.finfo(cdt).smallest_normal * h
    after = _cpu(cache)
    for b in range(batch):
        r = slice(int(cu[b]), int(cu[b + 1]))
        pos = torch.arange(r.stop - r.start) + past[b] + shift[b]
        for got, want in zip((q, k, v), cut(x)):
            want, off = ref.rotate(want[r], pos, theta) if got is not v else (want[r].double(), 0.0)
            assert ((got[r].cpu().double() - want).abs() <= h * want.abs() + 1.01 * off + tiny).all()
        # the cache holds exactly the 16-bit rows, each full block rounded once
        for name, rows in (("k", k), ("v", v)):
            turn = (lambda t: t) if name == "k" else (lambda t: t.transpose(-1, -2))
            old = turn(getattr(before, name + "_tail")[b])[:, :past[b] % BLOCK]
            every = torch.cat([old, rows[r].cpu().transpose(0, 1)], 1)
            n, held = divmod(every.shape[1], BLOCK)
            for hh in range(kv):
                touched = []
                for j in range(n):
                    at = int(after.blocks[b, hh, past[b] // BLOCK + j])
                    touched.append(at)
                    want8, sc = ref.to8(every[hh, j * BLOCK:(j + 1) * BLOCK].reshape(-1))
                    assert getattr(after, name + "_scale")[b, hh, at] == sc
                    assert torch.equal(turn(getattr(after, name)[b, hh, at]).reshape(-1).float(), want8.float())
                rest = [i for i in range(after.k.shape[2]) if i not in touched]
                assert torch.equal(getattr(after, name)[b, hh, rest].view(torch.uint8),
                                   getattr(before, name)[b, hh, rest].view(torch.uint8))
            tail, was = turn(getattr(after, name + "_tail")[b]), turn(getattr(before, name + "_tail")[b])
            assert torch.equal(tail[:, :held], every[:, n * BLOCK:])
            assert torch.equal(tail[:, held:], was[:, held:])


def test_append_pieces_and_tokens_give_the_same_bits(dev):
    heads, kv, D, n = 4, 2, 128, 333
    x = _rows(n, heads, kv, D, F32, 6).to(dev)
    cut = lambda x: (x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:])
    new = lambda: HelixKV8Cache.empty(1, kv, D, 400, device=dev)
    whole = new()
    whole.append(*cut(x), _i32([0], dev), _i32([0, n], dev), theta=1e6)
    pieces, at = new(), 0
    for m in (1, 62, 1, 1, 130, 64, 74):
        pieces.append(*cut(x[at:at + m]), _i32([at], dev), _i32([0, m], dev), theta=1e6)
        at += m
    assert at == n
    _same_bits(pieces, whole, [n])
    tokens = new()
    for t in range(n):
        tokens.attend(*cut(x[t:t + 1]), _i32([t], dev), theta=1e6)
    _same_bits(tokens, whole, [n])


def test_append_special_values(dev):
    """NaN and infinities become NaN and do not set the scale; a block of zeros; the borders of the
    scale; subnormal results."""
    D, kv = 64, 1
    x = torch.zeros(6 * BLOCK, kv, D, dtype=BF)
    x[:64] = torch.randn(64, 1, D, generator=_gen(7)).to(BF)
    x[5, 0, 7], x[6, 0, 8], x[7, 0, 9] = math.nan, math.inf, -math.inf
    x[128:192] = 448.0                    # scale 1
    x[192:256] = 450.0                    # scale 2
    x[256:320] = torch.logspace(-40, 30, 64 * D, base=2.0).view(64, 1, D).to(BF)
    x[320:384, 0, 0], x[320, 0, 0] = 2.0 ** -120, -(2.0 ** -105)
    cache = HelixKV8Cache.empty(1, kv, D, 512, device=dev)
    _, k, v = cache.append(None, x.to(dev), x.to(dev), _i32([0], dev), _i32([0, 384], dev))
    assert torch.equal(k.cpu().view(torch.int16), x.view(torch.int16))
    c = _cpu(cache)
    for j in range(6):
        want, sc = ref.to8(x[j * 64:(j + 1) * 64, 0].reshape(-1))
        for name in "kv":
            got = getattr(c, name)[0, 0, j]
            got = (got if name == "k" else got.t()).reshape(-1).float()
            assert float(getattr(c, name + "_scale")[0, 0, j]) == float(sc), (j, name)
            assert torch.equal(got.isnan(), want.float().isnan()), (j, name)
            assert torch.equal(got.nan_to_num(), want.float().nan_to_num()), (j, name)


def test_append_without_room_and_skipped(dev):
    """Tokens past the cache are not stored, the rows come out all the same; a sequence of negative
    count is left alone."""
    kv, D = 2, 64
    cache = HelixKV8Cache.empty(3, kv, D, 128, device=dev)
    was = _cpu(cache)
    x = _rows(90, 2, kv, D, BF, 8).to(dev)
    q, k, v = (x[:, :2], x[:, 2:4], x[:, 4:])
    outs = tuple(torch.full((90, 2, D), 9.0, dtype=BF, device=dev) for _ in range(3))
    cache.append(q, k, v, _i32([100, -1, 0], dev), _i32([0, 40, 60, 90], dev), theta=1e6, outs=outs)
    assert (outs[0][40:60] == 9).all() and (outs[2][40:60] == 9).all()
    assert torch.equal(outs[2][:40], v[:40])
    c = _cpu(cache)
    for n in ("k", "v", "k_tail", "v_tail"):
        a, b = getattr(c, n), getattr(was, n)
        assert torch.equal(a[1].view(torch.uint8), b[1].view(torch.uint8))
    assert (c.k_tail[0] == 0).all()       # block 1 got its 64 tokens, the 12 behind have no room
    assert c.k[0, :, 1].float().abs().sum() > 0 and c.k[0, :, 0].float().abs().sum() == 0
    assert torch.equal(c.k_tail[2][:, :30].transpose(0, 1), outs[1][60:].cpu())


# --- one token over the cache ------------------------------------------------------------------------
def _filled(batch, kv, D, cdt, past, n_blocks, dev, seed, table=True):
    """A cache of given counts, its blocks shuffled, filled by the prompt call."""
    cache = HelixKV8Cache.empty(batch, kv, D, n_blocks * BLOCK, dtype=cdt, device=dev, table=table)
    if table:
        _shuffled(cache, seed)
    lens = [max(p, 0) for p in past]
    x = _rows(sum(lens), 0, kv, D, F32, seed + 1).to(dev)
    if sum(lens):
        cache.append(None, x[:, :kv] * 0.6, x[:, kv:], _i32([0] * batch, dev), _ends(lens).to(dev),
                     theta=1e6)
    for t in (cache.k_tail, cache.v_tail):       # what is behind the last token must not matter
        for b, p in enumerate(lens):
            (t[b] if t is cache.k_tail else t[b].transpose(-1, -2))[:, p % BLOCK:] = math.nan
    return cache


def _check_attend(cache, x, heads, past, pos, got, weight, theta, odt, w0=0.0):
    c = _cpu(cache)
    kv, D = c.k.shape[1], c.k.shape[4]
    h, h16 = ref.half_step(odt), ref.half_step(c.k_tail.dtype)
    got = got.cpu().double()
    for b, n in enumerate(past):
        q, _ = ref.rotate(x[b:b + 1, :heads], torch.tensor([pos[b]]), theta)
        k, v = ref.cached_rows(c, b, n)
        # the new token as the cache took it
        nk, off = ref.rotate(x[b:b + 1, heads:heads + kv], torch.tensor([pos[b]]), theta)
        nv = x[b:b + 1, heads + kv:].to(c.k_tail.dtype).double()
        stored = ref.cached_rows(c, b, n + 1) if (n + 1) % BLOCK else None
        if stored is not None:
            assert torch.equal(stored[1][-1:], nv)
            assert ((stored[0][-1:] - nk).abs() <= h16 * nk.abs() + 1.01 * off + 1e-7).all()
            nk = stored[0][-1:]
            extra = 0.0
        else:
            nk = nk.to(c.k_tail.dtype).double()
            extra = 2 * float((q[0].abs().repeat(1, 1) * h16 * nk.abs().amax()).sum(-1).max()) * D ** -0.5
        out, p, spread, err = ref.attention(q, torch.cat([k, nk]), torch.cat([v, nv]), D ** -0.5,
                                            torch.ones(1, n + 1, dtype=torch.bool))
        # rotation of q in fp32 (2^-21 per element) joins the score's error
        err = 2 * (2 * err + 2.0 ** -21 * 4 * err / ((D + 8) * 2.0 ** -24)) + extra
        tol = h * out.abs() + (2.0 ** -16 + err + (n + 1) * 2.0 ** -24) * spread + 1e-12
        if odt == FP:
            tol = tol + 2.0 ** -25
        assert ((got[b] - out[0]).abs() <= tol[0]).all(), (b, float(((got[b] - out[0]).abs() / tol[0]).max()))
        if weight is not None:
            share = torch.nn.functional.pad(p[:, 0], (0, (-(n + 1)) % BLOCK)).view(heads, -1, BLOCK).sum(-1)
            share = share.view(kv, heads // kv, -1).sum(1)
            w = weight[b].cpu().double() - w0
            m = share.shape[1]
            tol = (err.amax() + (n + 68) * 2.0 ** -24) * share + 2.0 ** -23 * (1 + abs(w0))
            assert ((w[:, :m] - share).abs() <= tol).all(), (b, float((w[:, :m] - share).abs().max()))
            assert (w[:, m:].abs() <= 2.0 ** -23 * abs(w0)).all()


@pytest.mark.parametrize("cdt,dt,odt", [(BF, F32, BF), (FP, FP, F32), (BF, BF, F32), (FP, F32, FP)])
@pytest.mark.parametrize("heads,kv,D", [(16, 2, 128), (7, 1, 128), (4, 4, 64), (20, 2, 64), (16, 1, 128)])
@pytest.mark.parametrize("past", [[0, 1, 62], [63, 64, 65], [127, 200, 300]])
def test_attend(dev, cdt, dt, odt, heads, kv, D, past):
    cache = _filled(3, kv, D, cdt, past, 6, dev, 11)
    x = _rows(3, heads, kv, D, dt, 12)
    x[:, heads:heads + kv] *= 0.3
    before = _cpu(cache)
    xd = x.to(dev)
    pos = [p + 64 * i for i, p in enumerate(past)]
    w = torch.full((3, kv, 6), 0.5, device=dev)
    got, weight = cache.attend(xd[:, :heads], xd[:, heads:heads + kv], xd[:, heads + kv:],
                               _i32(past, dev), pos=_i32(pos, dev), theta=1e6, weight=w,
                               weight_out=torch.full_like(w, 9.0), out_dtype=odt)
    # the state before, with the token in the tail
    now = _cpu(cache)
    for b, p in enumerate(past):
        before.k_tail[b, :, p % BLOCK] = now.k_tail[b, :, p % BLOCK]
        before.v_tail[b, :, :, p % BLOCK] = now.v_tail[b, :, :, p % BLOCK]
    _check_attend(before, x, heads, past, pos, got, weight, 1e6, odt, w0=0.5)
    plain, _ = cache.attend(xd[:, :heads], xd[:, heads:heads + kv], xd[:, heads + kv:],
                            _i32(past, dev), pos=_i32(pos, dev), theta=1e6, out_dtype=odt)
    assert torch.equal(plain, got)        # the weights change nothing, a second call neither
    for b, p in enumerate(past):
        if p % BLOCK == BLOCK - 1:
            for name in "kv":
                turn = (lambda t: t) if name == "k" else (lambda t: t.transpose(-1, -2))
                for hh in range(kv):
                    at = int(now.blocks[b, hh, p // BLOCK])
                    want, sc = ref.to8(getattr(now, name + "_tail")[b, hh].reshape(-1))
                    assert torch.equal(getattr(now, name)[b, hh, at].reshape(-1).float(), want.float())
                    assert getattr(now, name + "_scale")[b, hh, at] == sc
        else:
            assert torch.equal(now.k[b].view(torch.uint8), before.k[b].view(torch.uint8))


@pytest.mark.parametrize("batch,past", [(1, 20000), (2, 9001)])
def test_attend_long(dev, batch, past):
    """Many splits, joined."""
    heads, kv, D = 16, 2, 128
    n = past // BLOCK + 3
    cache = _filled(batch, kv, D, BF, [past] * batch, n, dev, 13)
    x = _rows(batch, heads, kv, D, F32, 14)
    xd = x.to(dev)
    before = _cpu(cache)
    w = cache.new_weight()
    got, weight = cache.attend(xd[:, :heads], xd[:, heads:heads + kv], xd[:, heads + kv:],
                               _i32([past] * batch, dev), theta=1e6, weight=w, weight_out=w,
                               out_dtype=F32)
    now = _cpu(cache)
    before.k_tail[:, :, past % BLOCK] = now.k_tail[:, :, past % BLOCK]
    before.v_tail[:, :, :, past % BLOCK] = now.v_tail[:, :, :, past % BLOCK]
    _check_attend(before, x, heads, [past] * batch, [past] * batch, got, weight, 1e6, F32)


def test_attend_skipped_full_and_bad_table(dev):
    heads, kv, D = 4, 2, 64
    past = [-1, 128, 100, 70]
    cache = _filled(4, kv, D, BF, [0, 128, 100, 70], 2, dev, 15)
    x = _rows(4, heads, kv, D, BF, 16).to(dev)
    cache.blocks[2, 1, 0] = 7             # no such block
    was = _cpu(cache)
    out = torch.full((4, heads, D), 5.0, device=dev)
    w = torch.full((4, kv, 2), 0.25, device=dev)
    wo = torch.full((4, kv, 2), 3.0, device=dev)
    cache.attend(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], _i32(past, dev), out=out,
                 weight=w, weight_out=wo)
    assert (out[0] == 5).all() and (wo[0] == 3).all()
    assert out[1].isnan().all() and (wo[1] == 0.25).all()
    assert out[2, 2:].isnan().all() and torch.isfinite(out[2, :2]).all()
    assert torch.isfinite(out[3]).all()
    now = _cpu(cache)
    for n in ("k", "v", "k_tail", "v_tail"):
        for b in (0, 1):
            assert torch.equal(getattr(now, n)[b].view(torch.uint8), getattr(was, n)[b].view(torch.uint8))


def test_attend_nan_in_the_cache_is_seen(dev):
    heads, kv, D = 2, 1, 64
    cache = _filled(1, kv, D, BF, [130], 4, dev, 17)
    at = int(cache.blocks[0, 0, 1])
    cache.v.view(torch.uint8)[0, 0, at, 3, 10] = 0x7F
    x = _rows(1, heads, kv, D, BF, 18).to(dev)
    out, _ = cache.attend(x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:], _i32([130], dev))
    assert out[0, :, 3].isnan().all()
    assert torch.isfinite(out[0][:, [d for d in range(D) if d != 3]]).all()


# --- eviction ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("n_blocks,cached,keep,sink,recent", [
    (1, [64, 0, 10], 1, 0, 0), (9, [64 * 9, 64 * 8 + 5, 64 * 3], 4, 1, 1), (40, [64 * 39 + 63, 100, 64 * 40], 7, 0, 7),
    (1500, [64 * 1400 + 1, 64 * 1500, 64 * 700], 700, 3, 20), (2300, [64 * 2200, 64 * 2048, 64 * 2300], 1, 0, 0)])
def test_evict(dev, n_blocks, cached, keep, sink, recent):
    g = _gen(21)
    w = torch.randn(3, 2, n_blocks, generator=g)
    w[1] = torch.randint(0, 3, (2, n_blocks), generator=g).float()       # ties
    w[2, 0, ::3], w[2, 1, ::5] = math.nan, -0.0
    w[2, 1, 1::5] = 0.0
    blocks = torch.stack([torch.randperm(n_blocks, generator=g) for _ in range(6)]).view(3, 2, -1).to(torch.int32)
    cnt = torch.tensor(cached, dtype=torch.int32)
    got = kv8_evict(w.to(dev), blocks.to(dev), cnt.to(dev), keep, sink, recent)
    want = ref.evict(w, blocks, cnt, keep, sink, recent)
    assert torch.equal(got[0].cpu(), want[0])
    assert torch.equal(got[1].cpu().nan_to_num(99.0), want[1].nan_to_num(99.0))
    assert torch.equal(got[2].cpu(), want[2])
    plain = kv8_evict(w.to(dev), None, cnt.to(dev), keep, sink, recent)
    assert torch.equal(plain[0].cpu(), ref.evict(w, torch.arange(n_blocks, dtype=torch.int32).expand(3, 2, -1).contiguous(),
                                                 cnt, keep, sink, recent)[0])


# --- together --------------------------------------------------------------------------------------------
def test_prompt_then_tokens_then_eviction(dev):
    """A prompt, tokens that collect weight, eviction, tokens behind it: every token's attention is
    that over the blocks that stayed."""
    heads, kv, D, n, theta = 8, 2, 128, 500, 1e6
    cut = lambda x: (x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:])
    cache = HelixKV8Cache.empty(1, kv, D, 1024, device=dev)
    x = _rows(n, heads, kv, D, BF, 31)
    cu = _i32([0, n], dev)
    q, k, v = cache.append(*cut(x.to(dev)), _i32([0], dev), cu, theta=theta)
    o = attn_prompt(q, k, v, cu)
    _check_prompt(o, q.cpu(), k.cpu(), v.cpu(), cu.cpu(), cu.cpu())
    rk, rv = cache.read(0, n)
    want = ref.cached_rows(_cpu(cache), 0, n)
    assert torch.equal(rk.cpu().double(), want[0]) and torch.equal(rv.cpu().double(), want[1])
    cached, pos, w = _i32([n], dev), _i32([n], dev), cache.new_weight()
    count = n
    for step in range(40):
        t = _rows(1, heads, kv, D, F32, 100 + step)
        if step == 20:
            old = _cpu(cache)
            full = count // BLOCK
            keys = [old.blocks[0, h, :full].tolist() for h in range(kv)]
            cached = cache.evict(w, cached, keep=4, sink=1, recent=1)
            count = 4 * BLOCK + count % BLOCK
            assert int(cached) == count
            kept = [cache.blocks[0, h, :4].tolist() for h in range(kv)]
            for h in range(kv):
                assert [b for b in keys[h] if b in kept[h]] == kept[h]
                assert kept[h][0] == keys[h][0] and kept[h][-1] == keys[h][-1]
        before = _cpu(cache)
        out, _ = cache.attend(*cut(t.to(dev)), cached, pos=pos, theta=theta, weight=w, weight_out=w)
        now = _cpu(cache)
        before.k_tail[:, :, count % BLOCK] = now.k_tail[:, :, count % BLOCK]
        before.v_tail[:, :, :, count % BLOCK] = now.v_tail[:, :, :, count % BLOCK]
        _check_attend(before, t, heads, [count], [n + step], out, None, theta, F32)
        cached += 1
        pos += 1
        count += 1
    assert abs(float(w.sum()) - 0) > 0


def test_captured_and_replayed(dev):
    """One token per replay, counts advanced on the device; two graphs over one cache; eager work
    between the replays; every replay equals the eager result."""
    heads, kv, D, theta = 16, 2, 128, 1e6
    cut = lambda x: (x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:])
    make = lambda: _filled(2, kv, D, BF, [190, 700], 14, dev, 41)
    eager, graphed = make(), make()
    xs = [_rows(2, heads, kv, D, F32, 50 + i).to(dev) for i in range(8)]
    cached, w = _i32([190, 700], dev), eager.new_weight()
    want = []
    for x in xs:
        want.append((eager.attend(*cut(x), cached, theta=theta, weight=w, weight_out=w)[0].clone(), w.clone()))
        cached += 1
    x, cached, w = xs[0].clone(), _i32([190, 700], dev), graphed.new_weight()
    s = torch.cuda.Stream(device=dev)
    graphs = []
    for _ in range(2):
        g, out = torch.cuda.CUDAGraph(), torch.empty(2, heads, D, device=dev)
        s.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
            graphed.attend(*cut(x), cached, theta=theta, weight=w, weight_out=w, out=out)
            cached.add_(1)
        torch.cuda.current_stream(dev).wait_stream(s)
        graphs.append((g, out))
    for i, (o, ww) in enumerate(want):
        x.copy_(xs[i])
        g, out = graphs[i % 2]
        g.replay()
        junk = torch.randn(1 << 20, device=dev).sum()
        torch.cuda.synchronize()
        assert torch.equal(out, o) and torch.equal(w, ww), i
        del junk
    _same_bits(eager, graphed, [198, 708])


def test_on_another_stream(dev):
    lens = [100, 333]
    q, k, v, cu, _ = _prompt_case(lens, 8, 2, 128, BF, 61)
    a = [t.to(dev) for t in (q, k, v, cu)]
    want = attn_prompt(*a)
    s = torch.cuda.Stream(device=dev)
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s):
        got = attn_prompt(*a)
    s.synchronize()
    assert torch.equal(got, want)


def test_attend_and_append_offsets_past_32_bits(dev):
    """A cache of 4.9 GB of keys: the first blocks of the order lie at its end."""
    kv, D, n, heads, past = 1, 128, 600_000, 4, 200
    big = HelixKV8Cache.empty(1, kv, D, n * BLOCK, device=dev)
    big.blocks.copy_(big.blocks.flip(-1))
    small = HelixKV8Cache.empty(1, kv, D, 5 * BLOCK, device=dev)
    x = _rows(past, heads, kv, D, BF, 71).to(dev)
    t = _rows(1, heads, kv, D, F32, 72).to(dev)
    cut = lambda x: (x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:])
    outs = []
    for c in (big, small):
        c.append(*cut(x), _i32([0], dev), _i32([0, past], dev), theta=1e6)
        outs.append(c.attend(*cut(t), _i32([past], dev), theta=1e6)[0])
    assert torch.equal(*outs)
    assert big.k.numel() > 1 << 32
    assert torch.equal(big.k[0, 0, n - 3:].flip(0).view(torch.uint8), small.k[0, 0, :3].view(torch.uint8))


def test_two_calls_at_once(dev):
    """Two streams: prompts and tokens of different caches, each as alone."""
    heads, kv, D, past = 16, 2, 128, 3000
    cut = lambda x: (x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:])
    caches = [_filled(1, kv, D, BF, [past], 50, dev, 80 + i) for i in range(2)]
    xs = [_rows(1, heads, kv, D, F32, 90 + i).to(dev) for i in range(2)]
    prompts = [_prompt_case([9], heads, kv, D, BF, 95 + i, [4000]) for i in range(2)]
    prompts = [[t.to(dev) for t in p] for p in prompts]
    run = lambda i: (caches[i].attend(*cut(xs[i]), _i32([past], dev), theta=1e6,
                                      weight_out=caches[i].new_weight()), attn_prompt(*prompts[i]))
    want = [run(i) for i in range(2)]
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(run(i))
        torch.cuda.synchronize()
        for (a, p), (b, r) in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(p, r)


def test_prompt_captured_and_replayed(dev):
    """The form with split keys, its workspace from the graph's pool."""
    q, k, v, cu, cu_k = (t.to(dev) for t in _prompt_case([5, 40], 16, 2, 128, BF, 99, [3000, 2000]))
    want = attn_prompt(q, k, v, cu, cu_k)
    s, g = torch.cuda.Stream(device=dev), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        out = attn_prompt(q, k, v, cu, cu_k)
    torch.cuda.current_stream(dev).wait_stream(s)
    for i in range(4):
        out.zero_()
        g.replay()
        torch.randn(1 << 20, device=dev).sum().item()
        assert torch.equal(out, want)


def test_prompt_over_its_queries(dev):
    """out may be q."""
    q, k, v, cu, _ = _prompt_case([300, 77], 8, 2, 128, BF, 101)
    a = [t.to(dev) for t in (q, k, v, cu)]
    want = attn_prompt(*a)
    assert torch.equal(attn_prompt(*a, out=a[0]), want) and torch.equal(a[0], want)


def test_refusals_of_the_wrappers(dev):
    q, k, v, cu, _ = (t.to(dev) for t in _prompt_case([20], 4, 2, 64, BF, 102))
    with pytest.raises(RuntimeError, match="one dtype"):
        attn_prompt(q, k.half(), v, cu)
    with pytest.raises(RuntimeError, match="one dtype"):
        attn_prompt(q, k, v, cu, out=torch.empty_like(q, dtype=F32))
    with pytest.raises(ValueError, match="shapes"):
        attn_prompt(q, k, v[:, :1], cu)
    with pytest.raises(RuntimeError, match="int32"):
        attn_prompt(q, k, v, cu.long())
    with pytest.raises(RuntimeError, match="device tensors"):
        attn_prompt(q, k, v, cu.cpu())
    with pytest.raises(ValueError, match="cu_q and cu_k"):
        attn_prompt(q, k, v, cu, cu[:1])
    with pytest.raises(ValueError, match="as many rows"):
        attn_prompt(q, k[:10], v[:10], cu)
    with pytest.raises(RuntimeError, match="multiples of 16"):
        attn_prompt(q, k.view(-1)[4:4 + 19 * 128].view(19, 2, 64), v[:19], cu, cu)
    with pytest.raises(RuntimeError, match="head_dim"):
        attn_prompt(*(t[..., :32].contiguous() for t in (q, k, v)), cu)
    cache = HelixKV8Cache.empty(2, 2, 64, 128, device=dev)
    n = _i32([0, 0], dev)
    with pytest.raises(ValueError, match="of the cache"):
        cache.attend(q[:3], k[:3], v[:3], n)
    with pytest.raises(RuntimeError, match="int32"):
        cache.attend(q[:2], k[:2], v[:2], n.long())
    with pytest.raises(RuntimeError, match="int32"):
        cache.attend(q[:2], k[:2], v[:2], n[:1])
    with pytest.raises(ValueError, match="fp32"):
        cache.attend(q[:2], k[:2], v[:2], n, weight_out=torch.zeros(2, 2, 3, device=dev))
    with pytest.raises(RuntimeError, match="weight_in"):
        cache.attend(q[:2], k[:2], v[:2], n, weight=cache.new_weight())
    with pytest.raises(ValueError, match="cu_rows"):
        cache.append(q, k, v, n, cu)
    with pytest.raises(ValueError, match="16-bit dtype"):
        cache.append(q, k, v, n, _i32([0, 5, 20], dev), outs=(q.float(), None, None))
    with pytest.raises(RuntimeError, match="one dtype"):
        cache.append(q.float(), k, v, n, _i32([0, 5, 20], dev))
    with pytest.raises(RuntimeError, match="must hold|keep"):
        kv8_evict(cache.new_weight(), cache.blocks, n, 1, sink=1, recent=1)
    with pytest.raises(RuntimeError, match="e4m3"):
        HelixKV8Cache(cache.k.view(torch.uint8), cache.v, cache.k_scale, cache.v_scale, cache.k_tail,
                      cache.v_tail)
    with pytest.raises(ValueError, match="fit together"):
        HelixKV8Cache(cache.k, cache.v, cache.k_scale[:1], cache.v_scale, cache.k_tail, cache.v_tail)
    with pytest.raises(ValueError, match="block table"):
        HelixKV8Cache.empty(1, 1, 64, 64, device=dev, table=False).evict(cache.new_weight(), n, 1)
    with pytest.raises(ValueError, match="within the cache"):
        cache.read(0, 129)
