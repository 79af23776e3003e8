"""Prompt attention, the 8-bit cache and eviction at their edges: the last row of memory, counts past
the cache, tables that name no block, values next to the end of a type, every dtype's instance.
Oracle and tolerances as in ``test_gpu_attention``."""
import math

import pytest
import torch

import attention_ref as ref
from helix_substrate import _hxq
from helix_substrate.attention import BLOCK, HelixKV8Cache, attn_prompt, kv8_evict, rope_rows
from test_gpu_attention import (BF, F32, FP, _check_attend, _check_prompt, _cpu, _ends, _filled, _gen,
                                _i32, _prompt_case, _rows, _same_bits)
from test_gpu_attention import test_append as check_append

pytestmark = pytest.mark.gpu


# --- prompts ---------------------------------------------------------------------------------------
def _at_the_end(x, step):
    """x [rows, heads, D] with rows `step` elements apart, the last one ending with its allocation."""
    n, heads, D = x.shape
    out = torch.zeros((n - 1) * step + heads * D, dtype=x.dtype, device=x.device)
    out = out.as_strided((n, heads, D), (step, D, 1))
    out.copy_(x)
    return out


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dt,heads,kv,D,lens,past", [
    (BF, 16, 2, 128, [1], [129]), (FP, 4, 4, 64, [3], [127]),                    # each wave its own keys
    (BF, 16, 2, 128, [3], [2000]), (FP, 4, 4, 64, [5], [1500]),                  # and split
    (BF, 16, 2, 128, [1], [0]), (BF, 64, 8, 128, [70], [0]), (FP, 64, 8, 64, [40, 45], [0, 0]),              # 128 queries a block
    (BF, 64, 8, 128, [100], [6001]), (FP, 64, 8, 64, [100], [9001]),             # and split
    (BF, 64, 8, 128, [2100], [3101])])                                           # 256 queries a block
def test_prompt_values_that_are_not_finite_in_the_last_row(dev, dt, heads, kv, D, lens, past, causal):
    """Behind the last row of v there is no memory: what marks a row as not finite names rows that the
    sequence has, also where the last row stands for those behind it in a step of 64."""
    q, k, v, cu, cu_k = (t.to(dev) for t in _prompt_case(lens, heads, kv, D, dt, 7, past))
    want = attn_prompt(q, k, v, cu, cu_k, causal=causal)
    v[-1, 0, 3], v[-1, 0, D - 1] = math.nan, math.inf
    got = attn_prompt(q, k, _at_the_end(v, 1 << 18), cu, cu_k, causal=causal)
    group, first = heads // kv, int(cu[-1] - 1 if causal else cu[-2])   # the queries that see it
    assert got[first:, :group, 3].isnan().all() and not got[first:, :group, D - 1].isfinite().any()
    got, want = got.clone(), want.clone()
    got[first:, :group, 3] = want[first:, :group, 3] = 0
    got[first:, :group, D - 1] = want[first:, :group, D - 1] = 0
    assert torch.equal(got, want)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,D,lens,past", [
    (64, 8, 64, [1000], [0]), (64, 8, 128, [1000], [0]),      # 128 queries a block
    (64, 8, 64, [100], [9000]), (64, 8, 128, [100], [6000]),    # and split
    (4, 4, 64, [90], [60]), (16, 2, 128, [3], [2000]),        # each wave its own keys; split
    (64, 8, 128, [2100], [3100])])                            # 256 queries a block
def test_prompt_many_small_weights_beside_a_great_one(dev, heads, kv, D, lens, past, causal):
    """fp16: a key of weight 1 and value 0, all others of weight w = e^-18 < 2^-25 and value c: out is
    n w c / (1 + n w) of the n that a query sees.  A weight is rounded as 2^7 w, a subnormal: half of
    2^-24 at most, 2^-32 c in all for each of them (the sum of weights is 1 at least)."""
    n_q, n_k = lens[0], lens[0] + past[0]
    q = torch.ones(n_q, heads, D, dtype=FP)
    k, v = torch.zeros(n_k, kv, D, dtype=FP), torch.empty(n_k, kv, D, dtype=FP)
    k[0] = 144 / D
    v[:] = (32 + torch.arange(D) * 0.5).to(FP)
    v[0] = 0
    assert float((q[0, 0] * k[0, 0]).sum()) == 144
    got = attn_prompt(q.to(dev), k.to(dev), v.to(dev), _i32([0, n_q], dev), _i32([0, n_k], dev), scale=0.125,
                      causal=causal).cpu().double()
    n = (torch.arange(n_q) + n_k - n_q if causal else torch.full((n_q,), n_k - 1)).double()[:, None]
    c, w, h = v[-1, 0].double()[None], math.exp(-18.0), ref.half_step(FP)
    want = n * w * c / (1 + n * w)
    tol = h * want + 2.0 ** -25 + n * c * (2.0 ** -32 + w * (2 * 18 * (D + 8) * 2.0 ** -24 + n_k * 2.0 ** -24))
    assert ((got - want[:, None]).abs() <= tol[:, None]).all()


@pytest.mark.parametrize("D,heads", [(64, 4), (128, 4), (64, 64), (128, 64)])
@pytest.mark.parametrize("top", [16, 19, 20, 21, 24, 26])
def test_prompt_scores_of_many_millions(dev, D, heads, top):
    """fp16: scores that rise to 2^top powers of two, 2^(top - 9) a key: a query gets the value of its
    last key, through one rounding of its weight and one of the output."""
    n = 512
    _, _, v, cu, _ = _prompt_case([n], heads, 2, D, FP, 71)
    q = torch.ones(n, heads, D, dtype=FP)
    k = torch.arange(1, n + 1).to(FP)[:, None, None].expand(n, 2, D).contiguous()
    scale = 2.0 ** (top - 9) * math.log(2.0) / D
    got = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev), scale=scale).cpu().double()
    want = v.double().repeat_interleave(heads // 2, 1)
    assert ((got - want).abs() <= 2.01 * ref.half_step(FP) * want.abs() + 2.0 ** -24).all()


# --- eviction ------------------------------------------------------------------------------------------
def _cut(x, heads, kv):
    return x[:, :heads], x[:, heads:heads + kv], x[:, heads + kv:]


@pytest.mark.parametrize("n_blocks,cached,keep", [
    (2, [128 + 12, 128, 2 * 128 + 3], 1), (2, [128 + 5, 64, 3 * 64 + 3], 2),
    (9, [9 * 64 + 5, 10 * 64 + 3, 64], 4), (1100, [1100 * 64 + 63, 2 ** 31 - 1, 5], 7)])
def test_evict_counts_past_the_cache(dev, n_blocks, cached, keep):
    """Tokens past the cache were never stored: the count that comes out names stored ones only."""
    g = _gen(51)
    w = torch.randn(3, 2, n_blocks, generator=g)
    blocks = torch.stack([torch.randperm(n_blocks, generator=g) for _ in range(6)]).view(3, 2, -1).to(torch.int32)
    cnt = torch.tensor(cached, dtype=torch.int32)
    got = kv8_evict(w.to(dev), blocks.to(dev), cnt.to(dev), keep)
    want = ref.evict(w, blocks, cnt.clamp(max=n_blocks * BLOCK), keep, 0, 0)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


def test_evict_after_a_prompt_that_had_no_room(dev):
    """128 tokens of 140 fit; after eviction a token sees the block that stayed and itself."""
    heads, kv, D = 4, 2, 64
    cache = HelixKV8Cache.empty(1, kv, D, 128, device=dev)
    x = _rows(140, heads, kv, D, BF, 52).to(dev)
    cached, w = _i32([0], dev), cache.new_weight()
    for a, b in ((0, 100), (100, 140)):
        cache.append(*_cut(x[a:b], heads, kv), cached, _i32([0, b - a], dev), theta=1e6)
        cached += b - a
    t = _rows(1, heads, kv, D, F32, 53)
    out, _ = cache.attend(*_cut(t.to(dev), heads, kv), cached, theta=1e6, weight=w, weight_out=w)
    assert out.isnan().all() and (w == 0).all()
    cached = cache.evict(w, cached, keep=1)
    assert int(cached) == 64
    before = _cpu(cache)
    out, _ = cache.attend(*_cut(t.to(dev), heads, kv), cached, pos=_i32([140], dev), theta=1e6, out_dtype=F32)
    now = _cpu(cache)
    before.k_tail[:, :, 0], before.v_tail[..., 0] = now.k_tail[:, :, 0], now.v_tail[..., 0]
    _check_attend(before, t, heads, [64], [140], out, None, 1e6, F32)


@pytest.mark.parametrize("n_blocks", [1, 9, 1500])
def test_evict_leaves_skipped_sequences(dev, n_blocks):
    """A negative count skips a sequence: its blocks, weights and count come out as they were."""
    g = _gen(54)
    w = torch.rand(3, 2, n_blocks, generator=g)
    blocks = torch.stack([torch.randperm(n_blocks, generator=g) for _ in range(6)]).view(3, 2, -1).to(torch.int32)
    cnt = torch.tensor([-1, 64 * n_blocks, -(2 ** 31)], dtype=torch.int32)
    got = [t.cpu() for t in kv8_evict(w.to(dev), blocks.to(dev), cnt.to(dev), 1)]
    want = ref.evict(w[1:2], blocks[1:2], cnt[1:2], 1, 0, 0)
    for out, src, one in zip(got, (blocks, w, cnt), want):
        assert torch.equal(out[[0, 2]], src[[0, 2]]) and torch.equal(out[1:2], one)
    order = kv8_evict(w.to(dev), None, cnt.to(dev), 1)[0].cpu()
    assert torch.equal(order[[0, 2]], torch.arange(n_blocks, dtype=torch.int32).expand(2, 2, -1))


# --- what a cache holds, in 16 bits ----------------------------------------------------------------------
@pytest.mark.parametrize("entry", [-1, 4, 2 ** 31 - 1, -(2 ** 31)])
def test_read_of_blocks_that_the_table_does_not_place(dev, entry):
    """An entry outside the cache reads as NaN, as `attend` takes it; the other heads as they were."""
    kv, D, n = 2, 64, 150
    cache = HelixKV8Cache.empty(2, kv, D, 4 * BLOCK, device=dev)
    x = _rows(2 * n, 0, kv, D, BF, 61).to(dev)
    cache.append(None, *_cut(x, 0, kv)[1:], _i32([0, 0], dev), _i32([0, n, 2 * n], dev))
    want = cache.read(1, n)
    cache.blocks[1, 1, 0] = entry
    for got, was in zip(cache.read(1, n), want):
        assert got[:BLOCK, 1].isnan().all()
        assert torch.equal(got[BLOCK:], was[BLOCK:]) and torch.equal(got[:, 0], was[:, 0])


def test_read_next_to_the_end_of_fp16(dev):
    """63488 lies half way between the e4m3 values 240 and 256 times 256 and goes to the even one, 65536,
    which fp16 does not hold: it reads as 65504, not as infinity.  NaN stays NaN."""
    D, ends = 64, [65504.0, -65504.0, 63488.0, -63488.0, 63456.0]
    x = torch.zeros(BLOCK, 1, D, dtype=FP)
    x[0, 0, :5] = torch.tensor(ends, dtype=FP)
    x[1, 0, 0] = math.nan
    cache = HelixKV8Cache.empty(1, 1, D, 2 * BLOCK, dtype=FP, device=dev)
    cache.append(None, x.to(dev), x.to(dev), _i32([0], dev), _i32([0, BLOCK], dev))
    for got in cache.read(0, BLOCK):
        assert got[0, 0, :5].tolist() == [65504.0, -65504.0, 65504.0, -65504.0, 61440.0]
        assert got[1, 0, 0].isnan() and (got[2:] == 0).all()


@pytest.mark.parametrize("dt", [F32, BF, FP])
@pytest.mark.parametrize("cdt", [BF, FP])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("table", [True, False])
def test_the_same_bits_however_tokens_come(dev, dt, cdt, D, table):
    """One prompt, pieces of it, tokens one by one, and pieces with tokens between them: rows, blocks and
    tails of every kernel instance, at positions that turn a pair many times, with a table and without."""
    heads, kv, n, at = 4, 2, 200, 70_000
    x = _rows(n, heads, kv, D, dt, 81).to(dev)
    new = lambda: HelixKV8Cache.empty(1, kv, D, 256, dtype=cdt, device=dev, table=table)
    put = lambda c, a, b: c.append(*_cut(x[a:b], heads, kv), _i32([a], dev), _i32([0, b - a], dev),
                                   pos=_i32([at + a], dev), theta=1e4)
    one = lambda c, a: c.attend(*_cut(x[a:a + 1], heads, kv), _i32([a], dev), pos=_i32([at + a], dev), theta=1e4)
    whole, pieces, tokens, mixed = (new() for _ in range(4))
    rows = put(whole, 0, n)
    cut = [put(pieces, a, b) for a, b in ((0, 1), (1, 63), (63, 128), (128, 131), (131, n))]
    for i, t in enumerate(rows):
        assert torch.equal(torch.cat([c[i] for c in cut]), t)
    for t in range(n):
        one(tokens, t)
    put(mixed, 0, 60)
    for t in range(60, 66):
        one(mixed, t)
    put(mixed, 66, 190)
    for t in range(190, n):
        one(mixed, t)
    for c in (pieces, tokens, mixed):
        _same_bits(c, whole, [n])


# --- forms that nothing else reaches -----------------------------------------------------------------------
@pytest.mark.parametrize("dt,cdt", [(BF, FP), (FP, BF)])
@pytest.mark.parametrize("heads,kv,D", [(16, 2, 128), (5, 5, 64)])
def test_append_of_the_other_16_bit_type(dev, dt, cdt, heads, kv, D):
    check_append(dev, dt, cdt, heads, kv, D, [100, 5, 0], [28, 300, 0])


@pytest.mark.parametrize("cdt,dt,odt", [(BF, F32, BF), (FP, F32, F32)])
@pytest.mark.parametrize("heads,kv,D", [(16, 2, 128), (20, 2, 64)])
def test_attend_without_a_table(dev, cdt, dt, odt, heads, kv, D):
    past = [0, 63, 300]
    cache = _filled(3, kv, D, cdt, past, 6, dev, 91, table=False)
    assert cache.blocks is None
    x = _rows(3, heads, kv, D, dt, 92)
    before = _cpu(cache)
    got, weight = cache.attend(*_cut(x.to(dev), heads, kv), _i32(past, dev), theta=1e6,
                               weight_out=cache.new_weight(), out_dtype=odt)
    now = _cpu(cache)
    for b, p in enumerate(past):
        before.k_tail[b, :, p % BLOCK] = now.k_tail[b, :, p % BLOCK]
        before.v_tail[b, :, :, p % BLOCK] = now.v_tail[b, :, :, p % BLOCK]
    _check_attend(before, x, heads, past, past, got, weight, 1e6, odt)
    at = 63 // BLOCK
    for name in "kv":      # the second sequence's token ended its first block, which lies in its place
        want, sc = ref.to8(getattr(now, name + "_tail")[1].reshape(kv, -1))
        assert torch.equal(getattr(now, name)[1, :, at].reshape(kv, -1).float(), want.float())
        assert torch.equal(getattr(now, name + "_scale")[1, :, at], sc)


@pytest.mark.parametrize("dt", [F32, BF, FP])
@pytest.mark.parametrize("out", [BF, FP])
@pytest.mark.parametrize("heads,kv,D,theta", [(16, 2, 128, 1e6), (5, 5, 64, 1e4), (4, 1, 64, 0.0)])
def test_rope_rows(dev, dt, out, heads, kv, D, theta):
    """Rows rotated without a cache: values, positions far out, given outputs, rows that are left alone."""
    lens, pos = [70, 0, 5, 64], [0, 9, -1, 131_072]
    x = _rows(sum(lens) + 3, heads, kv, D, dt, 95)
    cu = _ends(lens)
    q, k, v = rope_rows(*_cut(x.to(dev), heads, kv), cu.to(dev), _i32(pos, dev), theta, dtype=out)
    outs = tuple(torch.full_like(t, 7.0) for t in (q, k, v))
    same = rope_rows(*_cut(x.to(dev), heads, kv), cu.to(dev), _i32(pos, dev), theta, dtype=out, outs=outs)
    h, tiny = ref.half_step(out), torch.finfo(out).smallest_normal * ref.half_step(out)
    for got, mine, src in zip((q, k, v), same, _cut(x, heads, kv)):
        assert got.dtype == out
        for s in range(len(lens)):
            r = slice(int(cu[s]), int(cu[s + 1]))
            if pos[s] < 0:
                assert (mine[r] == 7).all()
                continue
            want, off = (src[r].double(), 0.0) if got is v else ref.rotate(
                src[r], pos[s] + torch.arange(lens[s]), theta)
            assert ((got[r].cpu().double() - want).abs() <= h * want.abs() + 1.01 * off + tiny).all()
            assert torch.equal(got[r], mine[r])
        assert (mine[int(cu[-1]):] == 7).all()


def _splits(lens, past, heads, D, dev):
    """Into how many parts a prompt call cuts the keys: from its workspace."""
    n = sum(lens)
    return max(1, _hxq._prompt_workspace(n, n + sum(past), len(lens), heads, D, dev.index or 0) // (n * heads * (D * 4 + 8)))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dt,heads,kv,D,lens,past,splits", [
    (FP, 16, 4, 64, [512, 130, 1, 400, 257, 512], [7000, 6500, 7100, 0, 5000, 7000], 2),   # by die, tiles of 128
    (BF, 28, 4, 128, [300, 129, 40], [3000, 2500, 900], 3),
    (BF, 64, 8, 128, [100, 64], [6000, 5000], 4),
    (FP, 4, 4, 64, [40, 3], [900, 1200], 3)])                                            # each wave its own keys
def test_prompt_splits_of_ragged_batches(dev, dt, heads, kv, D, lens, past, splits, causal):
    """Several sequences of several tiles with their keys in parts, on 256 compute units."""
    if torch.cuda.get_device_properties(dev).multi_processor_count == 256:
        assert _splits(lens, past, heads, D, dev) == splits
    q, k, v, cu, cu_k = _prompt_case(lens, heads, kv, D, dt, 97, past)
    got = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev), cu_k.to(dev), causal=causal)
    _check_prompt(got, q, k, v, cu, cu_k, causal=causal)


def test_a_cache_on_another_device_is_refused(dev):
    """Rows on one device, the cache on another: its addresses mean nothing there."""
    heads, kv, D = 4, 2, 64
    cache = HelixKV8Cache.empty(1, kv, D, 128, device=dev)
    x, n = _rows(1, heads, kv, D, BF, 99).to(dev), _i32([0], dev)
    assert cache._desc.device == x.get_device()
    cache._desc.device += 1      # as of a cache there
    with pytest.raises(RuntimeError, match="cache is on"):
        cache.attend(*_cut(x, heads, kv), n)
    with pytest.raises(RuntimeError, match="cache is on"):
        cache.append(*_cut(x, heads, kv), n, _i32([0, 1], dev))


def test_a_prompt_a_token_and_an_eviction_captured(dev):
    """The whole run in one graph, replayed over a cache that each replay cuts again, with eager work
    between; every replay equals the eager run."""
    heads, kv, D, n, theta = 8, 2, 128, 150, 1e6
    xs = [_rows(n + 1, heads, kv, D, BF, 110 + i).to(dev) for i in range(4)]
    cu = _i32([0, n], dev)

    def step(cache, x, cached, pos, w):
        q, k, v = cache.append(*_cut(x[:n], heads, kv), cached, cu, pos=pos, theta=theta)
        o = attn_prompt(q, k, v, cu)
        cached += n
        pos += n
        one, _ = cache.attend(*_cut(x[n:], heads, kv), cached, pos=pos, theta=theta, weight=w, weight_out=w)
        cached += 1
        pos += 1
        cached.copy_(cache.evict(w, cached, keep=3, sink=1, recent=1))
        return o, one

    def fresh():
        cache = HelixKV8Cache.empty(1, kv, D, 512, device=dev)
        return cache, _i32([0], dev), _i32([0], dev), cache.new_weight()

    cache, cached, pos, w = fresh()
    want = []
    for x in xs:
        o, one = step(cache, x, cached, pos, w)
        want.append([t.clone() for t in (o, one, cached, pos, w, cache.blocks, cache.k.view(torch.uint8), cache.v_scale)])
    assert int(want[-1][2]) == 192 + (4 * (n + 1)) % 64
    cache, cached, pos, w = fresh()
    x = xs[0].clone()
    s, g = torch.cuda.Stream(device=dev), torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(s), torch.cuda.graph(g, stream=s):
        o, one = step(cache, x, cached, pos, w)
    torch.cuda.current_stream(dev).wait_stream(s)
    for i, right in enumerate(want):
        x.copy_(xs[i])
        g.replay()
        torch.randn(1 << 20, device=dev).sum().item()
        for a, b in zip((o, one, cached, pos, w, cache.blocks, cache.k.view(torch.uint8), cache.v_scale), right):
            assert torch.equal(a, b), i


# --- many sequences, wide groups, extreme arguments --------------------------------------------------------
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dt,heads,kv,D,long", [
    (BF, 1, 1, 128, False), (FP, 2, 1, 64, False),     # each wave its own keys; split and not
    (BF, 4, 2, 128, True), (FP, 4, 4, 64, True)])      # sequences of several tiles
def test_prompt_of_more_sequences_than_lanes(dev, dt, heads, kv, D, long, causal):
    """The tiles of 150 sequences, some without queries, some without keys, found in rounds of 64."""
    n = 150
    lens = [(37 * i) % 301 if long and i % 3 == 0 else (7 * i) % 6 for i in range(n)]
    past = [(53 * i) % 701 if i % 4 else -lens[i] for i in range(n)]
    q, k, v, cu, cu_k = _prompt_case(lens, heads, kv, D, dt, 121, past)
    got = attn_prompt(q.to(dev), k.to(dev), v.to(dev), cu.to(dev), cu_k.to(dev), causal=causal)
    _check_prompt(got, q, k, v, cu, cu_k, causal=causal)


@pytest.mark.parametrize("heads", [4, 64])
def test_prompt_without_any_key(dev, heads):
    q, _, _, cu, _ = _prompt_case([70, 3], heads, 2, 64, BF, 122)
    none = torch.empty(0, 2, 64, dtype=BF, device=dev)
    got = attn_prompt(q.to(dev), none, none, cu.to(dev), torch.zeros(3, dtype=torch.int32, device=dev))
    assert (got == 0).all()


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("heads", [4, 64])
def test_prompt_scale_at_its_ends(dev, dt, heads):
    """2^-100: the mean of what a query sees.  2^100 over products of 2^-100: as 1 over products of 1."""
    q, k, v, cu, _ = _prompt_case([200], heads, 2, 128, dt, 123)
    a = [t.to(dev) for t in (q, k, v, cu)]
    got = attn_prompt(*a, scale=2.0 ** -100)
    _check_prompt(got, q * 0, k, v, cu, cu)
    if dt == BF:
        small = attn_prompt(a[0] * 2.0 ** -50, a[1] * 2.0 ** -50, *a[2:], scale=2.0 ** 100)
        assert torch.equal(small, attn_prompt(*a, scale=1.0))


def test_append_and_attend_of_more_sequences_than_lanes(dev):
    """150 sequences, some skipped, some without rows: each as in a call of its own."""
    heads, kv, D, n, theta = 4, 2, 64, 150, 1e4
    lens = [(29 * i) % 140 if i % 3 else 0 for i in range(n)]
    cached = [-1 if i % 11 == 5 else (17 * i) % 100 for i in range(n)]
    cu, x = _ends(lens), _rows(sum(lens), heads, kv, D, BF, 131).to(dev)
    first = _rows(100, heads, kv, D, BF, 132).to(dev)
    t = _rows(n, heads, kv, D, F32, 133).to(dev)
    cache = HelixKV8Cache.empty(n, kv, D, 256, device=dev)
    fill = _ends([max(c, 0) for c in cached])
    rows = torch.cat([first[:max(c, 0)] for c in cached])
    cache.append(*_cut(rows, heads, kv), _i32([0] * n, dev), fill.to(dev), theta=theta)
    outs = tuple(torch.full((sum(lens), h, D), 7.0, dtype=BF, device=dev) for h in (heads, kv, kv))
    cache.append(*_cut(x, heads, kv), _i32(cached, dev), cu.to(dev), theta=theta, outs=outs)
    now = [c if c < 0 else c + m for c, m in zip(cached, lens)]
    w = torch.full((n, kv, 4), 3.0, device=dev)
    out = torch.full((n, heads, D), 5.0, device=dev)
    cache.attend(*_cut(t, heads, kv), _i32(now, dev), theta=theta, weight_out=w, out=out)
    for i in range(0, n):
        r = slice(int(cu[i]), int(cu[i + 1]))
        if cached[i] < 0:
            assert all((o[r] == 7).all() for o in outs) and (out[i] == 5).all() and (w[i] == 3).all()
            assert (cache.k[i].view(torch.uint8) == 0).all() and (cache.k_tail[i] == 0).all()
            continue
        if i % 7:
            continue
        one = HelixKV8Cache.empty(1, kv, D, 256, device=dev)
        one.append(*_cut(first[:cached[i]], heads, kv), _i32([0], dev), _i32([0, cached[i]], dev), theta=theta)
        mine = one.append(*_cut(x[r], heads, kv), _i32([cached[i]], dev), _i32([0, lens[i]], dev), theta=theta)
        for a, b in zip(mine, outs):
            assert torch.equal(a, b[r])
        o, ww = one.attend(*_cut(t[i:i + 1], heads, kv), _i32([now[i]], dev), theta=theta,
                           weight_out=one.new_weight(), out_dtype=F32)
        held = now[i] + 1
        assert torch.equal(cache.k[i].view(torch.uint8), one.k[0].view(torch.uint8))
        assert torch.equal(cache.v_tail[i][..., :held % BLOCK], one.v_tail[0][..., :held % BLOCK])
        assert torch.equal(out[i], o[0]) and torch.equal(w[i], ww[0])      # one split in both


@pytest.mark.parametrize("cdt,dt,odt", [(FP, F32, F32), (BF, FP, F32)])
@pytest.mark.parametrize("heads,kv,D", [(20, 2, 64), (16, 1, 128), (7, 7, 64), (9, 1, 64)])
def test_attend_long_of_other_groups(dev, cdt, dt, odt, heads, kv, D):
    """More than eight query heads a kv head over many splits, a token that ends its block among them."""
    past = [6000, 64 * 90 + 63, 0, 64 * 40]
    cache = _filled(4, kv, D, cdt, past, 96, dev, 141)
    x = _rows(4, heads, kv, D, dt, 142)
    x[:, heads:heads + kv] *= 0.3
    before = _cpu(cache)
    w = torch.full((4, kv, 96), 0.25, device=dev)
    got, weight = cache.attend(*_cut(x.to(dev), heads, kv), _i32(past, dev), theta=1e6, weight=w, weight_out=w,
                               out_dtype=odt)
    now = _cpu(cache)
    for b, p in enumerate(past):
        before.k_tail[b, :, p % BLOCK] = now.k_tail[b, :, p % BLOCK]
        before.v_tail[b, :, :, p % BLOCK] = now.v_tail[b, :, :, p % BLOCK]
    _check_attend(before, x, heads, past, past, got, weight, 1e6, odt, w0=0.25)
