"""The decoder over caches of more than a block: logits against the fp64 oracle that sees what the cache
holds, in pieces, token by token and after eviction.  What has no room is refused.

The bar is three times the most that bf16's roundings move the oracle's own logits by at the tokens that
are compared (all roundings but those of the softmax weights, a part of the output's; the kernels' sums
add in another order)."""
from dataclasses import replace

import numpy as np
import pytest

import decoder_cached_ref as plain
from test_gpu_decoder_prompt import PROMPT, _build

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
def test_prefill_counts_what_the_cache_holds(dev, kv):
    """Token by token as in one pass: a prompt that does not fit behind the cached tokens is refused,
    one that just fits is not."""
    dec = _build(dev, kv_cache=kv)
    room = dec.cfg.max_seq
    assert room == 64
    for feed in (dec.prefill, dec.prefill_prompt):
        dec.reset()
        feed(PROMPT)
        with pytest.raises(ValueError, match="longer than max_seq"):
            feed(PROMPT[:room - len(PROMPT) + 1])
        assert int(dec.pos.item()) == len(PROMPT)
        feed(PROMPT[:room - len(PROMPT)])
        assert int(dec.pos.item()) == room


class _Pair:
    """The decoder and its oracle, fed alike."""

    def __init__(self, dev, **change):
        cfg = replace(plain.CFG, **change)
        self.dec = plain.build(cfg, dev)
        weights = plain.dense_layers(self.dec)
        self.exact, self.rounded = (plain.CachedDecoder(cfg, weights, r) for r in (False, True))
        self.bar, self.worst = 0.0, 0.0

    def feed(self, ids, got):
        want, near = self.exact.feed(ids)[-1], self.rounded.feed(ids)[-1]
        if got is not None:
            self.bar = max(self.bar, 3 * float(plain.off(near, want)))
            self.worst = max(self.worst, float(plain.off(got.cpu().numpy(), want)))

    def token(self, t):
        self.dec.tok.fill_(t)
        self.dec._step_launches()
        self.feed([t], self.dec.logits)

    def check(self):
        print(f"off by {self.worst:.5f}, bar {self.bar:.5f}")
        assert self.worst <= self.bar <= 0.02, (self.worst, self.bar)


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("chunk", [70, 64, 4096])
def test_long_prompts_and_tokens_match_the_oracle(dev, kv, chunk):
    n, p = 220, _Pair(dev, kv_cache=kv)
    p.dec.prefill_prompt(plain.IDS[:n], chunk=chunk)
    for a in range(0, n, chunk):
        b = min(a + chunk, n)
        p.feed(plain.IDS[a:b], p.dec.logits if b == n else None)
    for t in plain.IDS[n:n + 40]:     # past the end of the fourth block
        p.token(t)
    p.check()


def test_tokens_from_the_first_match_the_oracle(dev):
    p = _Pair(dev, kv_cache="e4m3")
    for t in plain.IDS[:135]:
        p.token(t)
    p.check()


def test_tokens_after_an_eviction_match_the_oracle(dev):
    n, p = 330, _Pair(dev, kv_cache="e4m3", kv_weight=True)
    ids = (plain.IDS * 2)[:n + 60]
    p.dec.prefill_prompt(ids[:n])
    p.feed(ids[:n], p.dec.logits)
    for t in ids[n:n + 8]:
        p.token(t)
    before = [c.blocks[0].tolist() for c in p.dec.kv8]
    p.dec.evict(keep=3, sink=1, recent=1)
    after = [c.blocks[0].tolist() for c in p.dec.kv8]
    kept = [[[old.index(b) for b in new[:3]] for old, new in zip(*two)] for two in zip(before, after)]
    assert all(k[0] == 0 and k[2] == 4 and 0 < k[1] < 4 for heads in kept for k in heads)
    for m in (p.exact, p.rounded):
        m.keep(kept)
    for t in ids[n + 8:n + 60]:       # the unfinished block ends behind the three
        p.token(t)
    assert int(p.dec.cached.item()) == 3 * 64 + (n + 8) % 64 + 52 and int(p.dec.pos.item()) == n + 60
    p.dec.prefill_prompt(ids[:70])    # and a prompt goes on from there
    p.feed(ids[:70], p.dec.logits)
    p.check()
