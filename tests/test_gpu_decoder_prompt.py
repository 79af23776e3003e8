"""The decoder's one-pass prompt, its 8-bit cache and eviction, against the fp64 oracle of
transformers' Qwen2 math at the decoder's bf16 bar (2e-2 of max|logit|)."""
from dataclasses import replace

import numpy as np
import pytest
import torch

from helix_substrate import synth
from helix_substrate.decoder import HelixDecoder
from test_gpu_decoder import CFG, _oracle_logits

pytestmark = pytest.mark.gpu

PROMPT = [(37 * i * i + 11 * i + 5) % 1000 for i in range(60)]


def _build(dev, **change):
    mk = lambda o, i, s: synth.make_layer_np(o, i, seed=s, group_size=64)
    return HelixDecoder.synthetic(replace(CFG, **change), seed=0, device=dev, layer_fn=mk)


def _near(got, ref):
    return np.abs(got - ref).max() / np.abs(ref).max()


@pytest.mark.parametrize("kv", ["bf16", "e4m3"])
@pytest.mark.parametrize("n,chunk", [(1, 4096), (7, 4096), (60, 4096), (60, 17)])
def test_prompt_in_one_pass_matches_oracle(dev, kv, n, chunk):
    """Below 64 tokens the 8-bit cache holds its 16-bit tail only: the same bar."""
    dec = _build(dev, kv_cache=kv)
    dec.prefill_prompt(PROMPT[:n], chunk=chunk)
    ref = _oracle_logits(dec, PROMPT[:n] + [9, 8])
    assert int(dec.pos.item()) == n
    got = dec.logits.cpu().numpy()
    assert _near(got, ref[n - 1]) <= 2e-2
    assert int(dec.tok.item()) == int(np.argmax(got))
    for i, tok in enumerate((9, 8)):          # decoding goes on behind it
        dec.tok.fill_(tok)
        dec._step_launches()
        assert _near(dec.logits.cpu().numpy(), ref[n + i]) <= 2e-2
    assert int(dec.pos.item()) == n + 2


def test_token_by_token_e4m3_matches_oracle(dev):
    dec = _build(dev, kv_cache="e4m3")
    ref = _oracle_logits(dec, PROMPT[:9])
    for t, tok in enumerate(PROMPT[:9]):
        dec.tok.fill_(tok)
        dec._step_launches()
        assert _near(dec.logits.cpu().numpy(), ref[t]) <= 2e-2


def test_prompt_in_pieces_leaves_the_caches_of_one_pass(dev):
    """Layer 0's rows depend on their own tokens only: its cache is the same bit for bit however the
    prompt is cut, as long as every piece runs the same GEMM (rows of one length)."""
    ids = (PROMPT * 5)[:256]
    caches = []
    for chunk in (128, 64):
        dec = _build(dev, kv_cache="e4m3", max_seq=320)
        dec.prefill_prompt(ids, chunk=chunk)
        caches.append(dec.kv8[0].read(0, 256))
        assert int(dec.cached.item()) == int(dec.pos.item()) == 256
    for a, b in zip(*caches):
        # the two GEMM shapes may round a key differently: one e4m3 step at most, and rarely
        a, b = a.float(), b.float()
        step = 2.0 ** -3 * torch.maximum(a.abs(), b.abs()) + 1e-3 * a.abs().max()
        assert ((a - b).abs() <= step).all()
        assert (a != b).float().mean() <= 0.05


def test_e4m3_graph_equals_eager_and_evicts(dev):
    make = lambda: _build(dev, kv_cache="e4m3", kv_weight=True, max_seq=448)
    ids = (PROMPT * 7)[:400]
    eager, graphed = make(), make()
    outs = []
    for dec, graph in ((eager, False), (graphed, True)):
        dec.prefill_prompt(ids)
        if graph:
            dec.capture()
        first = dec.generate(20, use_graph=graph)
        with pytest.raises(ValueError, match="exceed"):
            dec.generate(100, use_graph=graph)
        blocks = [c.blocks.clone() for c in dec.kv8]
        dec.evict(keep=3, sink=1, recent=1)
        assert int(dec.cached.item()) == 3 * 64 + 420 % 64 and int(dec.pos.item()) == 420
        for old, cache in zip(blocks, dec.kv8):
            assert torch.equal(cache.blocks.sort(-1)[0], old.sort(-1)[0])
            assert torch.equal(cache.blocks[..., 0], old[..., 0])       # the sink
            assert torch.equal(cache.blocks[..., 2], old[..., 5])       # the last full one
        second = dec.generate(100, use_graph=graph)
        assert torch.isfinite(dec.logits).all()
        assert int(dec.cached.item()) == 3 * 64 + 420 % 64 + 100 and int(dec.pos.item()) == 520
        outs.append((first, second, dec.logits.clone(), [w.clone() for w in dec.kv_weight]))
        dec.close()
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert torch.equal(outs[0][2], outs[1][2])
    for a, b in zip(outs[0][3], outs[1][3]):
        assert torch.equal(a, b)


def test_eviction_that_keeps_all_changes_nothing(dev):
    a = _build(dev, kv_cache="e4m3", kv_weight=True, max_seq=448)
    a.prefill_prompt((PROMPT * 4)[:200])
    a.evict(keep=3, sink=1, recent=1)
    before = int(a.cached.item())
    b = _build(dev, kv_cache="e4m3", kv_weight=True, max_seq=448)
    b.prefill_prompt((PROMPT * 4)[:200])
    assert before == 200
    for dec in (a, b):
        dec._step_launches()
    assert torch.equal(a.logits, b.logits)


def test_refusals(dev):
    with pytest.raises(ValueError, match="kv_cache"):
        _build(dev, kv_cache="int8")
    dec = _build(dev)
    for bad in ([], [1000], [-1], list(range(65))):
        with pytest.raises(ValueError):
            dec.prefill_prompt(bad)
    with pytest.raises(ValueError, match="chunk"):
        dec.prefill_prompt([1], chunk=0)
    with pytest.raises(ValueError, match="evict"):
        dec.evict(4)
    dec8 = _build(dev, kv_cache="e4m3")
    with pytest.raises(ValueError, match="evict"):
        dec8.evict(4)
    with pytest.raises(ValueError, match="bf16"):
        dec8.persistent_init()
    with pytest.raises(ValueError, match="bf16"):
        dec8._step_launches(fused=False)
    dec8.prefill_prompt(PROMPT)
    dec8.reset()
    dec8.prefill_prompt(PROMPT)
    assert int(dec8.cached.item()) == 60
