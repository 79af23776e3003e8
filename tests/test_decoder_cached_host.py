"""The fp64 decoder with a cache (``decoder_cached_ref``): what its comparison with the kernels can tell
apart.  Mistakes are planted in the oracle, and each moves the logits past the bar that bf16's
roundings set."""
from dataclasses import replace

import numpy as np
import pytest

import oracle
import decoder_cached_ref as plain

N = 220


@pytest.fixture(scope="module")
def weights():
    return plain.dense_layers(plain.build(plain.CFG))


def run(weights, kv="e4m3", mistake=None, rounded=False):
    m = plain.CachedDecoder(replace(plain.CFG, kv_cache=kv), weights, rounded)
    out = [m.feed(plain.IDS[a:min(a + 70, N)]) for a in range(0, N, 70)]
    if mistake:
        mistake(m)
    return np.concatenate(out + [m.feed(plain.IDS[t:t + 1]) for t in range(N, N + 3)])


def test_without_8_bits_it_is_the_plain_decoder(weights):
    """But for keys and values in bf16."""
    c = plain.CFG
    want = oracle.qwen2_logits_np(plain.IDS[:N + 3], *weights, c.n_heads, c.n_kv_heads, c.head_dim, c.rope_theta,
                                  c.rms_eps)
    assert plain.off(run(weights, kv="bf16"), want).max() <= 5e-3


def _blocks(which):
    def change(m):
        for li, kv in enumerate(m.kv):
            kv = [x.copy() for x in kv]
            which(*kv)
            m.kv[li] = tuple(kv)
    return change


def _swap(k, v):
    v[64:128], v[128:192] = v[128:192].copy(), v[64:128].copy()


def _scale(k, v):
    k[128:192] *= 2


def _stale(k, v):
    v[192:210] = v[128:146]


def _head(k, v):
    v[64:128, 0] = v[64:128, 1]


def _drop(m):
    m.kv = [tuple(np.delete(x, slice(64, 128), 0) for x in kv) for kv in m.kv]


def _late(m):
    m.pos += 64


@pytest.mark.parametrize("mistake", [_blocks(_swap), _blocks(_scale), _blocks(_stale), _blocks(_head), _drop, _late])
def test_the_bar_tells_mistakes(weights, mistake):
    right = run(weights)
    bar = 3 * plain.off(run(weights, rounded=True), right).max()
    assert bar <= 0.02
    assert plain.off(run(weights, mistake=mistake), right)[N:].max() > bar
