"""The decoder in fp64, a piece of tokens at a time: what a query sees of earlier pieces is what the cache
holds of them (8-bit cache: blocks of 64 in e4m3, the rest in bf16); its own piece in bf16.

The model is HXQ-encoded noise, but its first norms are scaled by 9, so that attention is sharp and its
part of the logits large: a mistake in one block of the cache moves them by 2.4 % of the largest, what
bf16 roundings amount to by 0.5 % (``test_decoder_cached_host``)."""
import types

import numpy as np
import torch

import attention_ref as ref
import oracle
from helix_substrate import synth
from helix_substrate.decoder import DecoderConfig, HelixDecoder

CFG = DecoderConfig(hidden=512, n_layers=2, n_heads=4, n_kv_heads=2, head_dim=128, intermediate=768,
                    vocab=1000, rope_theta=1e6, rms_eps=1e-6, max_seq=448)
IDS = [(37 * i * i + 11 * i + 5) % 1000 for i in range(300)]


def build(cfg, dev=None):
    """The test's decoder on a device (None: its weights on the host only)."""
    make = HelixDecoder.synthetic
    if dev is None:
        made = lambda c, layers, embed, norm: types.SimpleNamespace(cfg=c, layers=layers, embed=embed,
                                                                    final_norm=norm)
        make = lambda *a, **k: HelixDecoder.synthetic.__func__(made, *a, **k)
    dec = make(cfg, seed=0, device=dev or "cpu",
               layer_fn=lambda o, i, s: synth.make_layer_np(o, i, seed=s, group_size=64))
    for L in dec.layers:
        L["in_norm"] *= 9
    return dec


def dense_layers(dec):
    """(embedding, layers, final norm) of a decoder as dense arrays on the host."""
    cpu = lambda t: None if t is None else t.detach().cpu().numpy()
    layers = []
    for L in dec.layers:
        d = {n: oracle.reconstruct(cpu(L[n].indices), cpu(L[n].codebook), cpu(L[n].group_scale),
                                   cpu(L[n].group_offset), L[n].group_size, cpu(L[n].sidecar_positions),
                                   cpu(L[n].sidecar_values))
             for n in ("q", "k", "v", "o", "gate", "up", "down")}
        d.update({"b" + n: cpu(L[n].bias) for n in "qkv"}, in_norm=cpu(L["in_norm"]), post_norm=cpu(L["post_norm"]))
        layers.append(d)
    return dec.embed.float().cpu().numpy().astype(np.float64), layers, cpu(dec.final_norm)


def _held(x, e4m3):
    """[tokens, kv heads, D] -> as the cache holds them."""
    x = torch.from_numpy(x).to(torch.bfloat16).double()
    n = len(x) // ref.BLOCK * ref.BLOCK if e4m3 else 0
    for a in range(0, n, ref.BLOCK):
        for h in range(x.shape[1]):
            v8, scale = ref.to8(x[a:a + ref.BLOCK, h].reshape(-1))
            x[a:a + ref.BLOCK, h] = (v8.double() * scale.double()).view(ref.BLOCK, -1)
    return x


def _bf16(x):
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.bfloat16).double().numpy()


class CachedDecoder:
    """kv[layer] = (keys, values) [tokens, kv heads, D] in bf16's rounding, each head's in the order of its
    block table.  rounded: the other roundings to bf16 that the decoder makes too (weights of the prompt's
    products, what enters and leaves a projection); the difference says what they amount to."""

    def __init__(self, cfg, weights, rounded=False):
        self.cfg, (self.embed, self.layers, self.norm) = cfg, weights
        self.r = _bf16 if rounded else lambda x: x
        if rounded:
            self.layers = [{n: _bf16(w) if np.ndim(w) == 2 else w for n, w in L.items()} for L in self.layers]
        c = cfg
        self.kv = [tuple(np.zeros((0, c.n_kv_heads, c.head_dim)) for _ in "kv") for _ in self.layers]
        self.pos = 0

    def feed(self, tokens):
        """Logits [len(tokens), vocab] of one piece."""
        c, E, r = self.cfg, self.embed, self.r
        T, D = len(tokens), c.head_dim
        x = E[np.asarray(tokens)]
        pos = self.pos + np.arange(T)
        for li, L in enumerate(self.layers):
            lin = lambda h, n: r(oracle.linear_np(h, L[n], L.get("b" + n)))
            h = r(oracle.rmsnorm_np(x, L["in_norm"], c.rms_eps))
            q, k, v = (lin(h, n).reshape(T, -1, D) for n in "qkv")
            q, k = (oracle.rope_np(t.transpose(1, 0, 2), pos, c.rope_theta).transpose(1, 0, 2) for t in (q, k))
            old = self.kv[li]
            k, v = _bf16(k), _bf16(v)
            keys, vals = (torch.cat([_held(o, c.kv_cache == "e4m3"), torch.from_numpy(n)]) for o, n in zip(old, (k, v)))
            a = ref.attention(torch.from_numpy(r(q)), keys, vals, D ** -0.5, ref.causal(T, len(keys)))[0]
            self.kv[li] = tuple(np.concatenate([o, n]) for o, n in zip(old, (k, v)))
            x = x + lin(r(a.reshape(T, -1).numpy()), "o")
            h = r(oracle.rmsnorm_np(x, L["post_norm"], c.rms_eps))
            x = x + lin(r(oracle.silu_np(lin(h, "gate")) * lin(h, "up")), "down")
        self.pos += T
        return oracle.linear_np(r(oracle.rmsnorm_np(x, self.norm, c.rms_eps)), E)

    def keep(self, blocks):
        """After an eviction: blocks[layer][head] are the full blocks that stay, by their place in order."""
        out = []
        for (k, v), heads in zip(self.kv, blocks):
            n = len(k) // ref.BLOCK * ref.BLOCK
            rows = [np.concatenate([np.arange(b * ref.BLOCK, (b + 1) * ref.BLOCK) for b in bs] + [np.arange(n, len(k))])
                    for bs in heads]
            out.append(tuple(np.stack([t[r, h] for h, r in enumerate(rows)], 1) for t in (k, v)))
        self.kv = out


def off(a, b):
    """Largest difference of every token's logits, relative to its largest logit."""
    return np.abs(a - b).max(-1) / np.abs(b).max(-1)
