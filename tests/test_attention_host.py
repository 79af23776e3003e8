"""Refusals of the attention operators (validation runs before any HIP call: no GPU), and their plain
forms against closed cases."""
import ctypes
import math

import pytest
import torch

import attention_ref as ref
from helix_substrate import _hxq
from helix_substrate.attention import HelixKV8Cache, attn_prompt, kv8_evict

A = 1 << 20    # an aligned address that nothing reads


@pytest.fixture(scope="module")
def lib():
    return _hxq.lib()


def _message(lib):
    return lib.hxq_last_error().decode()


PROMPT = dict(q=A, q_row=2048, q_head=128, k=A, k_row=256, k_head=128, v=A, v_row=256, v_head=128,
              dtype=_hxq.HXQ_BF16, cu_q=A, cu_k=None, n=1, rows_q=8, rows_k=8, heads=16, kv=2, D=128,
              scale=0.1, causal=1, out=A, o_row=2048, o_head=128, ws=None, ws_bytes=0,
              stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=_hxq.HXQ_F32), "bf16 or fp16"), (dict(dtype=9), "bf16 or fp16"),
    (dict(D=96), "head_dim"), (dict(heads=15), "multiple"), (dict(kv=0), "multiple"),
    (dict(q=A + 2), "16 bytes"), (dict(k_row=257), "16 bytes"), (dict(v_head=4), "16 bytes"),
    (dict(o_row=2052), "16 bytes"), (dict(q=None), "required"), (dict(out=None), "required"),
    (dict(cu_q=None), "required"), (dict(k=None), "required"), (dict(n=-1), "sizes"),
    (dict(rows_q=1 << 31), "sizes"), (dict(rows_k=-1), "sizes"), (dict(scale=math.nan), "scale"),
    (dict(scale=0.0), "scale"), (dict(scale=math.inf), "scale"),
    (dict(k_row=1 << 24), "row strides"), (dict(v_row=-8), "row strides"),
    (dict(rows_k=8192), "workspace"), (dict(rows_k=8192, ws=A, ws_bytes=64), "workspace"),
    (dict(rows_k=8192, ws=A + 8, ws_bytes=1 << 40), "workspace")])
def test_prompt_refuses(lib, change, text):
    assert lib.hxq_attn_prompt(*{**PROMPT, **change}.values()) == 1
    assert text in _message(lib)


@pytest.mark.parametrize("change,text", [
    (dict(scale=2.0 ** -101), "scale"), (dict(scale=2.0 ** 101), "scale"),
    (dict(n=1 << 21), "too many"),                                # 2^21 sequences, 16 heads, 256 threads
    (dict(heads=64, kv=64, rows_k=(1 << 30), n=1 << 19, ws=A, ws_bytes=1 << 40), "too many")])
def test_prompt_refuses_what_a_launch_cannot_hold(lib, change, text):
    assert lib.hxq_attn_prompt(*{**PROMPT, **change}.values()) == 1
    assert text in _message(lib)


def test_cache_launches_too_large(lib):
    assert _append(lib, _desc(batch=1 << 24)) == 1 and "too many" in _message(lib)
    assert _attend(lib, _desc(batch=65535, n_blocks=1 << 24), ws_bytes=1 << 60) == 1 and "too large" in _message(lib)
    assert lib.hxq_kv8_evict(*{**EVICT, "batch": 1 << 21}.values()) == 1 and "sizes" in _message(lib)
    assert _attend(lib, _desc(), scale=2.0 ** 101) == 1 and "scale" in _message(lib)
    assert lib.hxq_kv8_attn_decode_workspace_bytes(1, 16, 2, 96, 4, 0) == -1


def test_prompt_of_nothing(lib):
    assert lib.hxq_attn_prompt(*{**PROMPT, "n": 0}.values()) == 0
    assert lib.hxq_attn_prompt(*{**PROMPT, "rows_q": 0, "q": None}.values()) == 0


def test_prompt_workspace(lib):
    need = lib.hxq_attn_prompt_workspace_bytes
    assert need(8, 8, 1, 16, 128) == 0 and need(4096, 4096, 1, 16, 128) == 0
    assert need(0, 8, 1, 16, 128) == 0 and need(8, 8, 0, 16, 128) == 0
    assert need(8, 8, 1, 16, 96) == -1 and need(-1, 8, 1, 16, 128) == -1
    rest, bytes_a_split = divmod(need(8, 8192, 1, 16, 128), 8 * 16 * (128 * 4 + 8))
    assert rest > 1 and bytes_a_split == 0


def _desc(**change):
    d = dict(k=A, v=A, k_scale=A, v_scale=A, k_tail=A, v_tail=A, blocks=None, dtype=_hxq.HXQ_BF16,
             batch=2, n_kv_heads=2, head_dim=128, n_blocks=4)
    return _hxq.HxqKv8(*{**d, **change}.values())


BAD_CACHES = [dict(v=None), dict(k=A + 8), dict(k_tail=A + 2), dict(v_tail=None), dict(k_scale=None),
              dict(dtype=_hxq.HXQ_F32), dict(batch=0), dict(n_kv_heads=0), dict(head_dim=80),
              dict(n_blocks=0)]
APPEND = dict(q=A, q_row=2048, q_head=128, k=A, k_row=256, k_head=128, v=A, v_row=256, v_head=128,
              dtype=_hxq.HXQ_F32, cu=A, rows=8, heads=16, cached=A, pos=None, theta=1e6, cache=None,
              q_out=A, k_out=A, v_out=A, stream=None)


def _append(lib, desc, **change):
    args = {**APPEND, "cache": ctypes.byref(desc), **change}
    return lib.hxq_kv8_append(*args.values())


@pytest.mark.parametrize("change", BAD_CACHES)
def test_append_refuses_caches(lib, change):
    assert _append(lib, _desc(**change)) == 1 and "bad cache" in _message(lib)


@pytest.mark.parametrize("change,text", [
    (dict(k=None), "required"), (dict(q=None), "required"), (dict(cu=None), "required"),
    (dict(cached=None), "required"), (dict(dtype=3), "dtype"), (dict(heads=3), "multiple"),
    (dict(rows=-1), "sizes"), (dict(rows=1 << 31), "sizes"), (dict(theta=-1.0), "theta"),
    (dict(theta=math.nan), "theta"), (dict(v_row=130), "16 bytes"), (dict(q=A + 4), "16 bytes"),
    (dict(k_out=A + 4), "aligned"), (dict(cache=None), "bad cache")])
def test_append_refuses(lib, change, text):
    assert _append(lib, _desc(), **change) == 1 and text in _message(lib)


def test_append_of_nothing(lib):
    assert _append(lib, _desc(), rows=0, q=None, k=None, v=None) == 0


ATTEND = dict(q=A, q_row=2048, q_head=128, k=A, k_row=256, k_head=128, v=A, v_row=256, v_head=128,
              dtype=_hxq.HXQ_F32, heads=16, cached=A, pos=None, theta=1e6, scale=0.1, cache=None,
              w_in=None, w_out=A, out=A, out_dtype=_hxq.HXQ_BF16, ws=A, ws_bytes=1 << 40, stream=None)


def _attend(lib, desc, **change):
    return lib.hxq_kv8_attn_decode(*{**ATTEND, "cache": ctypes.byref(desc), **change}.values())


@pytest.mark.parametrize("change", [*BAD_CACHES, dict(k=None)])
def test_attend_refuses_caches(lib, change):
    assert _attend(lib, _desc(**change)) == 1 and "bad cache" in _message(lib)


@pytest.mark.parametrize("change,text", [
    (dict(q=None), "required"), (dict(out=None), "required"), (dict(cached=None), "required"),
    (dict(dtype=4), "dtype"), (dict(out_dtype=-1), "dtype"), (dict(heads=5), "multiple"),
    (dict(scale=math.nan), "finite"), (dict(theta=-2.0), "finite"),
    (dict(w_in=A, w_out=None), "weight_in"), (dict(ws=None), "workspace"),
    (dict(ws_bytes=16), "workspace"), (dict(ws=A + 4), "workspace")])
def test_attend_refuses(lib, change, text):
    assert _attend(lib, _desc(), **change) == 1 and text in _message(lib)


def test_attend_workspace(lib):
    need = lib.hxq_kv8_attn_decode_workspace_bytes
    assert need(0, 16, 2, 128, 4, 0) == -1 and need(1, 15, 2, 128, 4, 0) == -1
    assert need(1, 16, 2, 128, 0, 1) == -1
    assert need(1, 16, 2, 128, 4, 0) == 0                  # one split, no weights
    assert need(1, 16, 2, 128, 2048, 1) > need(1, 16, 2, 128, 2048, 0) > 0


EVICT = dict(w=A, b=None, c=A, batch=1, kv=2, n=8, keep=4, sink=1, recent=1, wo=2 * A, bo=3 * A,
             co=4 * A, stream=None)


@pytest.mark.parametrize("change,text", [
    (dict(w=None), "required"), (dict(wo=None), "required"), (dict(bo=None), "required"),
    (dict(co=None), "required"), (dict(wo=A), "must not be"), (dict(b=A, bo=A), "must not be"),
    (dict(co=A), "must not be"), (dict(keep=0), "keep"), (dict(sink=-1), "keep"),
    (dict(sink=3, recent=2), "keep"), (dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1), "keep"),
    (dict(batch=0), "sizes"), (dict(n=0), "sizes")])
def test_evict_refuses(lib, change, text):
    assert lib.hxq_kv8_evict(*{**EVICT, **change}.values()) == 1
    assert text in _message(lib)


def test_host_tensors_are_refused():
    x, cu = torch.zeros(4, 2, 64, dtype=torch.bfloat16), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="device tensors"):
        attn_prompt(x, x, x, cu)
    with pytest.raises(RuntimeError, match="device tensors"):
        HelixKV8Cache.empty(1, 2, 64, 64, device="cpu")
    with pytest.raises(RuntimeError, match="device tensors"):
        kv8_evict(torch.zeros(1, 1, 4), None, torch.zeros(1, dtype=torch.int32), 2)
    with pytest.raises(ValueError, match="positive"):
        HelixKV8Cache.empty(1, 2, 64, 0, device="cpu")
    with pytest.raises(ValueError, match="head_dim contiguous"):
        attn_prompt(x.transpose(1, 2), x, x, cu)


def test_plain_attention_closed_cases():
    """Equal keys: the running mean of v; one key: v; nothing seen: zeros."""
    v = torch.randn(5, 1, 8, dtype=torch.float64)
    q, k = torch.randn(5, 2, 8, dtype=torch.float64), torch.ones(5, 1, 8, dtype=torch.float64)
    out, p, _, _ = ref.attention(q, k, v, 0.3, ref.causal(5, 5))
    mean = v.cumsum(0) / torch.arange(1, 6)[:, None, None]
    assert torch.allclose(out, mean.expand(5, 2, 8))
    assert torch.allclose(p.sum(-1), torch.ones(2, 5, dtype=torch.float64))
    out, _, _, _ = ref.attention(q, k[:3], v[:3], 0.3, ref.causal(5, 3))
    assert (out[:2] == 0).all() and torch.allclose(out[2], v[0].expand(2, 8))


def test_plain_scales():
    x = torch.tensor([[448.0, 1.0], [450.0, 0.0], [0.0, 0.0], [3.5, -7.0], [math.inf, 2.0 ** -6]])
    assert ref.scale_of(x).tolist() == [1.0, 2.0, 2.0 ** -110, 2.0 ** -6, 2.0 ** -14]
    rot, _ = ref.rotate(torch.tensor([[[1.0, 0.0]]]), torch.tensor([2]), 1e4)
    assert torch.allclose(rot, torch.tensor([[[math.cos(2.0), math.sin(2.0)]]], dtype=torch.float64))
