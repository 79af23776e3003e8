"""Prompt attention, the 8-bit cache and eviction at their edges: the last row of memory, counts past
the cache, tables that name no block, values next to the end of a type, every dtype's instance.
Oracle and tolerances as in ``test_gpu_attention``."""
import math

import pytest
import torch

import attention_ref as ref
from helix_substrate import _hxq
from helix_substrate.attention import attn_prompt
from test_gpu_attention import BF, FP, _check_prompt, _prompt_case

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
