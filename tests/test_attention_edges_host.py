"""Refusals of the attention wrappers that need no device."""
import pytest
import torch

from helix_substrate.attention import kv8_evict


@pytest.mark.parametrize("change", [dict(keep=2 ** 32 + 5), dict(sink=2 ** 32), dict(recent=2 ** 31)])
def test_evict_numbers_that_32_bits_do_not_hold(change):
    """They are refused, not taken modulo 2^32."""
    w, n = torch.zeros(1, 1, 8), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="less than"):
        kv8_evict(w, None, n, **{"keep": 4, **change})
