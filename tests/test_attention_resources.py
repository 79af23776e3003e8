"""The attention kernels whose loops live in registers do not spill there (metadata of the built code
object, no GPU)."""
from test_kernel_resources import kernels  # noqa: F401 (the fixture)


def test_cache_attention_does_not_spill(kernels):  # noqa: F811
    found = {n: k for n, k in kernels.items() if "kv8_" in n}
    assert len(found) >= 30
    spilled = {n: k[".private_segment_fixed_size"] for n, k in found.items()
               if k[".private_segment_fixed_size"] or k[".vgpr_spill_count"]}
    assert not spilled, spilled


def test_prompt_attention_spills_no_more_than_constants(kernels):  # noqa: F811
    """A few lane constants that only the steps at the diagonal and the end use may be kept in
    scratch; the accumulators, operands and staged rows (16 to 256 bytes each) may not."""
    found = {n: k for n, k in kernels.items() if "attn_prompt_kernel" in n}
    assert len(found) == 36
    assert all(k[".private_segment_fixed_size"] <= 16 for k in found.values())
