"""Register budgets of the scoring and paged-cache kernels, from the compiler's metadata (hipcc cross-compiles without a GPU): they hold
a tile or a row's columns in registers and live from many waves per CU."""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))
sys.path.insert(0, ROOT)

import kernel_resources as kr  # noqa: E402


def test_paged_kernels_fit():
    for name, r in kr.resources("paged.hip"):
        assert r["spill"] == 0 and r["scratch"] == 0, (name, r)
        if "attn_paged_decode_kernel" in name:      # a wave's tile in flight: 128 columns at least two waves per SIMD, 64 four, 32 five
            assert r["vgpr"] <= (256 if "Li128E" in name else 128 if "Li64E" in name else 96), (name, r)


def test_scoring_kernels_fit():
    for name, r in kr.resources("scoring.hip"):
        assert r["spill"] == 0 and r["scratch"] == 0, (name, r)
        if "_fwd_kernel" in name or "logprobs_bwd" in name:      # eight waves per SIMD
            assert r["vgpr"] <= 64, (name, r)
        elif "top_kernel" in name:                  # eight workgroups of four waves per CU
            assert r["vgpr"] <= 64 and (r["wg"] > 256 or 8 * r["lds"] <= 160 * 1024), (name, r)
        else:
            assert r["vgpr"] <= 85, (name, r)
