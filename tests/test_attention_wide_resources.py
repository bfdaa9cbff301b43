"""Scratch (register spill) budget of the attention kernels that the budget of the wide bf16 ones leaves out: heads of 96 and the
fp32 kernels, which run one wave per SIMD with up to 512 registers; only dk and dv spill, in front of and behind their walks."""
import os

import pytest

from test_kernel_resources import LIBDIR, LLVM, _kernels

BUDGET = [("k_ba_fwd<unsigned short, 3,", 0), ("k_ba_dq<unsigned short, 1,", 0), ("k_ba_dq<unsigned short, 3,", 0),
          ("k_ba_dkv<unsigned short, 3>", 36), ("k_ba_fwd<float,", 0), ("k_ba_dq<float,", 0), ("k_ba_dkv<float, 1>", 0),
          ("k_ba_dkv<float, 2>", 0), ("k_ba_dkv<float, 3>", 36), ("k_ba_dkv<float, 4>", 44)]


@pytest.mark.skipif(not (os.path.exists(f"{LLVM}/llvm-readelf") and os.path.exists(os.path.join(LIBDIR, "biased_attention.o"))),
                    reason="ROCm LLVM tools or built objects not present")
def test_heads_of_96_and_fp32_stay_within_their_scratch_budget():
    kernels = _kernels(os.path.join(LIBDIR, "biased_attention.o"))
    for name, limit in BUDGET:
        found = [(k, s) for k, s in kernels if name in k]
        assert found, name
        for k, s in found:
            assert s <= limit, f"{k}: {s} bytes of scratch per lane, {limit} allowed"
