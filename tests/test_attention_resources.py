"""Scratch (register spill) budget of the attention operators' kernels, read from the built objects (no GPU).  The bf16 kernels of
wide heads sit at the 256-register line of two waves per SIMD; a spill inside their walks costs a third (dk and dv of heads of
128: 195 us with what is allowed here, 281 us with 132 bytes in the loop)."""
import os

import pytest

from test_kernel_resources import LIBDIR, LLVM, _kernels

# (object, kernel, largest scratch in bytes per lane): what the sources need, before and behind the walks
BUDGET = [
    ("biased_attention.o", "k_ba_fwd<unsigned short, 1,", 0),
    ("biased_attention.o", "k_ba_fwd<unsigned short, 2,", 0),
    ("biased_attention.o", "k_ba_fwd<unsigned short, 4,", 0),
    ("biased_attention.o", "k_ba_dq<unsigned short, 2,", 0),
    ("biased_attention.o", "k_ba_dq<unsigned short, 4,", 32),
    ("biased_attention.o", "k_ba_dkv<unsigned short, 1>", 0),
    ("biased_attention.o", "k_ba_dkv<unsigned short, 2>", 0),
    ("biased_attention.o", "k_ba_dkv<unsigned short, 4>", 68),
    ("token_attention.o", "k_token<", 0),
    ("qk_rotary.o", "k_qk<", 0),
]


@pytest.mark.skipif(not (os.path.exists(f"{LLVM}/llvm-readelf") and os.path.exists(os.path.join(LIBDIR, "token_attention.o"))),
                    reason="ROCm LLVM tools or built objects not present")
@pytest.mark.parametrize("obj", sorted({o for o, _, _ in BUDGET}))
def test_attention_kernels_stay_within_their_scratch_budget(obj):
    kernels = _kernels(os.path.join(LIBDIR, obj))
    for _, name, limit in (b for b in BUDGET if b[0] == obj):
        found = [(k, s) for k, s in kernels if name in k]
        assert found, f"{name} not in {obj}"
        for k, s in found:
            assert s <= limit, f"{k}: {s} bytes of scratch per lane, {limit} allowed"
