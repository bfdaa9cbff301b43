"""What counts as seen: mask != 0, whatever the mask's type"""
import ctypes

import pytest
import torch

from test_attention_saved_tensors import Recorder

gpu = pytest.mark.gpu
VALUES = [0.0, 1.0, 0.5, -0.25, 1e-30, -0.0, 3.0, float("nan"), float("inf"), -1.0]


class Masks(Recorder):
    """the struct's mask as the library would read it"""

    def __call__(self, name, args, stream):
        self.mask = list((ctypes.c_int64 * (args._obj.batch * args._obj.k_len)).from_address(args._obj.mask))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16, torch.int32, torch.int64, torch.uint8, torch.bool])
def test_masks_of_any_type(monkeypatch, dtype):
    from nonauto_lm_amd import ops
    lib = Masks(monkeypatch)
    values = torch.tensor(VALUES if dtype.is_floating_point else [0, 1, 0, 1, 2, 0, 3, 1, 1, 0]).to(dtype)
    x = torch.zeros(1, len(values), 32)
    ops.biased_attention(x, x, x, 2, mask=values[None])
    assert [m != 0 for m in lib.mask] == values.ne(0).tolist()


@gpu
def test_float_mask_on_the_gpu():
    from nonauto_lm_amd import ops
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(2, 40, 64, device="cuda", generator=g)
    mask = torch.rand(2, 40, device="cuda", generator=g) * (torch.arange(40, device="cuda") % 3 > 0)
    assert torch.equal(ops.biased_attention(x, x, x, 2, mask=mask), ops.biased_attention(x, x, x, 2, mask=mask.ne(0)))
