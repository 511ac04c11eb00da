"""What the operators on rows of logits refuse or take at the ends of their
arguments, and what their source has to keep, as far as no device is needed."""
import ctypes
import math
import os
import re

import pytest
import torch

import torch_dbs_extension as ext
from conftest import PKG


def test_dynamic_shared_memory_is_aligned_for_16_byte_accesses():
    """Lists and slices there are read 16 bytes at a time; an array declared with a smaller type's alignment may start 8 bytes off."""
    source = open(os.path.join(PKG, "csrc", "logits_kernels.cu")).read()
    arrays = re.findall(r"extern __shared__ ([^;]*);", source)
    assert len(arrays) >= 7
    assert [a for a in arrays if not a.startswith(("uint4 ", "__align__(16) "))] == []


@pytest.mark.parametrize("values,dtype,want", [
    ([5, 2 ** 32 + 5, -2 ** 32 + 5], torch.int64, [5, 2 ** 31 - 1, 0]),
    ([2 ** 63 - 1, -2 ** 63, 2 ** 31], torch.int64, [2 ** 31 - 1, 0, 2 ** 31 - 1]),
    ([math.inf, -math.inf, math.nan], torch.float32, [2 ** 31 - 1, 0, 0]),
    ([3e9, 7.0, -3e9], torch.float32, [2 ** 31 - 1, 7, 0]),
    ([40, -1, 0], torch.int32, [40, -1, 0]),
    ([40, 3, 0], torch.uint8, [40, 3, 0]),
])
def test_sample_top_k_of_each_row_reaches_the_library_unwrapped(values, dtype, want, monkeypatch):
    seen = []

    def call(name, device, *args):
        seen.extend(ctypes.cast(args[8], ctypes.POINTER(ctypes.c_int32))[:3])

    monkeypatch.setattr(ext, "_cuda_device_for", lambda t: torch.device("cpu"))
    monkeypatch.setattr(ext, "_call", call)
    ext.sample(torch.randn(3, 16), torch.rand(3), top_k=torch.tensor(values, dtype=dtype))
    assert seen == want


@pytest.mark.parametrize("grad", [True, False])
def test_distillation_refuses_tangents(grad):
    x, lq, at = torch.randn(3, 16), torch.full((3, 4), -2.0), torch.arange(4).expand(3, 4)
    ad = torch.autograd.forward_ad
    with ad.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(RuntimeError, match="forward-mode"):
            ext.distillation_loss(ad.make_dual(x, torch.ones_like(x)), lq, at)
        with pytest.raises(ValueError, match="takes no gradient"):
            ext.distillation_loss(x, ad.make_dual(lq, torch.ones_like(lq)), at)
