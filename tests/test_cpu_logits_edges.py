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


# Host memory stands in for the device's: every call here is refused before a kernel is launched.
BUF = (ctypes.c_float * 64)()
P = ctypes.c_void_p((ctypes.addressof(BUF) + 15) // 16 * 16)
ODD, FOUR = ctypes.c_void_p(P.value + 2), ctypes.c_void_p(P.value + 4)
ROWS = (P, 0, 1, 16, 16)


def refused(lib, rc, message):
    assert rc == -2
    assert message in lib.dbs_last_global_error().decode()


def changed(args, at, value):
    return [value if i == at else a for i, a in enumerate(args)]


@pytest.mark.parametrize("entry,args,names", [
    ("dbs_device_sample", [*ROWS, P, P, 1.0, P, 0, P, 1.0, P, 0.0, P, P, None],
     {5: "uniforms", 6: "temperatures", 8: "top_ks", 10: "top_ps", 12: "min_ps", 14: "tokens"}),
    ("dbs_device_top_log_probs", [*ROWS, 4, 1.0, P, P, None, None], {7: "log_probs", 8: "tokens"}),
    ("dbs_device_distill", [*ROWS, P, P, 4, 2, 1.0, 1, 1, 1.0, P, P, P, P, None],
     {5: "teacher_log_probs", 6: "teacher_tokens", 13: "row_losses", 14: "loss"}),
    ("dbs_device_distill_backward", [*ROWS, 2, 1.0, 1, 1, 1.0, P, P, 0, 0, P, None], {11: "grad_loss"}),
])
def test_c_pointers_that_are_not_aligned(libdbs, entry, args, names):
    """A kernel that reads or writes there would fault."""
    for at, name in names.items():
        refused(libdbs, getattr(libdbs, entry)(*changed(args, at, ODD)), name + " is not aligned")
    if entry == "dbs_device_distill":
        refused(libdbs, libdbs.dbs_device_distill(*changed(changed(args, 7, 8), 6, FOUR)), "teacher_tokens is not aligned")


def test_c_more_rows_than_an_int_counts(libdbs):
    """The loss' rows are counted in an int, a scan's rows are listed as ints: 2^31 rows (of one repeated row, or without a gradient) fit
    the memory of a GPU. A workspace for them is not asked for, as they are not scanned."""
    many, size = (P, 0, 2 ** 31, 16, 0), ctypes.c_int64(-1)
    refused(libdbs, libdbs.dbs_device_distill(*many, P, P, 4, 2, 1.0, 1, 2, 1.0, P, P, P, None, None), "at most 2147483647 rows")
    refused(libdbs, libdbs.dbs_device_distill_backward(*many, 2, 1.0, 1, 2, 1.0, P, P, 0, 0, P, None), "at most 2147483647 rows")
    assert libdbs.dbs_device_distill_state_bytes(2 ** 31, 1, ctypes.byref(size)) == -1
    assert libdbs.dbs_device_distill_state_bytes(2 ** 31 - 1, 1024, ctypes.byref(size)) == 0 and size.value > 2 ** 45
    for rows in (2 ** 31, 2 ** 62):
        assert libdbs.dbs_device_sample_workspace_bytes(0, rows, 32000, 8, 0.9, ctypes.byref(size)) == 0 and size.value == 0
        assert libdbs.dbs_device_top_log_probs_workspace_bytes(0, rows, 32000, 8, ctypes.byref(size)) == 0 and size.value == 0


def test_c_workspace_of_a_common_top_k_holds_no_chunk_sums(libdbs):
    """128 sums of 8 bytes for each part of a row are for rows that every token can come from; a top-k for all rows leaves none."""
    def bytes_of(rows, V, top_k, top_p):
        size = ctypes.c_int64()
        assert libdbs.dbs_device_sample_workspace_bytes(2, rows, V, top_k, top_p, ctypes.byref(size)) == 0
        return size.value

    # 4 parts of 128256 bf16 with the least share each: state and list, below 2 KB, and the row's place in the list of those left over
    assert 0 < bytes_of(2048, 128256, 8, 1.0) < 2048 * 4 * 1024 < bytes_of(2048, 128256, 0, 1.0)
    assert bytes_of(2048, 128256, 50, 1.0) == bytes_of(2048, 128256, 50, 0.9)
