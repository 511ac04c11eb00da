"""Refusals of the operators on rows of logits: the torch entry points' checks
(before any device is looked for) and the C entry points' (before any launch)."""
import ctypes

import pytest
import torch

import dbs_ctypes as dc
import torch_dbs_extension as ext

X = torch.randn(3, 16)
U = torch.rand(3)
LQ = torch.full((3, 4), -2.0)
AT = torch.arange(4, dtype=torch.int32).expand(3, 4)


@pytest.mark.parametrize("kwargs,message", [
    (dict(temperature=-0.5), "temperature cannot be negative"),
    (dict(temperature=float("nan")), "temperature must be finite"),
    (dict(temperature=float("inf")), "temperature must be finite"),
    (dict(top_k=-1), "top_k must be a non-negative integer"),
    (dict(top_k=2.5), "top_k must be a non-negative integer"),
    (dict(top_p=0.0), "top_p must be in"),
    (dict(top_p=1.5), "top_p must be in"),
    (dict(top_p=float("nan")), "top_p must be in"),
    (dict(min_p=-0.1), "min_p must be in"),
    (dict(min_p=1.1), "min_p must be in"),
])
def test_sample_settings(kwargs, message, monkeypatch):
    monkeypatch.setattr(ext, "_cuda_device_for", lambda t: torch.device("cpu"))
    with pytest.raises(ValueError, match=message):
        ext.sample(X, U, **kwargs)


@pytest.mark.parametrize("x,u,message", [
    (X.double(), U, "float32, float16 or bfloat16"),
    (torch.tensor(1.0), U, "shape"),
    (torch.empty(3, 0), U, "V must be positive"),
    (X, U[:2], "uniforms must have shape"),
    (X, U[:, None], "uniforms must have shape"),
    (X, U.double(), "uniforms must be float32"),
    (torch.empty(1, 750_001), U[:1], "takes at most"),
])
def test_sample_inputs(x, u, message):
    with pytest.raises(ValueError, match=message):
        ext.sample(x, u)


def test_sample_setting_of_another_shape(monkeypatch):
    monkeypatch.setattr(ext, "_cuda_device_for", lambda t: torch.device("cpu"))
    with pytest.raises(ValueError, match="top_k must have shape"):
        ext.sample(X, U, top_k=torch.tensor([1, 2]))


@pytest.mark.parametrize("n,kwargs,message", [
    (0, {}, "n must be in"), (17, {}, "n must be in"), (2.5, {}, "n must be in"),
    (4, dict(temperature=0.0), "temperature must be positive"),
    (4, dict(temperature=float("inf")), "temperature must be finite"),
])
def test_top_log_probs_arguments(n, kwargs, message):
    with pytest.raises(ValueError, match=message):
        ext.top_log_probs(X, n, **kwargs)


def test_top_log_probs_longest_list():
    with pytest.raises(ValueError, match="n must be in 1 .. 1024"):
        ext.top_log_probs(torch.empty(1, 5000), 1025)


@pytest.mark.parametrize("change,message", [
    (dict(teacher_tokens=AT.to(torch.int16)), "int32 or int64"),
    (dict(teacher_log_probs=LQ.long()), "floating-point"),
    (dict(teacher_tokens=AT[:2]), "teacher_tokens must have shape"),
    (dict(teacher_log_probs=LQ[:, :3]), "same shape"),
    (dict(teacher_tokens=AT[:, :0], teacher_log_probs=LQ[:, :0]), "1 .. 1024 slots"),
    (dict(teacher_tokens=torch.zeros(3, 1025, dtype=torch.int32), teacher_log_probs=torch.zeros(3, 1025)), "1 .. 1024 slots"),
    (dict(reduction="batchmean"), "reduction"),
    (dict(temperature=0.0), "temperature must be positive"),
    (dict(scale=float("nan")), "scale must be finite"),
    (dict(logits=X.double()), "float32, float16 or bfloat16"),
    (dict(logits=torch.empty(3, 260_001)), "takes at most 1040000 bytes"),
    (dict(teacher_log_probs=LQ.clone().requires_grad_(True)), "takes no gradient"),
])
def test_distillation_arguments(change, message):
    args = dict(logits=X, teacher_log_probs=LQ, teacher_tokens=AT)
    args.update(change)
    with pytest.raises(ValueError, match=message):
        ext.distillation_loss(**args)


@pytest.mark.skipif(torch.cuda.is_available(), reason="only meaningful without a CUDA device")
def test_no_cuda_device_fails_loudly():
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.sample(X, U)
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.top_log_probs(X, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        ext.distillation_loss(X, LQ, AT)


# Host memory stands in for the device's: every call here is refused before a kernel is launched.
BUF = (ctypes.c_float * 64)()
P = ctypes.c_void_p((ctypes.addressof(BUF) + 15) // 16 * 16)
ODD = ctypes.c_void_p(P.value + 1)


def refused(lib, rc, message):
    assert rc == -2
    assert message in lib.dbs_last_global_error().decode()


@pytest.mark.parametrize("change,message", [
    (dict(logits=None), "logits cannot be null"), (dict(dtype=7), "unknown data type"), (dict(rows=-1), "rows"),
    (dict(V=0), "vocab_size must be positive"), (dict(V=750_001), "at most 3000000 bytes"), (dict(stride=-1), "row_stride"),
    (dict(logits=ODD), "aligned"),
])
def test_c_rows(libdbs, change, message):
    a = dict(logits=P, dtype=0, rows=1, V=16, stride=16)
    a.update(change)
    rows = (a["logits"], a["dtype"], a["rows"], a["V"], a["stride"])
    refused(libdbs, libdbs.dbs_device_sample(*rows, P, None, 1.0, None, 0, None, 1.0, None, 0.0, P, P, None), message)
    refused(libdbs, libdbs.dbs_device_top_log_probs(*rows, 1, 1.0, P, P, P, None), message)
    refused(libdbs, libdbs.dbs_device_distill(*rows, P, P, 4, 2, 1.0, 1, 1, 1.0, P, P, P, None, None), message)
    refused(libdbs, libdbs.dbs_device_distill_backward(*rows, 2, 1.0, 1, 1, 1.0, P, P, 0, 0, P, None), message)


def test_c_arguments(libdbs):
    rows = (P, 0, 1, 16, 16)
    sample = libdbs.dbs_device_sample
    refused(libdbs, sample(*rows, None, None, 1.0, None, 0, None, 1.0, None, 0.0, P, P, None), "uniforms and tokens")
    refused(libdbs, sample(*rows, P, None, -1.0, None, 0, None, 1.0, None, 0.0, P, P, None), "temperature")
    refused(libdbs, sample(*rows, P, None, 1.0, None, -1, None, 1.0, None, 0.0, P, P, None), "top_k")
    refused(libdbs, sample(*rows, P, None, 1.0, None, 0, None, 0.0, None, 0.0, P, P, None), "top_p")
    refused(libdbs, sample(*rows, P, None, 1.0, None, 0, None, 1.0, None, 2.0, P, P, None), "min_p")
    assert sample(None, 0, 0, 16, 16, None, None, 1.0, None, 0, None, 1.0, None, 0.0, None, None, None) == 0
    top = libdbs.dbs_device_top_log_probs
    refused(libdbs, top(*rows, 0, 1.0, P, P, None, None), "n must be")
    refused(libdbs, top(*rows, 17, 1.0, P, P, None, None), "n must be")
    refused(libdbs, top(*rows, 4, 0.0, P, P, None, None), "temperature")
    refused(libdbs, top(*rows, 4, 1.0, None, P, None, None), "cannot be null")
    wide = (P, 0, 400, 32000, 32000)     # the rows' own scan passes its lists on
    refused(libdbs, sample(*wide, P, None, 1.0, None, 0, None, 1.0, None, 0.0, P, None, None), "workspace cannot be null")
    refused(libdbs, sample(*wide, P, None, 1.0, None, 0, None, 1.0, None, 0.0, P, ODD, None), "workspace is not aligned")
    refused(libdbs, top(*wide, 4, 1.0, P, P, None, None), "workspace cannot be null")
    size = ctypes.c_int64()
    for query, given in ((libdbs.dbs_device_sample_workspace_bytes, (8, 0.9)), (libdbs.dbs_device_top_log_probs_workspace_bytes, (8,))):
        assert query(0, 400, 32000, *given, ctypes.byref(size)) == 0 and size.value > 0
        assert query(0, 1, 32000, *given, ctypes.byref(size)) == 0 and size.value == 0
        refused(libdbs, query(0, 64, 32000, *given, None), "bytes cannot be null")
        refused(libdbs, query(9, 64, 32000, *given, ctypes.byref(size)), "data type")
    distill = libdbs.dbs_device_distill
    refused(libdbs, distill(*rows, None, P, 4, 2, 1.0, 1, 1, 1.0, P, P, P, None, None), "teacher_log_probs")
    refused(libdbs, distill(*rows, P, P, 2, 2, 1.0, 1, 1, 1.0, P, P, P, None, None), "token_bytes")
    refused(libdbs, distill(*rows, P, P, 4, 0, 1.0, 1, 1, 1.0, P, P, P, None, None), "slots")
    refused(libdbs, distill(*rows, P, P, 4, 2, 1.0, 1, 3, 1.0, P, P, P, None, None), "reduction")
    refused(libdbs, distill(*rows, P, P, 4, 2, 1.0, 1, 1, float("inf"), P, P, P, None, None), "scale")
    refused(libdbs, distill(*rows, P, P, 4, 2, 1.0, 1, 1, 1.0, None, P, P, None, None), "row_losses")
    refused(libdbs, distill(*rows, P, P, 4, 2, 1.0, 1, 1, 1.0, P, None, P, None, None), "needs a place")
    refused(libdbs, distill(*rows, P, P, 4, 2, 1.0, 1, 2, 1.0, P, P, None, None, None), "state cannot be null")
    refused(libdbs, distill(*rows, P, P, 4, 2, 1.0, 1, 2, 1.0, P, P, ODD, None, None), "state is not aligned")
    refused(libdbs, distill(P, 0, 1, 260_001, 260_001, P, P, 4, 2, 1.0, 1, 2, 1.0, P, P, P, None, None), "at most 1040000 bytes")
    assert libdbs.dbs_device_distill_state_bytes(3, 5, ctypes.byref(size)) == 0 and size.value >= 3 * 5 * 8
    assert libdbs.dbs_device_distill_state_bytes(3, 0, ctypes.byref(size)) == -1
    assert libdbs.dbs_device_distill_state_bytes(-1, 5, ctypes.byref(size)) == -1
    assert libdbs.dbs_device_distill_state_bytes(1, 5, None) == -1
    refused(libdbs, distill(*rows, P, P, 4, 2, 1.0, 1, 1, 1.0, P, P, P, ODD, None), "aligned")
    backward = libdbs.dbs_device_distill_backward
    refused(libdbs, backward(*rows, 2, 1.0, 1, 1, 1.0, P, None, 0, 0, P, None), "grad_loss")
    refused(libdbs, backward(*rows, 2, 1.0, 1, 1, 1.0, P, P, -1, 0, P, None), "stride")
    refused(libdbs, backward(*rows, 2, 1.0, 1, 1, 1.0, P, P, 0, 1, P, None), "flags")
    refused(libdbs, backward(*rows, 2, 1.0, 1, 2, 1.0, None, P, 0, 0, P, None), "state")
    assert dc.DBS_REDUCTIONS == {"none": 0, "sum": 1, "mean": 2}


@pytest.mark.parametrize("temperature", [1e-31, 1e31])
def test_temperatures_beyond_32_bits(libdbs, temperature):
    with pytest.raises(ValueError, match="1e-30"):
        ext.top_log_probs(X, 4, temperature=temperature)
    with pytest.raises(ValueError, match="1e-30"):
        ext.distillation_loss(X, LQ, AT, temperature=temperature)
    rows = (P, 0, 1, 16, 16)
    refused(libdbs, libdbs.dbs_device_top_log_probs(*rows, 4, temperature, P, P, None, None), "1e-30")
    refused(libdbs, libdbs.dbs_device_distill(*rows, P, P, 4, 2, temperature, 1, 1, 1.0, P, P, P, None, None), "1e-30")
    refused(libdbs, libdbs.dbs_device_distill_backward(*rows, 2, temperature, 1, 1, 1.0, P, P, 0, 0, P, None), "1e-30")
