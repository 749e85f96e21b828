"""The operators over tokens without a GPU: refusals before any CUDA call, sizes, the references the GPU tests compare with."""
import ctypes

import pytest
import torch

import cs2d
import gated_reference as R
from cs2d import _lib


def test_operators_reject_cpu_tensors_and_bad_arguments():
    u = torch.zeros(1, 4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        cs2d.gated_scan_1d(u, u)
    with pytest.raises(RuntimeError, match="CUDA"):
        cs2d.gated_scan_step(u[0], u[0], u[0])
    with pytest.raises(RuntimeError, match="CUDA"):
        cs2d.layer_norm(u)
    with pytest.raises(RuntimeError, match="form must be one of"):
        cs2d.gated_scan_1d(u, u, form="relu")


@pytest.mark.parametrize("form", ("sigmoid", "log", "direct"))
@pytest.mark.parametrize("weighted", (True, False))
def test_reference_gradient_against_differences(form, weighted):
    gen = torch.Generator().manual_seed(0)
    u, g, h = (torch.randn(*s, generator=gen, dtype=torch.float64).requires_grad_(True) for s in ((6, 3), (6, 3), (3,)))
    assert torch.autograd.gradcheck(lambda *a: R.scan(*a, form, weighted), (u, g, h))


class GScan(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_int32) for n in ("batch", "dim", "io_dtype", "form", "weighted", "n_seq", "offsets64")] + [("length", ctypes.c_int64)]
                + [("u", ctypes.c_void_p), ("u_bs", ctypes.c_int64), ("u_ls", ctypes.c_int64), ("gate", ctypes.c_void_p), ("gate_bs", ctypes.c_int64),
                   ("gate_ls", ctypes.c_int64), ("h0", ctypes.c_void_p), ("h0_bs", ctypes.c_int64), ("offsets", ctypes.c_void_p)])


class NormP(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_int32) for n in ("dim", "io_dtype", "param_dtype")] + [("eps", ctypes.c_float), ("outer", ctypes.c_int64), ("inner", ctypes.c_int64)]
                + [("x", ctypes.c_void_p)] + [(n, ctypes.c_int64) for n in ("x_os", "x_is", "x_cs")] + [("gate", ctypes.c_void_p)]
                + [(n, ctypes.c_int64) for n in ("g_os", "g_is")] + [("weight", ctypes.c_void_p), ("bias", ctypes.c_void_p)])


def _lib_with_types():
    L = ctypes.CDLL(_lib.LIB_PATH)
    L.cs2d_last_error.restype = ctypes.c_char_p
    L.cs2d_gscan_saved_bytes.restype = L.cs2d_norm_bwd_scratch_bytes.restype = ctypes.c_size_t
    return L


def _gscan(**over):
    p = GScan(batch=2, dim=64, io_dtype=_lib.BF16, length=1000, u=256, gate=256, u_bs=64000, u_ls=64, gate_bs=64000, gate_ls=64)
    for k, v in over.items():
        setattr(p, k, v)
    return p


def test_gated_scan_sizes():
    L = _lib_with_types()
    # checkpoints before rows 32, 64, ... 992 of two batch rows; 8 bytes per row with offsets; never nothing
    assert L.cs2d_gscan_saved_bytes(ctypes.byref(_gscan()), 1) == 2 * 31 * 64 * 4
    assert L.cs2d_gscan_saved_bytes(ctypes.byref(_gscan()), 0) == 16
    assert L.cs2d_gscan_saved_bytes(ctypes.byref(_gscan(length=32)), 1) == 16
    assert L.cs2d_gscan_saved_bytes(ctypes.byref(_gscan(length=33)), 1) == 2 * 64 * 4
    p = _gscan(batch=1, offsets=256, n_seq=3)
    assert L.cs2d_gscan_saved_bytes(ctypes.byref(p), 1) == 8 * 1000 + 31 * 64 * 4
    assert L.cs2d_gscan_saved_bytes(ctypes.byref(p), 0) == 8 * 1000


@pytest.mark.parametrize("over,msg", [(dict(batch=0), "positive"), (dict(length=0), "positive"), (dict(dim=-1), "positive"), (dict(io_dtype=3), "input type"),
                                      (dict(form=3), "form"), (dict(u=None), "must be given"), (dict(offsets=256), "batch is 1"),
                                      (dict(offsets=256, batch=1, n_seq=-1), "n_seq")])
def test_gated_scan_validation_happens_before_any_cuda_call(over, msg):
    L = _lib_with_types()
    p = _gscan(**over)
    assert L.cs2d_gscan_saved_bytes(ctypes.byref(p), 1) == 0 and msg in L.cs2d_last_error().decode()
    one = ctypes.c_void_p(256)
    i = ctypes.c_int64(64)
    assert L.cs2d_gscan_fwd(ctypes.byref(p), one, i, i, one, one, 1, None) == -1
    assert L.cs2d_gscan_bwd(ctypes.byref(p), one, i, i, None, i, one, one, one, None, None) == -1
    assert L.cs2d_gscan_fwd(ctypes.byref(_gscan()), None, i, i, one, one, 1, None) == -1
    assert L.cs2d_gscan_step(ctypes.byref(_gscan()), one, i, None, i, None) == -1


@pytest.mark.parametrize("over,msg", [(dict(dim=0), "positive"), (dict(inner=0), "positive"), (dict(io_dtype=-1), "input type"), (dict(param_dtype=_lib.F16), "weight"),
                                      (dict(x=None), "x must be given"), (dict(x_cs=2), "stride 1"), (dict(outer=1 << 31, inner=2), "rows")])
def test_norm_validation_happens_before_any_cuda_call(over, msg):
    L = _lib_with_types()
    p = NormP(dim=64, io_dtype=_lib.BF16, param_dtype=_lib.F32, eps=1e-5, outer=2, inner=10, x=256, x_os=640, x_is=64, x_cs=1)
    assert L.cs2d_norm_bwd_scratch_bytes(ctypes.byref(p)) >= 2 * 64 * 4
    for k, v in over.items():
        setattr(p, k, v)
    assert L.cs2d_norm_bwd_scratch_bytes(ctypes.byref(p)) == 0 and msg in L.cs2d_last_error().decode()
    assert L.cs2d_norm_fwd(ctypes.byref(p), ctypes.c_void_p(256), None, None) < 0


def test_counts_that_the_kernels_cannot_hold_are_refused():
    """Channels, rows and sequences are counted in 32 bits on the GPU: what such a count would pass is refused before any CUDA call."""
    L = _lib_with_types()
    scan = lambda **over: L.cs2d_gscan_saved_bytes(ctypes.byref(_gscan(**over)), 0)
    assert scan(dim=1 << 30) and scan(batch=1, length=1 << 30) and scan(batch=1, offsets=256, n_seq=(1 << 30) - 1)
    for over, msg in ((dict(dim=(1 << 30) + 1), "channels"), (dict(dim=(1 << 31) - 1), "channels"), (dict(batch=1, length=(1 << 30) + 1), "tokens"),
                      (dict(batch=1, offsets=256, n_seq=1 << 30), "sequences"), (dict(batch=1, offsets=256, n_seq=(1 << 31) - 1), "sequences")):
        assert scan(**over) == 0 and msg in L.cs2d_last_error().decode(), over
    norm = lambda dim: L.cs2d_norm_bwd_scratch_bytes(ctypes.byref(NormP(dim=dim, io_dtype=_lib.BF16, param_dtype=_lib.F32, eps=1e-5, outer=1, inner=1, x=256, x_cs=1)))
    assert norm(1 << 29)
    for dim in ((1 << 29) + 1, (1 << 31) - 1):
        assert norm(dim) == 0 and "channels" in L.cs2d_last_error().decode()
