"""Layer norm and RMSNorm with the library's host side and kernels emulated on the host, through the Python operators, against
the definition in float64 (bodies and tolerances in tests/norm_cases.py)."""

import ctypes as C

import pytest
import torch

import norm_cases as cases
import train_ops_emu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("n,hidden,dtype,wdtype,pitch", [
    (1, 1, FP32, FP32, 0), (3, 2, BF16, BF16, 0), (70, 5, FP16, FP32, 3), (67, 8, BF16, BF16, 0), (40, 24, BF16, FP32, 8),
    (33, 31, FP16, FP16, 0), (21, 33, BF16, BF16, 2), (37, 128, BF16, BF16, 0), (19, 132, FP32, FP32, 4), (13, 250, FP16, FP16, 6),
    (14, 264, BF16, BF16, 16), (9, 1001, FP32, FP32, 0), (8, 1024, FP32, FP32, 0), (5, 4104, BF16, FP32, 0), (4, 5000, FP16, FP16, 1),
    (2, 9000, FP32, FP32, 0), (2, 16387, BF16, BF16, 0), (2, 16392, FP16, FP32, 0)])
def test_matches_definition(kind, n, hidden, dtype, wdtype, pitch):
    with train_ops_emu.installed():
        cases.case_matches_definition("cpu", kind, n, hidden, dtype, wdtype, True, True, 0.0, pitch)


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("n,hidden,dtype,wdtype,pitch", [
    (101, 264, BF16, BF16, 16), (57, 520, FP16, FP32, 0), (27, 1024, FP32, FP32, 4), (11, 4104, BF16, BF16, 0), (7, 8200, FP16, FP16, 0),
    (300, 40, BF16, BF16, 0), (90, 33, FP16, FP16, 0), (31, 513, BF16, FP32, 1), (200, 12, BF16, BF16, 1)])
def test_more_rows_than_a_round_takes(kind, n, hidden, dtype, wdtype, pitch):
    with train_ops_emu.installed():
        cases.case_matches_definition("cpu", kind, n, hidden, dtype, wdtype, True, True, 0.0, pitch)


@pytest.mark.parametrize("kind,weight,bias,offset,mode", [
    ("layer", True, False, 1.0, "gemma"), ("layer", False, False, 0.0, "gemma"), ("layer", False, True, 0.0, "gemma"),
    ("rms", True, False, 1.0, "llama"), ("rms", False, False, 0.0, "llama"), ("rms", True, False, 1.0, "gemma")])
@pytest.mark.parametrize("hidden", [27, 40, 336, 777])
def test_parameters_and_casting(kind, weight, bias, offset, mode, hidden):
    with train_ops_emu.installed():
        cases.case_matches_definition("cpu", kind, 11, hidden, BF16, None, weight, bias, offset, 0, mode)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_gradient_against_differences(kind):
    with train_ops_emu.installed():
        cases.case_gradient_against_differences("cpu", kind)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_special_values_stay_in_their_row(kind):
    with train_ops_emu.installed():
        cases.case_special_values("cpu", kind)


def test_shapes_and_views():
    with train_ops_emu.installed():
        cases.case_shapes_and_views("cpu")


def test_refusals():
    with train_ops_emu.installed():
        cases.case_refusals("cpu")


def test_cpu_tensors_are_refused():
    import liger_kernel_b200 as lk

    with pytest.raises(RuntimeError, match="no CPU path"):
        lk.liger_layer_norm(torch.randn(2, 4))


def test_entry_points_check_their_arguments():
    """Every refusal of the C side comes before a launch; each case spoils one argument of a call that works."""
    from liger_kernel_b200 import _lib

    lib = train_ops_emu.load()
    buf = (C.c_float * 4096)()
    base = C.addressof(buf)
    base += -base % 64

    def norm(**kw):
        p = _lib.Norm(4, 16, 16, _lib.FLCE_LAYER_NORM, _lib.FLCE_FP32, _lib.FLCE_FP32, 0, 1e-6, 0.0, base, base + 1024, base + 2048)
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    def forward(p, y=base + 4096):
        return lib.flce_b200_norm_forward(C.byref(p) if p is not None else None, y, None, None, None)

    def backward(p, dy=base, ld=16, mean=base + 512, rstd=base + 640, dx=base + 4096, dw=base + 5120, db=None, ws=base + 8192, nbytes=4096):
        return lib.flce_b200_norm_backward(C.byref(p), dy, ld, mean, rstd, dx, dw, db, ws, nbytes, None)

    INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3
    assert forward(norm()) == 0 and backward(norm()) == 0
    assert forward(None) == INVALID
    for kw, code in ((dict(n_rows=-1), INVALID), (dict(n_rows=1 << 31), INVALID), (dict(hidden=0), INVALID), (dict(hidden=1 << 31), INVALID),
                     (dict(kind=2), INVALID), (dict(dtype=3), INVALID), (dict(dtype=-1), INVALID), (dict(weight_dtype=_lib.FLCE_BF16), UNSUPPORTED),
                     (dict(ld_x=-1), INVALID), (dict(x=base + 2), INVALID), (dict(weight=base + 1), INVALID), (dict(bias=base + 2), INVALID),
                     (dict(kind=_lib.FLCE_RMS_NORM), INVALID)):
        before = lib.emu_launches()
        assert forward(norm(**kw)) == code and backward(norm(**kw)) == code, kw
        assert lib.flce_b200_norm_workspace_bytes(C.byref(norm(**kw))) == 0
        assert lib.emu_launches() == before
    assert forward(norm(x=None)) == INVALID and forward(norm(), None) == INVALID
    assert backward(norm(), dy=None) == INVALID and backward(norm(), rstd=None) == INVALID and backward(norm(), mean=None) == INVALID
    assert backward(norm(), dx=None) == INVALID and backward(norm(), ld=-1) == INVALID and backward(norm(), dy=base + 2) == INVALID
    assert backward(norm(), nbytes=15) == WORKSPACE and backward(norm(), ws=None) == WORKSPACE and backward(norm(), ws=base + 2) == WORKSPACE
    assert b"workspace" in lib.flce_b200_last_error()
    assert backward(norm(), dw=None, ws=None, nbytes=0) == 0
    rms = norm(kind=_lib.FLCE_RMS_NORM, bias=None)
    assert backward(rms, mean=None) == 0 and backward(rms, db=base + 5120) == INVALID
    assert lib.flce_b200_norm_workspace_bytes(C.byref(norm())) >= 2 * 16 * 4


def test_autograd():
    with train_ops_emu.installed():
        cases.case_autograd("cpu")


def test_forward_mode():
    with train_ops_emu.installed():
        cases.case_forward_mode("cpu")
