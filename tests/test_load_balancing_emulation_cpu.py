"""The router's load-balancing loss with the library's host side and kernels emulated on the host, through the Python operator,
against the definition in float64 (bodies and tolerances in tests/balance_cases.py)."""

import ctypes as C

import pytest
import torch

import balance_cases as cases
import train_ops_emu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _emulation():
    with train_ops_emu.installed() as lib:
        yield lib


@pytest.mark.parametrize("layers,tokens,experts,top_k,dtype,pitch", [
    (1, 70, 8, 2, BF16, 0), (3, 33, 8, 2, FP32, 0), (2, 50, 16, 4, FP16, 8), (2, 35, 60, 4, FP16, 0), (1, 41, 64, 6, BF16, 0),
    (2, 40, 128, 8, BF16, 0), (1, 19, 128, 8, FP32, 0), (1, 9, 160, 6, BF16, 0), (1, 9, 256, 8, BF16, 0), (1, 6, 257, 9, FP16, 0),
    (1, 5, 384, 8, FP32, 4), (1, 4, 512, 10, BF16, 0), (1, 3, 1000, 4, FP32, 0), (1, 3, 1024, 3, BF16, 0), (1, 37, 5, 1, BF16, 1),
    (1, 12, 32, 32, BF16, 0), (1, 10, 40, 33, FP32, 0), (1, 40, 64, 16, BF16, 0), (1, 33, 48, 11, FP32, 0), (1, 34, 32, 17, FP16, 0), (2, 7, 2, 1, FP32, 0)])
def test_matches_definition(layers, tokens, experts, top_k, dtype, pitch):
    cases.case_matches_definition("cpu", cases.make(layers, tokens, experts, dtype), top_k, z=1e-3, pitch=pitch, up=0.5)


@pytest.mark.parametrize("mask_dtype", [torch.bool, torch.uint8, torch.int32, torch.int64, torch.float32])
def test_masks(mask_dtype):
    mask = [1] * 5 + [0] * 4 + [1] * 9 + [0] * 9 + [0] * 9                  # four sequences of nine; the last one all padding
    cases.case_matches_definition("cpu", cases.make(2, 36, 24, BF16), 4, mask=mask, z=0.01, mask_dtype=mask_dtype, leading=(4, 9))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("experts,top_k", [(8, 2), (16, 5), (60, 4), (128, 8), (64, 12), (300, 8)])
def test_ties_and_masked_experts(dtype, experts, top_k):
    cases.case_ties("cpu", dtype, experts, top_k)
    cases.case_masked_experts("cpu", dtype, experts, top_k)


def test_more_layers_than_one_launch_takes():
    cases.case_matches_definition("cpu", cases.make(258, 2, 8, FP32), 2)


def test_empty():
    cases.case_empty("cpu")


def test_views_and_partial_gradients():
    cases.case_views_and_partial_gradients("cpu")


def test_gradient_against_differences():
    cases.case_gradient_against_differences("cpu")


def test_nan_reaches_the_loss():
    cases.case_nan_reaches_the_loss("cpu")


def test_refusals():
    cases.case_refusals("cpu")


def test_agrees_with_the_model_library():
    """The function of transformers that this replaces in the mixture-of-experts forwards, value and gradient."""
    mixtral = pytest.importorskip("transformers.models.mixtral.modeling_mixtral")
    import liger_kernel_b200 as lk

    x = cases.make(3, 24, 8, FP32, seed=21)
    mask = torch.ones(4, 6, dtype=torch.int64)
    mask[1, 4:] = 0
    for m in (None, mask):
        a = [t.clone().requires_grad_(True) for t in x]
        b = [t.clone().requires_grad_(True) for t in x]
        ours, theirs = lk.liger_load_balancing_loss(tuple(a), 8, 2, m), mixtral.load_balancing_loss_func(tuple(b), 8, 2, m)
        # theirs: fp32 means over n = 72 tokens, up to (n + 64) steps; ours within the bound of tests/balance_cases.py
        limit = 2 * (72 + 64 + 32) * cases.U
        assert abs(float(ours.detach()) - float(theirs.detach())) <= limit * float(theirs.detach())
        ga, gb = torch.autograd.grad(ours, a), torch.autograd.grad(theirs, b)
        for u, v in zip(ga, gb):
            # their gradient is a difference of terms a p with a of order E / n: absolute, not relative to what is left
            assert float((u - v).abs().max()) <= limit * 8 / 72


def test_entry_points_check_their_arguments(_emulation):
    from liger_kernel_b200 import _lib

    lib = _emulation
    buf = (C.c_float * 8192)()
    base = C.addressof(buf)
    base += -base % 64
    layers = (C.c_void_p * 2)(base, base + 1024)

    def balance(**kw):
        p = _lib.Balance(2, 4, 16, 2, 16, _lib.FLCE_FP32, 0, 0.0, 0.0, None)
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    def forward(p, logits=layers, loss=base + 2048, counts=base + 4096, coef=base + 2112, ws=base + 8192, nbytes=8192):
        return lib.flce_b200_balance_forward(C.byref(p) if p is not None else None, logits, loss, counts, coef, ws, nbytes, None)

    def backward(p, logits=layers, coef=base + 2112, up=base + 2048, grads=base + 16384):
        return lib.flce_b200_balance_backward(C.byref(p), logits, coef, up, grads, None)

    INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3
    assert forward(balance()) == 0 and backward(balance()) == 0 and forward(None) == INVALID
    for kw, code in ((dict(n_layers=0), INVALID), (dict(n_layers=1 << 17), INVALID), (dict(n_tokens=-1), INVALID),
                     (dict(n_tokens=1 << 31), INVALID), (dict(n_experts=0), INVALID), (dict(n_experts=1025), UNSUPPORTED),
                     (dict(top_k=0), INVALID), (dict(top_k=17), INVALID), (dict(ld=-1), INVALID), (dict(dtype=3), INVALID),
                     (dict(mask=base, mask_bytes=2), INVALID), (dict(mask=base + 4, mask_bytes=8), INVALID)):
        before = lib.emu_launches()
        assert forward(balance(**kw)) == code and backward(balance(**kw)) == code, kw
        assert lib.flce_b200_balance_workspace_bytes(C.byref(balance(**kw))) == 0 and lib.emu_launches() == before
    null, crooked = (C.c_void_p * 2)(base, None), (C.c_void_p * 2)(base, base + 2)
    for logits in (None, null, crooked):
        assert forward(balance(), logits) == INVALID and backward(balance(), logits) == INVALID
    assert forward(balance(), loss=None) == INVALID and forward(balance(), counts=None) == INVALID and forward(balance(), coef=None) == INVALID
    assert forward(balance(), ws=None) == WORKSPACE and forward(balance(), ws=base + 4) == WORKSPACE and forward(balance(), nbytes=64) == WORKSPACE
    assert b"workspace" in lib.flce_b200_last_error()
    assert backward(balance(), coef=None) == INVALID and backward(balance(), up=None) == INVALID and backward(balance(), grads=None) == INVALID
    assert backward(balance(), grads=base + 2) == INVALID
    assert backward(balance(n_tokens=0)) == 0


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("experts,top_k", [(8, 2), (24, 4), (32, 4), (60, 4), (64, 6), (128, 8), (256, 8), (300, 8)])
def test_rows_far_from_zero(dtype, experts, top_k):
    cases.case_far_rows("cpu", dtype, experts, top_k)


def test_counts_out_of_range():
    cases.case_counts_out_of_range("cpu")


def test_forward_mode():
    cases.case_forward_mode("cpu")
