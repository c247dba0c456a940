"""A second copy of the library beside the installed one launches kernels of its own (see tests/test_library_copies_cpu.py)."""

import shutil

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_second_copy_gives_the_same_results(tmp_path):
    import liger_kernel_b200 as lk
    from liger_kernel_b200 import _lib, _torch_ops

    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(300, 4096, generator=g, device="cuda").bfloat16().requires_grad_(True)
    logits = torch.randn(500, 64, generator=g, device="cuda", requires_grad=True)

    def run():
        y = lk.liger_rms_norm(x)
        loss = lk.liger_load_balancing_loss(logits, 64, 6)
        return [y.detach(), *torch.autograd.grad(y, x, torch.ones_like(y)), loss.detach(), *torch.autograd.grad(loss, logits)]

    want = run()
    copy = shutil.copy(_lib.LIB_PATH, tmp_path / "another.so")
    _torch_ops.bind(copy)
    try:
        got = run()
    finally:
        _torch_ops.bind(_lib.LIB_PATH)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
