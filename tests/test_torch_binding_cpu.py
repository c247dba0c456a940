"""A package whose torch binding is missing, was built against another torch or cannot be loaded: the operators that do not need it are
there, those that do say what is wrong when they are called, and the build script builds it anew."""

import importlib.util
import os
import subprocess
import sys

import pytest

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_PACKAGE = os.path.join(_ROOT, "liger-kernel_b200", "liger_kernel_b200")
_BINDING = "libflce_b200_torch.so"

_SCRIPT = """
import torch
import liger_kernel_b200 as lk
x, w = torch.randn(2, 8), torch.ones(8)
for call in (lambda: lk.liger_layer_norm(x, w), lambda: lk.LigerRMSNorm(8)(x), lambda: lk.liger_load_balancing_loss(x, 8)):
    try:
        call()
    except ImportError as e:
        print("refused:", e)
try:
    lk.liger_fused_linear_cross_entropy(x, torch.randn(16, 8), torch.tensor([1, 2]))
except RuntimeError as e:
    print("head:", e)
"""


def _package_with(tmp_path, binding):
    package = tmp_path / "liger_kernel_b200"
    package.mkdir()
    for name in os.listdir(_PACKAGE):
        if name not in (_BINDING, "__pycache__"):
            os.symlink(os.path.join(_PACKAGE, name), package / name)
    if binding is not None:
        (package / _BINDING).write_bytes(binding)
    done = subprocess.run([sys.executable, "-c", _SCRIPT], cwd=tmp_path, env=dict(os.environ, PYTHONPATH=str(tmp_path)),
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
    return done.stdout.splitlines()


def _binding():
    with open(os.path.join(_PACKAGE, _BINDING), "rb") as f:
        return f.read()


@pytest.mark.parametrize("state,says", [("missing", "is missing"), ("other torch", "another torch"), ("unreadable", "cannot be loaded")])
def test_package_without_a_usable_binding(tmp_path, state, says):
    import torch

    version = torch.__version__.encode()
    binding = {"missing": None, "other torch": _binding().replace(b"against torch " + version + b";", b"against torch " + b"0" * len(version) + b";"),
               "unreadable": b"liger_b200 built against torch " + version + b";"}[state]
    lines = _package_with(tmp_path, binding)
    assert len(lines) == 4 and all(line.startswith("refused:") and says in line and "build.py" in line for line in lines[:3]), lines
    assert lines[3].startswith("head:") and "CUDA" in lines[3]          # there, and refuses tensors on the CPU as ever


def test_build_notices_another_torch(monkeypatch):
    spec = importlib.util.spec_from_file_location("flce_b200_build", os.path.join(_ROOT, "liger-kernel_b200", "build.py"))
    build = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(build)
    monkeypatch.setattr(build, "_deps", lambda: [])                      # the sources' age is another matter
    assert not build.needs_build()
    monkeypatch.setattr(build, "_torch_version", lambda: "0.0.0")
    assert build.needs_build()
