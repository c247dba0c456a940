"""Shared bodies of the tests of layer norm and RMSNorm: run on a B200 (tests/test_norm_gpu.py) and, with the library's host side
and kernels emulated, on CPU tensors (tests/test_norm_emulation_cpu.py).  They are held to the definition in float64.

Tolerances.  u = 2^-24, h = half a step of the result's type (finfo.eps / 2).  A row's sums are added in at most 32 + 5 + 16
steps (elements of a thread, lanes, warps), the rest of an element is below ten operations: C = 64 steps of u against the
magnitudes that meet in it.  The mean's error is C u mean|x|, which in units of xhat is C u mean|x| rstd <= C u max|x| rstd; the
same holds for x - mean.  So, with k = 1 + max|x| rstd of the row,
    y :  h |y|  +  C u k (|xhat g| + |b| + |g|)
    dx:  h |dx| +  C u k rstd (|m| + mean|m| + (1 + |xhat|) mean(|m| (1 + |xhat|)))
    dw:  h |dw| +  (n + C) u k sum|dy| (1 + |xhat|)          db:  h |db| + (n + C) u sum|dy|
(n rows, added one after the other at worst).  "llama" casting rounds xhat once more: h |xhat g| in y and h sum|dy xhat| in dw."""

import torch
import torch.utils.checkpoint

U, C = 2.0 ** -24, 64


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(n, hidden, dtype, wdtype, weight=True, bias=True, offset=0.0, pitch=0, seed=0, leading=None):
    g = torch.Generator().manual_seed(seed + 31 * n + hidden)
    wide = torch.randn(n, hidden + pitch, generator=g) * 2.0 + 0.3
    wide[:, ::7] *= 8.0
    x = wide.to(dtype)[:, :hidden]
    w = (1.0 - offset + 0.2 * torch.randn(hidden, generator=g)).to(wdtype) if weight else None
    b = (0.3 * torch.randn(hidden, generator=g)).to(wdtype) if bias else None
    dy = (torch.randn(n, hidden, generator=g) * 0.5).to(dtype)
    return x, w, b, dy


def reference(x, w, b, dy, eps, offset, centered):
    x, dy = x.double(), dy.double()
    n, hidden = x.shape
    mean = x.mean(-1, keepdim=True) if centered else torch.zeros(n, 1, dtype=torch.float64)
    rstd = 1 / torch.sqrt((x - mean).square().mean(-1, keepdim=True) + eps)
    xhat = (x - mean) * rstd
    g = torch.ones(hidden, dtype=torch.float64) if w is None else w.double() + offset
    bb = torch.zeros(hidden, dtype=torch.float64) if b is None else b.double()
    m = dy * g
    dx = rstd * (m - (m.mean(-1, keepdim=True) if centered else 0) - xhat * (m * xhat).mean(-1, keepdim=True))
    k = 1 + x.abs().amax(-1, keepdim=True) * rstd if n else rstd
    tol = dict(
        y=C * U * k * ((xhat * g).abs() + bb.abs() + g.abs()),
        dx=C * U * k * rstd * (m.abs() + m.abs().mean(-1, keepdim=True)
                               + (1 + xhat.abs()) * (m.abs() * (1 + xhat.abs())).mean(-1, keepdim=True)),
        dw=(n + C) * U * (k * dy.abs() * (1 + xhat.abs())).sum(0), db=(n + C) * U * dy.abs().sum(0))
    return dict(y=xhat * g + bb, dx=dx, dw=(dy * xhat).sum(0), db=dy.sum(0), tol=tol, xhat=xhat, g=g, dy=dy)


def compare(name, got, want, tol):
    got = got.detach().cpu()
    assert got.shape == want.shape, name
    limit = tol + half_step(got.dtype) * want.abs() * (1 + 2.0 ** -8)       # the rounding acts on the value just computed
    # below the smallest normal number a step is that number's
    limit = limit + torch.finfo(got.dtype).tiny * half_step(got.dtype) * 2
    off = (got.double() - want).abs() - limit
    assert not torch.isnan(got).any(), name
    assert off.numel() == 0 or float(off.max()) <= 0, (name, float(off.max()), int(off.argmax()))


def case_matches_definition(device, kind, n, hidden, dtype, wdtype=None, weight=True, bias=True, offset=0.0, pitch=0,
                            casting_mode="gemma", eps=1e-6, seed=0):
    import liger_kernel_b200 as lk

    wdtype = wdtype or dtype
    centered = kind == "layer"
    bias = bias and centered
    x, w, b, dy = make(n, hidden, dtype, wdtype, weight, bias, offset, pitch, seed)
    ref = reference(x, w, b, dy, eps, offset, centered)
    wide = torch.empty(n, hidden + pitch, dtype=dtype, device=device)
    xd = wide[:, :hidden]
    xd.copy_(x)
    xd.requires_grad_(True)
    wd = None if w is None else w.to(device).requires_grad_(True)
    bd = None if b is None else b.to(device).requires_grad_(True)
    if centered:
        y = lk.liger_layer_norm(xd, wd, bd, eps, offset=offset)
    else:
        y = lk.liger_rms_norm(xd, wd, eps, offset=offset, casting_mode=casting_mode)
    assert y.dtype == dtype and y.is_contiguous()
    leaves = [t for t in (xd, wd, bd) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy.to(device))
    tol = ref["tol"]
    if casting_mode == "llama" and not centered:
        tol["y"] = tol["y"] + half_step(dtype) * (ref["xhat"] * ref["g"]).abs()
        tol["dw"] = tol["dw"] + half_step(dtype) * (ref["dy"] * ref["xhat"]).abs().sum(0)
    compare("y", y, ref["y"], tol["y"])
    names = ["dx"] + ["dw"] * (w is not None) + ["db"] * (b is not None)
    for name, got, leaf in zip(names, grads, leaves):
        assert got.dtype == leaf.dtype and got.shape == leaf.shape, name
        compare(name, got, ref[name], tol[name])
    return y, grads


def case_gradient_against_differences(device, kind):
    """A directional derivative of sum(y * r) in float64 differences of the definition against the operator's gradients."""
    import liger_kernel_b200 as lk

    n, hidden, eps = 6, 40, 1e-5
    x, w, b, r = make(n, hidden, torch.float32, torch.float32, True, kind == "layer", 0.0, 0, 5)
    centered = kind == "layer"

    def f(xx, ww, bb):
        return float((reference(xx, ww, bb, r, eps, 0.0, centered)["y"] * r.double()).sum())

    leaves = [t for t in (x, w, b) if t is not None]
    moved = [t.to(device, copy=True).requires_grad_(True) for t in leaves]
    y = lk.liger_layer_norm(*moved, eps) if centered else lk.liger_rms_norm(*moved, eps)
    grads = torch.autograd.grad(y, moved, r.to(device))
    g = torch.Generator().manual_seed(1)
    for i, leaf in enumerate(leaves):
        direction = torch.randn(leaf.shape, generator=g, dtype=torch.float64)
        step = 1e-5
        plus, minus = list(leaves), list(leaves)
        plus[i], minus[i] = leaf.double() + step * direction, leaf.double() - step * direction
        fill = [None] * (3 - len(leaves))
        slope = (f(*plus, *fill) - f(*minus, *fill)) / (2 * step)
        got = float((grads[i].double().cpu() * direction).sum())
        # the differences are off by about step^2 times a third derivative of order |x| rstd^3: 1e-8 of the slope's terms
        size = float((grads[i].double().cpu().abs() * direction.abs()).sum())
        assert abs(got - slope) <= 1e-5 * size, (i, got, slope)


def case_special_values(device, kind):
    """A row with an infinity or a NaN is lost, its neighbours in the same block are what they are without it."""
    import liger_kernel_b200 as lk

    for n, hidden in ((9, 24), (5, 300), (4, 1000), (400 if device == "cuda" else 60, 520)):
        x, w, b, dy = make(n, hidden, torch.bfloat16, torch.bfloat16, True, False, 0.0, 0, 3)
        bad = x.clone()
        bad[1, 3], bad[2, 0] = float("inf"), float("nan")
        keep = [i for i in range(n) if i not in (1, 2)]
        out = []
        for t in (x, bad):
            td = t.to(device).requires_grad_(True)
            wd = w.to(device)
            y = lk.liger_layer_norm(td, wd, None, 1e-6) if kind == "layer" else lk.liger_rms_norm(td, wd, 1e-6)
            (dx,) = torch.autograd.grad(y, (td,), dy.to(device))
            out.append((y.detach()[keep], dx[keep], y.detach()[1:3].float()))
        assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
        assert bool(torch.isnan(out[1][2]).any(-1).all())


def case_shapes_and_views(device):
    """Leading dimensions, no rows, one element, a broadcast gradient, a transposed input, a gradient for the weight alone."""
    import liger_kernel_b200 as lk

    g = torch.Generator().manual_seed(0)
    x3 = torch.randn(2, 3, 5, 16, generator=g).to(device).requires_grad_(True)
    w = torch.randn(16, generator=g).to(device).requires_grad_(True)
    y = lk.liger_layer_norm(x3, w, None, 1e-6)
    assert y.shape == x3.shape
    y.sum().backward()                                           # an expanded gradient
    flat = x3.detach().reshape(-1, 16).clone().requires_grad_(True)
    w2 = w.detach().clone().requires_grad_(True)
    lk.liger_layer_norm(flat, w2, None, 1e-6).backward(torch.ones(30, 16, device=device))
    assert torch.equal(x3.grad.reshape(-1, 16), flat.grad) and torch.equal(w.grad, w2.grad)
    for fn in (lambda t, p: lk.liger_layer_norm(t, p, p, 1e-6), lambda t, p: lk.liger_rms_norm(t, p, 1e-6)):
        empty = torch.empty(0, 16, device=device, requires_grad=True)
        w.grad = None
        out = fn(empty, w)
        assert out.shape == (0, 16)
        out.sum().backward()
        assert empty.grad.shape == (0, 16) and torch.equal(w.grad, torch.zeros_like(w))
        one = torch.full((3, 1), 2.0, device=device, requires_grad=True)
        gain = torch.full((1,), 3.0, device=device, requires_grad=True)
        fn(one, gain).sum().backward()
        assert torch.isfinite(one.grad).all()
        t = torch.randn(16, 7, generator=g).to(device).t()       # [7, 16] with rows of stride 1
        assert torch.equal(fn(t, w.detach()), fn(t.contiguous(), w.detach()))
        frozen = torch.randn(4, 16, generator=g).to(device)
        w.grad = None
        fn(frozen, w).sum().backward()
        assert w.grad is not None
        row = torch.randn(16, generator=g).to(device).requires_grad_(True)       # one row seen as five
        fn(row.expand(5, 16), w.detach()).square().sum().backward()
        five = row.detach().repeat(5, 1).requires_grad_(True)
        fn(five, w.detach()).square().sum().backward()
        assert float((row.grad - five.grad.sum(0)).abs().max()) <= 8 * U * float(five.grad.abs().sum(0).max())
        assert torch.equal(fn(row.detach(), w.detach()), fn(row.detach()[None], w.detach())[0])
    same = torch.randn(3, 16, generator=g).to(device)
    assert torch.equal(lk.liger_layer_norm(torch.full((2, 8), 5.0, device=device), None, None, 1e-6), torch.zeros(2, 8, device=device))
    layer, rms = lk.LigerLayerNorm(16, bias=True).to(device), lk.LigerRMSNorm(16, offset=1.0, init_fn="zeros").to(device)
    assert torch.equal(layer(same), lk.liger_layer_norm(same, layer.weight, layer.bias, 1e-6))
    assert torch.equal(rms(same), lk.liger_rms_norm(same, None, 1e-6))
    assert lk.LigerRMSNorm(16, elementwise_affine=False).weight is None


def case_refusals(device):
    import pytest

    import liger_kernel_b200 as lk

    x = torch.randn(4, 16).to(device)
    w = torch.ones(16, device=device)
    with pytest.raises(TypeError, match="unsupported dtype"):
        lk.liger_layer_norm(x.double(), w, None, 1e-6)
    with pytest.raises(TypeError, match="unsupported weight dtype"):
        lk.liger_rms_norm(x, w.double(), 1e-6)
    with pytest.raises(ValueError, match=r"weight must be \[16\]"):
        lk.liger_layer_norm(x, w[:15], None, 1e-6)
    with pytest.raises(ValueError, match=r"bias must be \[16\]"):
        lk.liger_layer_norm(x, w, w[None], 1e-6)
    with pytest.raises(ValueError, match="H >= 1"):
        lk.liger_rms_norm(x[:, :0], None, 1e-6)
    with pytest.raises(NotImplementedError, match="casting_mode"):
        lk.liger_rms_norm(x, w, 1e-6, casting_mode="none")
    with pytest.raises(AssertionError, match="init_fn"):
        lk.LigerLayerNorm(8, init_fn="twos")
    xg = x.clone().requires_grad_(True)
    (first,) = torch.autograd.grad(lk.liger_layer_norm(xg, w, None, 1e-6).square().sum(), (xg,), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first.sum().backward()


def case_autograd(device):
    """A graph kept and used twice, a recomputed one, hooks on what is saved, an input changed in between, a weight alone."""
    import pytest

    import liger_kernel_b200 as lk

    g = torch.Generator().manual_seed(8)
    x = torch.randn(12, 40, generator=g).to(device).requires_grad_(True)
    w = torch.randn(40, generator=g).to(device).requires_grad_(True)
    b = torch.randn(40, generator=g).to(device).requires_grad_(True)
    dy = torch.randn(12, 40, generator=g).to(device)
    y = lk.liger_layer_norm(x, w, b, 1e-6)
    want = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(want, torch.autograd.grad(y, (x, w, b), dy)))
    with pytest.raises(RuntimeError, match="second time"):
        y.backward(dy)
    again = torch.utils.checkpoint.checkpoint(lambda t: lk.liger_layer_norm(t, w, b, 1e-6), x, use_reentrant=False)
    assert all(torch.equal(p, q) for p, q in zip(want, torch.autograd.grad(again, (x, w, b), dy)))
    packed = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: packed.append(t) or t, lambda t: t):
        y = lk.liger_layer_norm(x, w, b, 1e-6)
    assert len(packed) == 3 and all(torch.equal(p, q) for p, q in zip(want, torch.autograd.grad(y, (x, w, b), dy)))
    (only,) = torch.autograd.grad(lk.liger_layer_norm(x, w, b, 1e-6), (b,), dy)
    assert torch.equal(only, want[2])
    for fn in (lambda: lk.liger_layer_norm(x, w, b, 1e-6), lambda: lk.liger_rms_norm(x, w, 1e-6)):
        y = fn()
        with torch.no_grad():
            x.mul_(1.5)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward(dy)
    with torch.no_grad():
        assert not lk.liger_rms_norm(x, w, 1e-6).requires_grad
    with torch.inference_mode():
        assert lk.liger_layer_norm(x, w, b, 1e-6).shape == x.shape


def case_forward_mode(device):
    """A tangent on the input or on a parameter is refused: dropped, it would be a derivative of zero."""
    import pytest
    import torch.autograd.forward_ad as fa

    import liger_kernel_b200 as lk

    x, w, b = torch.randn(3, 16).to(device), torch.randn(16).to(device), torch.randn(16).to(device)
    want = lk.liger_layer_norm(x, w, b)
    with fa.dual_level():
        for i in range(3):
            args = [x, w, b]
            args[i] = fa.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError, match="forward"):
                lk.liger_layer_norm(*args)
            if i < 2:
                with pytest.raises(NotImplementedError, match="forward"):
                    lk.liger_rms_norm(*args[:2])
        assert torch.equal(lk.liger_layer_norm(x, w, b), want)
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(lambda t: lk.liger_rms_norm(t, w), (x,), (torch.ones_like(x),))
