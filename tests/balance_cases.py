"""Shared bodies of the tests of the router's load-balancing loss: run on a B200 (tests/test_load_balancing_gpu.py) and, with the
library's host side and kernels emulated, on CPU tensors (tests/test_load_balancing_emulation_cpu.py).  They are held to the
definition in float64, the choice of experts a sort by (logit, index).

Tolerances.  u = 2^-24.  With d_j = max - x_j: the exponent d_j log2(e) carries two roundings, 2 u d_j in e^-d_j, the device's
exp2 is good to 2^-22 = 4 u, the sum over a row takes at most 32 + 5 steps and the quotient two more: a probability is off by
at most r_j = (64 + 4 d_j) u of itself.  S_e adds n of them, one after the other at worst, the loss is summed in fp64 from
there and rounded once: (n + 64 + 4 max d) u of the loss.  lse is off by 8 u (1 + |lse|) (log2 of the device: 2^-22).  A
gradient p_j (a_j - sum a p + c lse) is off by 2 r_j p_j (|a_j| + sum |a| p + |c| (1 + |lse|)), a and c being rounded once,
and by half a step of its type."""

import math

import torch

U = 2.0 ** -24


def make(layers, tokens, experts, dtype, seed=0, steps=None, spread=1.5):
    """steps: logits are multiples of 1 / steps, so that many are equal."""
    g = torch.Generator().manual_seed(seed + 7 * layers + 13 * tokens + experts)
    x = torch.randn(layers, tokens, experts, generator=g) * spread + torch.randn(layers, 1, experts, generator=g) * 0.5
    if steps:
        x = torch.round(x * steps) / steps
    return x.to(dtype)


def reference(x, top_k, keep, z):
    """x [layers, tokens, experts]; keep [tokens] bool."""
    layers, tokens, experts = x.shape
    x = x[:, keep].double()
    n = x.shape[0] * x.shape[1]
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :top_k]
    counts = torch.nn.functional.one_hot(order, experts).sum((1, 2)) if n else torch.zeros(layers, experts, dtype=torch.int64)
    if n == 0:
        return dict(loss=0.0, z=0.0, counts=counts, grads=torch.zeros(layers, 0, experts, dtype=torch.float64),
                    tol_loss=0.0, tol_z=0.0, tol_grads=torch.zeros(layers, 0, experts, dtype=torch.float64))
    d = x.amax(-1, keepdim=True) - x
    p = torch.softmax(x, -1)
    lse = torch.logsumexp(x, -1, keepdim=True)
    c = counts.sum(0).double()
    a = experts * (c - c.mean()) / n ** 2
    zc = 2 * z / n
    grads = p * (a - (a * p).sum(-1, keepdim=True)) + zc * lse * p
    balance = experts * (c * p.sum((0, 1))).sum() / n ** 2
    z_loss = z * (lse ** 2).sum() / n
    dmax = float(d[torch.isfinite(d)].max())
    d = torch.where(torch.isfinite(d), d, 0.0)            # an expert that is masked out has probability zero exactly
    r = (64 + 4 * d) * U
    tol_grads = 2 * r * p * (a.abs() + (a.abs() * p).sum(-1, keepdim=True) + abs(zc) * (1 + lse.abs()))
    tol_z = float(z / n * (lse.abs() * 2 * 8 * U * (1 + lse.abs())).sum() + (n + 64) * U * z_loss)
    tol_loss = float((n + 64 + 4 * dmax) * U * balance) + tol_z
    return dict(loss=float(balance + z_loss), z=float(z_loss), counts=counts, grads=grads, tol_loss=tol_loss, tol_z=tol_z,
                tol_grads=tol_grads)


def case_matches_definition(device, x, top_k, mask=None, z=0.0, pitch=0, up=1.0, mask_dtype=torch.int64, leading=None):
    """mask: list of 0 / 1 per token.  What padding holds is garbage."""
    import liger_kernel_b200 as lk

    layers, tokens, experts = x.shape
    keep = torch.ones(tokens, dtype=torch.bool) if mask is None else torch.tensor(mask) != 0
    ref = reference(x, top_k, keep, z)
    given = x.clone()
    if mask is not None:
        garbage = torch.tensor([float("nan"), float("inf"), -float("inf"), torch.finfo(x.dtype).min]).to(x.dtype)
        given[:, ~keep] = garbage[torch.arange(int((~keep).sum())) % 4].view(1, -1, 1)
    leaves = []
    for l in range(layers):
        wide = torch.empty(tokens, experts + pitch, dtype=x.dtype, device=device)
        t = wide[:, :experts]
        t.copy_(given[l])
        leaves.append(t.requires_grad_(True))
    logits = tuple(leaves if leading is None else [t.reshape(*leading, experts) for t in leaves])
    m = None if mask is None else torch.tensor(mask).to(mask_dtype).to(device)
    out = lk.liger_load_balancing_loss(logits, experts, top_k, m, lse_square_scale=z, return_z_loss=True, return_expert_counts=True)
    assert out.loss.dtype == torch.float32 and out.loss.dim() == 0 and out.expert_counts.dtype == torch.int64
    assert torch.equal(out.expert_counts.cpu(), ref["counts"]), (out.expert_counts, ref["counts"])
    assert abs(float(out.loss.detach()) - ref["loss"]) <= ref["tol_loss"] + U * abs(ref["loss"]), (float(out.loss.detach()), ref["loss"])
    assert abs(float(out.z_loss) - ref["z"]) <= ref["tol_z"] + U * ref["z"]
    grads = torch.autograd.grad(out.loss * up, leaves)
    half = torch.finfo(x.dtype).eps / 2
    for l, got in enumerate(grads):
        assert got.dtype == x.dtype and got.shape == (tokens, experts)
        got = got.cpu().double()
        assert not got[~keep].any() and not torch.isnan(got).any()        # exact zeros for what the mask leaves out
        want, tol = ref["grads"][l] * up, ref["tol_grads"][l] * abs(up)
        tol = tol * 1.01 + half * want.abs() * (1 + 2.0 ** -8) + 2 * U * want.abs() + torch.finfo(x.dtype).tiny * half * 2
        off = (got[keep] - want).abs() - tol
        assert off.numel() == 0 or float(off.max()) <= 0, (l, float(off.max()))
    return out, grads


def case_ties(device, dtype, experts, top_k):
    """Logits on a coarse grid: most rows have several equal ones at the border of the chosen set; -0 equals +0."""
    x = make(2, 61, experts, dtype, seed=3, steps=1)
    x[0, ::3] = torch.where(x[0, ::3] == 0, torch.tensor(-0.0, dtype=dtype), x[0, ::3])
    x[1, 5] = 0.25                                                          # a row of equal logits
    case_matches_definition(device, x, top_k)


def case_masked_experts(device, dtype, experts, top_k):
    """Experts switched off by -inf or by the type's lowest value, in some rows more than leave top_k."""
    x = make(1, 40, experts, dtype, seed=4)
    x[0, :20, experts // 2:] = -float("inf")
    x[0, 20:30, 1:] = -float("inf")
    x[0, 30:, :experts // 2] = torch.finfo(dtype).min
    case_matches_definition(device, x, top_k)


def case_empty(device):
    import liger_kernel_b200 as lk

    x = make(2, 6, 16, torch.bfloat16)
    out, grads = case_matches_definition(device, x, 4, mask=[0] * 6, z=0.1)
    assert float(out.loss.detach()) == 0.0 and float(out.z_loss) == 0.0 and not out.expert_counts.any()
    none = torch.empty(0, 16, device=device, requires_grad=True)
    out = lk.liger_load_balancing_loss(none, 16, 2, torch.empty(0, device=device), return_expert_counts=True)
    assert float(out.loss.detach()) == 0.0 and out.expert_counts.shape == (16,) and not out.expert_counts.any()
    out.loss.backward()
    assert none.grad.shape == (0, 16)
    case_matches_definition(device, make(1, 1, 8, torch.float32), 2, z=0.5)
    case_matches_definition(device, make(1, 3, 1, torch.float32), 1)


def case_views_and_partial_gradients(device):
    """One tensor in the place of a tuple, leading dimensions, layers of different pitch, a transposed layer, a layer without a
    gradient, the loss unused, the module."""
    import liger_kernel_b200 as lk

    x = make(3, 24, 20, torch.float32, seed=9)
    whole = [t.clone().to(device).requires_grad_(True) for t in x]
    base = lk.liger_load_balancing_loss(tuple(whole), 20, 3)
    want = torch.autograd.grad(base, whole)
    wide = torch.empty(24, 28, device=device)
    wide[:, :20].copy_(x[0])
    mixed = [wide[:, :20].requires_grad_(True), x[1].clone().to(device), x[2].t().contiguous().to(device).t().requires_grad_(True)]
    loss = lk.liger_load_balancing_loss([t.view(4, 6, 20) if t.is_contiguous() else t for t in mixed], 20, 3)
    assert torch.equal(loss, base)
    got = torch.autograd.grad(loss, (mixed[0], mixed[2]))
    # the rows may be read in other pieces (their alignment differs): the same sums in another order, a few u of p |a|
    for a, b in zip(got, (want[0], want[2])):
        assert a.shape == b.shape and float((a - b).abs().max()) <= 64 * U * float(b.abs().max())
    one = lk.LigerLoadBalancingLoss(20, 3, return_expert_counts=True)(whole[0])
    assert one.expert_counts.shape == (20,) and one.z_loss is None and int(one.expert_counts.sum()) == 24 * 3
    assert not one.expert_counts.requires_grad and not lk.liger_load_balancing_loss(whole[0].detach(), 20, 3).requires_grad
    none = lk.LigerLoadBalancingLossFunction.apply(20, 3, None, 0.0, whole[0])
    assert len(none) == 3 and none[0].requires_grad and not none[1].requires_grad


def case_gradient_against_differences(device):
    import liger_kernel_b200 as lk

    x = make(2, 9, 12, torch.float32, seed=11)
    z = 0.05
    leaves = [t.clone().to(device).requires_grad_(True) for t in x]
    grads = torch.autograd.grad(lk.liger_load_balancing_loss(tuple(leaves), 12, 3, lse_square_scale=z), leaves)
    keep = torch.ones(9, dtype=torch.bool)
    counts = reference(x, 3, keep, z)["counts"].sum(0).double()

    def f(t):
        p = torch.softmax(t, -1)
        return float(12 * (counts * p.sum((0, 1))).sum() / 18 ** 2 + z * torch.logsumexp(t, -1).square().mean())

    direction = torch.randn(x.shape, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    step = 1e-5
    slope = (f(x.double() + step * direction) - f(x.double() - step * direction)) / (2 * step)
    got = sum(float((g.double().cpu() * dd).sum()) for g, dd in zip(grads, direction))
    size = sum(float((g.double().cpu().abs() * dd.abs()).sum()) for g, dd in zip(grads, direction))
    assert abs(got - slope) <= 1e-5 * size


def case_nan_reaches_the_loss(device):
    import liger_kernel_b200 as lk

    for experts in (16, 64):
        for bad in (float("nan"), float("inf")):              # softmax of an infinite logit is inf / inf
            x = make(1, 12, experts, torch.bfloat16)
            x[0, 3, 2] = bad
            t = x[0].to(device).requires_grad_(True)
            loss = lk.liger_load_balancing_loss(t, experts, 4)
            assert math.isnan(float(loss.detach()))
            (grad,) = torch.autograd.grad(loss, (t,))
            assert bool(torch.isnan(grad[3]).any())
            # the same row left out: nothing of it shows
            mask = torch.ones(12, dtype=torch.int64)
            mask[3] = 0
            case_matches_definition(device, make(1, 12, experts, torch.bfloat16), 4, mask=mask.tolist())


def case_refusals(device):
    import pytest

    import liger_kernel_b200 as lk

    x = torch.randn(6, 8).to(device)
    with pytest.raises(TypeError, match="unsupported dtype"):
        lk.liger_load_balancing_loss(x.double(), 8)
    with pytest.raises(ValueError, match="at least one layer"):
        lk.liger_load_balancing_loss((), 8)
    with pytest.raises(ValueError, match="router logits must be"):
        lk.liger_load_balancing_loss(x, 9)
    with pytest.raises(ValueError, match="top_k must be in"):
        lk.liger_load_balancing_loss(x, 8, 9)
    with pytest.raises(ValueError, match="top_k must be in"):
        lk.liger_load_balancing_loss(x, 8, 0)
    with pytest.raises(ValueError, match="must agree"):
        lk.liger_load_balancing_loss((x, x[:5]), 8)
    with pytest.raises(ValueError, match="must agree"):
        lk.liger_load_balancing_loss((x, x.half()), 8)
    with pytest.raises(ValueError, match="attention mask has 5 elements"):
        lk.liger_load_balancing_loss(x, 8, 2, torch.ones(5, device=device))
    with pytest.raises(NotImplementedError, match="at most 1024"):
        lk.liger_load_balancing_loss(torch.zeros(2, 1025, device=device), 1025)
    with pytest.raises(AssertionError, match="top_k must be between"):
        lk.LigerLoadBalancingLoss(8, 9)
    xg = x.clone().requires_grad_(True)
    (first,) = torch.autograd.grad(lk.liger_load_balancing_loss(xg, 8).square(), (xg,), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first.sum().backward()
    loss = lk.liger_load_balancing_loss(xg, 8)
    loss.backward()
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward()
    loss = lk.liger_load_balancing_loss(xg, 8)
    with torch.no_grad():
        xg.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def case_far_rows(device, dtype, experts, top_k):
    """Whole rows of -1e10, of +1e10, of the type's lowest and of its largest finite value among ordinary ones: a softmax over equal
    logits is 1 / experts wherever they lie, and neither the loss nor the gradients of the other rows may suffer.  Then rows whose
    largest logit is 1e10 above or below the others, or at the other end of the type's range."""
    import liger_kernel_b200 as lk

    info = torch.finfo(dtype)
    far = [v for v in (-1e10, 1e10, info.min, info.max) if abs(v) <= info.max]
    x = make(2, 40, experts, dtype, seed=6)
    for i, v in enumerate(far):
        x[i % 2, 3 + i::13] = v
    case_matches_definition(device, x, top_k, up=0.5)
    if abs(far[0]) < info.max:                                    # with the lse^2 term, where the square is a finite fp32 number
        x = make(1, 40, experts, dtype, seed=6)
        x[0, 3], x[0, 17] = -1e10, 1e10
        case_matches_definition(device, x, top_k, z=1e-22)
    x = make(1, 40, experts, dtype, seed=7)
    x[0, 2, 1], x[0, 5, experts - 1], x[0, 9, 0], x[0, 9, 1] = far[1], far[-1], far[-1], info.min
    x[0, 12], x[0, 14] = far[0], info.min
    x[0, 12, 2], x[0, 14, 3] = 1.0, info.max
    ref = reference(x, top_k, torch.ones(40, dtype=torch.bool), 0.0)
    t = x[0].to(device).requires_grad_(True)
    out = lk.liger_load_balancing_loss(t, experts, top_k, return_expert_counts=True)
    (grad,) = torch.autograd.grad(out.loss, (t,))
    assert torch.equal(out.expert_counts.cpu(), ref["counts"][0])
    # beyond d = 104 a probability is below 2^-150 and zero in fp32: r_j p_j is largest before that
    assert abs(float(out.loss.detach()) - ref["loss"]) <= (40 + 64 + 4 * 104) * U * ref["loss"]
    limit = ref["tol_grads"][0] * 1.01 + info.eps / 2 * ref["grads"][0].abs() * 1.01 + info.tiny * info.eps
    assert bool(((grad.cpu().double() - ref["grads"][0]).abs() <= limit).all())


def case_counts_out_of_range(device):
    """No experts, or fewer than none, whatever the number of dimensions and tokens: refused before anything is divided by them."""
    import pytest

    import liger_kernel_b200 as lk

    for shape in ((0,), (4, 0), (2, 3, 0), (0, 3, 0), (2, 2, 2, 0)):
        with pytest.raises(ValueError, match="num_experts must be at least 1"):
            lk.liger_load_balancing_loss(torch.zeros(shape, device=device), 0, 1)
    with pytest.raises(ValueError, match="num_experts must be at least 1"):
        lk.liger_load_balancing_loss(torch.zeros(2, 3, 4, device=device), -4, 1)
    with pytest.raises(ValueError, match="router logits must be"):
        lk.liger_load_balancing_loss(torch.zeros(2, 3, 0, device=device), 4, 1)
    with pytest.raises(ValueError, match="router logits must be"):
        lk.liger_load_balancing_loss(torch.zeros((), device=device), 1, 1)


def case_forward_mode(device):
    """A tangent on any layer's logits is refused: dropped, it would be a derivative of zero."""
    import pytest
    import torch.autograd.forward_ad as fa

    import liger_kernel_b200 as lk

    x = make(2, 6, 8, torch.float32).to(device)
    want = lk.liger_load_balancing_loss(tuple(x), 8)
    with fa.dual_level():
        dual = fa.make_dual(x[1], torch.ones_like(x[1]))
        with pytest.raises(NotImplementedError, match="forward"):
            lk.liger_load_balancing_loss((x[0], dual), 8)
        with pytest.raises(NotImplementedError, match="forward"):
            lk.LigerLoadBalancingLoss(8)(dual.clone().requires_grad_(True))
        assert torch.equal(lk.liger_load_balancing_loss((x[0], fa.unpack_dual(dual).primal), 8), want)
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(lambda t: lk.liger_load_balancing_loss(t, 8), (x[0],), (torch.ones_like(x[0]),))
