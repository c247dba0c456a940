"""Shared bodies of the tests that trace, compile and transform the norms and the router's balance loss: what the tracers record, and
what torch.func's transforms compute, has to be what the operators compute when they are called.  Run on a B200
(tests/test_tracing_gpu.py) and, with the library's host side and kernels emulated, on CPU tensors
(tests/test_tracing_emulation_cpu.py).  The same kernels run on the same rows either way: results agree bit for bit, unless
the rows are grouped differently (vmap calls once per slice), where only sums over the rows move by roundings."""

import torch
from torch.fx.experimental.proxy_tensor import make_fx

EXPERTS, TOP_K = 24, 3


def _operators():
    import liger_kernel_b200 as lk

    return {
        "layer": lambda x, w, b: lk.liger_layer_norm(x, w, b, 1e-6),
        "rms": lambda x, w, b: lk.liger_rms_norm(x, w, 1e-6) + b,
        "balance": lambda x, w, b: lk.liger_load_balancing_loss((x, x * w + b), EXPERTS, TOP_K, lse_square_scale=1e-3),
    }


def _inputs(device, rows, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(rows, EXPERTS, generator=g).to(dtype).to(device)] + [torch.randn(EXPERTS, generator=g).to(dtype).to(device) for _ in range(2)]


def _gradients(f, args, allow_unused=False):
    args = [t.detach().clone().requires_grad_(True) for t in args]
    y = f(*args)
    up = torch.linspace(0.5, 1.5, y.numel(), device=y.device).reshape(y.shape).to(y.dtype)
    return y.detach(), torch.autograd.grad(y, args, up, allow_unused=allow_unused)


def case_make_fx(device, name, mode):
    """The traced program, run on other inputs, forward and backward."""
    f = _operators()[name]
    first, second = _inputs(device, 10, 1), _inputs(device, 10, 2)
    forward = make_fx(f, tracing_mode=mode)(*first)
    assert torch.equal(forward(*second), f(*second))
    assert not torch.equal(forward(*second), f(*first))

    def step(x, w, b):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = f(*leaves)
        return (y.detach(), *torch.autograd.grad(y.sum(), leaves))

    traced = make_fx(step, tracing_mode=mode)(*first)
    for got, want in zip(traced(*second), step(*second)):
        assert got.shape == want.shape and got.dtype == want.dtype and torch.equal(got, want)


def case_make_fx_of_a_bare_norm(device):
    """Without parameters, where the graph has nothing but the operator in it."""
    import liger_kernel_b200 as lk

    for f in (lambda x: lk.liger_layer_norm(x), lambda x: lk.liger_rms_norm(x), lambda x: lk.liger_load_balancing_loss(x, EXPERTS)):
        a, b = (_inputs(device, 5, s)[0] for s in (3, 4))
        assert torch.equal(make_fx(f)(a)(b), f(b))


def case_compile(device, name, backend="aot_eager"):
    """One graph, forward and backward, also where the number of rows is symbolic."""
    f = _operators()[name]
    torch._dynamo.reset()
    compiled = torch.compile(f, backend=backend, fullgraph=True)
    for rows in (10, 13, 7):                       # the second size makes the number of rows symbolic
        args = _inputs(device, rows, rows)
        (y, grads), (want, want_grads) = _gradients(compiled, args), _gradients(f, args)
        assert torch.equal(y, want) and all(torch.equal(p, q) for p, q in zip(grads, want_grads))
    with torch.no_grad():
        assert torch.equal(compiled(*_inputs(device, 10, 5)), f(*_inputs(device, 10, 5)))
    torch._dynamo.reset()


def case_compile_modules(device, backend="aot_eager"):
    """The modules inside a model, in the rows' type and with fp32 parameters beside bf16 rows, with a mask and all outputs."""
    import liger_kernel_b200 as lk

    torch._dynamo.reset()
    torch.manual_seed(0)

    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.norm, self.rms = lk.LigerLayerNorm(EXPERTS, bias=True), lk.LigerRMSNorm(EXPERTS, offset=1.0)
            self.bare = lk.LigerRMSNorm(EXPERTS, elementwise_affine=False, casting_mode="gemma")
            self.balance = lk.LigerLoadBalancingLoss(EXPERTS, TOP_K, lse_square_scale=1e-2, return_z_loss=True, return_expert_counts=True)

        def forward(self, x, mask):
            h = self.bare(self.rms(self.norm(x)))
            out = self.balance((h, h * 0.5), mask)
            return h, out.loss, out.z_loss, out.expert_counts

    for dtype in (torch.float32, torch.bfloat16):
        block = Block().to(device)
        compiled = torch.compile(block, backend=backend, fullgraph=True)
        x = _inputs(device, 12, 8, dtype)[0].reshape(3, 4, EXPERTS)
        mask = torch.ones(3, 4, dtype=torch.int64, device=device)
        mask[1, 2:] = 0
        results = []
        for fn in (block, compiled):
            xx = x.clone().requires_grad_(True)
            block.zero_grad()
            h, loss, z_loss, counts = fn(xx, mask)
            assert counts.dtype == torch.int64 and not z_loss.requires_grad
            (loss + h.float().square().sum()).backward()
            results.append([h.detach(), loss.detach(), z_loss, counts, xx.grad, *[p.grad for p in block.parameters()]])
        for got, want in zip(results[1], results[0]):
            assert got.dtype == want.dtype and torch.equal(got, want)
    torch._dynamo.reset()


def case_meta(device):
    """Shapes and types without data."""
    import liger_kernel_b200 as lk

    x = torch.empty(2, 5, EXPERTS, device="meta", dtype=torch.bfloat16, requires_grad=True)
    w = torch.empty(EXPERTS, device="meta", requires_grad=True)
    for y in (lk.liger_layer_norm(x, w, w), lk.liger_rms_norm(x, w)):
        assert y.device.type == "meta" and y.shape == x.shape and y.dtype == x.dtype
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == x.shape and dx.dtype == x.dtype and dw.shape == w.shape and dw.dtype == w.dtype
    out = lk.liger_load_balancing_loss((x, x), EXPERTS, TOP_K, return_expert_counts=True)
    assert out.loss.shape == () and out.loss.dtype == torch.float32 and out.expert_counts.shape == (2, EXPERTS)
    (dx,) = torch.autograd.grad(out.loss, (x,))
    assert dx.shape == x.shape and dx.dtype == x.dtype


def case_functional_gradients(device, name):
    """torch.func.grad and vjp, and several upstream gradients at once."""
    f = _operators()[name]
    args = _inputs(device, 6, 11)
    y, want = _gradients(f, args)
    up = torch.linspace(0.5, 1.5, y.numel(), device=y.device).reshape(y.shape)
    out, pull = torch.func.vjp(f, *args)
    assert torch.equal(out, y) and all(torch.equal(p, q) for p, q in zip(pull(up), want))
    grads = torch.func.grad(lambda *a: (f(*a) * up).sum(), argnums=(0, 1, 2))(*args)
    assert all(torch.equal(p, q) for p, q in zip(grads, want))
    if name != "balance":                          # torch's loop for operators without a batching rule takes no lists of tensors
        leaves = [t.clone().requires_grad_(True) for t in args]
        y = f(*leaves)
        ups = torch.stack([up, 2 * up, -up])
        batched = torch.autograd.grad(y, leaves, ups, is_grads_batched=True)
        for got, ref in zip(batched, want):
            for k, scale in enumerate((1.0, 2.0, -1.0)):
                assert torch.equal(got[k], ref * scale)          # multiplying by a power of two commutes with every rounding
        stacked = torch.stack(_inputs(device, 6, 12)[:1] + args[:1])
        assert torch.equal(torch.vmap(f, in_dims=(0, None, None))(stacked, *args[1:]), torch.stack([f(t, *args[1:]) for t in stacked]))


def case_second_derivative_is_refused(device):
    import pytest

    for name, f in _operators().items():
        args = _inputs(device, 6, 11)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            torch.func.grad(lambda x: torch.func.grad(lambda t: f(t, *args[1:]).square().sum())(x).sum())(args[0])


def case_outputs_are_as_described(device):
    """What the launching operators return against what tracers are told: shapes, types, strides, storage, alignment.  A compiled graph
    takes an operator's results for tensors of their own that start on 16-byte boundaries; the gradients of several layers in one
    buffer are cut from it where the compiler sees it."""
    op = torch.ops.liger_b200
    x, w, b = _inputs(device, 7, 1)
    y, statistics = op._norm_with_statistics(x, w, b, 0, 1e-6, 0.0, False)
    checks = ("test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_dynamic")
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    torch.library.opcheck(op.norm.default, (*leaves, 0, 1e-6, 0.0, False), test_utils=checks)
    torch.library.opcheck(op.norm.default, (x, None, None, 1, 1e-6, 0.0, True), test_utils=checks)
    torch.library.opcheck(op._norm_with_statistics.default, (*leaves, 0, 1e-6, 0.0, False), test_utils=checks)
    torch.library.opcheck(op._norm_backward.default, (y, x, w, b, statistics, 0, 1e-6, 0.0, False, True, False), test_utils=checks)
    up, coefficients = torch.ones((), device=device), torch.ones(61, device=device)
    for dtype, rows in ((torch.float32, 7), (torch.float16, 5)):          # 5 x 60 x 2 bytes are no whole vectors
        logits = [torch.randn(rows, 60, device=device).to(dtype) for _ in range(3)]
        for given in (logits, [logits[0], *(t.clone().requires_grad_(True) for t in logits[1:])]):
            torch.library.opcheck(op._load_balancing_loss.default, (given, 60, 4, None, 1e-3), test_utils=checks)
        torch.library.opcheck(op._load_balancing_loss_backward.default, (up, logits, None, coefficients, 60, 4, 0.0), test_utils=checks)
        for t in (*op._load_balancing_loss(logits, 60, 4, None, 0.0), op._load_balancing_loss_backward(up, logits, None, coefficients, 60, 4, 0.0)):
            assert t.numel() == 1 or t.data_ptr() % 16 == 0
        traced = make_fx(lambda *t: torch.autograd.grad(op.load_balancing_loss([v.requires_grad_(True) for v in t], 60, 4, None, 0.0)[0], t))(
            *[t.clone() for t in logits])
        assert any(n.target is op._load_balancing_loss_backward.default for n in traced.graph.nodes)
        want = [t.clone().requires_grad_(True) for t in logits]
        want = torch.autograd.grad(op.load_balancing_loss(want, 60, 4, None, 0.0)[0], want)
        for got, ref in zip(traced(*logits), want):
            assert got.shape == ref.shape == (rows, 60) and torch.equal(got, ref)


def case_plain_calls_take_the_short_way(device):
    """Without a tracer the loss and the layers' gradients are cut from their buffers without further operators."""
    import liger_kernel_b200 as lk

    logits = [t.requires_grad_(True) for t in torch.randn(3, 6, EXPERTS).to(device)]
    loss = lk.liger_load_balancing_loss(tuple(logits), EXPERTS)
    assert loss.grad_fn.name() == "LigerLoadBalancingLossBackward" and not loss._is_view()
    grads = torch.autograd.grad(loss, logits)
    assert not any(g._is_view() for g in grads)
    assert [g.storage_offset() for g in grads] == [i * 6 * EXPERTS for i in range(3)]
    with torch.autocast(device):
        assert lk.liger_load_balancing_loss(logits[0], EXPERTS).grad_fn.name() == "LigerLoadBalancingLossBackward"


def case_lazy_negatives(device):
    """Tensors whose negation is still pending (torch's views of a conjugate's imaginary part) count with their values, as inputs, as
    parameters and as upstream gradients."""
    import liger_kernel_b200 as lk

    def pending(t):
        lazy = torch.complex(torch.zeros_like(t), -t).conj().imag
        assert lazy.is_neg() and torch.equal(lazy, t)
        return lazy

    x, w, b = _inputs(device, 6, 13)
    for name, f in _operators().items():
        assert torch.equal(f(pending(x), pending(w), pending(b)), f(x, w, b)), name
        lazy, plain = pending(x).requires_grad_(True), x.clone().requires_grad_(True)
        up = torch.rand_like(f(x, w, b))
        (got,), (want,) = (torch.autograd.grad(f(t, w, b), t, u) for t, u in ((lazy, pending(up)), (plain, up)))
        assert torch.equal(got, want), name
    assert torch.equal(lk.liger_load_balancing_loss((x, pending(x)), EXPERTS), lk.liger_load_balancing_loss((x, x), EXPERTS))


def case_forward_over_reverse(device):
    """A tangent that only the upstream gradient carries is refused as well: the input's gradient would lose it."""
    import pytest
    import torch.autograd.forward_ad as fa

    for f in _operators().values():
        x, w, b = _inputs(device, 4, 21)
        x.requires_grad_(True)
        y = f(x, w, b)
        with fa.dual_level():
            up = fa.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(NotImplementedError, match="forward"):
                torch.autograd.grad(y, x, up, retain_graph=True)
        torch.autograd.grad(y, x, torch.ones_like(y))


def case_operators_check_what_belongs_together(device):
    """The launching operators by themselves: a gradient, statistics or coefficients that do not fit the input are refused before a
    kernel reads them; what fits but lies otherwise in memory is taken."""
    import pytest

    op = torch.ops.liger_b200
    x, w, b = _inputs(device, 6, 31)
    y, stats = op._norm_with_statistics(x, w, b, 0, 1e-6, 0.0, False)

    def backward(grad=y, statistics=stats, kind=0, need_weight=True, need_bias=True, weight=w, bias=b):
        return op._norm_backward(grad, x, weight, bias, statistics, kind, 1e-6, 0.0, False, need_weight, need_bias)

    want = backward()
    for grad in (y[:5], y[:, :12], y.reshape(12, 12), y.reshape(2, 3, EXPERTS), y.half(), torch.ones((), device=device)):
        with pytest.raises(ValueError, match="gradient"):
            backward(grad)
    for statistics in (stats[:1], stats[:, :5], stats.t(), stats.reshape(-1), stats.half(), stats.double()):
        with pytest.raises(ValueError, match="statistics"):
            backward(statistics=statistics)
    with pytest.raises(ValueError, match="statistics"):
        backward(kind=1, bias=None, need_bias=False)                       # RMSNorm has one row of them
    for missing in (dict(weight=None), dict(bias=None)):
        with pytest.raises(ValueError, match="gradient of a parameter"):
            backward(**missing)
    for got, ref in zip(backward(y.t().contiguous().t(), stats.t().contiguous().t()), want):
        assert torch.equal(got, ref)

    logits = [x, y]
    values, counts = op._load_balancing_loss(logits, EXPERTS, TOP_K, None, 0.0)

    def balance_backward(grad=torch.ones((), device=device), v=values):
        return op._load_balancing_loss_backward(grad, logits, None, v, EXPERTS, TOP_K, 0.0)

    want = balance_backward()
    assert want.shape == (2, 6, EXPERTS) and torch.equal(balance_backward(v=torch.stack([values, values]).t()[:, 0]), want)
    for v in (values[:EXPERTS], values.half(), values[None], values[:0]):
        with pytest.raises(ValueError, match="coefficients"):
            balance_backward(v=v)
    for grad in (torch.ones(2, device=device), torch.ones(0, device=device)):
        with pytest.raises(ValueError, match="gradient"):
            balance_backward(grad)
