"""Which function the mixture-of-experts forwards take their router's auxiliary loss from: this package's operator for plain logits on
the GPU, the model library's for everything that the operator would refuse or define otherwise, with the library's results.
Logits on the CPU stand in for those on the GPU; the operator's library is emulated."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import train_ops_emu

mixtral = pytest.importorskip("transformers.models.mixtral.modeling_mixtral")

E, K, B, S = 8, 2, 3, 5


@pytest.fixture
def calls(monkeypatch):
    import liger_kernel_b200 as lk
    import liger_kernel_b200.transformers.model.causal_lm as causal_lm

    seen = []
    monkeypatch.setattr(causal_lm, "_on_gpu", lambda t: True)
    monkeypatch.setattr(causal_lm, "liger_load_balancing_loss", lambda *a: seen.append(a) or lk.liger_load_balancing_loss(*a))
    with train_ops_emu.installed():
        yield seen


def _logits(layers=2, dtype=torch.float32):
    g = torch.Generator().manual_seed(4)
    return tuple(torch.randn(B * S, E, generator=g).to(dtype) for _ in range(layers))


def _loss(*args):
    from liger_kernel_b200.transformers.model.causal_lm import router_balancing_loss

    return router_balancing_loss(*args)


def _mask():
    m = torch.ones(B, S, dtype=torch.int64)
    m[1, 3:] = 0
    return m


@pytest.mark.parametrize("mask", [None, _mask(), _mask().bool(), _mask().int()], ids=["none", "int64", "bool", "int32"])
def test_plain_logits_take_the_operator(calls, mask):
    x = _logits()
    got, want = _loss(x, E, K, mask), mixtral.load_balancing_loss_func(x, E, K, None if mask is None else mask.long())
    # sums of 30 probabilities and of a row of 8, in fp32 on both sides: below 128 roundings each
    assert len(calls) == 1 and abs(float(got) - float(want)) <= 2 * 128 * 2.0 ** -24 * float(want)


def _library_cases():
    ragged = (_logits()[0], _logits()[1][:4])
    mixed = (_logits()[0], _logits()[1].bfloat16())
    weights = _mask().float()
    weights[0, 1], weights[2, 2] = 0.25, 3.0
    return {"float mask": (_logits(), E, K, weights), "layers of other lengths": (ragged, E, K), "layers of other types": (mixed, E, K),
            "one tensor per sequence": (tuple(t.view(B, S, E) for t in _logits()), E, 1), "not a tuple": (list(_logits()), E, K),
            "nothing": (None, E, K), "fp64": (_logits(dtype=torch.float64), E, K)}


@pytest.mark.parametrize("name", _library_cases())
def test_the_rest_keeps_the_library_function(calls, name):
    args = _library_cases()[name]
    got, want = _loss(*args), mixtral.load_balancing_loss_func(*args)
    assert not calls and type(got) is type(want) and (got == want if isinstance(want, int) else torch.equal(got, want))


def test_forward_mode_and_transforms_keep_the_library_function(calls):
    x = _logits()
    t = tuple(torch.ones_like(v) * (i + 1) * torch.arange(E) for i, v in enumerate(x))
    with forward_ad.dual_level():
        duals = tuple(forward_ad.make_dual(a, b) for a, b in zip(x, t))
        want = forward_ad.unpack_dual(mixtral.load_balancing_loss_func(duals, E, K)).tangent
        assert torch.equal(forward_ad.unpack_dual(_loss(duals, E, K)).tangent, want)
    stacked = torch.stack(x)
    want = torch.vmap(lambda v: mixtral.load_balancing_loss_func((v,), E, K))(stacked)
    assert torch.equal(torch.vmap(lambda v: _loss((v,), E, K))(stacked), want)
    second = [torch.func.hessian(lambda v: f((v,), E, K))(x[0][:3]) for f in (_loss, mixtral.load_balancing_loss_func)]
    assert torch.equal(*second) and second[0].any() and not calls


def test_distributed_tensors_keep_the_library_function(calls):
    import torch.distributed as dist
    from torch.distributed.device_mesh import init_device_mesh
    from torch.distributed.tensor import DTensor, Replicate

    dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    try:
        mesh = init_device_mesh("cpu", (1,))
        x = _logits()
        d = tuple(DTensor.from_local(t, mesh, [Replicate()], run_check=False) for t in x)
        want = mixtral.load_balancing_loss_func(x, E, K)
        assert torch.equal(_loss(d, E, K).to_local(), want) and not calls
    finally:
        dist.destroy_process_group()
