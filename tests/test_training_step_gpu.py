"""The norms, the router's balance loss and the fused head together, as a training step of a small mixture-of-experts decoder uses
them, against the same step in float64; and the mixture-of-experts forward of a Hugging Face model with the balance loss on
this package's operator against the unpatched model."""

import copy

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

EXPERTS, TOP_K, COEF = 12, 3, 0.5


def _step(p, ids, targets, mask, norm1, rms, head, balance):
    x = p["embedding"][ids]
    h = x + norm1(x, p["ln_w"], p["ln_b"]) @ p["a"]
    n1 = rms(h, p["rms_w"])
    r1 = n1 @ p["router1"]
    h = h + torch.tanh(n1 @ p["b"])
    n2 = rms(h, p["rms_w"])
    r2 = n2 @ p["router2"]
    return head(n2.reshape(-1, n2.shape[-1]), p["lm_head"], targets.reshape(-1)) + COEF * balance((r1, r2), mask)


def _balance64(logits, mask):
    x = torch.stack([t.reshape(-1, EXPERTS) for t in logits])[:, mask.reshape(-1) != 0]
    chosen = torch.sort(x, dim=-1, descending=True, stable=True).indices[..., :TOP_K]
    share = F.one_hot(chosen, EXPERTS).sum(-2).double().mean((0, 1))
    return EXPERTS * (share * torch.softmax(x, -1).mean((0, 1))).sum()


def test_step_matches_float64():
    import liger_kernel_b200 as lk

    g = torch.Generator().manual_seed(3)
    hidden, vocab, batch, seq = 72, 515, 5, 33
    p = {"embedding": torch.randn(vocab, hidden, generator=g), "ln_w": 1 + 0.1 * torch.randn(hidden, generator=g),
         "ln_b": 0.1 * torch.randn(hidden, generator=g), "a": torch.randn(hidden, hidden, generator=g) * hidden ** -0.5,
         "rms_w": 0.1 * torch.randn(hidden, generator=g), "b": torch.randn(hidden, hidden, generator=g) * hidden ** -0.5,
         "router1": torch.randn(hidden, EXPERTS, generator=g) * hidden ** -0.5, "router2": torch.randn(hidden, EXPERTS, generator=g) * hidden ** -0.5,
         "lm_head": torch.randn(vocab, hidden, generator=g) * 0.1}
    ids, targets = torch.randint(0, vocab, (2, batch, seq), generator=g)
    mask = (torch.arange(seq) < torch.tensor([33, 20, 0, 1, 31])[:, None]).long()
    targets = torch.where(mask != 0, targets, -100)

    ours = {k: v.cuda().requires_grad_(True) for k, v in p.items()}
    loss = _step(ours, ids.cuda(), targets.cuda(), mask.cuda(), lambda x, w, b: lk.liger_layer_norm(x, w, b, 1e-6),
                 lambda x, w: lk.liger_rms_norm(x, w, 1e-6, offset=1.0), lk.liger_fused_linear_cross_entropy,
                 lambda logits, m: lk.liger_load_balancing_loss(logits, EXPERTS, TOP_K, m))
    loss.backward()

    exact = {k: v.double().requires_grad_(True) for k, v in p.items()}
    want = _step(exact, ids, targets, mask, lambda x, w, b: F.layer_norm(x, (hidden,), w, b, 1e-6),
                 lambda x, w: x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * (1 + w),
                 lambda x, w, t: F.cross_entropy(x @ w.t(), t, ignore_index=-100), _balance64)
    want.backward()
    # The head's gradients in fp32 are good to 2e-5 of their largest entry (three bf16 products per product), its loss to 1e-5;
    # what is passed back goes through two norms and two matrix products whose gains are of order one.  A factor of ten for both.
    loss, want = float(loss.detach()), float(want.detach())
    assert abs(loss - want) <= 1e-4 * want
    for k in p:
        got, ref = ours[k].grad.double().cpu(), exact[k].grad
        assert float((got - ref).abs().max()) <= 2e-4 * float(ref.abs().max()), k


def test_step_trains_with_modules_in_bf16():
    """Modules in a bf16 step: every parameter gets a finite gradient of its own type and shape."""
    import liger_kernel_b200 as lk

    torch.manual_seed(0)
    norm = lk.LigerLayerNorm(64, bias=True).cuda().bfloat16()
    rms = lk.LigerRMSNorm(64).cuda()                                    # fp32 weights beside bf16 rows
    router = torch.nn.Linear(64, 8, bias=False).cuda().bfloat16()
    head = torch.nn.Linear(64, 300, bias=False).cuda().bfloat16()
    x = torch.randn(4, 50, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    h = rms(norm(x))
    out = lk.LigerLoadBalancingLoss(8, 2, lse_square_scale=1e-3, return_z_loss=True, return_expert_counts=True)(router(h))
    loss = lk.LigerFusedLinearCrossEntropyLoss()(head.weight, h.reshape(-1, 64), torch.randint(0, 300, (200,), device="cuda")) + out.loss
    loss.backward()
    assert int(out.expert_counts.sum()) == 400 and float(out.z_loss) > 0
    for t in (x, *norm.parameters(), *rms.parameters(), *router.parameters(), *head.parameters()):
        assert t.grad is not None and t.grad.dtype == t.dtype and t.grad.shape == t.shape and torch.isfinite(t.grad).all()


@pytest.mark.parametrize("padded", [False, True])
def test_mixture_of_experts_forward_uses_the_operator(padded, monkeypatch):
    transformers = pytest.importorskip("transformers")
    import liger_kernel_b200 as lk
    import liger_kernel_b200.transformers.model.causal_lm as causal_lm

    torch.manual_seed(1)
    base = transformers.MixtralForCausalLM(transformers.MixtralConfig(
        hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, vocab_size=515,
        max_position_embeddings=128, num_local_experts=4, num_experts_per_tok=2, output_router_logits=True, router_aux_loss_coef=1.0)).cuda()
    patched = copy.deepcopy(base)
    lk._apply_liger_kernel_to_instance(patched, rope=False, rms_norm=False, swiglu=False)
    calls = []
    monkeypatch.setattr(causal_lm, "liger_load_balancing_loss", lambda *a: calls.append(a) or lk.liger_load_balancing_loss(*a))
    ids = torch.randint(1, 515, (3, 40), device="cuda")
    mask = torch.ones_like(ids)
    if padded:
        mask[1, 25:] = 0
    labels = torch.where(mask != 0, ids, -100)
    outs = []
    for model in (base, patched):
        model.train()
        out = model(input_ids=ids, attention_mask=mask if padded else None, labels=labels)
        out.loss.backward()
        outs.append(out)
    assert len(calls) == 1 and outs[1].logits is None
    # both in fp32 on the same router logits: means over 240 tokens, in another order
    ours, theirs = float(outs[1].aux_loss.detach()), float(outs[0].aux_loss.detach())
    assert abs(ours - theirs) <= 1e-5 * theirs
    ours, theirs = float(outs[1].loss.detach()), float(outs[0].loss.detach())
    assert abs(ours - theirs) <= 1e-4 * theirs
    gates = [(n, p) for n, p in base.named_parameters() if "gate" in n and p.grad is not None and p.dim() == 2 and p.shape[0] == 4]
    assert gates
    patched_parameters = dict(patched.named_parameters())
    for n, p in gates:
        assert float((patched_parameters[n].grad - p.grad).abs().max()) <= 1e-3 * float(p.grad.abs().max()), n
