"""What is measured of the norms and of the router's balance loss: cases, inputs, plain forms, the framework's calls.

Three operators of a training step around the language-model head:

* layer norm over the rows of ``[rows, hidden]``, forward and backward, weight and bias optional;
* RMSNorm over the same rows, weight ``offset + w``, everything in 32 bits and one rounding ("gemma" casting);
* the load-balancing loss of a mixture-of-experts router over the logits of all layers, with the number of tokens that
  each expert of each layer was chosen by, and the gradient of every layer's logits.

``run`` computes them in elementary torch operations, or, with ``own`` set, through ``liger_kernel_b200``.
"""

import math
import os
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_package = None


def _lk():
    global _package
    if _package is None:
        path = os.path.join(_ROOT, "liger-kernel_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import liger_kernel_b200

        _package = liger_kernel_b200
    return _package


# ---------------------------------------------------------------------------------------------------------------- cases
def _norm(name, op, rows, hidden, dtype, wdtype, train, weight=True, bias=False, offset=0.0, pitch=0):
    """pitch: elements from one row of x to the next beyond `hidden` (0: dense)."""
    return {"name": name, "op": op, "rows": rows, "hidden": hidden, "dtype": dtype, "wdtype": wdtype, "train": train,
            "weight": weight, "bias": bias, "offset": offset, "pitch": pitch}


def _balance(name, layers, batch, seq, experts, top_k, dtype, train, masked, z=0.0):
    return {"name": name, "op": "balance", "layers": layers, "batch": batch, "seq": seq, "experts": experts, "top_k": top_k,
            "dtype": dtype, "train": train, "masked": masked, "z": z}


def listed():
    return [
        # one training step's norm in front of the Llama-3-8B head (8 sequences of 4096 tokens, hidden size 4096)
        _norm("layer_norm_train_8b", "layer_norm", 32768, 4096, "bf16", "bf16", True, bias=True),
        # the 70B head's hidden size, master weights in fp32, weight stored as its distance from one
        _norm("layer_norm_train_70b", "layer_norm", 8192, 8192, "bf16", "fp32", True, bias=True, offset=1.0),
        # ragged packed batch of an encoder-like block, rows of odd length in a wider buffer
        _norm("layer_norm_train_odd", "layer_norm", 10007, 1537, "fp16", "fp16", True, bias=True, pitch=31),
        # narrow rows, many of them: a norm over each attention head's 128 elements
        _norm("layer_norm_train_heads", "layer_norm", 262144, 128, "bf16", "bf16", True),
        # evaluation of a short prompt, no parameters: where the call's latency counts
        _norm("layer_norm_eval_small", "layer_norm", 64, 1024, "fp32", "fp32", False, weight=False),
        # the norm of the Gemma-2-9B configuration (4 sequences of 4096 tokens, hidden size 3584, weight 1 + w)
        _norm("rms_norm_train_9b", "rms_norm", 16384, 3584, "bf16", "bf16", True, offset=1.0),
        # the small fp32 configuration (2 sequences of 512 tokens, hidden size 1024)
        _norm("rms_norm_train_fp32", "rms_norm", 1024, 1024, "fp32", "fp32", True),
        # one new token of the 70B width
        _norm("rms_norm_eval_token", "rms_norm", 1, 8192, "bf16", "bf16", False),
        # every layer's router of a wide mixture of experts, padded batch
        _balance("balance_train_wide", 48, 4, 4096, 128, 8, "bf16", True, True),
        # eight experts, two per token, routers in fp32
        _balance("balance_train_eight", 32, 8, 4096, 8, 2, "fp32", True, False),
        # an expert count that fills no vector, an odd number of tokens, padding, and the penalty on the log-sum-exp
        _balance("balance_train_odd", 5, 3, 1367, 60, 4, "fp16", True, True, 1e-3),
        # counts and loss of one layer's router for a short batch
        _balance("balance_eval_small", 1, 2, 32, 32, 4, "bf16", False, False),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over the logarithm; half of the time a round one."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.5:
        step = 1 << max(0, n.bit_length() - 3)
        n = n // step * step
    return min(high, max(low, n))


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if rng.random() < 0.6:
        op = rng.choice(["layer_norm", "rms_norm"])
        # from 16 elements: in rows of a few the gradient is what is left of nearly equal terms, in any arithmetic
        hidden = _spread(rng, 16, 16384)
        rows = _spread(rng, 1, min(262144, 32768 * 4096 // hidden // (2 if dtype == "fp32" else 1)))
        weight = op == "rms_norm" or rng.random() < 0.85
        return {"op": op, "rows": rows, "hidden": hidden, "dtype": dtype, "wdtype": rng.choice([dtype, "fp32"]),
                "train": rng.random() < 0.75, "weight": weight, "bias": op == "layer_norm" and weight and rng.random() < 0.7,
                "offset": rng.choice([0.0, 1.0]), "pitch": rng.choice([0, 0, 0, 5, 64])}
    # fewer chosen than half of the experts and some tokens at least: equal counts leave a gradient of zero
    experts = _spread(rng, 8, 512)
    top_k = min(experts // 2, rng.choice([1, 2, 4, 6, 8, 8, 10]))
    layers = _spread(rng, 1, 48)
    batch = rng.randint(1, 8)
    seq = _spread(rng, 16, min(4096, 96 * 1024 * 1024 // (experts * layers * batch)))
    return {"op": "balance", "layers": layers, "batch": batch, "seq": seq, "experts": experts, "top_k": top_k, "dtype": dtype,
            "train": rng.random() < 0.75, "masked": rng.random() < 0.5, "z": rng.choice([0.0, 1e-3])}


# --------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = _TYPES[case["dtype"]]
    train = case["train"]
    if case["op"] == "balance":
        return _prepare_balance(case, g, dtype, train)
    rows, hidden = case["rows"], case["hidden"]
    # hidden states: a few channels far larger than the others, rows of different scale and a mean that is not zero
    channel = torch.rand(hidden, generator=g, device="cuda")
    scale = torch.where(channel > 0.995, 20.0, 1.0)
    x = torch.empty((rows, hidden + case["pitch"]), dtype=dtype, device="cuda")[:, :hidden]
    row_scale = torch.exp(torch.randn((rows, 1), generator=g, device="cuda") * 0.3)
    x.copy_((torch.randn((rows, hidden), generator=g, device="cuda") * scale + 0.1) * row_scale)
    wdtype = _TYPES[case["wdtype"]]
    w = b = None
    if case["weight"]:
        w = (torch.randn(hidden, generator=g, device="cuda") * 0.1 + 1.0 - case["offset"]).to(wdtype)
    if case["bias"]:
        b = (torch.randn(hidden, generator=g, device="cuda") * 0.1).to(wdtype)
    dy = (torch.randn((rows, hidden), generator=g, device="cuda") * 0.05).to(dtype) if train else None
    leaves = [t.requires_grad_(train) for t in (x, w, b) if t is not None]
    return {"op": case["op"], "x": x, "w": w, "b": b, "dy": dy, "leaves": leaves, "train": train, "offset": case["offset"], "eps": 1e-6}


def _prepare_balance(case, g, dtype, train):
    layers, batch, seq, experts = (case[k] for k in ("layers", "batch", "seq", "experts"))
    tokens = batch * seq
    # routers prefer some experts: a bias per expert and layer under the tokens' own spread
    bias = torch.randn((layers, 1, experts), generator=g, device="cuda") * 0.7
    x = (torch.randn((layers, tokens, experts), generator=g, device="cuda") * 1.5 + bias).to(dtype)
    logits = tuple(t.clone().requires_grad_(train) for t in x.unbind(0))
    mask = None
    if case["masked"]:
        length = torch.randint(0, seq + 1, (batch, 1), generator=g, device="cuda")
        length[0] = seq                                     # the longest sequence has no padding
        mask = (torch.arange(seq, device="cuda") < length).to(torch.int64)
    # training in fp16 scales its loss, or the gradients of a mean over many tokens vanish
    go = torch.tensor(16384.0 if dtype == torch.float16 else 1.0, device="cuda")
    return {"op": "balance", "logits": logits, "mask": mask, "experts": experts, "top_k": case["top_k"], "train": train,
            "z": case["z"], "go": go}


# ------------------------------------------------------------------------------------------------------------------ run
def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "balance":
        return _balance_plain(state)
    with torch.no_grad():
        return _norm_plain(state)


def _run_own(s):
    lk = _lk()
    if s["op"] == "balance":
        out = lk.liger_load_balancing_loss(s["logits"], s["experts"], s["top_k"], s["mask"], lse_square_scale=s["z"],
                                           return_expert_counts=True)
        result = {"loss": out.loss, "counts": out.expert_counts}
        if s["train"]:
            result["grads"] = list(torch.autograd.grad(out.loss, s["logits"], s["go"]))
        return result
    if s["op"] == "layer_norm":
        y = lk.liger_layer_norm(s["x"], s["w"], s["b"], s["eps"], offset=s["offset"])
    else:
        y = lk.liger_rms_norm(s["x"], s["w"], s["eps"], offset=s["offset"], casting_mode="gemma")
    result = {"y": y}
    if s["train"]:
        result["grads"] = list(torch.autograd.grad(y, s["leaves"], s["dy"]))
    return result


def _norm_plain(s):
    x, w, b, dy = s["x"], s["w"], s["b"], s["dy"]
    xf = x.float()
    if s["op"] == "layer_norm":
        xf = xf - xf.mean(-1, keepdim=True)
    rstd = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + s["eps"])
    xhat = xf * rstd
    y = xhat
    if w is not None:
        gain = w.float() + s["offset"]
        y = y * gain
    if b is not None:
        y = y + b.float()
    result = {"y": y.to(x.dtype)}
    if s["train"]:
        dyf = dy.float()
        m = dyf if w is None else dyf * gain
        dx = m - xhat * (m * xhat).mean(-1, keepdim=True)
        if s["op"] == "layer_norm":
            dx = dx - m.mean(-1, keepdim=True)
        grads = [(dx * rstd).to(x.dtype)]
        if w is not None:
            grads.append((dyf * xhat).sum(0).to(w.dtype))
        if b is not None:
            grads.append(dyf.sum(0).to(b.dtype))
        result["grads"] = grads
    return result


def _balance_plain(s):
    with torch.no_grad():
        x = torch.stack(s["logits"])                        # [layers, tokens, experts]
        layers, tokens, experts = x.shape
        k = s["top_k"]
        xf = x.float()
        chosen = torch.sort(xf, dim=-1, descending=True, stable=True).indices[..., :k]
        keep = torch.ones(tokens, dtype=torch.bool, device=x.device) if s["mask"] is None else s["mask"].reshape(-1) != 0
        weight = keep.to(torch.int64).view(1, tokens, 1).expand(layers, tokens, k)
        counts = torch.zeros((layers, experts), dtype=torch.int64, device=x.device)
        counts.scatter_add_(1, chosen.reshape(layers, -1), weight.reshape(layers, -1))
        n = keep.sum().double() * layers
        top = xf.max(-1, keepdim=True).values
        e = torch.exp(xf - top)
        total = e.sum(-1, keepdim=True)
        p = e / total
        lse = (top + torch.log(total))[..., 0]
        kept = keep.view(1, tokens, 1)
        mass = torch.where(kept, p, 0.0).sum((0, 1), dtype=torch.float64)
        per_expert = counts.sum(0).double()
        loss = experts * (per_expert * mass).sum() / (n * n)
        if s["z"]:
            loss = loss + s["z"] * torch.where(keep, lse * lse, 0.0).sum(dtype=torch.float64) / n
        result = {"loss": loss.float(), "counts": counts}
        if s["train"]:
            # a shift of all coefficients changes nothing, as the probabilities of a row sum to one: take the mean out
            a = (s["go"].double() * experts * (per_expert - per_expert.mean()) / (n * n)).float()
            grad = p * (a - (p * a).sum(-1, keepdim=True))
            if s["z"]:
                grad = grad + p * (lse.unsqueeze(-1) * (s["go"].double() * 2.0 * s["z"] / n).float())
            result["grads"] = list(torch.where(kept, grad, 0.0).to(x.dtype).unbind(0))
        return result


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] == "balance":
        n = case["layers"] * case["batch"] * case["seq"] * case["experts"]
        moved = n * size * (2 if case["train"] else 1) + 8 * case["layers"] * case["experts"] + 4
        moved += 8 * case["batch"] * case["seq"] if case["masked"] else 0
        return {"bytes": moved, "flops": n * (12 if case["train"] else 6)}
    n = case["rows"] * case["hidden"]
    parameters = (int(case["weight"]) + int(case["bias"])) * case["hidden"] * _BYTES[case["wdtype"]]
    sides = 2 if case["train"] else 1
    return {"bytes": sides * (2 * n * size + parameters), "flops": n * (20 if case["train"] else 8)}


# ---------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The operators' definitions in 64 bits, gradients by automatic differentiation of the loss's own definition."""
    s = prepare(case, seed)
    if case["op"] == "balance":
        return _exact_balance(s)
    x = s["x"].detach().double().requires_grad_(s["train"])
    w = None if s["w"] is None else s["w"].detach().double().requires_grad_(s["train"])
    b = None if s["b"] is None else s["b"].detach().double().requires_grad_(s["train"])
    if s["op"] == "layer_norm":
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + s["eps"])
    else:
        y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + s["eps"])
    if w is not None:
        y = y * (s["offset"] + w)
    if b is not None:
        y = y + b
    out = {"y": y.detach()}
    if s["train"]:
        out["grads"] = list(torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], s["dy"].double()))
    return out


def _exact_balance(s):
    x = torch.stack([t.detach().double() for t in s["logits"]]).requires_grad_(s["train"])
    layers, tokens, experts = x.shape
    kept = torch.ones(tokens, dtype=torch.bool, device=x.device) if s["mask"] is None else s["mask"].flatten().bool()
    with torch.no_grad():
        # round by round, the largest logit that is left; the first of several
        left, counts = x.detach()[:, kept].clone(), torch.zeros((layers, experts), dtype=torch.int64, device=x.device)
        place = torch.arange(experts, device=x.device)
        for _ in range(s["top_k"]):
            best = torch.where(left == left.max(-1, keepdim=True).values, place, experts).min(-1, keepdim=True).values
            counts += (place == best).sum(1)
            left.scatter_(2, best, -math.inf)
    logits = x[:, kept]
    n = logits.shape[0] * logits.shape[1]
    fraction = counts.sum(0).double() / n
    loss = experts * (fraction * torch.softmax(logits, -1).mean((0, 1))).sum()
    if s["z"]:
        loss = loss + s["z"] * torch.logsumexp(logits, -1).square().mean()
    out = {"loss": loss.detach(), "counts": counts}
    if s["train"]:
        out["grads"] = list(torch.autograd.grad(loss, x, s["go"].double())[0].unbind(0))
    return out
