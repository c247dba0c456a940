"""The router's load-balancing loss on a B200 against the definition in float64 (bodies and tolerances in
tests/balance_cases.py)."""

import pytest
import torch

import balance_cases as cases

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("layers,tokens,experts,top_k,dtype,pitch", [
    (1, 700, 8, 2, BF16, 0), (3, 3333, 8, 2, FP32, 0), (2, 5000, 16, 4, FP16, 8), (2, 3500, 60, 4, FP16, 0), (1, 4100, 64, 6, BF16, 0),
    (4, 4000, 128, 8, BF16, 0), (2, 1900, 128, 8, FP32, 0), (1, 900, 160, 6, BF16, 0), (3, 900, 256, 8, BF16, 0),
    (1, 600, 257, 9, FP16, 0), (1, 500, 384, 8, FP32, 4), (1, 400, 512, 10, BF16, 0), (1, 300, 1000, 4, FP32, 0),
    (1, 300, 1024, 3, BF16, 0), (1, 3700, 5, 1, BF16, 1), (1, 1200, 32, 32, BF16, 0), (1, 1000, 40, 33, FP32, 0), (2, 70, 2, 1, FP32, 0),
    (40, 257, 96, 8, BF16, 0), (2, 1000, 128, 1, BF16, 0), (2, 1000, 128, 5, FP16, 0), (2, 1000, 128, 16, BF16, 0), (3, 1000, 128, 10, BF16, 0), (2, 700, 256, 12, FP32, 0), (2, 700, 64, 17, BF16, 0),
    (2, 1000, 120, 8, BF16, 8), (2, 1001, 127, 8, BF16, 1)])
def test_matches_definition(layers, tokens, experts, top_k, dtype, pitch):
    cases.case_matches_definition("cuda", cases.make(layers, tokens, experts, dtype), top_k, z=1e-3, pitch=pitch, up=0.5)


@pytest.mark.parametrize("mask_dtype", [torch.bool, torch.uint8, torch.int32, torch.int64, torch.float32])
@pytest.mark.parametrize("experts", [8, 24, 128])
def test_masks(mask_dtype, experts):
    mask = [1] * 50 + [0] * 40 + [1] * 90 + [0] * 90 + [0] * 90
    cases.case_matches_definition("cuda", cases.make(2, 360, experts, BF16), 4, mask=mask, z=0.01, mask_dtype=mask_dtype, leading=(4, 90))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("experts,top_k", [(8, 2), (16, 5), (60, 4), (64, 8), (128, 8), (128, 3), (128, 12), (256, 8), (300, 8)])
def test_ties_and_masked_experts(dtype, experts, top_k):
    cases.case_ties("cuda", dtype, experts, top_k)
    cases.case_masked_experts("cuda", dtype, experts, top_k)


def test_more_layers_than_one_launch_takes():
    cases.case_matches_definition("cuda", cases.make(258, 20, 8, FP32), 2)


def test_empty():
    cases.case_empty("cuda")


def test_views_and_partial_gradients():
    cases.case_views_and_partial_gradients("cuda")


def test_gradient_against_differences():
    cases.case_gradient_against_differences("cuda")


def test_nan_reaches_the_loss():
    cases.case_nan_reaches_the_loss("cuda")


def test_refusals():
    cases.case_refusals("cuda")


@pytest.mark.parametrize("experts", [8, 128])
def test_same_bits_on_another_stream_and_replayed(experts):
    """Two eager runs, a run on a side stream and a captured, replayed forward and backward give the same bits; the graph reads
    the values its inputs hold at replay."""
    import liger_kernel_b200 as lk

    x = [t.cuda().requires_grad_(True) for t in cases.make(3, 2000, experts, BF16)]
    mask = (torch.arange(2000, device="cuda") % 7 != 0).long()

    def step():
        out = lk.liger_load_balancing_loss(tuple(x), experts, 2, mask, return_expert_counts=True)
        return (out.loss.detach(), out.expert_counts) + torch.autograd.grad(out.loss, x)

    first, second = step(), step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        third = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    with torch.no_grad():
        saved = [t.clone() for t in x]
        for t in x:
            t.neg_()
    graph.replay()
    fourth = step()
    torch.cuda.synchronize()
    for a, c in zip(captured, fourth):
        assert torch.equal(a, c)
    with torch.no_grad():
        for t, s in zip(x, saved):
            t.copy_(s)
    graph.replay()
    torch.cuda.synchronize()
    for a, c, d, e in zip(first, second, third, captured):
        assert torch.equal(a, c) and torch.equal(a, d) and torch.equal(a, e)


@pytest.mark.parametrize("tokens,experts", [(16_000_000, 136), (17_000_000, 128)])
def test_offsets_beyond_32_bits(tokens, experts):
    """More than 2^31 logits in a layer, by tiles and without: every expert's count, and the last rows' gradient from the counts."""
    import liger_kernel_b200 as lk

    x = torch.zeros(tokens, experts, dtype=BF16, device="cuda")
    favourite = torch.arange(tokens, device="cuda") % 7 * 3                  # 0, 3, .. 18, then the lowest others
    x.scatter_(1, favourite[:, None], 4.0)
    x.requires_grad_(True)
    out = lk.liger_load_balancing_loss(x, experts, 2, return_expert_counts=True)
    first = torch.bincount(favourite, minlength=experts)
    second = torch.zeros_like(first)
    second[0], second[1] = int((favourite != 0).sum()), int((favourite == 0).sum())
    assert torch.equal(out.expert_counts, first + second)
    (grad,) = torch.autograd.grad(out.loss, (x,), torch.tensor(1e6, device="cuda"))
    rows = slice(tokens - 4, tokens)
    c = out.expert_counts.double()
    a = 1e6 * experts * (c - c.mean()) / tokens ** 2
    p = torch.softmax(x.detach()[rows].double(), -1)
    want = p * (a - (a * p).sum(-1, keepdim=True))
    # probabilities to (64 + 4 d) u with d = 4, bf16 results to half a step
    limit = 2 * (64 + 16) * cases.U * p * (a.abs() + (a.abs() * p).sum(-1, keepdim=True)) + 2.0 ** -8 * 1.01 * want.abs()
    assert bool(((grad[rows].double() - want).abs() <= limit).all())


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("experts,top_k", [(8, 2), (24, 4), (32, 4), (60, 4), (64, 6), (128, 8), (128, 12), (256, 8), (300, 8), (512, 10)])
def test_rows_far_from_zero(dtype, experts, top_k):
    cases.case_far_rows("cuda", dtype, experts, top_k)


def test_counts_out_of_range():
    cases.case_counts_out_of_range("cuda")


def test_forward_mode():
    cases.case_forward_mode("cuda")
