"""Layer norm and RMSNorm on a B200 against the definition in float64 (bodies and tolerances in tests/norm_cases.py)."""

import pytest
import torch

import norm_cases as cases

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("n,hidden,dtype,wdtype,pitch", [
    (1, 1, FP32, FP32, 0), (3, 2, BF16, BF16, 0), (700, 5, FP16, FP32, 3), (670, 8, BF16, BF16, 0), (400, 24, BF16, FP32, 8),
    (3300, 31, FP16, FP16, 0), (2100, 33, BF16, BF16, 2), (20000, 128, BF16, BF16, 0), (1900, 132, FP32, FP32, 4),
    (1300, 250, FP16, FP16, 6), (1400, 264, BF16, BF16, 16), (1, 4096, BF16, BF16, 0), (900, 1001, FP32, FP32, 0),
    (1024, 1024, FP32, FP32, 0), (1000, 1537, FP16, FP16, 31), (700, 3584, BF16, BF16, 0), (513, 4096, BF16, FP32, 0),
    (500, 4104, FP16, FP16, 8), (400, 5000, FP16, FP16, 1), (700, 8192, BF16, BF16, 0), (200, 9000, FP32, FP32, 0),
    (150, 16384, BF16, BF16, 0), (60, 16384, FP32, FP32, 0), (50, 16383, BF16, BF16, 0), (20, 16387, BF16, BF16, 0),
    (20, 40000, FP16, FP32, 0)])
def test_matches_definition(kind, n, hidden, dtype, wdtype, pitch):
    cases.case_matches_definition("cuda", kind, n, hidden, dtype, wdtype, True, True, 0.0, pitch)


@pytest.mark.parametrize("kind,weight,bias,offset,mode", [
    ("layer", True, False, 1.0, "gemma"), ("layer", False, False, 0.0, "gemma"), ("layer", False, True, 0.0, "gemma"),
    ("rms", True, False, 1.0, "llama"), ("rms", False, False, 0.0, "llama"), ("rms", True, False, 1.0, "gemma")])
@pytest.mark.parametrize("hidden", [27, 40, 336, 777, 8192])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_parameters_and_casting(kind, weight, bias, offset, mode, hidden, dtype):
    cases.case_matches_definition("cuda", kind, 311, hidden, dtype, None, weight, bias, offset, 0, mode)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_gradient_against_differences(kind):
    cases.case_gradient_against_differences("cuda", kind)


@pytest.mark.parametrize("kind", ["layer", "rms"])
def test_special_values_stay_in_their_row(kind):
    cases.case_special_values("cuda", kind)


def test_shapes_and_views():
    cases.case_shapes_and_views("cuda")


def test_refusals():
    cases.case_refusals("cuda")


@pytest.mark.parametrize("hidden", [96, 1000, 4096])
def test_same_bits_on_another_stream_and_replayed(hidden):
    """Two eager runs, a run on a side stream and a captured, replayed forward and backward give the same bits; the graph reads
    the values its inputs hold at replay."""
    import liger_kernel_b200 as lk

    x, w, b, dy = (t.cuda() for t in cases.make(777, hidden, BF16, BF16))
    for t in (x, w, b):
        t.requires_grad_(True)

    def step():
        y = lk.liger_layer_norm(x, w, b, 1e-6)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)

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
        saved = x.clone()
        x.mul_(2.0).add_(0.25)
    graph.replay()
    fourth = step()
    with torch.no_grad():
        x.copy_(saved)
    torch.cuda.synchronize()
    for a, c in zip(captured, fourth):
        assert torch.equal(a, c)
    graph.replay()
    torch.cuda.synchronize()
    for a, c, d, e in zip(first, second, third, captured):
        assert torch.equal(a, c) and torch.equal(a, d) and torch.equal(a, e)


@pytest.mark.parametrize("kind,hidden,rows", [("layer", 4096, 540000), ("rms", 128, 17_000_000), ("layer", 4097, 530000)])
def test_offsets_beyond_32_bits(kind, hidden, rows):
    """More than 2^31 elements, one path each for wide, narrow and unaligned rows: the first and the last rows against the
    definition (they differ from each other: an offset that wraps would show)."""
    import liger_kernel_b200 as lk

    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.empty(rows, hidden, dtype=BF16, device="cuda")
    dy = torch.empty(rows, hidden, dtype=BF16, device="cuda")
    x.zero_()
    dy.zero_()
    some = list(range(5)) + list(range(rows - 5, rows))
    x[some] = torch.randn(10, hidden, generator=g, device="cuda").to(BF16)
    dy[some] = torch.randn(10, hidden, generator=g, device="cuda").to(BF16)
    w = (1 + 0.1 * torch.randn(hidden, generator=g, device="cuda")).to(BF16)
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = lk.liger_layer_norm(x, w, None, 1e-6) if kind == "layer" else lk.liger_rms_norm(x, w, 1e-6, casting_mode="gemma")
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    ref = cases.reference(x.detach()[some].cpu(), w.detach().cpu(), None, dy[some].cpu(), 1e-6, 0.0, kind == "layer")
    cases.compare("y", y.detach()[some], ref["y"], ref["tol"]["y"])
    cases.compare("dx", dx[some], ref["dx"], ref["tol"]["dx"])
    cases.compare("dw", dw, ref["dw"], ref["tol"]["dw"])          # all other rows are zero: they add nothing
    assert not y.detach()[5:-5:9973].any() and not dx[5:-5:9973].any()


def test_autograd():
    cases.case_autograd("cuda")


def test_two_streams_at_once():
    """Norms and balance losses under way on two streams at the same time do not touch each other's scratch."""
    import liger_kernel_b200 as lk

    def inputs(seed):
        x, w, b, dy = (t.cuda() for t in cases.make(3000, 2048, BF16, BF16, seed=seed))
        logits = tuple(t.requires_grad_(True) for t in torch.randn(4, 3000, 64, generator=torch.Generator().manual_seed(seed)).to(BF16).cuda())
        return [t.requires_grad_(True) for t in (x, w, b)], dy, logits

    def step(leaves, dy, logits):
        y = lk.liger_layer_norm(*leaves, 1e-6)
        out = lk.liger_load_balancing_loss(logits, 64, 4, return_expert_counts=True)
        return [y.detach(), out.loss.detach(), out.expert_counts, *torch.autograd.grad(y, leaves, dy), *torch.autograd.grad(out.loss, logits)]

    data = [inputs(1), inputs(2)]
    want = [step(*d) for d in data]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k] = step(*data[k])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_forward_mode():
    cases.case_forward_mode("cuda")
