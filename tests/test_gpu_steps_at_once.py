"""Training steps of experts, router and adapters that run at the same time: streams, host threads, captured graphs."""
import threading

import pytest
import torch

from flydsl_b200.kernels.grouped_gemm import grouped_linear
from flydsl_b200.kernels.lora import lora_add
from flydsl_b200.kernels.moe_routing import moe_combine, moe_permute, route_rows, topk_gating

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def adapters(rows, count, mixed, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(dtype)

    y, x, a, b, dout = r(rows, 264), r(rows, 136).requires_grad_(), r(count, 24, 136).requires_grad_(), \
        r(count, 264, 24).requires_grad_(), r(rows, 264)
    ids = torch.randint(-1, count, (rows,), generator=g, device="cuda") if mixed else torch.arange(rows, device="cuda") * count // rows
    scaling = torch.rand(count, generator=g, device="cuda") + 0.5

    def step():
        out = lora_add(y, x, a, b, ids.int(), scaling)
        return (out.detach(), *torch.autograd.grad(out, (x, a, b), dout))

    return step


def experts(tokens, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape):
        return torch.randn(shape, generator=g, device="cuda").to(BF)

    leaves = [r(tokens, 128), torch.randn((tokens, 16), generator=g, device="cuda"), r(16, 72, 128), r(16, 128, 72)]
    x, logits, w1, w2 = (t.requires_grad_() for t in leaves)
    dout = r(tokens, 128)

    def step():
        weights, ids = topk_gating(logits, 4)
        plan = route_rows(ids, 16)
        z = grouped_linear(torch.nn.functional.silu(grouped_linear(moe_permute(x, plan), w1, plan.offsets)), w2, plan.offsets)
        out = moe_combine(z, weights, plan)
        return (out.detach(), *torch.autograd.grad(out, (x, logits, w1, w2), dout))

    return step


def equal(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.fixture(scope="module")
def steps():
    made = [adapters(1500, 6, False, BF, 1), adapters(1500, 30, True, HF, 2), adapters(60, 30, True, BF, 3),
            adapters(700, 4, False, HF, 4), experts(700, 5), experts(40, 6)]
    want = [step() for step in made]
    torch.cuda.synchronize()
    return made, want


def test_on_streams(steps):
    made, want = steps
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(5):
        got = []
        for stream, step in zip(streams, made):
            with torch.cuda.stream(stream):
                got.append(step())
        torch.cuda.synchronize()
        assert all(equal(a, b) for a, b in zip(got, want))


def test_in_threads(steps):
    made, want = steps
    off = []

    def run(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got = made[k]()
                    torch.cuda.current_stream().synchronize()
                    if not equal(got, want[k]):
                        off.append(k)
        except Exception as e:                   # a thread's exception would be lost
            off.append(repr(e))

    threads = [threading.Thread(target=run, args=(k,)) for k in range(len(made))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not off


def test_in_graphs(steps):
    made, want = steps
    graphs, results = [], []
    for step in made:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in made]
    for _ in range(5):
        for result in results:
            for t in result:
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(equal(a, b) for a, b in zip(results, want))
