"""Grouped products over ragged rows and their gradients, against a plain 64-bit implementation."""
import pytest
import torch

from flydsl_b200.kernels._call import on
from flydsl_b200.kernels.grouped_gemm import grouped_gemm, grouped_gemm_dgrad, grouped_gemm_wgrad, grouped_linear

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def make(counts, k, n, dtype, front=0, behind=0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = front + sum(counts) + behind
    x = torch.randn((rows, k), generator=g, device="cuda").to(dtype)
    dy = torch.randn((rows, n), generator=g, device="cuda").to(dtype)
    w = (torch.randn((len(counts), n, k), generator=g, device="cuda") * k ** -0.5).to(dtype)
    off = torch.tensor([front] + counts, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()
    return x, w, dy, off


def exact(x, w, dy, off):
    """Results in 64 bits, and the sums of absolute products that bound a summation's error."""
    o = off.tolist()
    x, w, dy = x.double(), w.double(), dy.double()
    y, dx, dw = torch.zeros_like(dy), torch.zeros_like(x), torch.zeros_like(w)
    ys, dxs, dws = torch.zeros_like(dy), torch.zeros_like(x), torch.zeros_like(w)
    for e in range(w.shape[0]):
        r = slice(o[e], o[e + 1])
        y[r], ys[r] = x[r] @ w[e].t(), x[r].abs() @ w[e].abs().t()
        dx[r], dxs[r] = dy[r] @ w[e], dy[r].abs() @ w[e].abs()
        dw[e], dws[e] = dy[r].t() @ x[r], dy[r].abs().t() @ x[r].abs()
    return (y, ys), (dx, dxs), (dw, dws)


def check(got, want, terms, what):
    """One rounding to the type (half a step, eps / 2 of the value, or half the smallest subnormal) after `terms` fp32
    additions that are off by at most one fp32 step (2^-23) of the sum of absolute products each."""
    ref, mag = want
    fi = torch.finfo(got.dtype)
    tol = fi.eps / 2 * ref.abs() + fi.smallest_normal * fi.eps / 2 + (1 + fi.eps) * terms * 2.0 ** -23 * mag
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), f"{what}: {int((~(err <= tol)).sum())} of {err.numel()} off, worst {float(err.max()):.3g}"


SHAPES = [
    ([64, 3, 0, 61], 64, 64, 0, 0),              # the smallest widths of a full K block; an expert without rows
    ([1], 8, 8, 0, 0),                           # one row, the smallest widths
    ([0, 0, 1, 0], 136, 72, 2, 3),               # empty experts at both ends, rows of no expert
    ([128, 127, 129, 1, 255, 257], 256, 264, 0, 0),
    ([63, 64, 65, 15, 16, 17, 47, 48, 49], 200, 328, 5, 77),    # every kind of last K block of the weight gradient
    ([300] * 3, 1024, 520, 0, 0),
    ([0] * 200 + [33, 1] * 100 + [0], 72, 88, 0, 9),             # many experts
    ([2500, 0, 71], 1048, 2104, 0, 0),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("counts,k,n,front,behind", SHAPES)
def test_forms_against_64_bits(counts, k, n, front, behind, dtype):
    x, w, dy, off = make(counts, k, n, dtype, front, behind)
    (y, ys), (dx, dxs), (dw, dws) = exact(x, w, dy, off)
    check(grouped_gemm(x, w, off), (y, ys), k, "y")
    check(grouped_gemm_dgrad(dy, w, off), (dx, dxs), n, "dx")
    check(grouped_gemm_wgrad(dy, x, off), (dw, dws), max(counts), "dw")


# (rows per expert, k, n) and the kernels that they take, forward and for the input gradient
KINDS = [
    ([1024, 700, 1300, 1100], 2048, 2048, 0, 0), ([130, 100, 150, 90, 0] * 5, 1000, 1032, 1, 1),
    ([80, 100, 129, 90, 0] * 5, 1544, 1032, 1, 2), ([100, 120] * 10, 264, 1800, 2, 2),
    ([5, 33, 0, 64, 31, 32] * 2, 520, 1544, 3, 4), ([1, 2], 2048, 1048, 4, 4),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("counts,k,n,forward,backward", KINDS)
def test_every_kernel(lib, counts, k, n, forward, backward, dtype):
    rows, e = sum(counts), len(counts)
    kinds = tuple(lib.flymoe_grouped_gemm_tile(rows, e, n, k, g) for g in (0, 1))
    assert kinds == (forward, backward)
    x, w, dy, off = make(counts, k, n, dtype, 0, 40)
    (y, ys), (dx, dxs), _ = exact(x, w, dy, off)
    check(grouped_gemm(x, w, off), (y, ys), k, "y")
    check(grouped_gemm_dgrad(dy, w, off), (dx, dxs), n, "dx")


@pytest.mark.parametrize("experts", [1, 1024])
def test_no_rows(experts):
    w = torch.randn((experts, 64, 72), device="cuda").to(BF)
    off = torch.zeros(experts + 1, dtype=torch.int32, device="cuda")
    x, dy = torch.empty((0, 72), dtype=BF, device="cuda"), torch.empty((0, 64), dtype=BF, device="cuda")
    assert grouped_gemm(x, w, off).shape == (0, 64)
    assert grouped_gemm_dgrad(dy, w, off).shape == (0, 72)
    out = torch.full((experts, 64, 72), 7.0, dtype=BF, device="cuda")
    assert not bool(grouped_gemm_wgrad(dy, x, off, out=out).any())
    # rows, but none that belongs to an expert
    x, dy = torch.randn((5, 72), device="cuda").to(BF), torch.randn((5, 64), device="cuda").to(BF)
    assert not bool(grouped_gemm(x, w, off).any()) and not bool(grouped_gemm_dgrad(dy, w, off).any())
    out.fill_(7.0)
    assert not bool(grouped_gemm_wgrad(dy, x, off, out=out).any())


def test_rows_of_no_expert_are_left_in_the_callers_result():
    x, w, dy, off = make([40, 0, 90], 128, 256, BF, front=3, behind=130)
    out = torch.full((x.shape[0], 256), 5.0, dtype=BF, device="cuda")
    assert grouped_gemm(x, w, off, out=out) is out
    assert bool((out[:3] == 5).all()) and bool((out[133:] == 5).all())
    assert torch.equal(out[3:133], grouped_gemm(x, w, off)[3:133])
    dx = torch.full((x.shape[0], 128), 5.0, dtype=BF, device="cuda")
    grouped_gemm_dgrad(dy, w, off, out=dx)
    assert bool((dx[:3] == 5).all()) and bool((dx[133:] == 5).all())


@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_what_stands_in_other_rows_stays_there(poison):
    counts = [50, 1, 77, 64]
    x, w, dy, off = make(counts, 192, 136, BF, front=2, behind=9)
    clean = grouped_gemm(x, w, off), grouped_gemm_dgrad(dy, w, off), grouped_gemm_wgrad(dy, x, off)
    xp, dyp, wp = x.clone(), dy.clone(), w.clone()
    lo, hi = off[2].item(), off[3].item()        # everything but expert 2 is poisoned
    for t in (xp, dyp):
        t[:lo], t[hi:] = poison, poison
    wp[:2], wp[3:] = poison, poison
    assert torch.equal(grouped_gemm(xp, wp, off)[lo:hi], clean[0][lo:hi])
    assert torch.equal(grouped_gemm_dgrad(dyp, wp, off)[lo:hi], clean[1][lo:hi])
    assert torch.equal(grouped_gemm_wgrad(dyp, xp, off)[2], clean[2][2])


def test_offsets_out_of_order_stay_inside():
    x, w, dy, _ = make([100, 100], 64, 64, BF)
    off = torch.tensor([-7, 150, 120, 999], dtype=torch.int32, device="cuda")
    w = torch.cat([w, w[:1]])
    taken = torch.tensor([0, 150, 150, 200], dtype=torch.int32, device="cuda")
    for f, a, b in ((grouped_gemm, x, w), (grouped_gemm_dgrad, dy, w), (grouped_gemm_wgrad, dy, x)):
        assert torch.equal(f(a, b, off), f(a, b, taken))


def test_autograd_and_differences():
    x, w, dy, off = make([33, 0, 20], 64, 72, HF, behind=4)
    x.requires_grad_()
    w.requires_grad_()
    y = grouped_linear(x, w, off)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    assert torch.equal(dx, grouped_gemm_dgrad(dy, w.detach(), off))
    assert torch.equal(dw, grouped_gemm_wgrad(dy, x.detach(), off))
    assert not bool(dx[53:].any())
    # differences of the 64-bit form along one direction, which is linear in x and in w
    g = torch.Generator(device="cuda").manual_seed(9)
    px, pw = (torch.randn(t.shape, generator=g, device="cuda", dtype=torch.float64) for t in (x, w))
    h = 1e-4

    def f(xx, ww):
        return sum(float(((xx[a:b] @ ww[e].t()) * dy[a:b].double()).sum())
                   for e, (a, b) in enumerate(((0, 33), (33, 33), (33, 53))))

    xd, wd = x.detach().double(), w.detach().double()
    num = (f(xd + h * px, wd + h * pw) - f(xd - h * px, wd - h * pw)) / (2 * h)
    ana = float((dx.double() * px).sum() + (dw.double() * pw).sum())
    # each gradient element is rounded to fp16 once: half a step 2^-11 of it, 2^-10 with its fp32 sum, all the same way
    slack = 2.0 ** -10 * float((dx.double() * px).abs().sum() + (dw.double() * pw).abs().sum())
    assert abs(num - ana) <= slack
    # only what is asked for; a gradient that arrives as a broadcast view
    (only,) = torch.autograd.grad(grouped_linear(x, w.detach(), off).sum(), (x,))
    assert torch.equal(only, grouped_gemm_dgrad(torch.ones_like(dy), w.detach(), off))


def test_another_stream_and_a_captured_step():
    sets = [make([70, 0, 130], 256, 192, BF, seed=s) for s in range(3)]
    eager = [(grouped_gemm(x, w, o), grouped_gemm_dgrad(dy, w, o), grouped_gemm_wgrad(dy, x, o)) for x, w, dy, o in sets]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    x, w, dy, o = sets[1]
    got = grouped_gemm(x, w, o, stream=side), grouped_gemm(x, w, o, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(got[0], eager[1][0]) and torch.equal(got[1], eager[1][0])
    st = [t.clone() for t in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = grouped_gemm(st[0], st[1], st[3]), grouped_gemm_dgrad(st[2], st[1], st[3]), grouped_gemm_wgrad(st[2], st[0], st[3])
    for i in (1, 2, 0):
        for d, s in zip(st, sets[i]):
            d.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(res, eager[i]))


def test_results_apart_from_inputs_and_streams_of_their_device():
    x, w = torch.ones((12, 64), dtype=BF, device="cuda"), torch.ones((2, 64, 64), dtype=BF, device="cuda")
    off = torch.tensor([0, 4, 12], dtype=torch.int32, device="cuda")
    for out in (x, w.view(-1, 64)[10:22]):
        with pytest.raises(ValueError, match="share memory"):
            grouped_gemm(x, w, off, out=out)
        with pytest.raises(ValueError, match="share memory"):
            grouped_gemm_dgrad(x, w, off, out=out)
    with pytest.raises(ValueError, match="share memory"):
        grouped_gemm_wgrad(w.view(-1, 64)[:12], x, off, out=w)
    with pytest.raises(ValueError, match="stream is on"):
        on(torch.device("cuda", torch.cuda.current_device() + 1), torch.cuda.Stream())


def test_weight_gradient_over_millions_of_rows():
    rows = 2 ** 24 + 37
    x, dy = torch.zeros((rows, 8), dtype=BF, device="cuda"), torch.ones((rows, 8), dtype=BF, device="cuda")
    x[0], x[rows // 2], x[rows - 1] = 1, 4, 2
    offsets = torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    assert bool((grouped_gemm_wgrad(dy, x, offsets) == 7).all())
