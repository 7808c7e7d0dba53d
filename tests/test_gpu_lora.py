"""Low-rank adapters beside a projection, against a plain 64-bit implementation."""
import pytest
import torch

from flydsl_b200.kernels.lora import lora_add
from kernels.blockscale_preshuffle_gemm import compile_blockscale_preshuffle_gemm

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def make(rows, k, n, rank, adapters, dtype, mix, seed=0, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if mix == "tokens":
        ids = torch.randint(-1, adapters + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
    elif mix == "one":
        ids = torch.full((rows,), adapters // 2, dtype=torch.int32, device="cuda")
    elif mix == "none":
        ids = torch.full((rows,), -1, dtype=torch.int32, device="cuda")
    else:                                        # runs of uneven length, one adapter skipped
        ids = (torch.arange(rows, device="cuda") * max(1, adapters - 1) // max(1, rows)).int()
    return dict(y=r(rows, n).to(dtype), x=(r(rows, k) * size).to(dtype), a=(r(adapters, rank, k) * k ** -0.5).to(dtype),
                b=(r(adapters, n, rank) * rank ** -0.5).to(dtype), adapter_ids=ids,
                scaling=torch.rand(adapters, generator=g, device="cuda") + 0.5), r(rows, n).to(dtype)


def exact(p, dout):
    """Results in 64 bits and, for each, the sums of absolute products that bound what fp32 steps may lose."""
    y, x, a, b = (p[s].double() for s in ("y", "x", "a", "b"))
    do = dout.double()
    out, dx, da, db = y.clone(), torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    mo, mx, ma, mb = y.abs(), torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for l in range(a.shape[0]):
        s = (p["adapter_ids"] == l).nonzero()[:, 0]
        if s.numel() == 0:
            continue
        sc = p["scaling"][l].double()
        v, va = x[s] @ a[l].t(), x[s].abs() @ a[l].abs().t()
        dv, dva = do[s] @ b[l], do[s].abs() @ b[l].abs()
        out[s] += sc * (v @ b[l].t())
        mo[s] += sc * (va @ b[l].abs().t())
        dx[s], mx[s] = sc * (dv @ a[l]), sc * (dva @ a[l].abs())
        da[l], ma[l] = sc * (dv.t() @ x[s]), sc * (dva.t() @ x[s].abs())
        db[l], mb[l] = sc * (do[s].t() @ v), sc * (do[s].abs().t() @ va)
    return (out, mo), (dx, mx), (da, ma), (db, mb)


def check(got, want, terms, what):
    """One rounding of the result (half a step, or half the smallest subnormal) after two chained fp32 sums of `terms` terms in
    all, off by at most one fp32 step (2^-23) of the absolute products each, and a middle factor held as two 16-bit numbers:
    bf16 keeps 2 * 8 bits of it (half a step of a half step, 2^-17), fp16 2 * 11 (2^-23)."""
    ref, mag = want
    fi = torch.finfo(got.dtype)
    rel = terms * 2.0 ** -23 + (2.0 ** -17 if got.dtype == BF else 2.0 ** -23)
    tol = fi.eps / 2 * ref.abs() + fi.smallest_normal * fi.eps / 2 + (1 + fi.eps) * rel * mag
    err = (got.double() - ref).abs()
    assert bool((err <= tol).all()), f"{what}: {int((~(err <= tol)).sum())} of {err.numel()} off, worst {float(err.max()):.3g}"


SIZES = [
    (1, 8, 8, 8, 1, "requests"), (1, 7168, 2112, 16, 4, "tokens"), (17, 264, 136, 24, 40, "tokens"),
    (64, 1024, 520, 16, 32, "tokens"), (33, 40, 1032, 128, 5, "tokens"), (130, 512, 256, 64, 3, "requests"),
    (1000, 328, 200, 32, 6, "requests"), (1500, 256, 264, 72, 2, "tokens"), (2100, 136, 72, 8, 1, "requests"), (700, 1096, 392, 48, 150, "tokens"), (512, 64, 72, 16, 1, "none"),
    (640, 1288, 328, 128, 3, "requests"), (900, 72, 64, 8, 2, "requests"), (2600, 1032, 136, 56, 5, "requests"),
    (50, 64, 64, 40, 3, "none"), (600, 2048, 136, 104, 9, "tokens"), (900, 264, 584, 16, 8, "tokens"),
    (777, 1032, 264, 64, 7, "tokens"), (1100, 520, 72, 56, 9, "tokens"), (640, 136, 264, 72, 4, "tokens"), (600, 72, 520, 88, 5, "tokens"),
    (1200, 256, 264, 16, 40, "one"), (300, 200, 1096, 120, 33, "tokens"), (40, 64, 72, 8, 3000, "tokens"), (5000, 64, 72, 8, 300, "tokens"),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,k,n,rank,adapters,mix", SIZES)
def test_forward_and_gradients(rows, k, n, rank, adapters, mix, dtype):
    p, dout = make(rows, k, n, rank, adapters, dtype, mix)
    (out, mo), (dx, mx), (da, ma), (db, mb) = exact(p, dout)
    got = lora_add(**p)
    check(got, (out, mo), k + rank, "out")
    none = (p["adapter_ids"] < 0) | (p["adapter_ids"] >= adapters)
    assert torch.equal(got[none], p["y"][none])
    q = {s: (t.clone().requires_grad_() if s in "yxab" else t) for s, t in p.items()}
    res = lora_add(**q)
    check(res.detach(), (out, mo), k + rank, "out in autograd")
    gy, gx, ga, gb = torch.autograd.grad(res, (q["y"], q["x"], q["a"], q["b"]), dout)
    assert torch.equal(gy, dout) and not bool(gx[none].any())
    check(gx, (dx, mx), n + rank, "dx")
    check(ga, (da, ma), n + rows, "da")
    check(gb, (db, mb), k + rows, "db")
    # each gradient alone is the same
    for name, ref in (("x", gx), ("a", ga), ("b", gb)):
        one = {s: (t.clone().requires_grad_() if s == name else t) for s, t in p.items()}
        (alone,) = torch.autograd.grad(lora_add(**one), (one[name],), dout)
        assert torch.equal(alone, ref), name


@pytest.mark.parametrize("size", [2.0 ** -12, 2.0 ** 9])
def test_fp16_rows_far_from_one(size):
    """The middle factor leaves fp16's range of full precision; the result does not."""
    p, dout = make(300, 512, 128, 32, 3, HF, "requests", seed=2, size=size)
    p["b"] = (p["b"].float() / max(size, 1.0)).half()
    p["y"].zero_()
    (out, mo), (dx, mx), (da, ma), (db, mb) = exact(p, dout)
    q = {s: (t.clone().requires_grad_() if s in "xab" else t) for s, t in p.items()}
    res = lora_add(**q)
    gx, ga, gb = torch.autograd.grad(res, (q["x"], q["a"], q["b"]), dout)
    check(res.detach(), (out, mo), 512 + 32, "out")
    check(gx, (dx, mx), 128 + 32, "dx")
    check(ga, (da, ma), 128 + 300, "da")
    check(gb, (db, mb), 512 + 300, "db")


@pytest.mark.parametrize("dtype", [BF, HF])
def test_many_column_tiles_with_several_adapters_in_a_row_tile(dtype):
    """Blocks walk through a dozen column tiles while some of their warps have no row of the adapter at hand."""
    rows, k, n, rank, adapters = 2048, 256, 7168, 32, 4
    p, dout = make(rows, k, n, rank, adapters, dtype, "requests", seed=4)
    p["adapter_ids"] = ((torch.arange(rows, device="cuda") // 40) % (adapters + 1)).int()       # three or four of them in a tile
    (out, mo), (dx, mx), (da, ma), (db, mb) = exact(p, dout)
    q = {s: (t.clone().requires_grad_() if s in "xab" else t) for s, t in p.items()}
    for _ in range(3):
        res = lora_add(**q)
        gx, ga, gb = torch.autograd.grad(res, (q["x"], q["a"], q["b"]), dout)
        check(res.detach(), (out, mo), k + rank, "out")
        check(gx, (dx, mx), n + rank, "dx")
        check(ga, (da, ma), n + rows, "da")
        check(gb, (db, mb), k + rows, "db")


def test_no_rows():
    p, dout = make(0, 64, 72, 16, 2, BF, "tokens")
    assert lora_add(**p).shape == (0, 72)
    q = {s: (t.clone().requires_grad_() if s in "yxab" else t) for s, t in p.items()}
    gy, gx, ga, gb = torch.autograd.grad(lora_add(**q), (q["y"], q["x"], q["a"], q["b"]), dout)
    assert gx.shape == (0, 64) and not bool(ga.any()) and not bool(gb.any())


@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_one_request_does_not_reach_another(poison):
    p, dout = make(100, 136, 200, 16, 4, BF, "tokens", seed=5)
    mine = p["adapter_ids"] == 2
    def run(q):
        q = {s: (t.clone().requires_grad_() if s in "xab" else t) for s, t in q.items()}
        out = lora_add(**q)
        return (out.detach(), *torch.autograd.grad(out, (q["x"], q["a"], q["b"]), dout))
    clean = run(p)
    for s in ("y", "x"):
        p[s][~mine] = poison
    for s in ("a", "b"):
        p[s][:2], p[s][3:] = poison, poison
    p["scaling"][:2] = poison
    dirty = run(p)
    assert torch.equal(dirty[0][mine], clean[0][mine]) and torch.equal(dirty[1][mine], clean[1][mine])
    assert torch.equal(dirty[2][2], clean[2][2]) and torch.equal(dirty[3][2], clean[3][2])


def test_in_place_buffers_and_streams():
    p, _ = make(70, 256, 520, 32, 5, HF, "tokens", seed=6)
    want = lora_add(**p)
    buf = torch.full_like(want, 3.0)
    assert lora_add(**p, out=buf) is buf and torch.equal(buf, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    res = lora_add(**p, stream=side)
    side.synchronize()
    assert torch.equal(res, want)
    y = p["y"].clone()
    assert lora_add(y, *(p[s] for s in ("x", "a", "b", "adapter_ids", "scaling")), out=y) is y and torch.equal(y, want)
    with pytest.raises(ValueError, match="for inference"):
        lora_add(p["y"].clone().requires_grad_(), *(p[s] for s in ("x", "a", "b", "adapter_ids", "scaling")), out=buf)
    with pytest.raises(ValueError, match="dtype"):
        lora_add(p["y"].bfloat16(), *(p[s] for s in ("x", "a", "b", "adapter_ids", "scaling")))
    rest = [p[s] for s in ("a", "b", "adapter_ids", "scaling")]
    store = torch.zeros(71 * 520, dtype=HF, device="cuda")
    whole, shifted = store[: 70 * 520].view(70, 520), store[520:].view(70, 520)
    for y, x, out in ((whole, p["x"], shifted), (p["y"], store[: 70 * 256].view(70, 256), whole)):
        with pytest.raises(ValueError, match="share memory"):
            lora_add(y, x, *rest, out=out)
    with pytest.raises(ValueError, match="scaling has no gradient"):
        lora_add(*(p[s] for s in ("y", "x", "a", "b", "adapter_ids")), p["scaling"].clone().requires_grad_())


def test_rows_alone_equal_rows_in_a_batch_of_their_block():
    """A row's result does not depend on the adapters around it."""
    p, _ = make(16, 512, 256, 16, 8, BF, "tokens", seed=7)
    whole = lora_add(**p)
    other = dict(p, adapter_ids=p["adapter_ids"].clone())
    other["adapter_ids"][1:] = -1
    (out, mo), *_ = exact(p, p["y"])
    check(lora_add(**other)[:1], (out[:1], mo[:1]), 528, "row 0")
    check(whole[:1], (out[:1], mo[:1]), 528, "row 0 in the batch")


def test_differences():
    p, dout = make(40, 64, 72, 8, 3, HF, "requests", seed=8)
    q = {s: (t.clone().requires_grad_() if s in "xab" else t) for s, t in p.items()}
    grads = torch.autograd.grad(lora_add(**q), (q["x"], q["a"], q["b"]), dout)
    g = torch.Generator(device="cuda").manual_seed(1)
    dirs = [torch.randn(p[s].shape, generator=g, device="cuda", dtype=torch.float64) for s in "xab"]
    h = 1e-4

    def f(t):
        x, a, b = (p[s].double() + t * d for s, d in zip("xab", dirs))
        total = 0.0
        for l in range(3):
            s = p["adapter_ids"] == l
            total += float((p["scaling"][l].double() * (x[s] @ a[l].t()) @ b[l].t() * dout[s].double()).sum())
        return total

    num = (f(h) - f(-h)) / (2 * h)               # exact up to the cubic term, h^2 of a product of three directions
    cubic = h * h * sum(float((dirs[0][s].abs() @ dirs[1][l].abs().t() @ dirs[2][l].abs().t() * dout[s].double().abs()).sum())
                        * float(p["scaling"][l]) for l in range(3) for s in [p["adapter_ids"] == l])
    ana = sum(float((gr.double() * d).sum()) for gr, d in zip(grads, dirs))
    slack = 2.0 ** -10 * sum(float((gr.double() * d).abs().sum()) for gr, d in zip(grads, dirs))   # one fp16 rounding each
    assert abs(num - ana) <= slack + cubic


def test_beside_the_shared_projection_in_a_graph():
    """The block-scaled dense projection and the adapters on top of its output, in place, captured and replayed."""
    M, N, K, r, L = 48, 2112, 1024, 16, 6
    p, _ = make(M, K, N, r, L, BF, "tokens", seed=9)
    g = torch.Generator().manual_seed(3)
    w = (torch.rand((N, K), generator=g) / 10).to(torch.float8_e4m3fn).cuda()
    sb = torch.rand(((N + 127) // 128, K // 128), generator=g).cuda()
    xq = [(torch.rand((M, K), generator=g) / 10).to(torch.float8_e4m3fn).cuda() for _ in range(2)]
    sa = torch.rand((K // 128, M), generator=g).cuda()
    exe = compile_blockscale_preshuffle_gemm(M=M, N=N, K=K, tile_m=64, tile_n=128, tile_k=128, w_layout="plain")
    ids = [p["adapter_ids"], p["adapter_ids"].flip(0).contiguous()]

    def step(c, q, i):
        exe(c, q, w, sa, sb, M, N)
        return lora_add(c, p["x"], p["a"], p["b"], i, p["scaling"], out=c)

    eager = []
    for q, i in zip(xq, ids):
        c = torch.empty((M, N), dtype=BF, device="cuda")
        exe(c, q, w, sa, sb, M, N)
        base = c.clone()
        step(c, q, i)
        (want, mag), *_ = exact(dict(p, y=base, adapter_ids=i), base)
        check(c, (want, mag), K + r, "projection with adapters")
        eager.append(c)
    static_q, static_i, c = xq[0].clone(), ids[0].clone(), torch.zeros((M, N), dtype=BF, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(c, static_q, static_i)
    for j in (1, 0, 1):
        static_q.view(torch.uint8).copy_(xq[j].view(torch.uint8))
        static_i.copy_(ids[j])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c, eager[j])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("adapters", [3, 40])
def test_in_place_where_tiles_have_no_adapter(adapters, dtype):
    """Runs of rows without an adapter longer than a tile, beside tiles of few adapters and of many."""
    p, _ = make(1700, 136, 392, 24, adapters, dtype, "tokens", seed=12)
    ids = p["adapter_ids"]
    ids[:300] = -1
    ids[300:700] = 1
    ids[1100:1450] = adapters                    # names no adapter either
    want = lora_add(**p)
    (out, mag), *_ = exact(p, want)
    check(want, (out, mag), 136 + 24, "out")
    none = (ids < 0) | (ids >= adapters)
    assert torch.equal(want[none], p["y"][none])
    y = p["y"].clone()
    rest = [p[s] for s in ("x", "a", "b", "adapter_ids", "scaling")]
    assert lora_add(y, *rest, out=y) is y and torch.equal(y, want)
    ids.fill_(-1)
    assert torch.equal(lora_add(y, *rest, out=y), want) and torch.equal(lora_add(want, *rest), want)


@pytest.mark.parametrize("rank", [64, 128])
def test_gradient_of_a_alone_behind_other_launches(rank):
    """Without dx the kernel of the adapters' gradients follows the shrink of dv directly, and tiles of up to eight adapters want
    all of TMEM: steps queued one behind the other, then captured."""
    rows, k, n, adapters = 20000, 136, 264, 8
    p, dout = make(rows, k, n, rank, adapters, BF, "requests", seed=13)
    p["adapter_ids"] = ((torch.arange(rows, device="cuda") // 30) % adapters).int()
    *_, (da, ma), _ = exact(p, dout)
    a = p["a"].clone().requires_grad_()

    def step():
        out = lora_add(p["y"], p["x"], a, p["b"], p["adapter_ids"], p["scaling"])
        return torch.autograd.grad(out, (a,), dout)[0]

    torch.cuda.synchronize()
    grads = [step() for _ in range(20)]
    check(grads[0], (da, ma), n + rows, "da")
    assert all(torch.equal(g, grads[0]) for g in grads)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(5):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, grads[0])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows,rank,adapters,mix", [(100, 24, 4, "requests"), (700, 24, 4, "requests"), (1500, 128, 3, "requests"),
                                                    (700, 16, 40, "tokens"), (900, 72, 3, "requests")])
def test_infinities_stay_infinities(rows, rank, adapters, mix, dtype):
    """One entry of a tensor is infinite: what the formulas make infinite, NaN or finite comes out as that."""
    k, n, inf = 136, 200, float("inf")
    for place, sign in (("x", 1), ("a", -1), ("b", 1), ("dout", -1), ("b", -1), ("x", -1)):
        p, dout = make(rows, k, n, rank, adapters, dtype, mix, seed=14)
        row = int((p["adapter_ids"] == 1).nonzero()[-1])
        {"x": p["x"][row], "a": p["a"][1, rank - 1], "b": p["b"][1, n - 1], "dout": dout[row]}[place][3] = sign * inf
        want = exact(p, dout)
        q = {s: (t.clone().requires_grad_() if s in "xab" else t) for s, t in p.items()}
        res = lora_add(**q)
        got = (res.detach(), *torch.autograd.grad(res, (q["x"], q["a"], q["b"]), dout))
        for name, out, (ref, mag), terms in zip(("out", "dx", "da", "db"), got, want, (k + rank, n + rank, n + rows, k + rows)):
            what = f"{name}, {place} {sign * inf}"
            assert torch.equal(out.isnan(), ref.isnan()), what
            odd = ~ref.isfinite()
            assert torch.equal(out[ref.isinf()].double(), ref[ref.isinf()]), what
            check(out[~odd], (ref[~odd], mag[~odd]), terms, what)


@pytest.mark.parametrize("rows", [40, 600, 20000])
def test_what_a_graph_keeps(rows):
    """The middle factor once, where the gradient of b wants it, and nothing else that the call made."""
    p, dout = make(rows, 2048, 136, 24, 5, BF, "requests", seed=15)
    want = lora_add(**p)
    given = {t.untyped_storage().data_ptr() for t in p.values()}
    for names, floats in (("yxab", rows * 24), ("b", rows * 24), ("y", 0), ("xa", 0)):
        q = {s: (t.detach().requires_grad_() if s in names else t) for s, t in p.items()}
        out = lora_add(**q)
        kept = [t for t in out.grad_fn.saved_tensors if t is not None and t.untyped_storage().data_ptr() not in given]
        assert sum(t.untyped_storage().nbytes() for t in kept) <= floats * 4 + (rows + 127) // 128 * 4
        grads = torch.autograd.grad(out, [q[s] for s in names], dout)
        if names == "yxab":
            full = dict(zip(names, grads))
            (ref, mag), (dx, mx), (da, ma), (db, mb) = exact(p, dout)
            check(full["b"], (db, mb), 2048 + rows, "db")
        assert all(torch.equal(g, full[s]) for s, g in zip(names, grads))
        check(out.detach(), (ref, mag), 2048 + 24, "out")
        check(want, (ref, mag), 2048 + 24, "out")


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), "lowest"])
@pytest.mark.parametrize("rows,rank,adapters,mix,dtype", [(100, 16, 4, "tokens", HF), (700, 24, 4, "tokens", BF), (700, 24, 4, "tokens", HF),
                                                          (1500, 128, 4, "requests", BF), (1500, 128, 4, "requests", HF),
                                                          (900, 64, 40, "tokens", BF), (900, 64, 40, "tokens", HF)])
def test_one_request_does_not_reach_another_on_tiles(rows, rank, adapters, mix, dtype, poison):
    if poison == "lowest":
        poison = torch.finfo(dtype).min
    p, dout = make(rows, 136, 200, rank, adapters, dtype, mix, seed=16)
    mine = p["adapter_ids"] == 2
    def run():
        q = {s: (t.clone().requires_grad_() if s in "xab" else t) for s, t in p.items()}
        out = lora_add(**q)
        return (out.detach(), *torch.autograd.grad(out, (q["x"], q["a"], q["b"]), dout))
    clean = run()
    for t in (p["y"], p["x"], dout):
        t[~mine] = poison
    for t in (p["a"], p["b"], p["scaling"]):
        t[:2], t[3:] = poison, poison
    dirty = run()
    assert torch.equal(dirty[0][mine], clean[0][mine]) and torch.equal(dirty[1][mine], clean[1][mine])
    assert torch.equal(dirty[2][2], clean[2][2]) and torch.equal(dirty[3][2], clean[3][2])


@pytest.mark.parametrize("rows,n,rank", [(700, 200, 24), (1500, 72, 128), (30000, 136, 16), (30000, 136, 88)])
def test_fp16_rows_of_every_size_beside_each_other(rows, n, rank):
    """Each row of a tile, and each tile that a block goes through, has a power of two of its own."""
    k = 72
    p, dout = make(rows, k, n, rank, 4, HF, "requests", seed=17)
    p["x"] *= (2.0 ** (torch.arange(rows, device="cuda") * 7 % 21 - 11))[:, None].half()
    dout = dout * (2.0 ** (torch.arange(rows, device="cuda") * 5 % 19 - 10))[:, None].half()
    p["b"] /= 64
    p["y"].zero_()
    (out, mo), (dx, mx), (da, ma), (db, mb) = exact(p, dout)
    q = {s: (t.clone().requires_grad_() if s in "xab" else t) for s, t in p.items()}
    res = lora_add(**q)
    gx, ga, gb = torch.autograd.grad(res, (q["x"], q["a"], q["b"]), dout)
    fits = [bool((t.abs() < 6e4).all()) for t in (out, dx, da, db)]
    assert fits[0] and fits[1]                   # sums over thousands of rows may pass what fp16 holds
    check(res.detach(), (out, mo), k + rank, "out")
    check(gx, (dx, mx), n + rank, "dx")
    for got, ref, mag, terms, what in ((ga, da, ma, n + rows, "da"), (gb, db, mb, k + rows, "db")):
        held = ref.abs() < 6e4
        check(got[held], (ref[held], mag[held]), terms, what)


@pytest.mark.parametrize("rows,adapters", [(64, 30), (2048, 4), (700, 30)])
def test_calls_that_read_what_the_call_before_wrote(rows, adapters):
    """Thirty in a row, each of whose launches start while the one before still runs."""
    p, _ = make(rows, 264, 264, 16, adapters, BF, "tokens", seed=18)
    rest = (p["a"], p["b"], p["adapter_ids"], p["scaling"] / 16)

    def chain(wait):
        h = p["x"]
        for _ in range(30):
            h = lora_add(h, h, *rest)
            if wait:
                torch.cuda.synchronize()
        return h

    want = chain(True)
    assert bool(want.isfinite().all())
    for _ in range(10):
        assert torch.equal(chain(False), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain(False)
    for _ in range(10):
        got.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
