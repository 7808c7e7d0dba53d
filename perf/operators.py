"""Performance cases of the trainable 16-bit expert path and of the adapters beside a shared projection.

Four operators, each over the range of sizes it is used at:

* ``grouped``  one matrix product per expert over ragged, unpadded rows: ``y[r] = x[r] . w[e(r)]^T``; with
               ``train`` also both gradients.
* ``lora``     low-rank adapters of many requests beside a shared projection: ``out = y + s_l (x A_l^T) B_l^T``,
               one adapter index per row; with ``train`` also the gradients of x, A and B.
* ``gating``   top-k softmax gating and the gradient of its weights with respect to the logits.
* ``combine``  the weighted sum of a token's expert rows, and the gradients of the rows and of the weights.

``run`` computes the plain forms (fp32 products, sums and indexing, rounded once) or, where ``own`` is true, makes the
calls that a user makes.  Sizes are those of ``flydsl_b200.workloads`` and of the dense projection's tests, and
neighbours of them.
"""

from __future__ import annotations

import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _grouped(name, rows, experts, k, n, dtype, train, spread="even", behind=0):
    return {"name": name, "op": "grouped", "rows": rows, "experts": experts, "k": k, "n": n, "dtype": dtype,
            "train": train, "spread": spread, "behind": behind}


def _lora(name, rows, k, n, rank, adapters, dtype, train, mix):
    return {"name": name, "op": "lora", "rows": rows, "k": k, "n": n, "rank": rank, "adapters": adapters,
            "dtype": dtype, "train": train, "mix": mix}


def _gating(name, tokens, experts, topk, dtype, renormalize):
    return {"name": name, "op": "gating", "tokens": tokens, "experts": experts, "topk": topk, "dtype": dtype,
            "renormalize": renormalize}


def _combine(name, tokens, topk, dim, experts, dtype):
    return {"name": name, "op": "combine", "tokens": tokens, "topk": topk, "dim": dim, "experts": experts,
            "dtype": dtype}


def listed():
    return [
        # a small model's decode step, top-2 of 8 experts, 32 tokens: launch latency
        _grouped("grouped-tiny-r64", 64, 8, 1024, 1024, "f16", False),
        # one GPU's 32 of 256 experts in a decode step of 64 tokens: about two rows each, the weights are the traffic
        _grouped("grouped-decode-r64", 64, 32, 7168, 4096, "bf16", False),
        # a fine-tuning step on a short ragged batch: odd sizes, experts without rows, unused rows behind the last one
        _grouped("grouped-train-odd-r3109", 3109, 16, 2104, 1048, "f16", True, "holes", 91),
        # a training step of 4096 tokens, top-8, on 32 local experts: gate and up projection with both gradients
        _grouped("grouped-train-r32768", 32768, 32, 7168, 4096, "bf16", True),
        # one request decoding with its adapter beside the narrow projection
        _lora("lora-decode-m1", 1, 7168, 2112, 16, 4, "bf16", False, "tokens"),
        # a decode batch of 64 requests over 32 adapters, some requests without one
        _lora("lora-decode-m64", 64, 7168, 7168, 16, 32, "bf16", False, "tokens"),
        # prefill of several requests, each with its own adapter
        _lora("lora-prefill-m4096", 4096, 2304, 7168, 64, 8, "f16", False, "requests"),
        # a training step of four adapters at once
        _lora("lora-train-m8192", 8192, 4096, 4096, 32, 4, "bf16", True, "requests"),
        # the router of a small batch, weights not renormalised: latency
        _gating("gating-t64-e8", 64, 8, 2, "bf16", False),
        # the router of a training step
        _gating("gating-t16384-e256", 16384, 256, 8, "f32", True),
        # the end of an expert layer for a small batch, and for a training step
        _combine("combine-t64", 64, 2, 4096, 8, "f16"),
        _combine("combine-t4096", 4096, 8, 7168, 256, "bf16"),
    ]


# the most that a drawn case may cost: what the largest listed ones do
_MAX_FLOPS = 6.0 * 32768 * 7168 * 4096
_MAX_WEIGHTS = 32 * 7168 * 4096


def _log(rng, lo, hi, step=1):
    return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)


def draw(rng):
    op = rng.choice(["grouped", "grouped", "lora", "lora", "gating", "combine"])
    dtype = rng.choice(["bf16", "f16"])
    if op == "grouped":
        while True:
            train = rng.random() < 0.5
            c = _grouped("", _log(rng, 1, 32768), _log(rng, 1, 64), _log(rng, 64, 8192, 8), _log(rng, 64, 8192, 8), dtype,
                         train, rng.choice(["even", "zipf", "holes"]), rng.choice([0, 0, rng.randrange(1, 200)]))
            if (6.0 if train else 2.0) * c["rows"] * c["k"] * c["n"] <= 0.4 * _MAX_FLOPS and \
                    c["experts"] * c["k"] * c["n"] <= 0.7 * _MAX_WEIGHTS:
                break
    elif op == "lora":
        train = rng.random() < 0.4
        mix = rng.choice(["tokens", "requests"])
        rows = _log(rng, 64, 8192) if train else _log(rng, 1, 512) if mix == "tokens" else _log(rng, 64, 8192)
        c = _lora("", rows, _log(rng, 512, 8192, 8), _log(rng, 512, 8192, 8), 8 * _log(rng, 1, 16),
                  _log(rng, 1, 8 if train else 32), dtype, train, mix)
    elif op == "gating":
        experts = _log(rng, 2, 512)
        c = _gating("", _log(rng, 1, 16384), experts, rng.randrange(1, min(8, experts) + 1),
                    rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.5)
    else:
        topk = rng.randrange(1, 9)
        c = _combine("", _log(rng, 1, 4096), topk, _log(rng, 128, 7168, 8), rng.choice([8, 64, 256]), dtype)
    del c["name"]
    return c


# ------------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype, scale=1.0):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    return out.normal_(generator=g).mul_(scale)


def _shares(c):
    """Expected share of the rows that each expert receives."""
    e = torch.arange(c["experts"], dtype=torch.float32)
    if c["spread"] == "zipf":
        p = 1.0 / (1.0 + e)
    elif c["spread"] == "holes":                 # every third expert receives nothing
        p = (e % 3 != 1).float()
    else:
        p = torch.ones_like(e)
    return p / p.sum()


def prepare(case, seed):
    c, g = case, _gen(seed)
    dt = _DT[c["dtype"]]
    s = {"case": c}
    if c["op"] == "grouped":
        rows, e, k, n = c["rows"], c["experts"], c["k"], c["n"]
        ids = torch.multinomial(_shares(c).cuda(), rows, replacement=True, generator=g)
        counts = torch.bincount(ids, minlength=e)
        s["offsets"] = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
        s["offsets"][1:] = counts.cumsum(0)
        s["x"] = _randn(g, (rows + c["behind"], k), dt)
        s["w"] = _randn(g, (e, n, k), dt, k ** -0.5)
        if c["train"]:
            s["dy"] = _randn(g, (rows + c["behind"], n), dt)
            s["x"].requires_grad_()
            s["w"].requires_grad_()
    elif c["op"] == "lora":
        m, k, n, r, ads = c["rows"], c["k"], c["n"], c["rank"], c["adapters"]
        if c["mix"] == "tokens":                 # one request a row, any adapter or none
            s["ids"] = torch.randint(-1, ads, (m,), generator=g, device="cuda", dtype=torch.int32)
        else:                                    # consecutive requests of uneven length
            marks = torch.rand(m, generator=g, device="cuda") < 2.0 * ads / m
            pick = torch.randint(0, ads, (m,), generator=g, device="cuda", dtype=torch.int32)
            s["ids"] = pick[marks.cumsum(0).clamp(max=m - 1)]
        s["x"] = _randn(g, (m, k), dt)
        s["y"] = _randn(g, (m, n), dt)
        s["a"] = _randn(g, (ads, r, k), dt, k ** -0.5)
        s["b"] = _randn(g, (ads, n, r), dt, r ** -0.5)
        s["scaling"] = torch.rand(ads, generator=g, device="cuda") + 0.5
        if c["train"]:
            s["dout"] = _randn(g, (m, n), dt)
            for name in ("x", "a", "b"):
                s[name].requires_grad_()
    elif c["op"] == "gating":
        s["logits"] = _randn(g, (c["tokens"], c["experts"]), dt, 2.0).requires_grad_()
        s["dweights"] = _randn(g, (c["tokens"], c["topk"]), torch.float32)
    else:
        t, k, dim = c["tokens"], c["topk"], c["dim"]
        ids = torch.rand((t, c["experts"]), generator=g, device="cuda").argsort(1)[:, :k]
        order = ids.reshape(-1).argsort(stable=True)             # rows in expert order, pairs of one expert in token order
        s["sorted_ids"] = ((order % k) << 24 | (order // k)).int()
        s["num_valid_ids"] = torch.tensor([t * k, t], dtype=torch.int32, device="cuda")
        s["row_index"] = torch.empty(t * k, dtype=torch.int32, device="cuda")
        s["row_index"][order] = torch.arange(t * k, dtype=torch.int32, device="cuda")
        counts = torch.bincount(ids.reshape(-1), minlength=c["experts"])
        s["offsets"] = torch.zeros(c["experts"] + 1, dtype=torch.int32, device="cuda")
        s["offsets"][1:] = counts.cumsum(0)
        s["row_index"] = s["row_index"].view(t, k)
        s["rows"] = _randn(g, (t * k, dim), dt).requires_grad_()
        w = torch.rand((t, k), generator=g, device="cuda") + 0.05
        s["weights"] = (w / w.sum(1, keepdim=True)).requires_grad_()
        s["dout"] = _randn(g, (t, dim), dt)
    return s


# ------------------------------------------------------------------------------- the framework's calls
def _own_grouped(s):
    from flydsl_b200.kernels.grouped_gemm import grouped_gemm, grouped_linear
    if not s["case"]["train"]:
        return grouped_gemm(s["x"], s["w"], s["offsets"])
    y = grouped_linear(s["x"], s["w"], s["offsets"])
    return (y.detach(), *torch.autograd.grad(y, (s["x"], s["w"]), s["dy"]))


def _own_lora(s):
    from flydsl_b200.kernels.lora import lora_add
    out = lora_add(s["y"], s["x"], s["a"], s["b"], s["ids"], s["scaling"])
    if not s["case"]["train"]:
        return out
    return (out.detach(), *torch.autograd.grad(out, (s["x"], s["a"], s["b"]), s["dout"]))


def _own_gating(s):
    from flydsl_b200.kernels.moe_routing import topk_gating
    weights, ids = topk_gating(s["logits"], s["case"]["topk"], renormalize=s["case"]["renormalize"])
    return (weights.detach(), ids, *torch.autograd.grad(weights, s["logits"], s["dweights"]))


def _own_combine(s):
    from flydsl_b200.kernels.moe_routing import RoutedRows, moe_combine
    plan = RoutedRows(s["sorted_ids"], s["num_valid_ids"], s["offsets"], s["row_index"])
    out = moe_combine(s["rows"], s["weights"], plan)
    return (out.detach(), *torch.autograd.grad(out, (s["rows"], s["weights"]), s["dout"]))


# ------------------------------------------------------------------------------- the plain forms
def _plain_grouped(s):
    """Experts padded to the longest one, one batched product for all of them."""
    c, x, w = s["case"], s["x"].detach(), s["w"].detach()
    rows, e, off = c["rows"], c["experts"], s["offsets"].long()
    counts = off[1:] - off[:-1]
    longest = int(counts.max())
    expert = torch.repeat_interleave(torch.arange(e, device="cuda"), counts, output_size=rows)
    at = expert * longest + torch.arange(rows, device="cuda") - off[expert]

    def padded(t):
        p = torch.zeros((e * longest, t.shape[1]), device="cuda")
        p[at] = t[:rows].float()
        return p.view(e, longest, -1)

    def ragged(p):
        t = torch.zeros((x.shape[0], p.shape[2]), dtype=x.dtype, device="cuda")
        t[:rows] = p.reshape(e * longest, -1)[at].to(x.dtype)
        return t

    xp, wf = padded(x), w.float()
    y = ragged(torch.bmm(xp, wf.transpose(1, 2)))
    if not c["train"]:
        return y
    dyp = padded(s["dy"])
    return y, ragged(torch.bmm(dyp, wf)), torch.bmm(dyp.transpose(1, 2), xp).to(w.dtype)


def _plain_lora(s):
    """Every row against every adapter, the other adapters' products masked out."""
    c, x, y = s["case"], s["x"].detach(), s["y"]
    a, b = s["a"].detach().float(), s["b"].detach().float()
    ads, r, k, n, m = c["adapters"], c["rank"], c["k"], c["n"], c["rows"]
    mine = s["ids"][:, None] == torch.arange(ads, device="cuda")                        # [m, adapters]
    a2, b2 = a.reshape(ads * r, k), b.permute(0, 2, 1).reshape(ads * r, n)
    xf = x.float()
    mask = mine[:, :, None].float()
    scale = mask * s["scaling"][None, :, None]
    v = ((xf @ a2.t()).view(m, ads, r) * mask).view(m, ads * r)
    vs = (v.view(m, ads, r) * scale).view(m, ads * r)
    out = (y.float() + vs @ b2).to(y.dtype)
    if not c["train"]:
        return out
    do = s["dout"].float()
    dv = ((do @ b2.t()).view(m, ads, r) * scale).view(m, ads * r)
    return (out, (dv @ a2).to(x.dtype), (dv.t() @ xf).view(ads, r, k).to(x.dtype),
            (vs.t() @ do).view(ads, r, n).transpose(1, 2).to(x.dtype))


def _plain_gating(s):
    c, logits = s["case"], s["logits"].detach().float()
    k = c["topk"]
    ids = torch.sort(logits, dim=1, descending=True, stable=True).indices[:, :k]
    ex = torch.exp(logits - logits.amax(1, keepdim=True))
    p = ex / ex.sum(1, keepdim=True)
    w = p.gather(1, ids)
    norm = w.sum(1, keepdim=True) if c["renormalize"] else torch.ones_like(w[:, :1])
    w = w / norm
    inner = (w * s["dweights"]).sum(1, keepdim=True)
    mine = torch.zeros_like(p).scatter_(1, ids, w * (s["dweights"] - inner) if c["renormalize"] else w * s["dweights"])
    d = mine if c["renormalize"] else mine - p * inner
    return w, ids.int(), d.to(s["logits"].dtype)


def _plain_combine(s):
    c, rows, w = s["case"], s["rows"].detach(), s["weights"].detach()
    at = s["row_index"].long()
    picked = rows.float()[at]                                                            # [t, k, dim]
    out = (picked * w[:, :, None]).sum(1).to(rows.dtype)
    do = s["dout"].float()
    drows = torch.empty_like(rows)
    drows[at.reshape(-1)] = (do[:, None, :] * w[:, :, None]).to(rows.dtype).reshape(-1, c["dim"])
    return out, drows, (picked * do[:, None, :]).sum(2)


_RUN = {"grouped": (_plain_grouped, _own_grouped), "lora": (_plain_lora, _own_lora),
        "gating": (_plain_gating, _own_gating), "combine": (_plain_combine, _own_combine)}


def run(state):
    plain, ours = _RUN[state["case"]["op"]]
    return ours(state) if own else plain(state)


# ------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "grouped":
        rows, k, n = float(c["rows"]), c["k"], c["n"]
        active = float((1.0 - (1.0 - _shares(c).double()) ** c["rows"]).sum())          # experts that receive a row
        ws = 2.0 * n * k * active
        if c["train"]:                           # x, w, dy read; y, dx, dw (of every expert) written
            return {"bytes": 4.0 * rows * (k + n) + ws + 2.0 * n * k * c["experts"], "flops": 6.0 * rows * k * n}
        return {"bytes": 2.0 * rows * (k + n) + ws, "flops": 2.0 * rows * k * n}
    if c["op"] == "lora":
        m, k, n, r, ads = float(c["rows"]), c["k"], c["n"], c["rank"], c["adapters"]
        if c["mix"] == "tokens":
            active = ads * (1.0 - (1.0 - 1.0 / (ads + 1)) ** m)
            with_one = m * ads / (ads + 1.0)
        else:
            active = ads * (1.0 - (1.0 - 1.0 / ads) ** (1.0 + min(m, 2.0 * ads)))
            with_one = m
        ws = 2.0 * r * (k + n) * active
        if c["train"]:                           # y, x, dout, A, B read; out, dx, dA, dB written
            return {"bytes": 2.0 * m * (2 * k + 3 * n) + ws + 2.0 * r * (k + n) * ads, "flops": 6.0 * with_one * r * (k + n)}
        return {"bytes": 2.0 * m * (k + 2 * n) + ws, "flops": 2.0 * with_one * r * (k + n)}
    if c["op"] == "gating":                      # logits read and their gradient written; weights, ids, weights' gradient
        size = {"f32": 4.0, "bf16": 2.0, "f16": 2.0}[c["dtype"]]
        return {"bytes": c["tokens"] * (2.0 * size * c["experts"] + 12.0 * c["topk"]), "flops": 4.0 * c["tokens"] * c["experts"]}
    t, k, dim = float(c["tokens"]), c["topk"], c["dim"]
    return {"bytes": 4.0 * t * k * dim + 4.0 * t * dim + 12.0 * t * k, "flops": 5.0 * t * k * dim}


# ------------------------------------------------------------------------------- 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "grouped":
        x, w, off = s["x"].detach(), s["w"].detach(), s["offsets"].tolist()
        y = torch.zeros((x.shape[0], c["n"]), dtype=torch.float64, device="cuda")
        dx = torch.zeros((x.shape[0], c["k"]), dtype=torch.float64, device="cuda") if c["train"] else None
        dw = torch.zeros(w.shape, dtype=torch.float64, device="cuda") if c["train"] else None
        for e in range(c["experts"]):
            i, j = off[e], off[e + 1]
            we, xe = w[e].double(), x[i:j].double()
            y[i:j] = torch.einsum("rk,nk->rn", xe, we)
            if c["train"]:
                de = s["dy"][i:j].double()
                dx[i:j] = torch.einsum("rn,nk->rk", de, we)
                dw[e] = torch.einsum("rn,rk->nk", de, xe)
        return (y, dx, dw) if c["train"] else y
    if c["op"] == "lora":
        x, a, b = (s[name].detach().double() for name in ("x", "a", "b"))
        out = s["y"].double()
        dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
        for i in range(c["adapters"]):
            sel = (s["ids"] == i).nonzero()[:, 0]
            if sel.numel() == 0:
                continue
            sc = s["scaling"][i].double()
            xi = x[sel]
            v = torch.einsum("mk,rk->mr", xi, a[i])
            out[sel] += sc * torch.einsum("mr,nr->mn", v, b[i])
            if c["train"]:
                do = s["dout"][sel].double() * sc
                dv = torch.einsum("mn,nr->mr", do, b[i])
                dx[sel] = torch.einsum("mr,rk->mk", dv, a[i])
                da[i] = torch.einsum("mr,mk->rk", dv, xi)
                db[i] = torch.einsum("mn,mr->nr", do, v)
        return (out, dx, da, db) if c["train"] else out
    if c["op"] == "gating":
        z = s["logits"].detach().double()
        order = torch.argsort(-z, dim=1, stable=True)[:, : c["topk"]]
        top = torch.gather(z, 1, order)
        base = top if c["renormalize"] else z
        log_norm = torch.logsumexp(base, dim=1, keepdim=True)
        w = torch.exp(top - log_norm)
        gw = s["dweights"].double() * w
        d = -torch.exp(base - log_norm) * gw.sum(1, keepdim=True)      # through the normaliser: all that it sums over
        if c["renormalize"]:
            full = torch.zeros_like(z).scatter_add(1, order, d + gw)
        else:
            full = d.scatter_add(1, order, gw)
        return w, None, full
    rows, w, do = s["rows"].detach().double(), s["weights"].detach().double(), s["dout"].double()
    at = s["row_index"].long()
    out = torch.zeros_like(do)
    drows = torch.zeros_like(rows)
    dw = torch.zeros_like(w)
    for j in range(c["topk"]):
        z = rows[at[:, j]]
        out += w[:, j : j + 1] * z
        drows[at[:, j]] = w[:, j : j + 1] * do
        dw[:, j] = torch.einsum("td,td->t", z, do)
    return out, drows, dw
