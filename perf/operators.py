"""Cases of the dense operators beside the embedding store: layer normalisation
of pooled or looked-up rows with its backward pass, and the Muon update of the
dense matrices that read them (an update orthogonalised by Newton-Schulz
products).

`listed` and `draw` give cases, `prepare` a case's inputs on the GPU, `run` one
pass (`own` chooses the framework's kernels, else the formulas in elementary
torch operations), `exact` the same results in 64 bits, `work` the bytes and
operations a pass cannot do without.
"""

from __future__ import annotations

import math

import torch

own = False

# The quintic of the Newton-Schulz iteration: X <- a X + (b A + c A A) X, A = X X^T.
NS_A, NS_B, NS_C = 3.4445, -4.7750, 2.0315
STEPS = 5

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}


def listed():
    return [
        # Serving: the 26 pooled rows of one sample, dim 128, on their way into the dense part.
        {"name": "norm sample 26x128 f32", "op": "norm", "rows": 26, "dim": 128, "pad": 0, "dtype": "float32", "param": "float32"},
        # Serving: one lookup batch of the weight-only store (262,144 keys, dim 256, bf16).
        {"name": "norm lookup 262144x256 bf16", "op": "norm", "rows": 262144, "dim": 256, "pad": 0, "dtype": "bfloat16", "param": "bfloat16"},
        # Training: the rows of the single-table train step (65,536 keys, dim 64, fp32).
        {"name": "norm bwd 65536x64 f32", "op": "norm_backward", "rows": 65536, "dim": 64, "pad": 0, "dtype": "float32", "param": "float32"},
        # Training: the pooled rows of a DLRM batch (8,192 samples x 26 tables, dim 128).
        {"name": "norm bwd 212992x128 f32", "op": "norm_backward", "rows": 212992, "dim": 128, "pad": 0, "dtype": "float32", "param": "float32"},
        # Training: an odd width inside wider rows, 16-bit rows with fp32 weights.
        {"name": "norm bwd 9973x1037 bf16", "op": "norm_backward", "rows": 9973, "dim": 1037, "pad": 3, "dtype": "bfloat16", "param": "float32"},
        # Training: wide hidden rows of a large batch.
        {"name": "norm bwd 32768x4096 bf16", "op": "norm_backward", "rows": 32768, "dim": 4096, "pad": 0, "dtype": "bfloat16", "param": "bfloat16"},
        # The update of one small projection behind dim-64 rows.
        {"name": "orth 128x64 bf16", "op": "orth", "batch": 1, "m": 128, "n": 64, "pad": 0, "dtype": "bfloat16"},
        # An odd matrix in full precision.
        {"name": "orth 1000x517 f32", "op": "orth", "batch": 1, "m": 1000, "n": 517, "pad": 0, "dtype": "float32"},
        # The largest: one square projection of a wide model.
        {"name": "orth 4096x4096 bf16", "op": "orth", "batch": 1, "m": 4096, "n": 4096, "pad": 0, "dtype": "bfloat16"},
        # A layer of a DLRM's tower: the whole optimizer step of one small matrix.
        {"name": "muon 512x256 f32", "op": "muon", "batch": 1, "m": 512, "n": 256, "pad": 0, "dtype": "float32", "grad": "float32"},
        # Eight equal layers (or experts) stepped in one call.
        {"name": "muon 8x1024x2048 bf16", "op": "muon", "batch": 8, "m": 1024, "n": 2048, "pad": 0, "dtype": "bfloat16", "grad": "bfloat16"},
        # fp32 master weights of a tall rectangular layer.
        {"name": "muon 4096x1024 f32", "op": "muon", "batch": 1, "m": 4096, "n": 1024, "pad": 0, "dtype": "float32", "grad": "float32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _ns_flops(c):
    s, w = min(c["m"], c["n"]), max(c["m"], c["n"])
    return c["batch"] * STEPS * (3 * s * s * w + s**3)


def draw(rng):
    op = rng.choice(["norm", "norm_backward", "orth", "muon"])
    dtype = rng.choice(["float32", "float16", "bfloat16"])
    if op in ("norm", "norm_backward"):
        dim = _log(rng, 8, 8192)
        rows = _log(rng, 1, min(262144, 32768 * 4096 // dim))
        if rng.random() < 0.5 and dim > 64:
            dim -= dim % 8
        return {"op": op, "rows": rows, "dim": dim, "pad": rng.choice([0, 0, 1, 8]), "dtype": dtype,
                "param": rng.choice([dtype, "float32"])}
    most = _ns_flops({"batch": 1, "m": 4096, "n": 4096}) // (1 if dtype == "bfloat16" else 4)
    while True:
        c = {"op": op, "batch": rng.choice([1, 1, 1, _log(rng, 2, 32)]), "m": _log(rng, 16, 6144), "n": _log(rng, 16, 6144),
             "pad": rng.choice([0, 0, 3]), "dtype": dtype}
        if rng.random() < 0.5:
            c["m"], c["n"] = -(-c["m"] // 16) * 16, -(-c["n"] // 16) * 16
        if _ns_flops(c) <= most and c["batch"] * c["m"] * c["n"] <= 1 << 25:
            break
    if op == "muon":
        c["grad"] = rng.choice([dtype, "float32"])
    return c


def _normal(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _rows_of(x, pad, dtype):
    """x's last axis as part of rows that are `pad` values longer."""
    if not pad:
        return x.to(dtype)
    wide = torch.zeros(*x.shape[:-1], x.shape[-1] + pad, dtype=dtype, device=x.device)
    wide[..., : x.shape[-1]] = x
    return wide[..., : x.shape[-1]]


def _matrix(gen, b, m, n):
    """Gradient-like matrices: a few strong directions whose weights fall off, above noise."""
    r = min(16, m, n)
    fall = torch.arange(1, r + 1, device="cuda", dtype=torch.float32) ** -1.0
    return 1e-3 * ((_normal(gen, b, m, r) * fall) @ _normal(gen, b, r, n) + 0.3 * _normal(gen, b, m, n))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] in ("norm", "norm_backward"):
        R, D = case["rows"], case["dim"]
        # pooled sums of embedding rows: each row has its own scale, the columns their own offsets
        x = _normal(gen, R, D) * (0.25 + torch.rand(R, 1, generator=gen, device="cuda") * 2) + 0.5 * _normal(gen, D)
        s["x"] = _rows_of(x, case["pad"], dt)
        pt = DTYPES[case["param"]]
        s["weight"] = (1 + 0.1 * _normal(gen, D)).to(pt)
        s["bias"] = (0.1 * _normal(gen, D)).to(pt)
        s["eps"] = 1e-5
        if case["op"] == "norm_backward":
            s["grad"] = _rows_of(1e-3 * _normal(gen, R, D), case["pad"], dt)
            xd = s["x"].double()  # the statistics that the forward pass left
            mean = xd.mean(1)
            s["mean"] = mean.float()
            s["rstd"] = (1 / torch.sqrt((xd - mean[:, None]).square().mean(1) + s["eps"])).float()
        return s
    b, m, n = case["batch"], case["m"], case["n"]
    if case["op"] == "orth":
        s["update"] = _rows_of(_matrix(gen, b, m, n), case["pad"], dt)
        return s
    s["weight"] = _rows_of(_normal(gen, b, m, n) / math.sqrt(n), case["pad"], dt)
    s["grad"] = _rows_of(_matrix(gen, b, m, n), case["pad"], DTYPES[case["grad"]])
    s["momentum"] = 5 * _matrix(gen, b, m, n)
    s["lr"], s["beta"], s["decay"] = 0.02, 0.95, 0.01
    return s


def _norm(s):
    x = s["x"].float()
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = 1 / torch.sqrt((d * d).mean(1) + s["eps"])
    y = d * rstd[:, None] * s["weight"].float() + s["bias"].float()
    return y.to(s["x"].dtype), mean, rstd


def _norm_backward(s):
    x, g = s["x"].float(), s["grad"].float()
    h = (x - s["mean"][:, None]) * s["rstd"][:, None]
    wg = g * s["weight"].float()
    dx = (wg - wg.mean(1)[:, None] - h * (wg * h).mean(1)[:, None]) * s["rstd"][:, None]
    pt = s["weight"].dtype
    return dx.to(s["x"].dtype), (g * h).sum(0).to(pt), g.sum(0).to(pt)


def _orthogonal(u, eps=1e-7):
    x = u.float()
    if x.shape[-2] > x.shape[-1]:
        x = x.transpose(-2, -1)
    x = x / (torch.sqrt((x * x).sum((-2, -1), keepdim=True)) + eps)
    for _ in range(STEPS):
        a = x @ x.transpose(-2, -1)
        x = NS_A * x + (NS_B * a + NS_C * (a @ a)) @ x
    return x.transpose(-2, -1) if u.shape[-2] > u.shape[-1] else x


def _muon(s):
    w, g, mom = s["weight"], s["grad"].float(), s["momentum"]
    mom.mul_(s["beta"]).add_(g)
    o = _orthogonal(g + s["beta"] * mom)
    scale = math.sqrt(max(1.0, w.shape[-2] / w.shape[-1]))
    w.copy_(w.float() * (1 - s["lr"] * s["decay"]) - (s["lr"] * scale) * o)
    return w, mom


def run(state):
    op = state["case"]["op"]
    if own:
        import sparse_embedding_b200 as se

        if op == "norm":
            return se.layer_norm(state["x"], state["weight"], state["bias"], eps=state["eps"], return_stats=True)
        if op == "norm_backward":
            return se.layer_norm_backward(state["grad"], state["x"], state["mean"], state["rstd"], state["weight"])
        if op == "orth":
            return se.orthogonalize(state["update"], steps=STEPS)
        se.muon_step(state["weight"], state["grad"], state["momentum"], lr=state["lr"], beta=state["beta"],
                     weight_decay=state["decay"], nesterov=True, steps=STEPS)
        return state["weight"], state["momentum"]
    if op == "norm":
        return _norm(state)
    if op == "norm_backward":
        return _norm_backward(state)
    if op == "orth":
        return _orthogonal(state["update"]).to(state["update"].dtype)
    return _muon(state)


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] in ("norm", "norm_backward"):
        R, D, p = case["rows"], case["dim"], BYTES[case["param"]]
        if case["op"] == "norm":
            return {"bytes": 2 * R * D * e + 8 * R + 2 * D * p, "flops": 8 * R * D}
        return {"bytes": 3 * R * D * e + 8 * R + 3 * D * p, "flops": 14 * R * D}
    values = case["batch"] * case["m"] * case["n"]
    moved = 2 * values * e if case["op"] == "orth" else values * (2 * e + 8 + BYTES[case["grad"]])
    return {"bytes": moved, "flops": _ns_flops(case)}


def _exact_orthogonal(u, eps=1e-7):
    """The iteration in 64 bits, from the polynomial's other side where that is the smaller one."""
    y = u / (torch.linalg.matrix_norm(u, keepdim=True) + eps)
    right = y.shape[-1] <= y.shape[-2]
    eye = torch.eye(min(y.shape[-2:]), dtype=torch.float64, device=y.device)
    for _ in range(STEPS):
        gram = torch.matmul(y.mT, y) if right else torch.matmul(y, y.mT)
        p = NS_A * eye + torch.matmul(gram, NS_B * eye + NS_C * gram)
        y = torch.matmul(y, p) if right else torch.matmul(p, y)
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "norm_backward"):
        x, w = s["x"].double(), s["weight"].double()
        if case["op"] == "norm":
            var, mean = torch.var_mean(x, dim=1, correction=0)
            rstd = torch.rsqrt(var + s["eps"])
            return (x.sub_(mean[:, None]).mul_(rstd[:, None]).mul_(w).add_(s["bias"].double()), mean, rstd)
        D = case["dim"]
        r = s["rstd"].double()[:, None]
        x.sub_(s["mean"].double()[:, None]).mul_(r)
        g = s["grad"].double()
        dw, db = torch.einsum("rd,rd->d", g, x), g.sum(0)
        g.mul_(w)
        c1, c2 = g.sum(1, keepdim=True) / D, torch.einsum("rd,rd->r", g, x)[:, None] / D
        return g.sub_(c1).sub_(x.mul_(c2)).mul_(r), dw, db
    if case["op"] == "orth":
        return _exact_orthogonal(s["update"].double())
    g, beta = s["grad"].double(), s["beta"]
    mom = beta * s["momentum"].double() + g
    o = _exact_orthogonal(g + beta * mom)
    scale = max(1.0, case["m"] / case["n"]) ** 0.5
    return s["weight"].double() * (1 - s["lr"] * s["decay"]) - s["lr"] * scale * o, mom
