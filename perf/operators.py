"""Performance cases of the operators at the two ends of a language model: token embedding with its gradient, layer
norm with its weight gradients, the top logits of a teacher and the distillation loss that reads them.

A case is a dict with `op` (which operator), its sizes and its options. `listed()` holds the cases that are followed,
`draw(rng)` makes one more of the same ranges. `run` computes the plain form, or where `own` is set makes the calls of
the package's own operators; `exact` is the definition in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed() -> list[dict]:
    return [
        # LayerNorm of the smoke-sized target (4 sequences of 128 tokens, 256 wide), forward and backward: launches count.
        dict(name="norm_small", op="norm", rows=512, d=256, x="bf16", w="bf16", grad=True),
        # LayerNorm of a 768-wide model at the headline batch (64 x 512 tokens), forward and backward: nine of these a step.
        dict(name="norm_768", op="norm", rows=32768, d=768, x="bf16", w="bf16", grad=True),
        # A wider stream in 32 bits with an odd width and a ragged number of rows, forward and backward.
        dict(name="norm_odd_fp32", op="norm", rows=6151, d=2047, x="fp32", w="fp32", grad=True),
        # Token embedding of the smoke-sized target: 32-bit master table, activations in bf16, forward and backward.
        dict(name="embed_small", op="embed", n=512, V=2000, d=256, table="fp32", out="bf16", grad=True),
        # Token embedding of the headline target at its batch, forward and backward.
        dict(name="embed_50k", op="embed", n=32768, V=50277, d=768, table="bf16", out="bf16", grad=True),
        # Odd width and ragged tokens over a wide vocabulary, 32-bit master table, forward and backward.
        dict(name="embed_odd_152k", op="embed", n=6151, V=151936, d=515, table="fp32", out="bf16", grad=True),
        # Eight best logits of a small vocabulary, a handful of rows: the smallest teacher.
        dict(name="top_small", op="top", n=127, V=2000, k=8, x="bf16", T=1.0),
        # Clean side of the headline target's output loss kept as 64 logits a position (16 sequences of 512).
        dict(name="top_50k", op="top", n=8192, V=50277, k=64, x="bf16", T=1.0),
        # The largest vocabulary, 32-bit logits at a raised temperature, two sequences of 512 and a ragged rest.
        dict(name="top_152k_fp32", op="top", n=1031, V=151936, k=256, x="fp32", T=2.0),
        # Next-token loss of a small vocabulary through autograd: one slot a position, some positions without a target.
        dict(name="kl_next_small", op="kl", n=512, V=2000, k=1, x="bf16", T=1.0, tail=False, form="autograd"),
        # Distillation of the headline target from 64 logits a position with the rest as one event: loss and gradient at once.
        dict(name="kl_50k", op="kl", n=8192, V=50277, k=64, x="bf16", T=1.0, tail=True, form="rows"),
        # Distillation over the largest vocabulary in 32 bits at a raised temperature, through autograd.
        dict(name="kl_152k_fp32", op="kl", n=1031, V=151936, k=32, x="fp32", T=2.0, tail=True, form="autograd"),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    """One more case: sizes spread over the logarithm of their ranges, any value of them."""
    op = rng.choice(["norm", "embed", "top", "kl"])
    while True:
        if op == "norm":
            x = rng.choice(["bf16", "bf16", "fp32"])
            c = dict(op=op, rows=_log_int(rng, 1, 65536), d=_log_int(rng, 32, 8192), x=x,
                     w=rng.choice(["fp32", x]), grad=rng.random() < 0.8)
            if c["rows"] * c["d"] <= 32768 * 768:
                return c
        elif op == "embed":
            table = rng.choice(["bf16", "fp32"])
            c = dict(op=op, n=_log_int(rng, 1, 65536), V=_log_int(rng, 50, 151936), d=_log_int(rng, 8, 2048), table=table,
                     out=rng.choice(["bf16", table]), grad=rng.random() < 0.8)
            if c["n"] * c["d"] <= 32768 * 768 and c["V"] * c["d"] <= 50277 * 768:
                return c
        else:
            c = dict(op=op, n=_log_int(rng, 1, 8192), V=_log_int(rng, 100, 151936), k=_log_int(rng, 1, 256),
                     x=rng.choice(["bf16", "bf16", "fp32"]), T=rng.choice([1.0, 1.0, 2.0]))
            if op == "kl":
                c.update(tail=rng.random() < 0.6, form=rng.choice(["rows", "autograd", "loss"]))
            if c["k"] < c["V"] and c["n"] * c["V"] * (2 if c["x"] == "fp32" else 1) <= 8192 * 50277:
                return c


# ---- states -----------------------------------------------------------------------------------------------------


def _zipf_tokens(g: torch.Generator, n: int, V: int) -> torch.Tensor:
    """Token ids as text has them: the r-th most frequent id comes up about as 1 / r."""
    p = 1.0 / torch.arange(1, V + 1, device="cuda", dtype=torch.float64)
    cdf = torch.cumsum(p / p.sum(), 0)
    rank = torch.searchsorted(cdf, torch.rand(n, device="cuda", generator=g, dtype=torch.float64)).clamp_(max=V - 1)
    return torch.randperm(V, device="cuda", generator=g)[rank]


def _logits(g: torch.Generator, n: int, V: int, dtype: torch.dtype) -> torch.Tensor:
    """Rows of logits that share a part, as a model's do (frequent tokens), and spread about a few units."""
    z = torch.randn(n, V, device="cuda", generator=g, dtype=torch.float32)
    return z.mul_(1.5).add_(torch.randn(V, device="cuda", generator=g) * 2.0).to(dtype)


def prepare(case: dict, seed: int):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, scale=1.0, shift=0.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(dtype)

    s: dict = dict(case=case)
    if case["op"] == "norm":
        n, d = case["rows"], case["d"]
        # residual streams have a mean and columns of their own size
        s["x"] = (randn(n, d, dtype=torch.float32) * randn(d, scale=0.5, shift=1.5, dtype=torch.float32)
                  + randn(d, scale=0.3, shift=0.2, dtype=torch.float32)).to(TYPES[case["x"]])
        s["w"], s["b"] = randn(d, scale=0.2, shift=1.0, dtype=TYPES[case["w"]]), randn(d, scale=0.2, dtype=TYPES[case["w"]])
        s["dy"] = randn(n, d, dtype=TYPES[case["x"]])
        for name in ("x", "w", "b"):
            s[name].requires_grad_(case["grad"])
    elif case["op"] == "embed":
        s["tokens"] = _zipf_tokens(g, case["n"], case["V"])
        s["table"] = randn(case["V"], case["d"], scale=0.02, dtype=TYPES[case["table"]]).requires_grad_(case["grad"])
        s["dy"] = randn(case["n"], case["d"], dtype=TYPES[case["out"]])
        s["scale"] = math.sqrt(case["d"])
    elif case["op"] == "top":
        s["z"] = _logits(g, case["n"], case["V"], TYPES[case["x"]])
    else:
        n, V, k = case["n"], case["V"], case["k"]
        z = _logits(g, n, V, torch.float32)
        if case["tail"]:  # a teacher near the student: its best logits and what is left
            t = z + torch.randn(n, V, device="cuda", generator=g)
            s["values"], s["indices"] = torch.topk(t, k, dim=1)
            t.scatter_(1, s["indices"], -math.inf)
            s["tail"] = torch.logsumexp(t / case["T"], 1)
            s["values"] = s["values"].to(TYPES[case["x"]])
        else:
            s["values"] = randn(n, k, scale=1.5, dtype=TYPES[case["x"]])
            start = torch.randint(V, (n, 1), device="cuda", generator=g)
            s["indices"] = (start + torch.arange(k, device="cuda") * (V // k)) % V  # the row's columns, all different
            s["tail"] = None
        s["indices"][torch.rand(n, device="cuda", generator=g) < 0.03] = -1  # positions without a target
        if case["tail"]:
            s["tail"][s["indices"][:, 0] < 0] = -math.inf
        s["z"] = z.to(TYPES[case["x"]]).requires_grad_(case["form"] == "autograd")
        s["dloss"] = torch.rand(n, device="cuda", generator=g) / n
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------


def _norm_plain(s: dict):
    x, w, b = s["x"].detach().float(), s["w"].detach().float(), s["b"].detach().float()
    c = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((c * c).mean(1, keepdim=True) + 1e-5)
    xh = c * rstd
    y = (xh * w + b).to(s["x"].dtype)
    if not s["case"]["grad"]:
        return y
    dy = s["dy"].float()
    gw = dy * w
    dx = rstd * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * xh).sum(0).to(s["w"].dtype), dy.sum(0).to(s["b"].dtype)


def _embed_plain(s: dict):
    tokens, table = s["tokens"], s["table"].detach()
    y = (table[tokens].float() * s["scale"]).to(s["dy"].dtype)
    if not s["case"]["grad"]:
        return y
    dE = torch.zeros(table.shape, device=table.device, dtype=torch.float32)
    dE.index_add_(0, tokens, s["dy"].float() * s["scale"])
    return y, dE.to(table.dtype)


def _top_plain(s: dict):
    z, k = s["z"].float(), s["case"]["k"]
    order = torch.sort(z, dim=1, descending=True, stable=True)[1][:, :k]  # equal logits stay in the order of their columns
    rest = (z / s["case"]["T"]).scatter(1, order, -math.inf)
    top = rest.amax(1, keepdim=True)
    total = torch.exp(rest - torch.where(torch.isfinite(top), top, 0.0)).sum(1)
    return torch.gather(s["z"], 1, order), order.to(torch.int32), torch.log(total) + torch.where(torch.isfinite(top), top, 0.0)[:, 0]


def _kl_plain(s: dict):
    case, idx = s["case"], s["indices"]
    z = s["z"].detach().float() / case["T"]
    used = idx >= 0
    col = idx.clamp(min=0)
    # The loss is a small difference of logarithms of long sums: the sums and what follows of them in 64 bits.
    low = torch.full((z.shape[0],), -math.inf, device=z.device)
    t = torch.where(used, s["values"].double() / case["T"], -math.inf)
    t = torch.cat([t, (low if s["tail"] is None else s["tail"]).double()[:, None]], 1)  # the K + 1 events of the teacher
    tmax = t.amax(1, keepdim=True)
    mass = torch.isfinite(tmax)
    e = torch.exp(t - torch.where(mass, tmax, 0.0))
    p = e / torch.where(mass, e.sum(1, keepdim=True), 1.0)
    zmax = z.amax(1, keepdim=True)
    ez = torch.exp(z - zmax)
    rest = ez.clone().scatter_reduce_(1, col, torch.where(used, 0.0, 1.0), "prod").sum(1, dtype=torch.float64)
    total = ez.sum(1, keepdim=True, dtype=torch.float64)
    named = torch.gather(s["z"].detach(), 1, col).double() / case["T"]
    log_all = torch.log(total) + zmax
    log_q = torch.cat([named - log_all, (torch.log(rest)[:, None] + zmax - log_all)], 1)
    terms = p * (torch.log(p) - log_q)
    loss = torch.where(p > 0, terms, 0.0).sum(1).float()
    if case["form"] == "loss":
        return loss
    live = mass.double()
    r = p[:, -1:]
    coef = live / total - torch.where(r > 0, r / rest[:, None], 0.0)
    dz = ez * coef.float()
    dz.scatter_(1, col, torch.where(used, (torch.exp(named - log_all) * live - p[:, :-1]).float(), torch.gather(dz, 1, col)))
    dz = dz / case["T"]
    if case["form"] == "autograd":
        dz = dz * s["dloss"][:, None]
    return loss, dz.to(s["z"].dtype)


def _own(s: dict):
    from param_decomp_b200.ops.elementwise import layer_norm
    from param_decomp_b200.ops.embedding import embedding
    from param_decomp_b200.ops.top_logits import top_kl, top_kl_rows, top_logits

    case = s["case"]
    if case["op"] == "norm":
        y = layer_norm(s["x"], s["w"], s["b"], 1e-5)
        return (y, *torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])) if case["grad"] else y
    if case["op"] == "embed":
        y = embedding(s["tokens"], s["table"], s["scale"], out_dtype=s["dy"].dtype)
        return (y, *torch.autograd.grad(y, (s["table"],), s["dy"])) if case["grad"] else y
    if case["op"] == "top":
        return tuple(top_logits(s["z"], case["k"], case["T"]))
    args = (s["z"], s["indices"], s["values"], s["tail"], case["T"])
    if case["form"] == "autograd":
        loss = top_kl(*args)
        return (loss, *torch.autograd.grad(loss, (s["z"],), s["dloss"]))
    loss, dz = top_kl_rows(*args, want_grad=case["form"] == "rows")
    return (loss, dz) if case["form"] == "rows" else loss


def run(s: dict):
    if own:
        return _own(s)
    return {"norm": _norm_plain, "embed": _embed_plain, "top": _top_plain, "kl": _kl_plain}[s["case"]["op"]](s)


def work(case: dict) -> dict:
    size = {"bf16": 2, "fp32": 4}
    if case["op"] == "norm":
        e, b, w = case["rows"] * case["d"], size[case["x"]], case["d"] * size[case["w"]]
        return {"bytes": e * b * (4 if case["grad"] else 2) + w * (4 if case["grad"] else 2),  # x, y (dy, dx), parameters (gradients)
                "flops": e * (22 if case["grad"] else 8)}
    if case["op"] == "embed":
        n, V, d, t, o = case["n"], case["V"], case["d"], size[case["table"]], size[case["out"]]
        back = n * d * o + V * d * t if case["grad"] else 0
        return {"bytes": n * 8 + min(n, V) * d * t + n * d * o + back, "flops": n * d * (3 if case["grad"] else 1)}
    n, V, k, b = case["n"], case["V"], case["k"], size[case["x"]]
    if case["op"] == "top":
        return {"bytes": n * V * b + n * k * (b + 4) + n * 4, "flops": n * V * 4}
    grad = case["form"] != "loss"
    return {"bytes": n * V * b * (2 if grad else 1) + n * k * (8 + b) + n * 4 * (2 + (case["form"] == "autograd")),
            "flops": n * V * (7 if grad else 4)}


# ---- the definition in 64 bits ----------------------------------------------------------------------------------


def _norm_exact(s: dict):
    x = s["x"].detach().double().requires_grad_(True)
    w, b = (s[k].detach().double().requires_grad_(True) for k in ("w", "b"))
    var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
    y = (x - mean) / torch.sqrt(var + 1e-5) * w + b
    if not s["case"]["grad"]:
        return y.detach()
    return (y.detach(), *torch.autograd.grad(y, (x, w, b), s["dy"].double()))


def _embed_exact(s: dict):
    tokens, table = s["tokens"], s["table"].detach().double()
    y = torch.index_select(table, 0, tokens) * s["scale"]
    if not s["case"]["grad"]:
        return y
    # rows gathered by token, then differences of their running sums at the ends of each token's run
    order = torch.argsort(tokens, stable=True)
    counts = torch.bincount(tokens, minlength=s["case"]["V"])
    total = torch.cumsum(s["dy"].double()[order], 0)
    total = torch.cat([torch.zeros_like(total[:1]), total])
    ends = torch.cumsum(counts, 0)
    return y, (total[ends] - total[ends - counts]) * s["scale"]


def _top_exact(s: dict):
    case, values, indices, tails = s["case"], [], [], []
    for z in s["z"].split(512):
        # one whole number a logit that orders by value first and by column second
        zf = z.float() + 0.0
        bits = zf.view(torch.int32).long()
        bits = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        key = bits * (1 << 20) + (case["V"] - torch.arange(case["V"], device=z.device))
        idx = torch.topk(key, case["k"], dim=1, sorted=True)[1]
        rest = z.double() / case["T"]
        rest[torch.arange(z.shape[0], device=z.device)[:, None], idx] = -math.inf
        values.append(torch.gather(z.double(), 1, idx))
        indices.append(idx.to(torch.int32))
        tails.append(torch.logsumexp(rest, 1))
    return torch.cat(values), torch.cat(indices), torch.cat(tails)


def _kl_exact(s: dict):
    case, losses, grads = s["case"], [], []
    n = case["n"]
    for a in range(0, n, 256):
        rows = slice(a, min(n, a + 256))
        z = s["z"].detach()[rows].double().requires_grad_(True)
        idx = s["indices"][rows]
        named = idx[:, 0] >= 0
        teacher = s["values"][rows].double() / case["T"]
        if s["tail"] is not None:
            teacher = torch.cat([teacher, s["tail"][rows].double()[:, None]], 1)
        logp = torch.log_softmax(torch.where(named[:, None], teacher, 0.0), 1)
        logq = torch.log_softmax(z / case["T"], 1)
        events = torch.gather(logq, 1, idx.clamp(min=0))
        if s["tail"] is not None:
            others = torch.ones_like(logq, dtype=torch.bool).scatter(1, idx.clamp(min=0), False)
            events = torch.cat([events, torch.logsumexp(logq.masked_fill(~others, -math.inf), 1, keepdim=True)], 1)
        p = torch.where(named[:, None], logp.exp(), 0.0)
        loss = torch.where(p > 0, p * (logp - events), 0.0).sum(1)
        losses.append(loss.detach())
        if case["form"] != "loss":
            up = s["dloss"][rows].double() if case["form"] == "autograd" else torch.ones_like(loss)
            grads.append(torch.autograd.grad(loss, z, up)[0])
    return (torch.cat(losses), torch.cat(grads)) if grads else torch.cat(losses)


def exact(case: dict, seed: int):
    return {"norm": _norm_exact, "embed": _embed_exact, "top": _top_exact, "kl": _kl_exact}[case["op"]](prepare(case, seed))
