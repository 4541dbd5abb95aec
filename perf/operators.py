"""The operators of a training step around the graph product, as measurable cases.

A graph model whose nodes carry learned vectors (and any model over tokens)
looks rows up in a table, normalises each row between its layers, and updates
its weight matrices; a case is one call of

  lookup      out[t] = scale table[tokens[t]]                  sporder.embedding
  lookup_grad dtable[v] = scale sum of grad[t], tokens[t] = v  sporder.embedding_grad
  norm        y = weight (x - mean) / sqrt(var + eps) + bias   sporder.layer_norm
  norm_grad   its gradients by x, weight and bias              sporder.layer_norm_grad
  ortho       X = G / (|G| + eps), then some times
              X <- a X + (b A + c A A) X with A = X X^T        sporder.newton_schulz

Where `own` is false the same is computed from elementary torch operations.
Tokens are drawn with weights 1/rank ("zipf": words, or the hubs of a
power-law graph) or uniformly.
"""

import math

import torch

own = False

DEVICE = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-5
ORTHO = (3.4445, -4.7750, 2.0315)
ORTHO_EPS = 1e-7
STEPS = 5


def listed():
    return [
        # A mini-batch of sampled nodes on a small graph: latency.
        {"name": "lookup_small", "op": "lookup", "tokens": 256, "rows": 20_000, "dim": 32,
         "type": "f32", "dist": "uniform", "scaled": False},
        # The input of a token batch in half precision, scaled by sqrt(dim).
        {"name": "lookup_tokens", "op": "lookup", "tokens": 65_536, "rows": 50_000, "dim": 2048,
         "type": "bf16", "dist": "zipf", "scaled": True},
        # The gradient of the small mini-batch: latency.
        {"name": "lookup_grad_small", "op": "lookup_grad", "tokens": 1000, "rows": 20_000,
         "dim": 32, "type": "f32", "out": "f32", "dist": "uniform", "scaled": False, "pad": 0.0},
        # A padded token batch: half-precision gradients, a table gradient in 32 bits.
        {"name": "lookup_grad_tokens", "op": "lookup_grad", "tokens": 32_768, "rows": 50_000,
         "dim": 1024, "type": "bf16", "out": "f32", "dist": "zipf", "scaled": True, "pad": 0.2},
        # Sampled neighbourhoods of the GCN's graph (its node count and feature
        # width): a large table, hubs with very many occurrences.
        {"name": "lookup_grad_nodes", "op": "lookup_grad", "tokens": 500_000, "rows": 2_449_029,
         "dim": 100, "type": "f32", "out": "f32", "dist": "zipf", "scaled": False, "pad": 0.0},
        # A few rows, as in serving: latency.
        {"name": "norm_small", "op": "norm", "rows": 64, "dim": 512, "type": "bf16",
         "weights": "bf16"},
        # Every node of the GCN's graph at its hidden width.
        {"name": "norm_nodes", "op": "norm", "rows": 2_449_029, "dim": 128, "type": "f32",
         "weights": "f32"},
        # A token batch in half precision with weights in 32 bits.
        {"name": "norm_grad_tokens", "op": "norm_grad", "rows": 16_384, "dim": 4096,
         "type": "bf16", "weights": "f32"},
        # Nodes at the GCN's feature width, an odd number of them.
        {"name": "norm_grad_nodes", "op": "norm_grad", "rows": 1_000_003, "dim": 100,
         "type": "f32", "weights": "f32"},
        # The GCN's first weight matrix: latency.
        {"name": "ortho_gcn", "op": "ortho", "batch": 1, "m": 100, "n": 128, "type": "f32"},
        # A mid-size layer's update in half precision.
        {"name": "ortho_mid", "op": "ortho", "batch": 1, "m": 1024, "n": 1536, "type": "bf16"},
        # A wide layer's update in 32 bits.
        {"name": "ortho_large", "op": "ortho", "batch": 1, "m": 4096, "n": 4096, "type": "f32"},
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def _dim(rng, lo, hi):
    """A size spread over [lo, hi]'s logarithm: a power of two, or any odd number, or a
    multiple of 4 that is none of 8."""
    v = _log(rng, lo, hi)
    kind = rng.randrange(3)
    if kind == 0:
        return min(hi, max(lo, 1 << round(math.log2(v))))
    return min(hi, max(lo, int(v) | 1 if kind == 1 else int(v) // 8 * 8 + 4))


def _count(rng, v):
    """About v, odd or a round number."""
    return int(v) | 1 if v < 10 or rng.random() < 0.5 else int(v) // 10 * 10


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "lookup_grad", "norm", "norm_grad", "norm_grad",
                     "ortho", "ortho"])
    t = rng.choice(["f32", "bf16", "bf16", "f16"])
    case = {"op": op, "type": t}
    if op in ("lookup", "lookup_grad"):
        case["dim"] = _dim(rng, 16, 4096)
        case["rows"] = _count(rng, min(_log(rng, 1000, 2_400_000), 200e6 / case["dim"]))
        case["tokens"] = _count(rng, min(_log(rng, 1, 500_000), 100e6 / case["dim"]))
        case["dist"] = rng.choice(["uniform", "zipf"])
        case["scaled"] = rng.random() < 0.5
        if op == "lookup_grad":
            case["out"] = rng.choice([t, "f32"])
            case["pad"] = rng.choice([0.0, 0.0, 0.3])
    elif op in ("norm", "norm_grad"):
        case["dim"] = _dim(rng, 16, 16384)
        most = (300e6 if op == "norm" else 64e6) / case["dim"]
        case["rows"] = _count(rng, _log(rng, 1, most))
        case["weights"] = rng.choice([t, "f32"])
    else:
        m, n = _dim(rng, 16, 2500), _dim(rng, 16, 2500)
        case["m"], case["n"] = m, n
        case["batch"] = rng.choice([1, 1, 1 if m * n > 1 << 18 else rng.randint(2, 12)])
    return case


# ---- the inputs ---------------------------------------------------------------


def _tokens(case, g):
    n, rows = case["tokens"], case["rows"]
    u = torch.rand(n, device=DEVICE, generator=g, dtype=torch.float64)
    if case["dist"] == "uniform":
        ids = (u * rows).long()
    else:  # rank r with probability close to 1 / (r log rows), ids scrambled
        rank = (torch.exp(u * math.log(rows + 1.0)) - 1.0).long().clamp_(0, rows - 1)
        ids = torch.randperm(rows, device=DEVICE, generator=g)[rank]
    ids = ids.clamp_(0, rows - 1)
    if case.get("pad", 0.0) > 0.0:
        ids[torch.rand(n, device=DEVICE, generator=g) < case["pad"]] = 0
    return ids


def _scale(case):
    return math.sqrt(case["dim"]) if case["scaled"] else 1.0


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    t = TYPES[case["type"]]
    state = {"case": case}

    def normal(*shape):
        return torch.randn(*shape, device=DEVICE, generator=g)

    if case["op"] in ("lookup", "lookup_grad"):
        state["tokens"] = _tokens(case, g)
        if case["op"] == "lookup":
            state["table"] = normal(case["rows"], case["dim"]).mul_(0.02).to(t)
        else:
            state["grad"] = normal(case["tokens"], case["dim"]).mul_(1e-3).to(t)
            state["padding"] = 0 if case["pad"] > 0.0 else None
    elif case["op"] in ("norm", "norm_grad"):
        r, d, w = case["rows"], case["dim"], TYPES[case["weights"]]
        # Activations with an offset and a spread of their own in each row.
        x = normal(r, d).mul_(normal(r, 1).exp_()).add_(normal(r, 1)).to(t)
        state["x"] = x
        state["weight"] = (1.0 + 0.1 * normal(d)).to(w)
        state["bias"] = (0.1 * normal(d)).to(w)
        if case["op"] == "norm_grad":
            state["grad"] = normal(r, d).mul_(1e-2).to(t)
            var, mean = torch.var_mean(x.float(), dim=1, correction=0)
            state["mean"], state["rstd"] = mean, (var + EPS).rsqrt()
    else:
        b, m, n = case["batch"], case["m"], case["n"]
        k = max(1, min(m, n) // 8)
        # A momentum of gradients: a few strong directions over noise.
        left, right = normal(b, m, k), normal(b, k, n)
        u = torch.bmm(left, right).div_(math.sqrt(k)).add_(normal(b, m, n), alpha=0.3)
        u = u.mul_(1e-3).to(t)
        state["g"] = u if b > 1 else u[0].clone()
    return state


# ---- one pass -----------------------------------------------------------------


def _own(s):
    from chunkedgreedy_amd import sporder

    case = s["case"]
    op = case["op"]
    if op == "lookup":
        return sporder.embedding(s["table"], s["tokens"], scale=_scale(case))
    if op == "lookup_grad":
        return sporder.embedding_grad(s["grad"], s["tokens"], case["rows"], scale=_scale(case),
                                      padding_idx=s["padding"], dtype=TYPES[case["out"]])
    if op == "norm":
        return sporder.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS)
    if op == "norm_grad":
        return sporder.layer_norm_grad(s["grad"], s["x"], s["mean"], s["rstd"], s["weight"])
    return sporder.newton_schulz(s["g"], steps=STEPS, coefficients=ORTHO, eps=ORTHO_EPS)


def run(s):
    if own:
        return _own(s)
    case = s["case"]
    op = case["op"]
    t = TYPES[case["type"]]
    if op == "lookup":
        return (s["table"][s["tokens"]].float() * _scale(case)).to(t)
    if op == "lookup_grad":
        grad = s["grad"].float() * _scale(case)
        if s["padding"] is not None:
            grad = grad * (s["tokens"] != s["padding"])[:, None]
        out = torch.zeros(case["rows"], case["dim"], device=grad.device)
        return out.index_add_(0, s["tokens"], grad).to(TYPES[case["out"]])
    if op == "norm":
        x = s["x"].float()
        mean = x.mean(1, keepdim=True)
        c = x - mean
        rstd = ((c * c).mean(1, keepdim=True) + EPS).rsqrt()
        y = c * rstd * s["weight"].float() + s["bias"].float()
        return y.to(t), mean[:, 0], rstd[:, 0]
    if op == "norm_grad":
        grad, rstd = s["grad"].float(), s["rstd"][:, None]
        xhat = (s["x"].float() - s["mean"][:, None]) * rstd
        gw = grad * s["weight"].float()
        dx = (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True)) * rstd
        w = s["weight"].dtype
        return dx.to(t), (grad * xhat).sum(0).to(w), grad.sum(0).to(w)
    x = s["g"].float()
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.mT.contiguous()
    x = x / ((x * x).sum((-2, -1), keepdim=True).sqrt() + ORTHO_EPS)
    a, b, c = ORTHO
    for _ in range(STEPS):
        gram = x @ x.mT.contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.mT.contiguous() if tall else x).to(t)


# ---- what a pass has to do, and its value in 64 bits ---------------------------


def _distinct(case):
    """Expected number of distinct tokens."""
    n, rows = case["tokens"], case["rows"]
    if case["dist"] == "uniform":
        return rows * -math.expm1(n * math.log1p(-1.0 / rows)) if rows > 1 else 1.0
    r = torch.arange(rows, dtype=torch.float64)
    p = torch.log1p(1.0 / (r + 1.0)) / math.log(rows + 1.0)
    return float(-torch.expm1(n * torch.log1p(-p)).sum()) if rows > 1 else 1.0


def work(case):
    e = BYTES[case["type"]]
    if case["op"] in ("lookup", "lookup_grad"):
        n, d = case["tokens"], case["dim"]
        if case["op"] == "lookup":
            return {"bytes": 8 * n + (_distinct(case) + n) * d * e, "flops": n * d}
        return {"bytes": 8 * n + (1 - case["pad"]) * n * d * e
                + case["rows"] * d * BYTES[case["out"]], "flops": n * d}
    if case["op"] in ("norm", "norm_grad"):
        r, d, w = case["rows"], case["dim"], BYTES[case["weights"]]
        if case["op"] == "norm":
            return {"bytes": 2 * r * d * e + 8 * r + 2 * d * w, "flops": 8 * r * d}
        return {"bytes": 3 * r * d * e + 8 * r + 3 * d * w, "flops": 14 * r * d}
    m, n = sorted((case["m"], case["n"]))
    # The Gram matrix and its square are symmetric: half of each is computed.
    step = m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n
    return {"bytes": case["batch"] * 2 * m * n * e, "flops": case["batch"] * STEPS * step}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "lookup":
        return torch.index_select(s["table"].double(), 0, s["tokens"]).mul_(_scale(case))
    if op == "lookup_grad":
        keep = s["tokens"] >= 0 if s["padding"] is None else s["tokens"] != s["padding"]
        ids, order = torch.sort(s["tokens"][keep], stable=True)
        sums = s["grad"][keep].double()[order].cumsum(0)
        sums = torch.cat([torch.zeros_like(s["grad"][:1], dtype=torch.float64), sums])
        v = torch.arange(case["rows"], device=ids.device)
        first, last = torch.searchsorted(ids, v), torch.searchsorted(ids, v, right=True)
        return (sums[last] - sums[first]) * _scale(case)
    if op == "norm":
        x = s["x"].double()
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        rstd = 1.0 / torch.sqrt(var + EPS)
        y = torch.addcmul(s["bias"].double(), (x - mean).mul_(rstd), s["weight"].double())
        return y, mean[:, 0], rstd[:, 0]
    if op == "norm_grad":
        x, grad = s["x"].double(), s["grad"].double()
        d = x.shape[1]
        var, mean = torch.var_mean(x, dim=1, correction=0, keepdim=True)
        rstd = 1.0 / torch.sqrt(var + EPS)
        xhat = x.sub_(mean).mul_(rstd)
        dweight, dbias = (grad * xhat).sum(0), grad.sum(0)
        grad.mul_(s["weight"].double())
        along = (grad * xhat).sum(1, keepdim=True) / d
        dx = grad.sub_(grad.sum(1, keepdim=True) / d).sub_(xhat.mul_(along)).mul_(rstd)
        return dx, dweight, dbias
    g = s["g"].double()
    tall = g.shape[-2] > g.shape[-1]
    x = g.transpose(-1, -2).contiguous() if tall else g
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + ORTHO_EPS)
    a, b, c = ORTHO
    for _ in range(STEPS):
        xt = x.transpose(-1, -2).contiguous()
        gram = torch.matmul(x, xt)
        once = torch.matmul(gram, x)
        x = a * x + b * once + c * torch.matmul(gram, once)
    return x.transpose(-1, -2).contiguous() if tall else x
