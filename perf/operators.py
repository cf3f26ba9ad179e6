"""The training-step operators beside the collectives, as cases to time: the AdamW step of a gradient
shard (between ReduceScatter and AllGather), the sum of squares its clipping needs (summed over the
ranks by AllReduce), and the experts' balance loss with its counts (beside AllToAll) and its gradient.

`run` computes a case with elementary torch operations, or with this package's operators where `own`
is set.  `exact` computes it in 64 bits from the definitions.

Definitions (every tensor of a layout takes the same step):

  AdamW   c = grad_scale * min(1, max_norm / (norm + 1e-6)), norm = grad_scale * sqrt(square sum);
          nothing at all changes where the square sum is not finite; else t = t + 1 and
          g = c * grad, p = p * (1 - lr * decay), m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2,
          p = p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps).
          In 8 bits a run of 256 values of a tensor holds m as e4m3 codes times one 32-bit scale, and
          sqrt(v) likewise (a second moment above zero never becomes a zero code).
  norm    the sum of the squares of every gradient.
  balance p_t = softmax(x_t), or sigmoid(x_t) over its sum; c_e the slots of valid tokens that chose
          expert e, P_e the sum of p_te over the N valid tokens;
          loss = coef * E / (k N^2) * sum_e c_e P_e (counts carry no gradient).
"""
import math

import torch

own = False

DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 256            # values that share a scale where states are held in 8 bits
TOP = 448.0            # the largest e4m3 value
LOW = 2.0 ** -9        # the smallest above zero
LR, B1, B2, EPS, DECAY, MAX_NORM = 3e-4, 0.9, 0.95, 1e-8, 0.1, 1.0
COEF = 0.01


def listed():
    return [
        # the vectors of a small model (norm weights, biases, a router): latency counts
        {"name": "adamw_vectors", "op": "adamw", "layout": "vectors", "hidden": 643, "ffn": 1715, "layers": 4,
         "param": "f32", "grad": "f32", "master": False, "bits": 32},
        # every tensor of a few layers, weights in 32 bits
        {"name": "adamw_layers", "op": "adamw", "layout": "layers", "hidden": 1280, "ffn": 3424, "layers": 3,
         "param": "f32", "grad": "f32", "master": False, "bits": 32},
        # one flat shard: half of the 256 MiB bfloat16 bucket of the ring workload, weights with a 32-bit copy
        {"name": "adamw_shard", "op": "adamw", "layout": "flat", "count": 67108864,
         "param": "bf16", "grad": "bf16", "master": True, "bits": 32},
        # fine-tuning with states in 8 bits and weights in bfloat16 alone: many tensors, ragged ends
        {"name": "adamw8_layers", "op": "adamw", "layout": "layers", "hidden": 1283, "ffn": 3421, "layers": 3,
         "param": "bf16", "grad": "bf16", "master": False, "bits": 8},
        # the whole 256 MiB bfloat16 bucket with states in 8 bits and a 32-bit copy of the weights
        {"name": "adamw8_shard", "op": "adamw", "layout": "flat", "count": 134217728,
         "param": "bf16", "grad": "bf16", "master": True, "bits": 8},
        # the gradient norm over every tensor of a few layers
        {"name": "norm_layers", "op": "norm", "layout": "layers", "hidden": 1283, "ffn": 3421, "layers": 3, "grad": "bf16"},
        # the gradient norm of a flat 32-bit shard with an odd end
        {"name": "norm_shard", "op": "norm", "layout": "flat", "count": 67108863, "grad": "f32"},
        # the balance loss of a short sequence over a few experts: latency counts
        {"name": "balance_small", "op": "balance", "tokens": 96, "experts": 8, "k": 2, "type": "f32",
         "score": "softmax", "masked": False},
        # a packed batch with padding, sigmoid scores
        {"name": "balance_batch", "op": "balance", "tokens": 16384, "experts": 64, "k": 6, "type": "bf16",
         "score": "sigmoid", "masked": True},
        # a long batch over many experts
        {"name": "balance_long", "op": "balance", "tokens": 131072, "experts": 256, "k": 8, "type": "bf16",
         "score": "softmax", "masked": False},
        # gradients: an odd number of experts and tokens, padding
        {"name": "balance_grad_odd", "op": "balance_grad", "tokens": 10007, "experts": 60, "k": 4, "type": "f16",
         "score": "softmax", "masked": True},
        # gradients of the long batch
        {"name": "balance_grad_long", "op": "balance_grad", "tokens": 131072, "experts": 256, "k": 8, "type": "bf16",
         "score": "softmax", "masked": False},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["adamw", "adamw", "norm", "balance", "balance_grad"])
    if op in ("adamw", "norm"):
        layout = rng.choice(["flat", "layers", "vectors"])
        c = {"op": op, "layout": layout}
        if layout == "flat":
            c["count"] = _spread(rng, 1, 60_000_000)
        else:
            hidden = _spread(rng, 17, 1300)
            c |= {"hidden": hidden, "ffn": int(hidden * rng.uniform(1.5, 2.7)), "layers": rng.randint(1, 3)}
        c["grad"] = rng.choice(["f32", "bf16", "f16"])
        if op == "adamw":
            c["param"] = rng.choice(["f32", "bf16", "f16"])
            c["master"] = c["param"] != "f32" and rng.random() < 0.6
            c["bits"] = rng.choice([32, 8])
        return c
    experts = rng.choice([rng.randint(2, 16), rng.randint(17, 96), rng.randint(97, 512)])
    return {"op": op, "tokens": _spread(rng, 1, 33_000_000 // max(256, experts)), "experts": experts,
            "k": rng.randint(1, min(8, experts)), "type": rng.choice(["f32", "bf16", "f16"]),
            "score": rng.choice(["softmax", "sigmoid"]), "masked": rng.random() < 0.5}


# ---- layouts -----------------------------------------------------------------------------------

def _sizes(case):
    """(element counts, how many of them, from the first on, take weight decay)"""
    if case["layout"] == "flat":
        return [case["count"]], 1
    h, f, n = case["hidden"], case["ffn"], case["layers"]
    matrices = [] if case["layout"] == "vectors" else [3 * h * h, h * h, h * f, f * h] * n
    vectors = [h, h, 3 * h, h, f, h] * n + [h, 1]
    return matrices + vectors, len(matrices)


def _layout(case):
    """(views, total, decayed): where each tensor lies in one flat buffer, at multiples of 256"""
    sizes, decayed = _sizes(case)
    spans, at, edge = [], 0, 0
    for i, n in enumerate(sizes):
        spans.append((at, n))
        at += -(-n // BLOCK) * BLOCK
        if i + 1 == decayed:
            edge = at
    return spans, at, edge


def _cut(flat, spans, per=1):
    """the tensors of a flat buffer (per: the values that share one of the buffer's)"""
    return [flat[a // per: a // per + -(-n // per)] for a, n in spans]


# ---- inputs ------------------------------------------------------------------------------------

def _device():
    return "cuda" if torch.cuda.is_available() else "cpu"


def _gen(seed):
    return torch.Generator(device=_device()).manual_seed(seed)


def _pads(spans, total, *flats):
    """zeros behind each tensor's end: what lies there belongs to nobody"""
    for (a, n), (b, _) in zip(spans, spans[1:] + [(total, 0)]):
        if a + n < b:
            for t in flats:
                t[a + n:b] = 0


def _prepare_tensors(case, seed):
    g, dev = _gen(seed), _device()
    spans, total, edge = _layout(case)
    # gradients of very different size from place to place, as layers have
    run = torch.exp(torch.randn(total // BLOCK, generator=g, device=dev) * 1.5).repeat_interleave(BLOCK)
    grad = (torch.randn(total, generator=g, device=dev) * run * 1e-3).to(DTYPE[case["grad"]])
    s = {"case": case, "spans": spans, "total": total, "edge": edge, "grad": grad}
    if case["op"] == "norm":
        _pads(spans, total, grad)
        return s
    w = torch.randn(total, generator=g, device=dev) * 0.02
    m = torch.randn(total, generator=g, device=dev) * run * 3e-4
    v = (torch.randn(total, generator=g, device=dev) * 3e-4 * run).square() + (run * 1e-4).square()
    _pads(spans, total, grad, w, m, v)
    s["param"] = w.to(DTYPE[case["param"]])
    s["master"] = w if case["master"] else None
    s["step"] = torch.full((1,), 20 + seed % 1000, dtype=torch.int64, device=dev)
    # the square sum over every rank, as AllReduce leaves it: here 1.7 times this shard's own
    s["square_sum"] = grad.double().square().sum().reshape(1) * 1.7
    if case["bits"] == 32:
        s["m"], s["v"], s["m_scale"], s["v_scale"] = m, v, None, None
    else:
        s["m"], s["m_scale"] = _to8(m)
        s["v"], s["v_scale"] = _to8(v.sqrt(), LOW)
    return s


def _prepare_balance(case, seed):
    g, dev = _gen(seed), _device()
    t, e, k = case["tokens"], case["experts"], case["k"]
    bias = torch.randn(e, generator=g, device=dev)
    logits = (torch.randn(t, e, generator=g, device=dev) * 1.5 + bias).to(DTYPE[case["type"]])
    s = {"case": case, "logits": logits, "valid": None,
         "index": logits.float().topk(k, dim=1).indices.to(torch.int32)}
    if case["masked"]:
        s["valid"] = torch.rand(t, generator=g, device=dev) < 0.9
    if case["op"] == "balance_grad":
        # the statistics over every rank, as AllReduce leaves them, and the loss's gradient
        here = torch.ones(t, device=dev) if s["valid"] is None else s["valid"].double()
        counts = torch.zeros(e + 1, dtype=torch.float64, device=dev)
        counts.scatter_add_(0, s["index"].long().reshape(-1), here.double().repeat_interleave(k))
        counts[e] = here.sum()
        s["counts"] = counts.long() * 2
        s["grad"] = torch.rand(1, generator=g, device=dev) + 0.5
        if case["type"] == "f16":  # times the loss scale that half precision needs
            s["grad"] = s["grad"] * 2.0 ** round(math.log2(16 * t * e))
    return s


def prepare(case, seed):
    s = _prepare_balance(case, seed) if case["op"].startswith("balance") else _prepare_tensors(case, seed)
    if own and not case["op"].startswith("balance"):
        # the plan over the tensors that the optimizer keeps
        from msccl_amd import ops
        spans = s["spans"]
        grads = _cut(s["grad"], spans)
        if case["op"] == "norm":
            s["plan"] = ops.SquareSum(grads)
        else:
            decay = [DECAY if a < s["edge"] else 0.0 for a, _ in spans]
            s["plan"] = ops.AdamW(
                _cut(s["param"], spans), grads, _cut(s["m"], spans), _cut(s["v"], spans), s["step"],
                masters=_cut(s["master"], spans) if case["master"] else None,
                exp_avg_scales=_cut(s["m_scale"], spans, BLOCK) if case["bits"] == 8 else None,
                exp_avg_sq_scales=_cut(s["v_scale"], spans, BLOCK) if case["bits"] == 8 else None,
                weight_decay=decay)
    return s


# ---- the plain forms ---------------------------------------------------------------------------

def _to8(x, low=0.0):
    """e4m3 codes and a scale for each run of 256 values; `low`: no value above zero gets a code below it"""
    x = x.reshape(-1, BLOCK)
    top = x.abs().amax(1, keepdim=True)
    y = x * torch.where(top > 0, TOP / top, 0.0)
    if low:
        y = torch.where(x > 0, y.clamp_min(low), y)
    return y.to(torch.float8_e4m3fn).reshape(-1), (top * (1 / TOP)).reshape(-1)


def _from8(code, scale):
    return (code.float().reshape(-1, BLOCK) * scale.reshape(-1, 1)).reshape(-1)


def _plain_adamw(s):
    case, edge = s["case"], s["edge"]
    ok = torch.isfinite(s["square_sum"])
    coef = (MAX_NORM / (s["square_sum"].sqrt() + 1e-6)).clamp_max(1.0).float()
    s["step"] += ok
    t = s["step"].double()
    rate = (LR / (1 - B1 ** t)).float()
    root = (1 - B2 ** t).sqrt().float()
    g = s["grad"].float() * coef
    old = s["param"].float() if s["master"] is None else s["master"]
    m, v = (s["m"], s["v"]) if case["bits"] == 32 else (_from8(s["m"], s["m_scale"]), _from8(s["v"], s["v_scale"]).square())
    m = B1 * m + (1 - B1) * g
    v = B2 * v + (1 - B2) * (g * g)
    r = v.sqrt()
    p = torch.cat([old[:edge] * (1 - LR * DECAY), old[edge:]]) if edge else old
    p = p - rate * (m / (r / root + EPS))
    if s["master"] is not None:
        torch.where(ok, p, s["master"], out=s["master"])
    s["param"].copy_(torch.where(ok, p, old))
    if case["bits"] == 32:
        torch.where(ok, m, s["m"], out=s["m"])
        torch.where(ok, v, s["v"], out=s["v"])
    else:
        for new, low, code, scale in ((m, 0.0, s["m"], s["m_scale"]), (r, LOW, s["v"], s["v_scale"])):
            c, x = _to8(new, low)
            code.view(torch.uint8).copy_(torch.where(ok, c.view(torch.uint8), code.view(torch.uint8)))
            torch.where(ok, x, scale, out=scale)
    return _state(s)


def _state(s):
    return {n: s[n] for n in ("param", "master", "m", "v", "m_scale", "v_scale", "step")}


def _plain_scores(logits, score):
    x = logits.float()
    z = torch.exp(x - x.amax(1, keepdim=True)) if score == "softmax" else 1 / (1 + torch.exp(-x))
    return z, z / z.sum(1, keepdim=True)


def _plain_balance(s):
    case, index = s["case"], s["index"].long()
    e, k = case["experts"], case["k"]
    p = _plain_scores(s["logits"], case["score"])[1]
    counts = torch.zeros(e + 1, dtype=torch.int64, device=p.device)
    if s["valid"] is None:
        counts.scatter_add_(0, index.reshape(-1), torch.ones_like(index).reshape(-1))
        counts[e] = len(p)
    else:
        here = s["valid"].long()
        counts.scatter_add_(0, index.reshape(-1), here.reshape(-1, 1).expand(-1, k).reshape(-1))
        counts[e] = here.sum()
        p = torch.where(s["valid"].reshape(-1, 1), p, 0.0)
    probs = p.sum(0, dtype=torch.float64)
    n = counts[e].double()
    loss = (counts[:e].double() * probs).sum() * (COEF * e / k) / (n * n).clamp_min(1.0)
    return {"counts": counts, "probs": probs.float(), "loss": loss.float().reshape(1)}


def _plain_balance_grad(s):
    case = s["case"]
    e, k = case["experts"], case["k"]
    z, p = _plain_scores(s["logits"], case["score"])
    n = s["counts"][e].double()
    w = (s["counts"][:e].double() * (COEF * e / k) / (n * n).clamp_min(1.0) * s["grad"]).float()
    d = p * (w - (p * w).sum(1, keepdim=True))
    if case["score"] == "sigmoid":
        d = d * (1 - z)
    if s["valid"] is not None:
        d = torch.where(s["valid"].reshape(-1, 1), d, 0.0)
    return d.to(s["logits"].dtype)


# ---- one pass ----------------------------------------------------------------------------------

def run(state):
    s, case = state, state["case"]
    op = case["op"]
    if not own:
        if op == "norm":
            return s["grad"].double().square().sum().reshape(1)
        return {"adamw": _plain_adamw, "balance": _plain_balance, "balance_grad": _plain_balance_grad}[op](s)
    from msccl_amd import ops
    if op == "norm":
        return s["plan"]()
    if op == "adamw":
        s["plan"].step(LR, betas=(B1, B2), eps=EPS, grad_square_sum=s["square_sum"], max_norm=MAX_NORM)
        return _state(s)
    if op == "balance":
        counts, probs = ops.balance_stats(s["logits"], s["index"], valid=s["valid"], score=case["score"])
        return {"counts": counts, "probs": probs, "loss": ops.balance_loss(counts, probs, case["k"], COEF)}
    return ops.balance_backward(s["logits"], s["counts"], case["k"], COEF, grad_output=s["grad"], valid=s["valid"],
                                score=case["score"])


# ---- what a pass cannot do without -------------------------------------------------------------

def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] in ("adamw", "norm"):
        n = sum(_sizes(case)[0])
        if case["op"] == "norm":
            return {"bytes": n * size[case["grad"]] + 8, "flops": 2 * n}
        each = size[case["grad"]] + size[case["param"]] * (1 if case["master"] else 2) + 8 * case["master"]
        each += 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": n * each + 24, "flops": 16 * n}
    t, e, k = case["tokens"], case["experts"], case["k"]
    rows = t * e * size[case["type"]] + t * case["masked"]
    if case["op"] == "balance":
        return {"bytes": rows + t * k * 4 + 12 * e + 12, "flops": 6 * t * e}
    return {"bytes": rows + t * e * size[case["type"]] + 8 * e + 12, "flops": 9 * t * e}


# ---- the definitions in 64 bits ----------------------------------------------------------------

def _exact8(x, floor):
    """the nearest e4m3 values (even on ties) of x over its run's scale, in 64 bits"""
    runs = x.reshape(-1, BLOCK)
    scale = runs.abs().amax(dim=1) / 448
    y = torch.where(scale[:, None] > 0, runs / scale[:, None], torch.zeros_like(runs))
    exponent = torch.frexp(y)[1].clamp(min=-5) - 1
    unit = torch.ldexp(torch.ones_like(y), exponent - 3)
    q = torch.round(y / unit) * unit
    if floor:
        q = torch.where((runs > 0) & (q < 2.0 ** -9), torch.full_like(q, 2.0 ** -9), q)
    return q.reshape(-1), scale


def _exact_adamw(s):
    case = s["case"]
    total = float(s["square_sum"])
    c = min(1.0, MAX_NORM / (math.sqrt(total) + 1e-6))
    t = int(s["step"]) + 1
    g = c * s["grad"].double()
    p = (s["param"] if s["master"] is None else s["master"]).double()
    m, v = s["m"].double(), s["v"].double()
    if case["bits"] == 8:
        m = m * s["m_scale"].double().repeat_interleave(BLOCK)
        v = (v * s["v_scale"].double().repeat_interleave(BLOCK)) ** 2
    m.mul_(B1).add_(g, alpha=1 - B1)
    v.mul_(B2).addcmul_(g, g, value=1 - B2)
    del g
    p[:s["edge"]] *= 1 - LR * DECAY
    p.addcdiv_(m, v.sqrt().div_(math.sqrt(1 - B2 ** t)).add_(EPS), value=-LR / (1 - B1 ** t))
    out = {"param": p, "master": p if case["master"] else None, "step": s["step"] + 1, "m": m, "v": v,
           "m_scale": None, "v_scale": None}
    if case["bits"] == 8:
        out["m"], out["m_scale"] = _exact8(m, False)
        out["v"], out["v_scale"] = _exact8(v.sqrt(), True)
    return out


def _exact_balance(s):
    case = s["case"]
    e, k = case["experts"], case["k"]
    rows = torch.arange(case["tokens"], device=s["logits"].device) if s["valid"] is None else s["valid"].nonzero()[:, 0]
    x = s["logits"].double()
    if case["score"] == "softmax":
        a = torch.exp(x - torch.logsumexp(x, 1, keepdim=True))
        slope = None
    else:
        z = torch.special.expit(x)
        a, slope = z / z.sum(1, keepdim=True), 1 - z
    if case["op"] == "balance":
        c = torch.bincount(s["index"][rows].reshape(-1).long(), minlength=e)
        sums, n = a[rows].sum(0), len(rows)
        loss = COEF * e * float((c.double() / k * sums).sum()) / (n * n) if n else 0.0
        return {"counts": torch.cat([c, c.new_tensor([n])]), "probs": sums,
                "loss": torch.tensor([loss], dtype=torch.float64)}
    n = int(s["counts"][e])
    w = s["counts"][:e].double() / (float(n) ** 2 or 1.0) * (COEF * e * float(s["grad"]) / k)
    d = a * w - a * (a @ w)[:, None]
    if slope is not None:
        d *= slope
    keep = torch.zeros(len(x), 1, dtype=torch.float64, device=x.device)
    keep[rows] = 1
    return d * keep


def exact(case, seed):
    s = _prepare_balance(case, seed) if case["op"].startswith("balance") else _prepare_tensors(case, seed)
    if case["op"] == "norm":
        x = s["grad"].double()
        return torch.dot(x, x).reshape(1)
    return _exact_adamw(s) if case["op"] == "adamw" else _exact_balance(s)
