"""Measured cases of the microscaled 4-bit matrices and of the move sampler.

Three operators, each in a plain form (elementary torch operations in 32
bits) and through the package's own entry points (`own`):

    values   x -> its microscaled 4-bit form -> the values that form holds
    product  relu?(Q(x) . Q(w)^T + bias), w quantised beforehand
    sample   one move per row of logits: legal mask, temperature, top-k,
             top-p and min-p, from given uniform numbers

Q is the 4-bit microscaled form: blocks of 32 along a row share the scale
2^(floor(log2(max |x|)) - 2) (exponent at least -127), and each element is
x / scale rounded to nearest even onto {0, .5, 1, 1.5, 2, 3, 4, 6}, at most
6. A block that holds an infinity or a NaN is NaN throughout.

The sampler: with l the legal, non-NaN logits above -inf and m their
maximum, x = 0 where l = m and (l - m) / T elsewhere. In descending order of
l (ties: lower index first) top-k keeps the first k, top-p of those the
shortest prefix whose share of their mass reaches p, min-p those with
exp(x) >= min_p; the first is always kept. Among the kept the move is the
argmax of x - log(-log u), u clamped into [2^-25, 1 - 2^-24] (ties: lower
index), and logprob is x[move] - log(sum exp x) over all of l. T <= 0 takes
the largest logit (logprob 0); a row without any l gives -1 and -inf.
"""
import math
import os
import sys

import torch

own = False

U_LOW, U_HIGH = 2.0 ** -25, 1.0 - 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "bf16": 2}


def _ops():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "alphazero-go_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import azb_ops

    return azb_ops


# ------------------------------------------------------------------- cases


def listed():
    return [
        # One position's policy features of the 19x19 head (2 x 361), as a
        # single-position evaluation quantises them.
        {"name": "values_one_row", "op": "values", "rows": 1, "cols": 722, "dtype": "f32"},
        # A self-play batch of encoded 19x19 positions (4 planes x 361).
        {"name": "values_batch", "op": "values", "rows": 1024, "cols": 1444, "dtype": "bf16"},
        # A weight matrix or a long prompt's activations, quantised in one go.
        {"name": "values_large", "op": "values", "rows": 16384, "cols": 8192, "dtype": "bf16"},
        # One token through a square layer: latency and weight streaming.
        {"name": "product_one_row", "op": "product", "m": 1, "n": 4096, "k": 4096, "dtype": "bf16", "bias": False,
         "relu": False},
        # A decode batch through a widening layer.
        {"name": "product_decode", "op": "product", "m": 32, "n": 16384, "k": 4096, "dtype": "bf16", "bias": False,
         "relu": True},
        # The 19x19 policy head's FC (722 -> 362) on a full self-play batch.
        {"name": "product_policy_fc", "op": "product", "m": 1024, "n": 362, "k": 722, "dtype": "f32", "bias": True,
         "relu": False},
        # Nothing a multiple of anything: a ragged batch.
        {"name": "product_ragged", "op": "product", "m": 333, "n": 1111, "k": 2501, "dtype": "f32", "bias": True,
         "relu": True},
        # A long prompt or a training-size batch: tensor-core bound.
        {"name": "product_large", "op": "product", "m": 8192, "n": 8192, "k": 8192, "dtype": "bf16", "bias": False,
         "relu": False},
        # The move of one 19x19 game.
        {"name": "sample_one_game", "op": "sample", "rows": 1, "cols": 362, "dtype": "f32", "legal": True,
         "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0},
        # The moves of a full self-play batch: opening rows at temperature 1,
        # later ones greedy ("mixed": per-row temperatures), filtered.
        {"name": "sample_selfplay", "op": "sample", "rows": 1024, "cols": 362, "dtype": "f32", "legal": True,
         "temperature": "mixed", "top_k": 40, "top_p": 0.95, "min_p": 0.01},
        # A few sequences over a wide vocabulary of odd size, all filters.
        {"name": "sample_wide", "op": "sample", "rows": 8, "cols": 50001, "dtype": "bf16", "legal": False,
         "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.02},
        # A large batch over a wide vocabulary, nucleus only.
        {"name": "sample_large", "op": "sample", "rows": 512, "cols": 131072, "dtype": "f32", "legal": False,
         "temperature": 1.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["values", "product", "product", "sample", "sample"])
    dtype = rng.choice(["f32", "bf16"])
    if op == "values":
        rows, cols = _log_int(rng, 1, 16384), _log_int(rng, 1, 8192)
        return {"op": op, "rows": rows, "cols": cols, "dtype": dtype if rows * cols <= 1 << 26 else "bf16"}
    if op == "product":
        return {"op": op, "m": _log_int(rng, 1, 8192), "n": _log_int(rng, 1, 8192), "k": _log_int(rng, 1, 8192),
                "dtype": dtype, "bias": rng.random() < 0.5, "relu": rng.random() < 0.5}
    cols = _log_int(rng, 1, 131072)
    rows = _log_int(rng, 1, max(1, min(1024, (1 << 26) // cols)))
    return {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "legal": rng.random() < 0.5,
            "temperature": rng.choice(["mixed", 0.5, 0.8, 1.0, 1.3]),
            "top_k": rng.choice([0, 0, _log_int(rng, 1, 1000)]),
            "top_p": rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
            "min_p": rng.choice([0.0, 0.0, round(rng.uniform(0.005, 0.2), 3)])}


def work(case):
    es = SIZES[case["dtype"]]
    if case["op"] == "values":
        n, blocks = case["rows"] * case["cols"], case["rows"] * -(-case["cols"] // 32)
        return {"bytes": 2 * es * n + 17 * blocks, "flops": 2 * n}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": es * m * k + 17 * n * -(-k // 32) + es * m * n + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    b, v = case["rows"], case["cols"]
    # Only kept tokens need their random number: k of them under top-k, some
    # number that the data decides (counted as one) under top-p or min-p.
    plain = case["top_p"] >= 1.0 and case["min_p"] <= 0.0
    kept = min(case["top_k"], v) if case["top_k"] else (v if plain else 1)
    return {"bytes": b * (v * (es + (1 if case["legal"] else 0)) + 4 * kept + 12), "flops": 4 * b * v}


# ------------------------------------------------------------------ inputs


def _activations(rows, cols, dtype, g):
    """Normal activations whose channels differ in scale, as a layer's do."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    return x.mul_(torch.randn(cols, generator=g, device="cuda").mul_(0.7).exp_()).to(DTYPES[dtype])


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "values":
        return {"x": _activations(case["rows"], case["cols"], case["dtype"], g)}
    if case["op"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        w = torch.randn(n, k, generator=g, device="cuda").mul_(k ** -0.5).to(DTYPES[case["dtype"]])
        return {"x": _activations(m, k, case["dtype"], g), "w": w,
                "bias": torch.randn(n, generator=g, device="cuda").mul_(0.1) if case["bias"] else None}
    b, v = case["rows"], case["cols"]
    s = {"logits": torch.randn(b, v, generator=g, device="cuda").mul_(3.0).to(DTYPES[case["dtype"]]),
         "noise": torch.rand(b, v, generator=g, device="cuda"), "legal": None}
    if case["legal"]:   # the pass (the last move) is always legal
        s["legal"] = torch.rand(b, v, generator=g, device="cuda") < 0.6
        s["legal"][:, -1] = True
    if case["temperature"] == "mixed":
        s["temperature"] = (torch.rand(b, generator=g, device="cuda") < 0.5).float()
    else:
        s["temperature"] = float(case["temperature"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if case["op"] == "product":   # the weights are laid out once
        w = s.pop("w")
        s["w"] = _ops().mx4_quantise(w) if own else _plain_quantised(w)
    return s


# ------------------------------------------------------------- plain forms


def _plain_quantised(x):
    """The values that x's 4-bit form holds, in 32 bits."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = torch.zeros(rows, blocks * 32, device=x.device)
    v[:, :cols] = x.float()
    v = v.view(rows, blocks, 32)
    top = v.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(top)
    _, e = torch.frexp(torch.where(bad, torch.ones_like(top), top))
    e = torch.where(top == 0, torch.full_like(e, -127), (e - 3).clamp(min=-127))
    a = torch.ldexp(v, -e)
    mag = torch.zeros_like(a)
    a = a.abs()
    for edge, step in ((0.25, 0.5), (1.25, 0.5), (2.5, 1.0), (5.0, 2.0)):   # ties go down
        mag += (a > edge) * step
    for edge, step in ((0.75, 0.5), (1.75, 0.5), (3.5, 1.0)):               # ties go up
        mag += (a >= edge) * step
    out = torch.ldexp(torch.copysign(mag, v), e)
    return out.masked_fill_(bad, float("nan")).view(rows, blocks * 32)[:, :cols]


def _plain_sample(logits, noise, legal, temperature, top_k, top_p, min_p):
    l = logits.float()
    out = torch.isnan(l)
    if legal is not None:
        out |= ~legal
    l = l.masked_fill(out, -math.inf)
    m = l.amax(-1, keepdim=True)
    t = torch.as_tensor(temperature, dtype=torch.float32, device=l.device).expand(l.shape[0]).unsqueeze(1)
    greedy = (t <= 0).squeeze(1)
    x = (l - m) / torch.where(t > 0, t, torch.ones_like(t))
    x = torch.where(l == m, torch.zeros_like(x), x).masked_fill(l == -math.inf, -math.inf)
    w = x.exp()
    z = w.sum(-1)
    _, order = torch.sort(l, dim=-1, descending=True, stable=True)
    ws = w.gather(1, order)
    if top_k > 0:
        ws[:, top_k:] = 0
    zk = ws.sum(-1, keepdim=True)
    before = ws.cumsum(-1) - ws
    keep = (before < top_p * zk) if top_p < 1 else torch.ones_like(ws, dtype=torch.bool)
    if top_k > 0:
        keep[:, top_k:] = False
    if min_p > 0:
        keep &= ws >= min_p
    keep[:, 0] = True
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    u = noise.clamp(U_LOW, U_HIGH)
    key = (x - torch.log(-torch.log(u))).masked_fill(~kept, -math.inf)
    move = torch.where(greedy, l.argmax(-1), key.argmax(-1))
    logprob = x.gather(1, move.unsqueeze(1)).squeeze(1) - z.log()
    logprob = torch.where(greedy, torch.zeros_like(logprob), logprob)
    none = m.squeeze(1) == -math.inf
    return [move.masked_fill(none, -1), logprob.masked_fill(none, -math.inf)]


def run(state):
    case = state["case"]
    if case["op"] == "values":
        x = state["x"]
        if own:
            ops = _ops()
            return ops.mx4_values(ops.mx4_quantise(x), x.dtype)
        return _plain_quantised(x).to(x.dtype)
    if case["op"] == "product":
        x = state["x"]
        if own:
            return _ops().mx4_product(x, state["w"], bias=state["bias"], relu=case["relu"], dtype=x.dtype)
        y = _plain_quantised(x) @ state["w"].t()
        if state["bias"] is not None:
            y += state["bias"]
        return (y.clamp_(min=0) if case["relu"] else y).to(x.dtype)
    args = (state["logits"], state["noise"])
    if own:
        move, logprob = _ops().sample_moves(*args, legal=state["legal"], temperature=state["temperature"],
                                            top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])
        return [move, logprob]
    return _plain_sample(*args, state["legal"], state["temperature"], case["top_k"], case["top_p"], case["min_p"])


# ------------------------------------------------------------------- exact


def _exact_quantised(x):
    """The 4-bit form's values in 64 bits: the scale from the block maximum's
    exponent field, each element the nearest of the eight magnitudes (of two
    equally near the one with the even code)."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    out = torch.empty(rows, cols, dtype=torch.float64, device=x.device)
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    chunk = max(1, (1 << 24) // (blocks * 32))
    for r in range(0, rows, chunk):
        v = torch.nn.functional.pad(x[r:r + chunk].float(), (0, blocks * 32 - cols)).view(-1, blocks, 32)
        field = (v.abs().amax(-1).view(torch.int32) >> 23) & 255
        e = (field - 127 - 2).clamp(min=-127)
        scale = ((e.long() + 1023) << 52).view(torch.float64).unsqueeze(-1)   # 2^e
        y = v.double() / scale
        a = y.abs()
        best = torch.zeros_like(a)
        gap = a.clone()
        for code in range(1, 8):
            d = (a - table[code]).abs()
            take = (d < gap) | ((d == gap) & (code % 2 == 0))
            best = torch.where(take, table[code], best)
            gap = torch.where(take, d, gap)
        y = torch.where(y < 0, -best, best) * scale
        y.masked_fill_((~torch.isfinite(v)).any(-1, keepdim=True), math.nan)
        out[r:r + chunk] = y.reshape(-1, blocks * 32)[:, :cols]
    return out


def _exact_sample(s, case):
    moves, logprobs = [], []
    for r in range(case["rows"]):
        l = s["logits"][r].double()
        open_ = ~torch.isnan(l) & (l > -math.inf)
        if s["legal"] is not None:
            open_ &= s["legal"][r]
        ids = open_.nonzero().squeeze(1)
        if ids.numel() == 0:
            moves.append(torch.full((), -1, dtype=torch.int64, device=l.device))
            logprobs.append(torch.full((), -math.inf, dtype=torch.float64, device=l.device))
            continue
        ls, place = torch.sort(l[ids], descending=True, stable=True)
        ids = ids[place]
        t = s["temperature"] if isinstance(s["temperature"], float) else float(s["temperature"][r])
        if t <= 0:
            moves.append(ids[0])
            logprobs.append(torch.zeros((), dtype=torch.float64, device=l.device))
            continue
        t = float(torch.tensor(t, dtype=torch.float32))
        x = torch.where(ls == ls[0], torch.zeros_like(ls), (ls - ls[0]) / t)
        w = torch.exp(x)
        n = min(case["top_k"], ids.numel()) if case["top_k"] > 0 else ids.numel()
        keep = torch.ones(n, dtype=torch.bool, device=l.device)
        if case["top_p"] < 1:
            ahead = torch.cat([w.new_zeros(1), w[:n].cumsum(0)[:-1]])
            keep &= ahead < float(torch.tensor(case["top_p"], dtype=torch.float32)) * w[:n].sum()
        if case["min_p"] > 0:
            keep &= w[:n] >= float(torch.tensor(case["min_p"], dtype=torch.float32))
        keep[0] = True
        u = s["noise"][r].double()[ids[:n]].clamp(U_LOW, U_HIGH)
        key = (x[:n] - torch.log(-torch.log(u))).masked_fill(~keep, -math.inf)
        best = ids[:n].masked_fill(key < key.max(), case["cols"]).min()   # ties: lower index
        moves.append(best)
        logprobs.append(x[(ids == best).nonzero()[0, 0]] - torch.log(w.sum()))
    return [torch.stack(moves), torch.stack(logprobs)]


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "values":
        return _exact_quantised(s["x"])
    if case["op"] == "product":
        y = _exact_quantised(s["x"]) @ _exact_quantised(s["w"]).t()
        if s["bias"] is not None:
            y = y + s["bias"].double()
        return torch.where(y > 0, y, torch.zeros_like(y)) if case["relu"] else y
    return _exact_sample(s, case)
