"""The 8-bit path through the end of a layer and of a model, operator by operator, in plain torch operations and in the
library's calls: which calls a serving program makes, at which sizes.

  norm      residual addition, root-mean-square norm and quantisation of the rows to 8 bits (``add_rmsnorm_i8``)
  quantize  quantisation of rows alone, the input of a projection that follows no norm (``quantize_i8``)
  matmul    product of 8-bit rows with 8-bit weights, scales per row and per channel (``matmul_i8``)
  logprobs  log probabilities of given tokens, entropy and the most likely tokens of each row (``logprobs``)

Sizes are those of the benchmark's configurations (hidden sizes 4096 and 8192, feed-forward sizes 14336 and 28672, 128256
tokens) and ragged ones between.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
HEAD = 128256


def listed():
    return [
        # one token's hidden state ahead of a layer's projections: nothing but latency
        {"name": "norm_1", "op": "norm", "m": 1, "k": 4096, "type": "f32", "residual": True},
        # a ragged batch whose rows start at odd addresses, first layer (no residual yet)
        {"name": "norm_301_odd", "op": "norm", "m": 301, "k": 5001, "type": "f16", "residual": False},
        # a long prompt through a 70B layer: the residual stream in float
        {"name": "norm_2048", "op": "norm", "m": 2048, "k": 8192, "type": "f32", "residual": True},
        # the input of a down projection, a prompt of 512 rows
        {"name": "quantize_512", "op": "quantize", "m": 512, "k": 14336, "type": "bf16"},
        # the key or value projection of one token
        {"name": "matmul_1", "op": "matmul", "m": 1, "n": 1024, "k": 4096, "type": "f32", "bias": False},
        # the output head of one token
        {"name": "matmul_head_1", "op": "matmul", "m": 1, "n": HEAD, "k": 4096, "type": "f32", "bias": False},
        # Q+K+V of a small batch, with the bias that some models have there
        {"name": "matmul_13", "op": "matmul", "m": 13, "n": 6144, "k": 4096, "type": "f32", "bias": True},
        # a short prompt, odd in every direction
        {"name": "matmul_203_odd", "op": "matmul", "m": 203, "n": 14335, "k": 4093, "type": "f16", "bias": False},
        # a long prompt through the up projection of a 70B layer: the largest
        {"name": "matmul_2048", "op": "matmul", "m": 2048, "n": 28672, "k": 8192, "type": "bf16", "bias": False},
        # the answer of one decoded token: its log probability and the twenty best
        {"name": "logprobs_1", "op": "logprobs", "m": 1, "v": HEAD, "type": "f32", "given": 1, "top": 20, "masked": False},
        # a batch under a grammar's mask, eight candidate tokens each, odd vocabulary
        {"name": "logprobs_48_masked", "op": "logprobs", "m": 48, "v": 32003, "type": "bf16", "given": 8, "top": 5, "masked": True},
        # scoring a prompt: the log probability of every next token, with entropy and the best five
        {"name": "logprobs_512", "op": "logprobs", "m": 512, "v": HEAD, "type": "f32", "given": 1, "top": 5, "masked": False},
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm", "quantize", "matmul", "matmul", "logprobs", "logprobs"])
    kind = rng.choice(["f32", "f32", "f16", "bf16"])
    if op in ("norm", "quantize"):
        case = {"op": op, "m": log_int(1, 2048), "k": log_int(256, 16384), "type": kind}
        case["m"] = min(case["m"], 2048 * 8192 // case["k"])
        return dict(case, residual=rng.random() < 0.7) if op == "norm" else case
    if op == "matmul":
        case = {"op": op, "m": log_int(1, 2048), "n": log_int(64, 32768), "k": log_int(256, 16384), "type": kind, "bias": rng.random() < 0.3}
        case["m"] = max(1, min(case["m"], 2048 * 28672 * 8192 // (case["n"] * case["k"])))
        return case
    v = log_int(1000, 131072)
    return {"op": op, "m": min(log_int(1, 512), 512 * HEAD // v), "v": v, "type": kind, "given": rng.choice([1, 1, 1, 4, 16]),
            "top": rng.choice([0, 1, 5, 8, 20, 32]), "masked": rng.random() < 0.3}


# ---- inputs ------------------------------------------------------------------------------------------------------------

def _codes(rows, k, gen):
    """Codes of rows that were quantised by their largest value: bell-shaped, about 30 wide.  Rows lie a multiple of 16 bytes
    apart; what is between them is never a row's."""
    pad = (k + 15) // 16 * 16
    c = torch.empty((rows, pad), dtype=torch.int8, device="cuda")
    for r in range(0, rows, 16384):
        c[r:r + 16384] = torch.randn((min(16384, rows - r), pad), generator=gen, device="cuda").mul_(30).round_().clamp_(-127, 127).to(torch.int8)
    return c[:, :k]


def _uniform(n, lo, hi, gen):
    return torch.empty(n, device="cuda").uniform_(lo, hi, generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    m, t = case["m"], DTYPE[case["type"]]
    s = dict(case)
    if case["op"] in ("norm", "quantize"):
        k = case["k"]
        # hidden states: most channels near one, some far larger, as residual streams are
        wide = torch.where(_uniform(k, 0, 1, gen) < 0.01, 20.0, 1.0)
        s["x"] = (torch.randn((m, k), generator=gen, device="cuda") * wide).to(t)
        if case["op"] == "norm":
            s["w"] = _uniform(k, 0.2, 2.0, gen)
            s["r"] = (torch.randn((m, k), generator=gen, device="cuda") * wide * 2).to(t) if case["residual"] else None
    elif case["op"] == "matmul":
        n, k = case["n"], case["k"]
        s["x"], s["sx"] = _codes(m, k, gen), _uniform(m, 0.005, 0.05, gen)
        s["w"], s["sw"] = _codes(n, k, gen), _uniform(n, 2e-4, 2e-3, gen)
        s["b"] = torch.randn(n, generator=gen, device="cuda") if case["bias"] else None
    else:
        v = case["v"]
        x = torch.randn((m, v), generator=gen, device="cuda") * 2.5
        x += 8.0 * (_uniform(m * v, 0, 1, gen).view(m, v) < 20.0 / v)       # a few tokens stand out
        if case["masked"]:
            live = _uniform(m * v, 0, 1, gen).view(m, v) < _uniform(m, 0, 0.05, gen).view(m, 1)
            live[m // 2] &= m < 8                                            # one row of a larger batch has no token left
            x.masked_fill_(~live, -math.inf)
        s["x"] = x.to(t)
        s["given"] = torch.randint(0, v, (m, case["given"]), generator=gen, device="cuda", dtype=torch.int32)
    return s


# ---- the operators ------------------------------------------------------------------------------------------------------

_contexts = {}


def _context():
    """One handle for the whole process, as a serving program keeps it."""
    import backpack_b200 as bp

    dev = torch.cuda.current_device()
    if dev not in _contexts:
        _contexts[dev] = bp.Q4KContext(dev)
    return _contexts[dev]


def _rows_own(s):
    ctx = _context()
    if s["op"] == "norm":
        rows, total = ctx.add_rmsnorm_i8(s["x"], s["w"], EPS, residual=s["r"])
        return {"values": rows.codes * rows.scales[:, None], "scales": rows.scales, "sum": total if s["r"] is not None else None}
    rows = ctx.quantize_i8(s["x"])
    return {"values": rows.codes * rows.scales[:, None], "scales": rows.scales}


def _rows_plain(s):
    v = s["x"].float()
    if s.get("r") is not None:
        v = v + s["r"].float()
    # the codes next to a border between two of them need the products in 64 bits; the norm is a factor of the whole row and of
    # its largest value, so it is in the scale alone
    p = v.double() * s["w"].double() if s["op"] == "norm" else v.double()
    a = p.abs().amax(dim=1, keepdim=True)
    codes = torch.round(127.0 * p / torch.where(a == 0, 1.0, a))
    scales = a / 127.0
    if s["op"] == "norm":
        scales = scales / torch.sqrt((v * v).mean(dim=1, keepdim=True) + EPS).double()
    out = {"values": (codes * scales).float(), "scales": scales[:, 0].float()}
    if s["op"] == "norm":
        out["sum"] = v.to(s["x"].dtype) if s["r"] is not None else None
    return out


def _matmul_own(s):
    import backpack_b200 as bp

    return _context().matmul_i8(bp.I8Rows(s["x"], s["sx"]), bp.I8Rows(s["w"], s["sw"]), bias=s["b"], dtype=DTYPE[s["type"]])


def _matmul_plain(s):
    y = (s["x"].float() @ s["w"].float().T) * s["sx"][:, None] * s["sw"]
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(DTYPE[s["type"]])


def _logprobs_own(s):
    r = _context().logprobs(s["x"], given=s["given"], top=s["top"])
    return {"given": r.given, "entropy": r.entropy, "top_ids": r.top_ids if s["top"] else None, "top": r.top if s["top"] else None}


def _logprobs_plain(s):
    x = s["x"].float()
    m = x.amax(dim=1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)                # a row with no token left: every log probability is -infinity
    u = x - m
    e = torch.exp(u)
    total = e.sum(dim=1, keepdim=True)
    lse = torch.log(total)

    def lp(ids):
        at = torch.gather(u, 1, ids)
        return torch.where(at == -math.inf, -math.inf, at - lse)

    mean = torch.where(e > 0, e * u, 0.0).sum(dim=1, keepdim=True) / torch.where(total == 0, 1.0, total)
    entropy = torch.where(total == 0, 0.0, lse - mean)[:, 0]
    out = {"given": lp(s["given"].long()), "entropy": entropy, "top_ids": None, "top": None}
    if s["top"]:
        # values in the order of whole numbers, the lowest index first among equal ones
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
        key = (order << 32) + (x.shape[1] - 1 - torch.arange(x.shape[1], device=x.device))
        best = torch.topk(key, s["top"], dim=1).values
        ids = x.shape[1] - 1 - (best & 0xFFFFFFFF)
        out["top_ids"], out["top"] = ids.int(), lp(ids)
    return out


def run(s):
    if own:
        return _rows_own(s) if s["op"] in ("norm", "quantize") else _matmul_own(s) if s["op"] == "matmul" else _logprobs_own(s)
    return _rows_plain(s) if s["op"] in ("norm", "quantize") else _matmul_plain(s) if s["op"] == "matmul" else _logprobs_plain(s)


def work(case):
    m, e = case["m"], BYTES[case["type"]]
    if case["op"] in ("norm", "quantize"):
        k, norm = case["k"], case["op"] == "norm"
        streams = 3 if norm and case["residual"] else 1
        return {"bytes": m * k * (streams * e + 1) + 4 * m + (4 * k if norm else 0), "flops": (8 if norm else 4) * m * k}
    if case["op"] == "matmul":
        n, k = case["n"], case["k"]
        return {"bytes": m * k + n * k + e * m * n + 4 * (m + n) + (4 * n if case["bias"] else 0), "flops": 2 * m * n * k}
    v = case["v"]
    return {"bytes": e * m * v + 8 * m * case["given"] + 4 * m + 8 * m * case["top"], "flops": 5 * m * v}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "quantize"):
        x = s["x"].double()
        residual = s.get("r")
        if residual is not None:
            x = (x + residual.double()).float().double()   # the stream is a float
        y = x * s["w"].double() if case["op"] == "norm" else x
        peak = y.abs().max(dim=1).values
        step = peak / 127
        if case["op"] == "norm":
            step = step * (x.square().sum(dim=1) / case["k"] + EPS).rsqrt()
        values = ((y * 127).div(peak[:, None]).round().nan_to_num(0.0)) * step[:, None]
        out = {"values": values, "scales": step}
        if case["op"] == "norm":
            out["sum"] = x if residual is not None else None
        return out
    if case["op"] == "matmul":
        out = []
        w = s["w"].double() * s["sw"].double()[:, None]
        for i in range(0, case["m"], 512):
            y = (s["x"][i:i + 512].double() * s["sx"][i:i + 512].double()[:, None]) @ w.t()
            out.append(y if s["b"] is None else y + s["b"].double())
        return torch.cat(out)
    given, entropy, top = [], [], []
    for i in range(case["m"]):
        x = s["x"][i].double()
        live = x > -math.inf
        if not bool(live.any()):
            given.append(torch.full((case["given"],), -math.inf, dtype=torch.float64, device=x.device))
            entropy.append(torch.zeros((), dtype=torch.float64, device=x.device))
            top.append(torch.full((case["top"],), -math.inf, dtype=torch.float64, device=x.device))
            continue
        logp = x - torch.logsumexp(x, 0)
        given.append(logp[s["given"][i].long()])
        p = logp[live].exp()
        entropy.append(-(p * logp[live]).sum())
        top.append(logp.sort(descending=True).values[:case["top"]])
    return {"given": torch.stack(given), "entropy": torch.stack(entropy), "top_ids": None,
            "top": torch.stack(top) if case["top"] else None}
