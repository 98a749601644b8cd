"""Measured cases of the int8 linear and of the linears grouped by expert.

Three operators:

* ``int8``: the dense W8A8 linear in 8-bit integers.  Activations are
  quantised per token (scale = largest magnitude / 127), weights carry one
  bf16 scale per output channel: out = bf16(sum(q * wq) * s[token] * ws[channel]).
* ``grouped``: products by expert over bf16 weights [E, N, K].  Slot
  ``t * topk + j`` is token t's j-th expert; the slots come sorted by expert
  in blocks padded to ``block_size`` (the layout of the framework's
  alignment).  Form ``up``: rows of x by token, N = 2 I channels, the SwiGLU
  of both halves as the output; form ``down``: one row of x per slot, the
  output times its route weight; form ``plain``: rows by token, no epilogue.
* ``grouped_int8``: the same over int8 weights with a bf16 scale per expert
  and channel, activations quantised per row as in ``int8``.

``run`` computes them in elementary torch operations, or with ``own`` through
the framework's entry points.
"""

import functools
import importlib
import math

import torch

own = False

CLAMP = 10.0
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK_SIZES = (8, 16, 32, 48, 64)


def _int8(name, m, n, k, dtype="bf16"):
    return {"name": name, "op": "int8", "m": m, "n": n, "k": k, "dtype": dtype}


def _grouped(name, op, form, tokens, topk, experts, n, k, skew=0.0, dtype="bf16"):
    return {"name": name, "op": op, "form": form, "tokens": tokens, "topk": topk, "experts": experts, "n": n, "k": k,
            "skew": skew, "dtype": dtype}


def listed():
    return [
        # one user's decode step through a square projection: latency and launches
        _int8("int8_m1", 1, 4096, 4096),
        # a ragged decode batch through the widest projection
        _int8("int8_m48", 48, 16384, 4096),
        # a chunk of a prompt, every size off the tiles' sizes, fp16 activations
        _int8("int8_m777_odd", 777, 4112, 2064, "fp16"),
        # a prompt of ordinary length
        _int8("int8_m2000", 2000, 4096, 4096),
        # the largest prefill batch through the widest projection
        _int8("int8_m8192", 8192, 16384, 4096),
        # bf16 experts: one user's decode step, six experts of 256 read
        _grouped("grouped_up_t1", "grouped", "up", 1, 6, 256, 4096, 4096),
        # the second product of a decode batch, route weights applied
        _grouped("grouped_down_t64", "grouped", "down", 64, 6, 256, 4096, 2048),
        # a chunk of a chunked prefill: some 23 slots per expert
        _grouped("grouped_up_t1000", "grouped", "up", 1000, 6, 256, 4096, 4096),
        # the largest prefill batch
        _grouped("grouped_up_t8192", "grouped", "up", 8192, 6, 256, 4096, 4096),
        # int8 experts: a few concurrent users
        _grouped("grouped_int8_up_t8", "grouped_int8", "up", 8, 6, 256, 4096, 4096),
        # a small model's experts, odd sizes, fp32 activations
        _grouped("grouped_int8_down_t301", "grouped_int8", "down", 301, 4, 40, 1936, 1424, 0.5, "fp32"),
        # a prompt over fewer, popular and unpopular, experts
        _grouped("grouped_int8_up_t4096", "grouped_int8", "up", 4096, 8, 64, 4096, 4096, 0.5),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("int8", "grouped", "grouped_int8"))
    dtype = "bf16" if op == "grouped" else rng.choice(("bf16", "bf16", "fp16", "fp32"))
    n = 32 * _log_int(rng, 8, 512 if op == "int8" else 128)
    k = 16 * _log_int(rng, 16, 512 if op == "int8" else 256)
    if op == "int8":
        m = _log_int(rng, 1, 8192)
        while m * n * k > 8192 * 16384 * 4096:
            m = m // 2 + 1
        c = _int8("", m, n, k, dtype)
    else:
        experts = rng.choice((8, 20, 64, 160, 256))
        c = _grouped("", op, rng.choice(("up", "down", "plain")), _log_int(rng, 1, 8192),
                     rng.randint(1, 8 if experts == 8 else 6), experts, n, k, rng.choice((0.0, 0.5)), dtype)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs, from the seed alone
# ---------------------------------------------------------------------------


def _gen(seed, what):
    return torch.Generator("cuda").manual_seed(seed * 1_000_003 + what)


def _randn(shape, seed, what):
    return torch.randn(shape, device="cuda", generator=_gen(seed, what))


def _activations(rows, k, seed, dtype):
    """Hidden states: unit normal, rows of unlike magnitude, a few loud channels."""

    x = _randn((rows, k), seed, 1) * torch.exp(0.5 * _randn((rows, 1), seed, 2))
    loud = torch.where(torch.rand(k, device="cuda", generator=_gen(seed, 3)) < 1 / 128, 8.0, 1.0)
    return (x * loud).to(DTYPES[dtype])


def _int8_weight(shape, seed, what):
    """(int8 codes [.., n, k], bf16 scales [.., n]) of Gaussian weights."""

    w = _randn(shape, seed, what) * 0.02
    s = (w.abs().amax(-1) / 127.0).to(torch.bfloat16)
    return torch.round(w / s.float()[..., None]).clamp_(-127, 127).to(torch.int8), s


def _weights(case, seed):
    n, k, count = case["n"], case["k"], case.get("experts")
    if case["op"] == "int8":
        return _int8_weight((n, k), seed, 10)
    if case["op"] == "grouped":
        w = torch.empty((count, n, k), dtype=torch.bfloat16, device="cuda")
        for e in range(count):
            w[e] = _randn((n, k), seed, 1000 + e) * 0.02
        return w, None
    w = torch.empty((count, n, k), dtype=torch.int8, device="cuda")
    s = torch.empty((count, n), dtype=torch.bfloat16, device="cuda")
    for e in range(count):
        w[e], s[e] = _int8_weight((n, k), seed, 1000 + e)
    return w, s


def _route(case, seed):
    """(expert ids int32 [T, topk], distinct in a row; route weights fp32 [T, topk])."""

    t, e = case["tokens"], case["experts"]
    scores = _randn((t, e), seed, 4) + case["skew"] * _randn((e,), seed, 5)
    top, ids = scores.topk(case["topk"], dim=-1)
    return ids.to(torch.int32), torch.softmax(top, dim=-1) * 1.5


def _align(ids, experts):
    """The framework's alignment of these ids: slots sorted by expert, each
    expert's run padded to whole blocks with the sentinel ``ids.numel()``."""

    slots = ids.numel()
    bs = next((b for b in BLOCK_SIZES if slots / experts / b < 0.9), BLOCK_SIZES[-1])
    capacity = min(slots + experts * (bs - 1), slots * bs if slots < experts else 1 << 62)
    flat = ids.flatten().long()
    order = torch.argsort(flat, stable=True)
    counts = torch.bincount(flat, minlength=experts)
    padded = (counts + bs - 1) // bs * bs
    ends, padded_ends = counts.cumsum(0), padded.cumsum(0)
    by = flat[order]
    at = torch.arange(slots, device="cuda") - (ends - counts)[by]
    sorted_ids = torch.full((capacity,), slots, dtype=torch.int32, device="cuda")
    sorted_ids[(padded_ends - padded)[by] + at] = order.to(torch.int32)
    first = torch.arange(-(-capacity // bs), device="cuda") * bs
    owner = torch.searchsorted(padded_ends, first, right=True)
    block_experts = torch.where(first < padded_ends[-1], owner, -1).to(torch.int32)
    position = torch.empty_like(at)  # of each slot among its expert's
    position[order] = at
    return {"sorted_token_ids": sorted_ids, "expert_ids": block_experts,
            "num_tokens_post_padded": padded_ends[-1:].to(torch.int32), "block_size": bs,
            "position": position, "most": int(counts.max())}


def prepare(case, seed):
    op, n, k = case["op"], case["n"], case["k"]
    weight, weight_scale = _weights(case, seed)
    s = {"case": case, "weight": weight, "weight_scale": weight_scale}
    if op == "int8":
        rows, out_rows, width = case["m"], case["m"], n
    else:
        out_rows = case["tokens"] * case["topk"]
        rows = out_rows if case["form"] == "down" else case["tokens"]
        width = n // 2 if case["form"] == "up" else n
        s["ids"], weights = _route(case, seed)
        s["route_weights"] = weights if case["form"] == "down" else None
        s["alignment"] = _align(s["ids"], case["experts"])
    s["x"] = _activations(rows, k, seed, case["dtype"])
    s["out"] = torch.empty((out_rows, width), dtype=torch.bfloat16, device="cuda")
    if op != "grouped":  # the quantised activations' storage
        s["quantized"] = torch.empty((rows, k), dtype=torch.int8, device="cuda")
        s["scale"] = torch.empty((rows,), dtype=torch.float32, device="cuda")
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


@functools.lru_cache(maxsize=1)
def _framework():
    importlib.import_module("gaiban-lite_amd")
    return importlib.import_module("gaiban_lite_amd.int8_linear"), importlib.import_module("gaiban_lite_amd.grouped_linear")


def _run_own(s):
    int8_linear, grouped_linear = _framework()
    c = s["case"]
    if c["op"] == "int8":
        plan = int8_linear.make_gemm_plan(c["m"], c["n"], c["k"])
        int8_linear.int8_linear_into(s["x"], s["weight"], s["weight_scale"], s["out"], s["quantized"], s["scale"],
                                     plan=plan)
        return s["out"]
    a = s["alignment"]
    plan = grouped_linear.make_grouped_plan(c["tokens"], c["topk"], c["experts"], c["n"], c["k"],
                                            block_size=a["block_size"], swiglu=c["form"] == "up",
                                            per_slot=c["form"] == "down")
    how = {"plan": plan, "sorted_token_ids": a["sorted_token_ids"], "expert_ids": a["expert_ids"],
           "num_tokens_post_padded": a["num_tokens_post_padded"], "route_weights": s["route_weights"],
           "clamp_limit": CLAMP if c["form"] == "up" else 0.0}
    if c["op"] == "grouped":
        grouped_linear.grouped_linear_into(s["x"], s["weight"], s["out"], **how)
    else:
        grouped_linear.grouped_int8_linear_into(s["x"], s["weight"], s["weight_scale"], s["out"], s["quantized"],
                                                s["scale"], **how)
    return s["out"]


def _quantise(x):
    """(codes as fp32, scales fp32 [rows, 1])."""

    x = x.float()
    s = x.abs().amax(-1, keepdim=True).clamp_min(1e-12) / 127.0
    return torch.round(x / s), s


def _by_expert(x, weight, ids, position, most):
    """Row i of x (fp32, one per slot) times the weights of its expert."""

    experts, n, k = weight.shape
    flat = ids.flatten().long()
    if flat.numel() <= experts:  # few slots: their experts' weights alone
        return torch.bmm(weight[flat].float(), x.unsqueeze(-1)).squeeze(-1)
    padded = torch.zeros((experts, most, k), device="cuda")
    padded[flat, position] = x
    return torch.bmm(padded, weight.float().transpose(1, 2))[flat, position]


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    quantised = c["op"] != "grouped"
    x, scale = _quantise(s["x"]) if quantised else (s["x"].float(), None)
    if c["op"] == "int8":
        return (x @ s["weight"].float().T * scale * s["weight_scale"].float()).to(torch.bfloat16)
    if c["form"] != "down":  # a row of x serves its token's slots
        x = x.repeat_interleave(c["topk"], 0)
        scale = scale.repeat_interleave(c["topk"], 0) if quantised else None
    y = _by_expert(x, s["weight"], s["ids"], s["alignment"]["position"], s["alignment"]["most"])
    if quantised:
        y = y * scale * s["weight_scale"].float()[s["ids"].flatten().long()]
    if c["form"] == "up":
        half = c["n"] // 2
        g, u = y[:, :half].clamp(max=CLAMP), y[:, half:].clamp(-CLAMP, CLAMP)
        y = g / (1.0 + torch.exp(-g)) * u
    if s["route_weights"] is not None:
        y = y * s["route_weights"].reshape(-1, 1)
    return y.to(torch.bfloat16)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    n, k, op = case["n"], case["k"], case["op"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if op == "int8":
        m = case["m"]
        return {"bytes": n * k + 2 * n + size * m * k + 2 * m * n, "flops": 2.0 * m * n * k}
    t, topk, experts = case["tokens"], case["topk"], case["experts"]
    slots = t * topk
    touched = experts * (1.0 - (1.0 - topk / experts) ** t)  # experts with slots, of a uniform routing
    per_expert = 2 * n * k if op == "grouped" else n * k + 2 * n
    rows = slots if case["form"] == "down" else t
    width = n // 2 if case["form"] == "up" else n
    return {"bytes": touched * per_expert + size * rows * k + 2 * slots * width + 4 * slots, "flops": 2.0 * slots * n * k}


# ---------------------------------------------------------------------------
# the same results in 64 bits
# ---------------------------------------------------------------------------


def _quantise64(x):
    """The codes and scales as defined: both quotients are fp32 numbers (a
    64-bit quotient of two fp32 numbers rounds to them exactly)."""

    x = x.double()
    s = (x.abs().amax(-1, keepdim=True).clamp_min(float(torch.tensor(1e-12))) / 127.0).float().double()
    return torch.round((x / s).float().double()), s


def exact(case, seed):
    weight, weight_scale = _weights(case, seed)
    k = case["k"]
    if case["op"] == "int8":
        q, s = _quantise64(_activations(case["m"], k, seed, case["dtype"]))
        return q @ weight.double().T * s * weight_scale.double()
    ids, route = _route(case, seed)
    slots, topk, n = ids.numel(), case["topk"], case["n"]
    down, up = case["form"] == "down", case["form"] == "up"
    x = _activations(slots if down else case["tokens"], k, seed, case["dtype"])
    x, s = _quantise64(x) if case["op"] == "grouped_int8" else (x.double(), None)
    out = torch.empty((slots, n // 2 if up else n), dtype=torch.float64, device="cuda")
    flat = ids.flatten()
    for e in torch.unique(flat).tolist():
        mine = (flat == e).nonzero().flatten()
        row = mine if down else mine // topk
        y = x[row] @ weight[e].double().T
        if s is not None:
            y = y * s[row] * weight_scale[e].double()
        if up:
            g, u = y[:, : n // 2].clamp(max=CLAMP), y[:, n // 2:].clamp(-CLAMP, CLAMP)
            y = g * torch.sigmoid(g) * u
        out[mine] = y * route.flatten()[mine].double()[:, None] if down else y
    return out
