"""Linears grouped by expert on the GPU, against 64-bit products.

bf16 tolerance, per element: the products of two bf16 numbers are exact in
fp32; K of them are added in K / 32 steps of up to 32 terms each, every
addition off by at most 2^-23 of the sum of magnitudes (twice half a step, so
that a truncating adder is covered), hence (K / 32 + 32) * 2^-23 * sum|x w|;
the output is rounded once to bf16: 2^-8.  Epilogue factors add two fp32
roundings.  int8 sums are exact: three fp32 roundings before bf16's.  SwiGLU:
silu's slope is at most 1.1, and its exponential, sum and quotient are off by
at most (|g| + 8) * 2^-22 relative.
"""

import pytest
import torch

from gaiban_lite_amd import deterministic_moe_align_block_size, grouped_linear as G, int8_linear as L, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def randn(shape, seed):
    return torch.randn(shape, device=DEV, generator=gen(seed))


def routed(tokens, topk, experts, seed, skew=1.0):
    scores = randn((tokens, experts), seed) + skew * randn((experts,), seed + 1)
    return scores.topk(topk, dim=-1).indices.to(torch.int32)


def align(ids, experts, block_size):
    a = deterministic_moe_align_block_size(ids, block_size=block_size, num_experts=experts)
    return {"sorted_token_ids": a.sorted_token_ids, "expert_ids": a.expert_ids,
            "num_tokens_post_padded": a.num_tokens_post_padded}


def reference(x, w, ids, *, per_slot, swiglu, route, clamp, xs=None, ws=None):
    """(output in 64 bits, its allowed error before the rounding to bf16)."""

    slots, topk = ids.numel(), ids.shape[1]
    experts, n, k = w.shape
    y = torch.zeros((slots, n), dtype=torch.float64, device=DEV)
    err = torch.zeros_like(y)
    flat = ids.flatten()
    for e in torch.unique(flat).tolist():
        mine = (flat == e).nonzero().flatten()
        rows = mine if per_slot else mine // topk
        xe, we = x[rows].double(), w[e].double()
        ye = xe @ we.T
        if xs is None:
            err[mine] = (k / 32 + 32) * 2.0**-23 * (xe.abs() @ we.abs().T)
        else:
            ye = ye * xs[rows].double()[:, None] * ws[e].double()
            err[mine] = 3 * 2.0**-24 * ye.abs()
        y[mine] = ye
    if swiglu:
        half = n // 2
        g, u, dg, du = y[:, :half], y[:, half:], err[:, :half], err[:, half:]
        if clamp > 0:
            g, u = g.clamp(max=clamp), u.clamp(-clamp, clamp)
        act = g * torch.sigmoid(g)
        y = act * u
        err = 1.1 * dg * (u.abs() + du) + act.abs() * du + ((g.abs() + 8) * 2.0**-22 + 2.0**-23) * y.abs()
    if route is not None:
        r = route.flatten().double()[:, None]
        y, err = y * r, err * r.abs() + 2.0**-23 * (y * r).abs()
    return y, err


def check(out, ref, err):
    d = (out.double() - ref).abs()
    allowed = err + 2.0**-8 * (ref.abs() + err) + 2.0**-133
    worst = (d - allowed).max().item()
    assert torch.isfinite(out).all()
    assert worst <= 0, f"off by {d.max().item()}, {worst} over what is allowed"


def make(tokens, topk, experts, n, k, form, int8, seed, ids=None, skew=1.0, block_size=None, dtype=BF16, clamp=1.5):
    ids = routed(tokens, topk, experts, seed, skew) if ids is None else ids
    swiglu, per_slot = form == "up", form == "down"
    plan = G.make_grouped_plan(tokens, topk, experts, n, k, block_size=block_size, swiglu=swiglu, per_slot=per_slot)
    x = randn(plan.activation_shape, seed + 2).to(dtype)
    w = randn(plan.weight_shape, seed + 3) / k**0.5
    route = torch.rand((tokens, topk), device=DEV, generator=gen(seed + 4)) if form == "down" else None
    kw = {"plan": plan, "route_weights": route, "clamp_limit": clamp if swiglu else 0.0,
          **align(ids, experts, plan.block_size)}
    ref = {"per_slot": per_slot, "swiglu": swiglu, "route": route, "clamp": kw["clamp_limit"]}
    out = torch.full(plan.output_shape, float("nan"), dtype=BF16, device=DEV)
    if not int8:
        w = w.to(BF16)
        return ids, (x, w, out), kw, (x, w, ids), ref
    ws = (w.abs().amax(-1) / 127).to(BF16)
    wq = torch.round(w / ws.float()[..., None]).clamp(-127, 127).to(torch.int8)
    q = torch.empty(plan.activation_shape, dtype=torch.int8, device=DEV)
    s = torch.empty(plan.activation_scale_shape, device=DEV)
    L.activation_quant_into(x, q, s, plan=L.make_gemm_plan(plan.rows, 16, k))
    return ids, (x, wq, ws, out, torch.empty_like(q), torch.empty_like(s)), kw, (q, wq, ids), {**ref, "xs": s, "ws": ws}


def run(args, kw, int8):
    (G.grouped_int8_linear_into if int8 else G.grouped_linear_into)(*args, **kw)
    return args[3] if int8 else args[2]


FORMS = ["plain", "up", "down"]
SHAPES = [
    # tokens, topk, experts, n, k
    (1, 1, 1, 32, 16), (1, 6, 256, 512, 512), (2, 2, 3, 96, 144), (8, 6, 16, 256, 1040), (33, 3, 20, 160, 272),
    (64, 6, 64, 512, 256), (300, 4, 8, 224, 400), (777, 2, 5, 288, 656), (1000, 8, 40, 256, 512),
    (2048, 6, 16, 512, 1024), (3000, 1, 2, 544, 144),
]


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("tokens,topk,experts,n,k", SHAPES)
def test_against_64_bits(tokens, topk, experts, n, k, form, int8):
    _, args, kw, data, ref = make(tokens, topk, experts, n, k, form, int8, tokens + n)
    check(run(args, kw, int8), *reference(*data, **ref))


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("block_size", G.BLOCK_SIZES)
@pytest.mark.parametrize("tokens", [5, 130, 1100])
def test_every_block_size_gives_the_same_bits(block_size, tokens, int8):
    bits = []
    for form in FORMS:
        _, args, kw, data, ref = make(tokens, 3, 7, 96, 336, form, int8, 50, block_size=block_size)
        out = run(args, kw, int8)
        check(out, *reference(*data, **ref))
        _, args, kw, _, _ = make(tokens, 3, 7, 96, 336, form, int8, 50)
        bits.append(torch.equal(out, run(args, kw, int8)))
    assert int8 is False or all(bits)  # exact sums: not even the tile shows


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("tokens,block_size", [(1, 8), (65, 8), (1500, 8), (1500, 16), (2500, 32), (900, 48), (5000, 64)])
def test_all_tokens_at_one_expert_of_many(tokens, block_size, int8):
    ids = torch.full((tokens, 1), 37, dtype=torch.int32, device=DEV)
    _, args, kw, data, ref = make(tokens, 1, 64, 64, 256, "plain", int8, 7, ids=ids, block_size=block_size)
    check(run(args, kw, int8), *reference(*data, **ref))


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_a_token_may_name_an_expert_twice(int8):
    ids = torch.tensor([[1, 1, 0], [2, 2, 2]], dtype=torch.int32, device=DEV)
    _, args, kw, data, ref = make(2, 3, 3, 32, 64, "plain", int8, 8, ids=ids)
    out = run(args, kw, int8)
    check(out, *reference(*data, **ref))
    assert torch.equal(out[0], out[1]) and torch.equal(out[3], out[5])


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_rows_without_work_keep_what_they_held(int8):
    """Ids out of range (num_tokens_post_padded -1), a block of an expert out
    of range, sorted ids out of range: nothing of theirs is written."""

    tokens, topk, experts = 40, 2, 5
    _, args, kw, data, ref = make(tokens, topk, experts, 64, 128, "plain", int8, 9, block_size=8)
    out = run(args, kw, int8).clone()
    args[3 if int8 else 2].fill_(7.0)
    run(args, {**kw, "num_tokens_post_padded": torch.full_like(kw["num_tokens_post_padded"], -1)}, int8)
    assert (args[3 if int8 else 2] == 7.0).all()
    hurt = kw["expert_ids"].clone()
    hurt[0], hurt[2] = experts, -5
    lost = torch.cat([kw["sorted_token_ids"][0:8], kw["sorted_token_ids"][16:24]]).long()
    ids = kw["sorted_token_ids"].clone()
    gone = ids[8].item()
    ids[8], ids[9] = -3, 1 << 30
    gone2 = kw["sorted_token_ids"][9].item()
    got = run(args, {**kw, "expert_ids": hurt, "sorted_token_ids": ids}, int8)
    untouched = {i for i in lost.tolist() + [gone, gone2] if i < tokens * topk}
    for i in range(tokens * topk):
        assert torch.equal(got[i], torch.full_like(got[i], 7.0) if i in untouched else out[i]), i


def test_what_is_not_finite_stays_in_its_rows_and_channels():
    _, args, kw, data, ref = make(30, 2, 4, 64, 200, "plain", False, 10)
    ids, x, w = data[2], args[0], args[1]
    clean = run(args, kw, False).clone()
    x[3, 199] = float("nan")
    w[1, 5, 0] = float("inf")
    out = run(args, kw, False)
    flat = ids.flatten()
    for i in range(60):
        bad = torch.zeros(64, dtype=torch.bool, device=DEV)
        if i // 2 == 3:
            bad[:] = True
        if flat[i] == 1:
            bad[5] = True
        assert not torch.isfinite(out[i][bad]).any()
        assert torch.equal(out[i][~bad], clean[i][~bad])


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_weights_past_four_gigabytes(int8):
    experts, n, k = 40, 8192, 8192 if not int8 else 16384
    w = torch.empty((experts, n, k), dtype=torch.int8 if int8 else BF16, device=DEV)
    last = experts - 1
    w[last] = (randn((n, k), 1) * 20).clamp(-127, 127).to(w.dtype)
    ids = torch.full((3, 1), last, dtype=torch.int32, device=DEV)
    plan = G.make_grouped_plan(3, 1, experts, n, k)
    kw = {"plan": plan, **align(ids, experts, plan.block_size)}
    x = randn((3, k), 2).to(BF16)
    out = torch.empty(plan.output_shape, dtype=BF16, device=DEV)
    one = {"per_slot": False, "swiglu": False, "route": None, "clamp": 0.0}
    only = torch.zeros_like(ids)
    if int8:
        ws = torch.full((experts, n), 0.01, dtype=BF16, device=DEV)
        q, s = torch.empty((3, k), dtype=torch.int8, device=DEV), torch.empty((3,), device=DEV)
        L.activation_quant_into(x, q, s, plan=L.make_gemm_plan(3, 16, k))
        G.grouped_int8_gemm_into(q, s, w, ws, out, **kw)
        check(out, *reference(q, w[last:], only, **one, xs=s, ws=ws[last:]))
    else:
        G.grouped_linear_into(x, w, out, **kw)
        check(out, *reference(x, w[last:], only, **one))


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("tokens", [1, 30, 700])
def test_experts_of_a_layer(tokens, int8):
    """Route, alignment, both products and the sum over the experts, as a
    layer uses them, against the same in 64 bits.  The intermediate h is
    rounded to bf16 (and to int8 with its row's scale), so the second
    product's reference starts from the h computed here; its own bar is the
    single product's."""

    topk, experts, hidden, inter = 4, 16, 512, 256
    x = randn((tokens, hidden), 20).to(BF16)
    logits = randn((tokens, experts), 21)
    ids = torch.empty((tokens, topk), dtype=torch.int32, device=DEV)
    route = torch.empty((tokens, topk), device=DEV)
    ops.route_topk_into(logits, None, topk=topk, score_func="sigmoid", route_scale=1.5, ids=ids, weights=route)
    up = G.make_grouped_plan(tokens, topk, experts, 2 * inter, hidden, swiglu=True)
    down = G.make_grouped_plan(tokens, topk, experts, hidden, inter, per_slot=True)
    a = align(ids, experts, up.block_size)
    w13, w2 = randn(up.weight_shape, 22) / hidden**0.5, randn(down.weight_shape, 23) / inter**0.5
    h = torch.empty(up.output_shape, dtype=BF16, device=DEV)
    y = torch.empty(down.output_shape, dtype=BF16, device=DEV)
    form = {"per_slot": False, "swiglu": True, "route": None, "clamp": 3.0}
    form2 = {"per_slot": True, "swiglu": False, "route": route, "clamp": 0.0}
    if int8:
        s13, s2 = ((w.abs().amax(-1) / 127).to(BF16) for w in (w13, w2))
        w13, w2 = (torch.round(w / s.float()[..., None]).clamp(-127, 127).to(torch.int8)
                   for w, s in ((w13, s13), (w2, s2)))
        q, s = torch.empty(up.activation_shape, dtype=torch.int8, device=DEV), torch.empty((tokens,), device=DEV)
        L.activation_quant_into(x, q, s, plan=L.make_gemm_plan(tokens, 16, hidden))
        G.grouped_int8_gemm_into(q, s, w13, s13, h, plan=up, clamp_limit=3.0, **a)
        qh, sh = torch.empty(down.activation_shape, dtype=torch.int8, device=DEV), torch.empty((down.rows,), device=DEV)
        G.grouped_int8_linear_into(h, w2, s2, y, qh, sh, plan=down, route_weights=route, **a)
        L.activation_quant_into(h, qh, sh, plan=L.make_gemm_plan(down.rows, 16, inter))
        check(h, *reference(q, w13, ids, **form, xs=s, ws=s13))
        ref, err = reference(qh, w2, ids, **form2, xs=sh, ws=s2)
    else:
        w13, w2 = w13.to(BF16), w2.to(BF16)
        G.grouped_linear_into(x, w13, h, plan=up, clamp_limit=3.0, **a)
        G.grouped_linear_into(h, w2, y, plan=down, route_weights=route, **a)
        check(h, *reference(x, w13, ids, **form))
        ref, err = reference(h, w2, ids, **form2)
    check(y, ref, err)
    total = y.view(tokens, topk, hidden).sum(1, dtype=torch.float32)
    allowed = (err + 2.0**-8 * (ref.abs() + err)).view(tokens, topk, hidden).sum(1) + topk * 2.0**-23 * ref.abs().view(
        tokens, topk, hidden).sum(1)
    assert ((total.double() - ref.view(tokens, topk, hidden).sum(1)).abs() <= allowed).all()


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
def test_graph_replays_with_new_routes(int8):
    """Alignment and product captured once; each replay routes anew."""

    tokens, topk, experts = 50, 4, 12
    ids, args, kw, data, ref = make(tokens, topk, experts, 128, 272, "up", int8, 30)
    from gaiban_lite_amd import allocate_deterministic_moe_alignment

    block = kw["plan"].block_size
    static = allocate_deterministic_moe_alignment(ids, block_size=block, num_experts=experts)
    kw |= {"sorted_token_ids": static.sorted_token_ids, "expert_ids": static.expert_ids,
           "num_tokens_post_padded": static.num_tokens_post_padded}

    def step():
        deterministic_moe_align_block_size(ids, block_size=block, num_experts=experts, output=static)
        return run(args, kw, int8)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        ids.copy_(routed(tokens, topk, experts, 60 + i))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.fill_(float("nan"))
        step()
        assert torch.equal(got, out), i
        check(got, *reference(data[0], data[1], ids, **ref))


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("tokens,block_size", [(3, 8), (40, 16), (200, 32), (300, 64), (20000, 64)])
def test_a_nan_passes_the_clamp(tokens, block_size, int8):
    """A NaN activation, gate channel or up channel is NaN in what it reaches
    and nowhere else, whatever the limits."""

    experts, half = 4, 96
    ids = torch.randint(0, experts, (tokens, 2), device=DEV, generator=gen(11)).to(torch.int32)
    ids[:, 0] = 1
    _, args, kw, data, ref = make(tokens, 2, experts, 2 * half, 272, "up", int8, 12, ids=ids, block_size=block_size)
    clean = run(args, kw, int8).clone()
    x, w = args[0], args[1]
    x[tokens - 1, 17] = float("nan")
    if int8:
        args[2][1, 5] = args[2][1, half + 40] = float("nan")
    else:
        w[1, 5, 3] = w[1, half + 40, 271] = float("nan")
    out = run(args, kw, int8)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[2 * (tokens - 1):] = True
    for ch in (5, 40):
        bad[:, ch] |= ids.flatten() == 1
    assert torch.isnan(out[bad]).all()
    assert torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("tokens,topk,experts,n,k", [
    (2048, 6, 16, 1056, 336), (4000, 6, 40, 1056, 336), (3000, 4, 64, 544, 528), (9000, 4, 24, 320, 656),
])
@pytest.mark.parametrize("form", FORMS)
def test_many_rows_ragged_channels(tokens, topk, experts, n, k, form, int8):
    _, args, kw, data, ref = make(tokens, topk, experts, n, k, form, int8, tokens + n)
    check(run(args, kw, int8), *reference(*data, **ref))


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("block_size", [48, 64])
def test_more_than_a_thousand_blocks(block_size, int8):
    """1300 blocks and more of three experts, then the same with blocks in the
    middle of an expert's run taken out."""

    tokens, topk, experts = 21000, 4, 3
    ids = torch.randint(0, experts, (tokens, topk), device=DEV, generator=gen(40)).to(torch.int32)
    _, args, kw, data, ref = make(tokens, topk, experts, 288, 64, "up", int8, 41, ids=ids, block_size=block_size)
    out = run(args, kw, int8).clone()
    check(out, *reference(*data, **ref))
    hurt = kw["expert_ids"].clone()
    lost = []
    for b in (1, 2, 700, 1023, 1024, 1100):
        hurt[b] = -1
        lost.append(kw["sorted_token_ids"][b * block_size:(b + 1) * block_size])
    lost = torch.cat(lost).long()
    lost = lost[lost < tokens * topk]
    args[3 if int8 else 2].fill_(7.0)
    got = run(args, {**kw, "expert_ids": hurt}, int8)
    assert (got[lost] == 7.0).all()
    kept = torch.ones(tokens * topk, dtype=torch.bool, device=DEV)
    kept[lost] = False
    assert torch.equal(got[kept], out[kept])


def test_output_past_four_gigabytes():
    tokens, n, k = 33000, 65536, 16
    ids = (torch.arange(tokens, device=DEV) % 2).to(torch.int32)[:, None]
    plan = G.make_grouped_plan(tokens, 1, 2, n, k)
    x, w = randn((tokens, k), 50).to(BF16), randn((2, n, k), 51).to(BF16)
    out = torch.empty(plan.output_shape, dtype=BF16, device=DEV)
    G.grouped_linear_into(x, w, out, plan=plan, **align(ids, 2, plan.block_size))
    one = {"per_slot": False, "swiglu": False, "route": None, "clamp": 0.0}
    for rows in (slice(0, 50), slice(tokens // 2, tokens // 2 + 50), slice(tokens - 50, tokens)):
        check(out[rows], *reference(x[rows], w, ids[rows], **one))


def test_calls_on_two_streams_at_once():
    calls = [make(t, 4, 16, 512, 528, "up", int8, 70 + i) for i, (t, int8) in
             enumerate([(20, False), (20, True), (1500, False), (1500, True)])]
    alone = [run(args, kw, i % 2 == 1).clone() for i, (_, args, kw, _, _) in enumerate(calls)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for turn in range(10):
        for i, (_, args, kw, _, _) in enumerate(calls):
            with torch.cuda.stream(streams[i]):
                run(args, kw, i % 2 == 1)
    torch.cuda.synchronize()
    for i, (_, args, kw, _, _) in enumerate(calls):
        assert torch.equal(args[3 if i % 2 else 2], alone[i])


def test_more_blocks_and_channels_than_one_launch_of_tiles_holds():
    """9000 blocks x 2048 channel tiles x 256 lanes: past 2^32; almost all
    blocks lie behind the last sequence."""

    tokens, n, k = 100, 65536, 8
    ids = (torch.arange(tokens, device=DEV) % 2).to(torch.int32)[:, None]
    plan = G.make_grouped_plan(tokens, 1, 2, n, k, block_size=8)
    x, w = randn((tokens, k), 80).to(BF16), randn((2, n, k), 81).to(BF16)
    a = align(ids, 2, 8)
    out = torch.full(plan.output_shape, float("nan"), dtype=BF16, device=DEV)
    long = torch.full((72000,), tokens, dtype=torch.int32, device=DEV)
    long[:plan.capacity] = a["sorted_token_ids"]
    experts = torch.zeros((9000,), dtype=torch.int32, device=DEV)
    experts[:a["expert_ids"].numel()] = a["expert_ids"]
    ops.grouped_gemm_into(x, w, out, tokens=tokens, topk=1, sorted_token_ids=long, expert_ids=experts,
                          num_tokens_post_padded=a["num_tokens_post_padded"], block_size=8)
    check(out, *reference(x, w, ids, per_slot=False, swiglu=False, route=None, clamp=0.0))


@pytest.mark.parametrize("int8", [False, True], ids=["bf16", "int8"])
@pytest.mark.parametrize("tokens,topk,experts,n,k", [
    (64, 4, 128, 2048, 512), (40, 4, 128, 1024, 1024), (40, 4, 20, 1056, 4608), (1000, 4, 128, 1024, 1024),
    (1500, 4, 128, 1024, 1024), (3000, 4, 128, 1024, 1024), (60, 2, 8, 2048, 8192),
])
@pytest.mark.parametrize("form", FORMS)
def test_a_hundred_megabytes_of_weights(tokens, topk, experts, n, k, form, int8):
    _, args, kw, data, ref = make(tokens, topk, experts, n, k, form, int8, tokens + n)
    out = run(args, kw, int8).clone()
    check(out, *reference(*data, **ref))
    assert torch.equal(run(args, kw, int8), out)
