"""W8A8 int8 linear and its per-token quantiser on the GPU.

The integer sum is exact, so the expected bits follow from the definition:
``bf16(fp32(fp32(fp32(S) * s[m]) * ws[n]))`` with S from a 64-bit product of
the codes, and codes and scales from IEEE fp32 quotients.  Both are compared
bit for bit.
"""

import pytest
import torch

from gaiban_lite_amd import int8_linear as L

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16 = torch.bfloat16


def gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def activations(m, k, dtype, seed):
    x = torch.randn((m, k), device=DEV, generator=gen(seed)) * torch.exp(
        torch.randn((m, 1), device=DEV, generator=gen(seed + 1)))
    return x.to(dtype)


def weights(n, k, seed):
    w = torch.randint(-127, 128, (n, k), device=DEV, generator=gen(seed), dtype=torch.int32).to(torch.int8)
    s = (torch.rand(n, device=DEV, generator=gen(seed + 1)) * 1e-3 + 1e-5).to(BF16)
    return w, s


def expected_codes(x):
    """Codes and scales as defined; the fp32 quotients are formed as rounded
    64-bit quotients, which round to the same fp32 numbers."""

    x = x.double()
    s = (x.abs().amax(-1).clamp_min(float(torch.tensor(1e-12))) / 127.0).float()
    q = torch.round((x / s.double()[:, None]).float()).to(torch.int8)
    return q, s


def expected(q, s, w, ws):
    total = q.double() @ w.double().T  # below 2^53: exact
    return ((total.float() * s[:, None]) * ws.float()).to(BF16)


def quantise(x):
    m, k = x.shape
    q = torch.empty((m, k), dtype=torch.int8, device=DEV)
    s = torch.empty((m,), dtype=torch.float32, device=DEV)
    L.activation_quant_into(x, q, s, plan=L.make_gemm_plan(m, 16, k))
    return q, s


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 16), (3, 4096), (5, 8208), (17, 65536), (1025, 528), (1500, 8192)])
def test_codes_and_scales(m, k, dtype):
    x = activations(m, k, dtype, m + k)
    x[m // 2] = 0
    q, s = quantise(x)
    qe, se = expected_codes(x)
    assert torch.equal(s, se)
    assert torch.equal(q, qe)
    assert q[m // 2].abs().max() == 0 and s[m // 2] > 0


def test_half_way_quotients_round_to_even():
    # scale 1 exactly: the codes are the values' roundings
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5] + [0.0] * 8], device=DEV)
    q, s = quantise(x)
    assert s.item() == 1.0
    assert q[0, :8].tolist() == [127, 0, 2, 2, 0, -2, -2, 126]


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("m", [4, 2000])
def test_rows_that_are_not_finite_give_nan(bad, m):
    x = activations(m, 512, torch.float32, 5)
    x[1, 511] = bad
    q, s = quantise(x)
    assert torch.isnan(s[1]) and torch.isfinite(s[[0, 2, m - 1]]).all()
    assert q[1].abs().max() == 0
    w, ws = weights(64, 512, 9)
    out = L.int8_linear(x, w, ws)
    assert torch.isnan(out[1]).all() and torch.isfinite(out[0]).all() and torch.isfinite(out[2:]).all()


def test_smallest_and_largest_magnitudes():
    x = torch.zeros((3, 32), device=DEV)
    x[0, 3] = 1e-30  # below the floor of the scale: codes 0
    x[1, 5] = 3.4e38
    x[2, 7] = -1e-12
    q, s = quantise(x)
    qe, se = expected_codes(x)
    assert torch.equal(q, qe) and torch.equal(s, se)
    assert q[0].abs().max() == 0 and q[1, 5] == 127 and q[2, 7] == -127


SHAPES = [
    (1, 16, 16), (1, 4096, 4096), (2, 48, 80), (7, 1040, 1040), (16, 256, 128), (16, 4096, 8208), (17, 64, 144),
    (33, 4112, 272), (64, 1024, 4096), (65, 272, 2064), (100, 4096, 512), (200, 1008, 1056), (257, 512, 1024),
    (300, 2064, 336), (777, 4112, 2064), (1000, 16, 128), (1024, 4096, 4096), (2000, 4096, 1040),
    (2050, 8192, 512), (4097, 1280, 656),
]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm_and_linear_bits(m, n, k):
    x = activations(m, k, BF16, m * 7 + n)
    w, ws = weights(n, k, m + n + k)
    plan = L.make_gemm_plan(m, n, k)
    q, s = quantise(x)
    out = torch.full((m, n), float("nan"), dtype=BF16, device=DEV)
    L.int8_gemm_into(q, s, w, ws, out, plan=plan)
    want = expected(q, s, w, ws)
    assert torch.equal(out, want)
    out2 = torch.full((m, n), float("nan"), dtype=BF16, device=DEV)
    L.int8_linear_into(x, w, ws, out2, torch.empty_like(q), torch.empty_like(s), plan=plan)
    assert torch.equal(out2, want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 272, 4096), (9, 64, 2064), (40, 512, 512), (600, 528, 304)])
def test_linear_of_other_activation_types(m, n, k, dtype):
    x = activations(m, k, dtype, 3)
    w, ws = weights(n, k, 4)
    q, s = expected_codes(x)
    assert torch.equal(L.int8_linear(x, w, ws), expected(q, s, w, ws))


@pytest.mark.parametrize("m,n", [(1, 32), (16, 16), (70, 144), (300, 256)])
def test_extreme_codes_at_the_longest_k(m, n):
    """|sum| up to 65536 * 128 * 128 = 2^30 stays in int32, minus 128 included."""

    k = 65536
    q = torch.full((m, k), -128, dtype=torch.int8, device=DEV)
    w = torch.full((n, k), -128, dtype=torch.int8, device=DEV)
    w[1::2] = 127
    s = torch.full((m,), 2.0**-20, device=DEV)
    ws = torch.full((n,), 1.0, dtype=BF16, device=DEV)
    out = torch.empty((m, n), dtype=BF16, device=DEV)
    L.int8_gemm_into(q, s, w, ws, out, plan=L.make_gemm_plan(m, n, k))
    assert torch.equal(out, expected(q, s, w, ws))


def test_rows_past_four_gigabytes_of_activations():
    m, n, k = 70_001, 16, 65536  # 4.6e9 bytes of codes
    q = torch.zeros((m, k), dtype=torch.int8, device=DEV)
    q[-300:] = torch.randint(-127, 128, (300, k), device=DEV, generator=gen(1), dtype=torch.int32).to(torch.int8)
    s = torch.ones((m,), device=DEV)
    w, ws = weights(n, k, 2)
    out = torch.empty((m, n), dtype=BF16, device=DEV)
    L.int8_gemm_into(q, s, w, ws, out, plan=L.make_gemm_plan(m, n, k))
    assert torch.equal(out[-300:], expected(q[-300:], s[-300:], w, ws))
    assert out[:-300].abs().max() == 0


def test_a_row_does_not_depend_on_its_batch():
    x = activations(2000, 1024, BF16, 8)
    w, ws = weights(512, 1024, 9)
    full = L.int8_linear(x, w, ws)
    for m in (1, 3, 16, 17, 64, 65, 300):
        assert torch.equal(L.int8_linear(x[:m].contiguous(), w, ws), full[:m]), m


def test_side_stream_and_graph_replays():
    cases = []
    for m in (1, 40, 300):
        x = activations(m, 1040, BF16, m)
        w, ws = weights(528, 1040, m + 1)
        plan = L.make_gemm_plan(m, 528, 1040)
        out = torch.empty(plan.output_shape, dtype=BF16, device=DEV)
        q, s = torch.empty((m, 1040), dtype=torch.int8, device=DEV), torch.empty((m,), device=DEV)
        cases.append((x, w, ws, out, q, s, plan))

    def step():
        for x, w, ws, out, q, s, plan in cases:
            L.int8_linear_into(x, w, ws, out, q, s, plan=plan)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        for case in cases:
            case[0].copy_(activations(*case[0].shape, BF16, 100 + i))
            case[3].fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        for x, w, ws, out, *_ in cases:
            assert torch.equal(out, L.int8_linear(x, w, ws)), i


def test_more_rows_than_one_launch_of_the_quantiser_holds():
    m = 2**25 + 7  # four rows of 64 lanes a workgroup: 2^31 lanes
    x = torch.zeros((m, 16), dtype=BF16, device=DEV)
    rows = torch.tensor([0, 1, 2**25 - 1, 2**25, 2**25 + 1, m - 1], device=DEV)
    x[rows] = activations(6, 16, BF16, 5)
    q, s = quantise(x)
    want_q, want_s = expected_codes(x[rows])
    assert torch.equal(q[rows], want_q) and torch.equal(s[rows], want_s)
    assert q.count_nonzero() == want_q.count_nonzero()
    assert (s > 0).all()


@pytest.mark.parametrize("m,n,k", [(1, 24592, 4096), (5, 24592, 4224), (16, 98320, 1024), (3, 7696, 14336)])
def test_few_tokens_over_a_hundred_megabytes(m, n, k):
    x = activations(m, k, BF16, m + n)
    w, ws = weights(n, k, m + k)
    q, s = expected_codes(x)
    assert torch.equal(L.int8_linear(x, w, ws), expected(q, s, w, ws))
