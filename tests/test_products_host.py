"""Plans and refusals of the int8 linear and of the linears grouped by
expert: everything is refused before a launch (CPU)."""

import ctypes

import pytest
import torch

from gaiban_lite_amd import _lib, grouped_linear as G, int8_linear as L, ops

FAKE = ctypes.c_void_p(0x1000)
ODD = ctypes.c_void_p(0x1008)


def einval(name, *args):
    lib = _lib.load()
    assert getattr(lib, name)(*args) == _lib.DSV4MOE_EINVAL
    return _lib.last_error()


def test_int8_plan():
    plan = L.make_gemm_plan(3, 48, 80)
    assert plan.activation_shape == (3, 80) and plan.weight_shape == (48, 80) and plan.output_shape == (3, 48)
    assert plan.activation_scale_shape == (3,) and plan.weight_scale_shape == (48,)
    for bad in ((0, 16, 16), (1, 8, 16), (1, 16, 24), (1, 16, 65552), (-1, 16, 16), (True, 16, 16), (1.0, 16, 16)):
        with pytest.raises(ValueError):
            L.make_gemm_plan(*bad)


def test_grouped_plan():
    plan = G.make_grouped_plan(10, 4, 8, 64, 24, swiglu=True)
    assert plan.block_size == ops.block_size_m(10, 4, 8)
    assert plan.activation_shape == (10, 24) and plan.output_shape == (40, 32) and plan.weight_shape == (8, 64, 24)
    assert G.make_grouped_plan(10, 4, 8, 64, 24, per_slot=True).activation_shape == (40, 24)
    for bad in ((0, 1, 1, 16, 8), (1, 0, 1, 16, 8), (1, 1, 0, 16, 8), (1, 1, 1, 24, 8), (1, 1, 1, 16, 12)):
        with pytest.raises(ValueError):
            G.make_grouped_plan(*bad)
    with pytest.raises(ValueError, match="multiple of 32"):
        G.make_grouped_plan(1, 1, 1, 48, 8, swiglu=True)
    with pytest.raises(ValueError, match="block_size"):
        G.make_grouped_plan(1, 1, 1, 16, 8, block_size=24)
    with pytest.raises(TypeError):
        G.make_grouped_plan(1, 1, 1, 16, 8, swiglu=1)


def test_int8_entry_refusals():
    quant, gemm, linear = "dsv4moe_act_quant_int8", "dsv4moe_int8_gemm", "dsv4moe_int8_linear"
    assert "x_dtype" in einval(quant, FAKE, 3, 1, 16, FAKE, FAKE, None)
    assert "multiple of 16" in einval(quant, FAKE, 0, 1, 24, FAKE, FAKE, None)
    assert "null" in einval(quant, FAKE, 0, 1, 16, None, FAKE, None)
    assert "aligned" in einval(quant, ODD, 0, 1, 16, FAKE, FAKE, None)
    assert "multiple of 16" in einval(gemm, FAKE, FAKE, 1, 24, 16, FAKE, FAKE, FAKE, None)
    assert "65536" in einval(gemm, FAKE, FAKE, 1, 16, 65552, FAKE, FAKE, FAKE, None)
    assert "2^31" in einval(gemm, FAKE, FAKE, 1, 1 << 20, 2048, FAKE, FAKE, FAKE, None)
    assert "m must be" in einval(gemm, FAKE, FAKE, -1, 16, 16, FAKE, FAKE, FAKE, None)
    assert "null" in einval(gemm, FAKE, FAKE, 1, 16, 16, FAKE, None, FAKE, None)
    assert "aligned" in einval(gemm, FAKE, FAKE, 1, 16, 16, ODD, FAKE, FAKE, None)
    assert "too large" in einval(gemm, FAKE, FAKE, (1 << 31) - 1, 1024, 16, FAKE, FAKE, FAKE, None)
    assert "null" in einval(linear, FAKE, 0, 1, 16, 16, FAKE, FAKE, FAKE, None, FAKE, None)
    lib = _lib.load()
    assert lib.dsv4moe_int8_linear(None, 0, 0, 16, 16, None, None, None, None, None, None) == _lib.DSV4MOE_OK


def grouped_args(tokens=4, topk=2, n=64, k=64, experts=3, capacity=29, block_size=8, swiglu=0, clamp=0.0, per_slot=0,
                 x=FAKE, out=FAKE, sorted_ids=FAKE):
    return (x, tokens, topk, per_slot, n, k, experts, FAKE, sorted_ids, capacity, FAKE, FAKE, block_size, swiglu, clamp,
            None, out, None)


@pytest.mark.parametrize("bad,said", [
    ({"tokens": -1}, "tokens"), ({"topk": 0}, "topk"), ({"tokens": 1 << 30, "topk": 2}, "topk"),
    ({"experts": 0}, "experts"), ({"n": 40}, "multiple of 16"), ({"n": 48, "swiglu": 1}, "multiple of 32"),
    ({"k": 12}, "16 bytes"), ({"n": 1 << 20, "k": 1024}, "weights"), ({"tokens": 1 << 20, "k": 1024}, "x must be"),
    ({"block_size": 24}, "block_size"), ({"capacity": 0}, "capacity"), ({"clamp": -1.0}, "clamp"),
    ({"clamp": float("nan")}, "clamp"), ({"x": None}, "null"), ({"sorted_ids": None}, "null"), ({"x": ODD}, "aligned"),
    ({"out": ODD}, "aligned"),
])
def test_grouped_entry_refusals(bad, said):
    assert said in einval("dsv4moe_grouped_gemm", *grouped_args(**bad))


def test_grouped_int8_entry_refusals():
    def args(k=64, xs=FAKE, ws=FAKE):
        return (FAKE, xs, 4, 2, 0, 64, k, 3, FAKE, ws, FAKE, 29, FAKE, FAKE, 8, 0, 0.0, None, FAKE, None)

    name = "dsv4moe_grouped_int8_gemm"
    assert "16 bytes" in einval(name, *args(k=24))
    assert "65536" in einval(name, *args(k=65552))
    assert "null" in einval(name, *args(xs=None))
    assert "null" in einval(name, *args(ws=None))
    linear = (FAKE, 5, 4, 2, 0, 64, 64, 3, FAKE, FAKE, FAKE, 29, FAKE, FAKE, 8, 0, 0.0, None, FAKE, FAKE, FAKE, None)
    assert "x_dtype" in einval("dsv4moe_grouped_int8_linear", *linear)
    lib = _lib.load()
    none = (None, 0, 0, 2, 0, 64, 64, 3, None, None, None, 29, None, None, 8, 0, 0.0, None, None, None, None, None)
    assert lib.dsv4moe_grouped_int8_linear(*none) == _lib.DSV4MOE_OK


def test_wrong_tensors_are_refused():
    plan = L.make_gemm_plan(2, 16, 32)
    x = torch.zeros((2, 32), dtype=torch.bfloat16)
    w, ws = torch.zeros((16, 32), dtype=torch.int8), torch.zeros(16, dtype=torch.bfloat16)
    out, q, s = torch.zeros((2, 16), dtype=torch.bfloat16), torch.zeros((2, 32), dtype=torch.int8), torch.zeros(2)
    with pytest.raises(ValueError, match="device"):  # host tensors
        L.int8_linear_into(x, w, ws, out, q, s, plan=plan)
    with pytest.raises(TypeError):
        L.int8_linear_into(None, w, ws, out, q, s, plan=plan)
    with pytest.raises(TypeError):
        L.int8_linear_into(x.to(torch.float64), w, ws, out, q, s, plan=plan)
    with pytest.raises(TypeError):
        L.int8_linear_into(x, w, ws, out, q, s, plan=(2, 16, 32))
    with pytest.raises(ValueError, match="shape"):
        L.int8_linear_into(x[:1], w, ws, out, q, s, plan=plan)
    with pytest.raises(ValueError, match="shape"):
        L.int8_gemm_into(q, s, w[:, :16], ws, out, plan=plan)
    g = G.make_grouped_plan(2, 2, 3, 32, 32)
    ids = torch.zeros(g.capacity, dtype=torch.int32)
    kw = {"plan": g, "sorted_token_ids": ids, "expert_ids": ids[:4], "num_tokens_post_padded": ids[:1]}
    gw, gx = torch.zeros((3, 32, 32), dtype=torch.bfloat16), torch.zeros((2, 32), dtype=torch.bfloat16)
    go = torch.zeros((4, 32), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device"):
        G.grouped_linear_into(gx, gw, go, **kw)
    with pytest.raises(TypeError):
        G.grouped_linear_into(gx, gw.to(torch.int8), go, **kw)
    with pytest.raises(TypeError):
        G.grouped_int8_gemm_into(gx.to(torch.int8), s, gw, ws, go, **kw)
    with pytest.raises(ValueError, match="sorted_token_ids"):
        G.grouped_linear_into(gx, gw, go, **{**kw, "sorted_token_ids": ids[:-1]})
    with pytest.raises(ValueError, match="weight"):
        G.grouped_linear_into(gx, gw[:2], go, **kw)


def at(value):
    return ctypes.c_void_p(value)


@pytest.mark.parametrize("out,q,scale,said", [
    (0x10000 + 2 * 64 - 16, 0x40000, 0x50000, "out and x"), (0x20000, 0x40000, 0x50000, "out and wq"),
    (0x30000, 0x40000, 0x50000, "out and ws"), (0x40010, 0x40000, 0x50000, "q and out"),
    (0x60000, 0x10000, 0x50000, "q and x"), (0x60000, 0x40000, 0x4003C, "scale and q"),
    (0x60000, 0x40000, 0x20004, "scale and wq"),
])
def test_int8_calls_that_overlap(out, q, scale, said):
    args = (at(0x10000), 0, 2, 32, 32, at(0x20000), at(0x30000), at(q), at(scale), at(out), None)
    assert said in einval("dsv4moe_int8_linear", *args)


def test_overlaps_of_the_parts():
    assert "q and x" in einval("dsv4moe_act_quant_int8", at(0x10000), 2, 2, 32, at(0x100F0), at(0x50000), None)
    gemm = (at(0x10000), at(0x20000), 2, 32, 32, at(0x30000), at(0x40000), at(0x10000), None)
    assert "out and a" in einval("dsv4moe_int8_gemm", *gemm)
    assert "out and x" in einval("dsv4moe_grouped_gemm", *grouped_args(x=at(0x20000), out=at(0x20000), sorted_ids=FAKE))
    assert "out and sorted_token_ids" in einval(
        "dsv4moe_grouped_gemm", *grouped_args(x=at(0x20000), out=at(0x80000), sorted_ids=at(0x80010)))
    linear = (at(0x10000), 0, 4, 2, 0, 64, 64, 3, at(0x20000), at(0x30000), at(0x40000), 29, at(0x41000), at(0x42000), 8,
              0, 0.0, None, at(0x43000), at(0x50000), at(0x43010), None)
    assert "q and out" in einval("dsv4moe_grouped_int8_linear", *linear)
