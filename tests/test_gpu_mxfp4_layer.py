"""Expert layers of MXFP4 weights as they are used, against the 64-bit oracle.

Tolerances, derived: a second product is off by at most `product`'s bound (its sum of K terms in fp32).  The weighted sum then rounds once for each product and once for each addition, both in
fp32: with the routes' and the shared expert's terms of magnitudes T, at most 2 (top_k + 1) * 2^-24 * T, for the shared expert's gate 4 * 2^-24 more of its term (exponential, sum and quotient).
The result is rounded once to its type, half a step of it."""
import numpy as np
import pytest
import torch

from oracle import mxfp4 as orc
from orinfer_amd import mxfp4, programs
from tests.gpu_util import dev, host, kernel
from tests.test_gpu_mxfp4 import check, product, rows_of, slots_of, weights

pytestmark = pytest.mark.gpu
DEV = "cuda"


def second_products(rows, chosen, down):
    """rows (slots, I) as the device has them, the slots' experts -> products and their bounds, 64 bits"""
    b = orc.values(*orc.quantise(rows.double().cpu().numpy()))
    y, dy = (np.empty((len(b), down[0].shape[1])) for _ in range(2))
    for e in np.unique(chosen):
        at = chosen == e
        y[at], dy[at] = product(b[at], orc.values(down[0][e], down[1][e]))
    return y, dy


def weighted(y, dy, slot, prob, shared=None, gate=None):
    """sum of the routes' products times their weights, and its bound before the result's own rounding"""
    p = prob.astype(np.float64)[:, :, None]
    want, bound, size = (y[slot] * p).sum(1), (dy[slot] * p).sum(1), (np.abs(y[slot]) * p).sum(1)
    if shared is not None:
        term = 1 / (1 + np.exp(-gate.double().cpu().numpy()))[:, None] * shared.double().cpu().numpy()
        want, size, bound = want + term, size + np.abs(term), bound + 4 * 2.0**-24 * np.abs(term)
    return want, bound + 2 * (prob.shape[1] + 1) * 2.0**-24 * size


@pytest.mark.parametrize("h", [8, 100, 2056, 4096])
@pytest.mark.parametrize("m,top_k,offset", [(1, 1, 0), (5, 8, 0), (33, 10, 1), (7, 3, 2)])
def test_sums_of_fp32_rows(h, m, top_k, offset):
    """Slots that are not there count nothing; rows and results at addresses of their types' own alignment; nothing behind the result."""
    rng = np.random.default_rng(h + m)
    slots = m * top_k + 2
    expert = (rng.standard_normal((slots, h)) * 1e6).astype(np.float32)
    slot = rng.integers(0, slots, (m, top_k)).astype(np.int32)
    slot[0, 0], slot[-1, -1] = -1, slots
    prob = (rng.random((m, top_k)) * 1e-3).astype(np.float32)
    there = (slot >= 0) & (slot < slots)
    shared, gate = torch.from_numpy(rng.standard_normal((m, h))).half().to(DEV), torch.from_numpy(rng.standard_normal(m)).half().to(DEV)
    moved = torch.empty(expert.size + offset, device=DEV)[offset:].view(slots, h).copy_(torch.from_numpy(expert))
    for more in ((None, None), (shared, gate)):
        out = torch.full((m * h + offset + 8,), -7.0, dtype=torch.float16, device=DEV)
        got = out[offset:offset + m * h].view(m, h)
        kernel("moe_combine", M=m, H=h, slots=slots, top_k=top_k, expert_dtype="float32")(Expert=moved, Output=got, Prob=dev(prob), Shared=more[0], SharedGate=more[1], SlotMap=dev(slot))
        y = expert.astype(np.float64)
        check(got, *weighted(y, np.zeros_like(y), np.where(there, slot, 0), prob * there, *more), torch.float16)
        assert (out[:offset] == -7).all() and (out[offset + m * h:] == -7).all()


@pytest.mark.parametrize("tokens,experts,top_k,hidden,inner,block_m", [(2, 64, 8, 288, 96, None), (40, 8, 2, 320, 160, 16), (64, 16, 6, 288, 128, 64), (300, 4, 2, 256, 544, 128), (300, 8, 4, 512, 256, 256)])
def test_second_products_outside_fp16_and_a_sum_within(tokens, experts, top_k, hidden, inner, block_m):
    """Products of both signs far beyond 65504 with small weights: their weighted sum is what fp16 holds."""
    rng = np.random.default_rng(tokens * 7 + inner)
    gate_up, down = weights(rng, experts, 2 * inner, hidden), weights(rng, experts, hidden, inner, low=136, high=140)
    layer = programs.Mxfp4MoeLayer(tokens, experts, top_k, hidden, inner, *map(dev, gate_up), *map(dev, down), block_m=block_m)
    ids = np.argsort(rng.random((tokens, experts)), 1)[:, :top_k].astype(np.int32)
    layer.place(dev(ids))
    order, slot = slots_of(ids)
    rows = torch.from_numpy(rng.standard_normal((tokens * top_k, inner))).half()
    prob = (rng.random((tokens, top_k)) * 2.0**-10).astype(np.float32)
    y, dy = second_products(rows, ids.reshape(-1)[order], down)
    want, bound = weighted(y, dy, slot, prob)
    assert (np.abs(y) > 65520).mean() > 0.05 and np.abs(want).max() < 60000
    check(layer.down(rows.to(DEV), dev(prob)), want, bound, torch.float16)


@pytest.mark.parametrize("tokens,experts,top_k,hidden,inner", [(1, 8, 2, 64, 32), (3, 128, 8, 512, 64), (64, 60, 6, 288, 128), (700, 8, 3, 512, 256)])
def test_a_weighted_sum_is_rounded_once(tokens, experts, top_k, hidden, inner):
    rng = np.random.default_rng(tokens)
    gate_up, down = weights(rng, experts, 2 * inner, hidden), weights(rng, experts, hidden, inner)
    layer = programs.Mxfp4MoeLayer(tokens, experts, top_k, hidden, inner, *map(dev, gate_up), *map(dev, down))
    ids = np.argsort(rng.random((tokens, experts)), 1)[:, :top_k].astype(np.int32)
    layer.place(dev(ids))
    order, slot = slots_of(ids)
    rows = rows_of(rng, tokens * top_k, inner, torch.float16)
    prob = rng.dirichlet(np.ones(top_k), tokens).astype(np.float32)
    y, dy = second_products(rows, ids.reshape(-1)[order], down)
    shared, gate = rows_of(rng, tokens, hidden, torch.float16).to(DEV), torch.from_numpy(rng.standard_normal(tokens)).half().to(DEV)
    for more in ((None, None), (shared, gate)):
        check(layer.down(rows.to(DEV), dev(prob), *more), *weighted(y, dy, slot, prob, *more), torch.float16)


def test_tiles_of_more_rows_than_32_bits_count_pieces():
    """2^32 pieces of eight values, 64 GiB, and some rows more: the first rows, some in the middle and the last ones, of which only three of a tile's sixteen are there."""
    rows, k = 2**32 // 640 // 16 * 16 + 19, 5120
    some = torch.randn((4096, k), device=DEV).half()
    x = torch.empty((rows, k), dtype=torch.float16, device=DEV)
    for first in range(0, rows, 4096):
        x[first:first + 4096] = some[:rows - first]
    x[-3:] *= 3
    tiles = -(-rows // 16)
    q, s = torch.empty((tiles, 20, 2048), dtype=torch.uint8, device=DEV), torch.empty((tiles, 20, 128), dtype=torch.uint8, device=DEV)
    kernel("mxfp4_quantization", K=k, layout="tiles", M=rows)(Q=q, S=s, X=x, rows=rows)
    for tile in (0, tiles // 2, tiles - 2, tiles - 1):
        part = x[16 * tile:16 * tile + 16].double().cpu().numpy()
        part = np.pad(part, ((0, 16 - len(part)), (0, 0)))
        want = mxfp4.tiles(*map(torch.from_numpy, orc.quantise(part)))
        assert torch.equal(q[tile].cpu().flatten(), want[0].flatten()) and torch.equal(s[tile].cpu().flatten(), want[1].flatten())
    del x, q, s
    torch.cuda.empty_cache()


@pytest.mark.parametrize("rows", [1, 4, 6, 40])
def test_a_linear_of_its_own_result(rows):
    rng = np.random.default_rng(rows)
    codes, exponents = weights(rng, 512, 512, low=114, high=120)
    linear = programs.Mxfp4Linear(dev(codes), dev(exponents), rows)
    x = rows_of(rng, rows, 512, torch.float16).to(DEV)
    w = orc.values(codes, exponents)
    for _ in range(3):
        once = linear.run(x).clone()
        want, bound = product(orc.values(*orc.quantise(once.double().cpu().numpy())), w)
        check(linear.run(linear.run(x)), want, bound, torch.float16)


def layer_case(tokens, experts, top_k, hidden, inner, dtype, powers=(113, 118), **options):
    rng = np.random.default_rng(tokens * 31 + experts)
    gate_up, down = weights(rng, experts, 2 * inner, hidden, low=powers[0], high=powers[1]), weights(rng, experts, hidden, inner)
    options["block_m"] = options.get("block_m")
    layer = programs.Mxfp4MoeLayer(tokens, experts, top_k, hidden, inner, *map(dev, gate_up), *map(dev, down), dtype=dtype, **options)
    x, shared = rows_of(rng, tokens, hidden, dtype).to(DEV), rows_of(rng, tokens, hidden, dtype).to(DEV)
    gate = torch.from_numpy(rng.standard_normal(tokens) * 2).to(dtype).to(DEV)
    logits = (rng.standard_normal((tokens, experts)) * 2).astype(np.float32)
    return layer, gate_up, down, x, logits, shared, gate


def check_run(layer, gate_up, down, x, logits, shared, gate, routing):
    """`run` step by step: routes and weights, activations from the rows, the result from the activations as the device left them."""
    got = layer.run(x, dev(logits), shared, gate)
    scale = {"scale": float(np.float32(routing["scale"]))} if "scale" in routing else {}
    ids, prob = orc.routes(logits, layer.top_k, **dict(routing, **scale))
    np.testing.assert_array_equal(host(layer.ids), ids)
    np.testing.assert_allclose(host(layer.prob), prob, rtol=2e-6 if not routing else 2.0**-23, atol=2.0**-149)
    order, slot = slots_of(ids)
    np.testing.assert_array_equal(host(layer.slot_map), slot)
    chosen, inner = ids.reshape(-1)[order], layer.inter
    a = orc.values(*orc.quantise(x.double().cpu().numpy()))[order // layer.top_k]
    want, bound = np.empty((order.size, inner)), np.empty((order.size, inner))
    for e in np.unique(chosen):
        at = chosen == e
        w = orc.values(gate_up[0][e], gate_up[1][e])
        (g, dg), (up, du) = product(a[at], w[:inner]), product(a[at], w[inner:])
        with np.errstate(over="ignore"):
            want[at] = orc.silu(g) * up
        bound[at] = 1.1 * dg * (np.abs(up) + du) + np.abs(g) * du + 8 * 2.0**-24 * np.abs(want[at])
    check(layer.act, want, bound, layer.dtype)
    assert torch.isfinite(layer.act).all()
    y, dy = second_products(layer.act, chosen, down)
    check(got, *weighted(y, dy, slot, host(layer.prob), shared, gate), layer.dtype)
    return want


ROUTINGS = [{}, dict(scoring="sigmoid", scale=2.5), dict(scoring="sigmoid", groups=8, top_groups=3, group_best=1), dict(scoring="softmax", groups=4, top_groups=2, renormalize=False)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("routing", range(4))
@pytest.mark.parametrize("tokens,experts,top_k,hidden,inner", [(1, 8, 2, 64, 32), (3, 128, 8, 512, 96), (48, 64, 6, 512, 160), (300, 16, 4, 288, 544), (1100, 8, 3, 256, 128)])
def test_a_whole_layer_with_and_without_a_shared_expert(tokens, experts, top_k, hidden, inner, routing, dtype):
    routing = dict(ROUTINGS[routing])
    if routing:
        routing["bias"] = np.linspace(-0.1, 0.1, experts).astype(np.float32)[::-1].copy()
    case = layer_case(tokens, experts, top_k, hidden, inner, dtype, **routing)
    check_run(*case, routing)
    check_run(*case[:5], None, None, routing)


@pytest.mark.parametrize("block_m", [16, 64, 128, 256])
@pytest.mark.parametrize("tokens", [40, 300])
def test_bf16_experts_in_units_of_every_size(tokens, block_m):
    case = layer_case(tokens, 8, 3, 320, 224, torch.bfloat16, block_m=block_m)
    check_run(*case, {})


@pytest.mark.parametrize("tokens,experts,top_k", [(2, 64, 8), (40, 16, 4), (300, 4, 2), (700, 2, 1)])
def test_activations_outside_fp16(tokens, experts, top_k):
    """Activations beyond 65504, which fp16 cannot hold, and results of the same layer."""
    case = layer_case(tokens, experts, top_k, 256, 96, torch.bfloat16, powers=(131, 136))
    act = check_run(*case, {})
    assert (np.abs(act) > 65520).mean() > 0.05
    # the layer's own parts and a graph of it give the same
    layer, _, _, x, logits, shared, gate = case
    logits = dev(logits)
    eager = layer.run(x, logits, shared, gate).clone()
    ids, prob = layer.route(logits)
    layer.place(ids)
    assert torch.equal(layer.down(layer.up(x), prob, shared, gate), eager)
    torch.cuda.synchronize()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=stream):
        out = layer.run(x, logits, shared, gate)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
        x.neg_()
        logits.copy_(logits.roll(1, 1))
        torch.cuda.synchronize()
        eager = layer.run(x, logits, shared, gate).clone()
        torch.cuda.synchronize()


@pytest.mark.parametrize("h", [8, 100, 2056])
def test_sums_in_bf16(h):
    rng = np.random.default_rng(h)
    m, top_k, slots = 9, 6, 40
    expert = (rng.standard_normal((slots, h)) * 1e6).astype(np.float32)
    slot, prob = rng.integers(0, slots, (m, top_k)).astype(np.int32), rng.random((m, top_k)).astype(np.float32)
    shared, gate = torch.from_numpy(rng.standard_normal((m, h)) * 1e5).bfloat16().to(DEV), torch.from_numpy(rng.standard_normal(m)).bfloat16().to(DEV)
    for more in ((None, None), (shared, gate)):
        for offset in (0, 1):
            out = torch.full((m * h + 9,), -7.0, dtype=torch.bfloat16, device=DEV)
            got = out[offset:offset + m * h].view(m, h)
            kernel("moe_combine", M=m, H=h, slots=slots, top_k=top_k, expert_dtype="float32", output_dtype="bfloat16")(
                Expert=dev(expert), Output=got, Prob=dev(prob), Shared=more[0], SharedGate=more[1], SlotMap=dev(slot))
            y = expert.astype(np.float64)
            check(got, *weighted(y, np.zeros_like(y), slot, prob, *more), torch.bfloat16)
            assert (out[:offset] == -7).all() and (out[offset + m * h:] == -7).all()


def test_a_layer_refuses_values_of_another_type():
    layer, _, _, x, logits, shared, gate = layer_case(4, 8, 2, 64, 32, torch.bfloat16)
    logits = dev(logits)
    _, prob = layer.route(logits)
    for call in (lambda: layer.up(x.half()), lambda: layer.down(layer.act.half(), prob), lambda: layer.down(layer.act, prob, shared.half(), gate),
                 lambda: layer.down(layer.act, prob, shared, gate.half()), lambda: layer.run(x.float(), logits)):
        with pytest.raises(ValueError):
            call()


def test_a_new_layer_lists_nothing():
    layer, *_ = layer_case(4, 8, 2, 64, 32, torch.float16)
    assert layer.tile_count.tolist() == [0] and (layer.slot_map == -1).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("tokens,experts,top_k", [(2, 16, 6), (50, 16, 6), (300, 16, 10)])
def test_closed_experts_of_nan_weights_count_nothing(tokens, experts, top_k, dtype):
    """A bias closes all experts but four, whose weights are numbers; the others' are not, and they fill up the routes."""
    bias = np.zeros(experts, np.float32)
    bias[4:] = -np.inf
    rng = np.random.default_rng(tokens)
    gate_up, down = weights(rng, experts, 512, 256, low=113, high=118), weights(rng, experts, 256, 256)
    gate_up[1][4:10], down[1][10:] = 255, 255
    layer = programs.Mxfp4MoeLayer(tokens, experts, top_k, 256, 256, *map(dev, gate_up), *map(dev, down), scoring="sigmoid", bias=bias, dtype=dtype)
    x, logits = rows_of(rng, tokens, 256, dtype).to(DEV), rng.standard_normal((tokens, experts)).astype(np.float32)
    got = layer.run(x, dev(logits))
    ids, _ = orc.routes(logits, top_k, scoring="sigmoid", bias=bias)
    np.testing.assert_array_equal(host(layer.ids), ids)
    prob = host(layer.prob)
    assert (prob[:, 4:] == 0).all() and (prob[:, :4] > 0).all()
    order, slot = slots_of(ids)
    chosen = ids.reshape(-1)[order]
    act = layer.act.clone()
    act[torch.from_numpy(chosen >= 4).to(DEV)] = 0
    numbers = down[0], np.where(np.arange(experts)[:, None, None] < 4, down[1], 0).astype(np.uint8)
    check(got, *weighted(*second_products(act, chosen, numbers), slot, prob), dtype)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("h", [64, 100])
def test_sums_without_the_rows_of_weight_0(h):
    expert = torch.full((6, h), float("nan"), device=DEV)
    expert[1], expert[4] = float("inf"), 3.0
    out = torch.empty((2, h), dtype=torch.float16, device=DEV)
    slot, prob = dev(np.array([[0, 1, 4], [2, 3, 5]], np.int32)), dev(np.array([[0, 0, 0.5], [0, 0, -0.0]], np.float32))
    kernel("moe_combine", M=2, H=h, slots=6, top_k=3, expert_dtype="float32")(Expert=expert, Output=out, Prob=prob, Shared=None, SharedGate=None, SlotMap=slot)
    assert (out[0] == 1.5).all() and (out[1] == 0).all()
