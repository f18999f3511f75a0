"""Layers of routed experts with int8 weights and with fp16 or bf16 weights, against 64 bits.

Tolerances, derived.  Int8 products: as in test_gpu_int8.py.  16-bit products: each product of two values is exact in fp32; a sum of K of them is at most K + 40 additions (the splits over waves
among them) of a relative 2^-24 of the sum of magnitudes S where they round to nearest; the matrix unit's own rounding is not documented, so 2^-23.  SwiGLU and the weighted sum: as in
test_gpu_mxfp4_layer.py.  The activations and the result are rounded once to their type."""
import numpy as np
import pytest
import torch

from oracle import int8 as orc
from oracle import mxfp4 as routing_oracle
from orinfer_amd import byte_tiles, int8, lib, programs
from tests.gpu_util import dev, host, kernel
from tests.test_gpu_int8 import check, product, rows_of, swiglu, weights_of
from tests.test_gpu_mxfp4 import slots_of
from tests.test_gpu_mxfp4_layer import weighted

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16
KINDS = [("int8", F16), ("int8", BF16), ("half", F16), ("half", BF16)]


class Bank:
    """Weights (E, N, K) of a kind: what a layer is given, and products in 64 bits."""

    def __init__(self, rng, kind, dtype, experts, n, k, size=1.0):
        self.kind = kind
        if kind == "int8":
            self.weight, self.scale = weights_of(rng, experts, n, k)
            self.scale *= np.float32(size / np.sqrt(k))
            self.given = torch.from_numpy(self.weight).to(DEV), torch.from_numpy(self.scale).to(DEV)
        else:
            held = torch.from_numpy((rng.standard_normal((experts, n, k)) * size / np.sqrt(k)).astype(np.float32)).to(dtype)
            self.weight, self.given = held.double().numpy(), (held.to(DEV),)

    def rows(self, x):
        x = x.detach().cpu().double().numpy()
        return orc.quantise(x) if self.kind == "int8" else (x,)

    def product(self, rows, at, e):
        if self.kind == "int8":
            return product(*(r[at] for r in rows), self.weight[e], self.scale[e])
        a, w = rows[0][at], self.weight[e]
        return a @ w.T, (np.abs(a) @ np.abs(w).T) * (w.shape[1] + 40) * 2.0**-23

    def products(self, x, chosen, row_of, finish=lambda *pair: pair):
        """Every slot's product (and its bound): of row row_of[slot] of x with expert chosen[slot]"""
        rows, out = self.rows(x), None
        for e in np.unique(chosen):
            at = np.nonzero(chosen == e)[0]
            pair = finish(*self.product(rows, row_of[at], e))
            if out is None:
                out = [np.empty((len(chosen), pair[0].shape[1])) for _ in range(2)]
            out[0][at], out[1][at] = pair
        return out


def make(kind, dtype, tokens, experts, top_k, hidden, inner, size=1.0, seed=0, **options):
    rng = np.random.default_rng(tokens * 31 + experts + seed)
    gate_up, down = Bank(rng, kind, dtype, experts, 2 * inner, hidden, size), Bank(rng, kind, dtype, experts, hidden, inner)
    if kind == "int8":
        layer = programs.Int8MoeLayer(tokens, experts, top_k, hidden, inner, *gate_up.given, *down.given, dtype=dtype, **options)
    else:
        layer = programs.HalfMoeLayer(tokens, experts, top_k, hidden, inner, *gate_up.given, *down.given, **options)
    x, shared = rows_of(rng, tokens, hidden, dtype).to(DEV), rows_of(rng, tokens, hidden, dtype).to(DEV)
    gate = torch.from_numpy(rng.standard_normal(tokens) * 2).to(dtype).to(DEV)
    logits = (rng.standard_normal((tokens, experts)) * 2).astype(np.float32)
    return layer, gate_up, down, x, logits, shared, gate


def check_run(layer, gate_up, down, x, logits, shared, gate, routing):
    """`run` step by step: routes and weights, activations from the rows, the result from the activations as the device left them."""
    got = layer.run(x, dev(logits), shared, gate)
    scale = {"scale": float(np.float32(routing["scale"]))} if "scale" in routing else {}
    ids, prob = routing_oracle.routes(logits, layer.top_k, **dict(routing, **scale))
    np.testing.assert_array_equal(host(layer.ids), ids)
    np.testing.assert_allclose(host(layer.prob), prob, rtol=2e-6 if not routing else 2.0**-23, atol=2.0**-149)
    check_parts(layer, gate_up, down, x, ids, shared, gate, got)


def check_parts(layer, gate_up, down, x, ids, shared, gate, got):
    order, slot = slots_of(ids)
    np.testing.assert_array_equal(host(layer.slot_map), slot)
    chosen = ids.reshape(-1)[order]
    with np.errstate(over="ignore", invalid="ignore"):
        check(layer.act, *gate_up.products(x, chosen, order // layer.top_k, swiglu), layer.dtype)
        y = down.products(layer.act, chosen, np.arange(len(order)))
        check(got, *weighted(*y, slot, host(layer.prob), shared, gate), layer.dtype)


ROUTINGS = [{}, dict(scoring="sigmoid", groups=4, top_groups=2, scale=2.5)]
SHAPES = [(1, 8, 2, 64, 32), (1, 60, 6, 256, 136), (3, 128, 8, 512, 96), (48, 64, 6, 512, 160), (300, 16, 4, 296, 264), (1100, 8, 3, 256, 128), (2, 16, 2, 5192, 72), (2, 16, 2, 72, 5192)]


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("routing", range(2))
@pytest.mark.parametrize("tokens,experts,top_k,hidden,inner", SHAPES)
def test_a_whole_layer_with_and_without_a_shared_expert(tokens, experts, top_k, hidden, inner, routing, kind, dtype):
    routing = dict(ROUTINGS[routing])
    if routing:
        routing["bias"] = np.linspace(-0.1, 0.1, experts).astype(np.float32)[::-1].copy()
    case = make(kind, dtype, tokens, experts, top_k, hidden, inner, **routing)
    check_run(*case, routing)
    check_run(*case[:5], None, None, routing)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,experts,top_k,hidden,inner", [(1, 5, 2, 65, 33), (2, 9, 3, 515, 100), (7, 3, 1, 100, 1), (40, 8, 2, 131, 70), (500, 4, 2, 301, 255)])
def test_int8_layers_of_any_width(tokens, experts, top_k, hidden, inner, dtype):
    check_run(*make("int8", dtype, tokens, experts, top_k, hidden, inner), {})


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,experts,top_k,hidden,inner", [(1, 5, 2, 8, 8), (2, 9, 3, 520, 72), (7, 3, 1, 2048, 24), (40, 8, 2, 136, 1000), (500, 4, 2, 72, 200)])
def test_16_bit_layers_whose_rows_end_within_a_step(tokens, experts, top_k, hidden, inner, dtype):
    check_run(*make("half", dtype, tokens, experts, top_k, hidden, inner), {})


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("block_m", [16, 64, 128])
@pytest.mark.parametrize("tokens,hidden,inner", [(40, 328, 224), (300, 64, 64), (900, 136, 520), (40, 5192, 72), (40, 72, 5192)])
def test_units_of_every_size(tokens, hidden, inner, block_m, kind, dtype):
    check_run(*make(kind, dtype, tokens, 8, 3, hidden, inner, block_m=block_m), {})


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_experts_without_rows_and_all_rows_to_one(kind, dtype):
    layer, gate_up, down, x, _, shared, gate = make(kind, dtype, 70, 16, 2, 264, 136)
    prob = torch.rand((70, 2), device=DEV)
    for ids in (np.tile(np.array([[15, 0]], np.int32), (70, 1)), np.stack([np.full(70, 7), np.arange(70) % 3], 1).astype(np.int32), np.full((70, 2), 3, np.int32)):
        layer.place(dev(ids))
        layer.up(x)
        layer.prob.copy_(prob)
        check_parts(layer, gate_up, down, x, ids, None, None, layer.down(layer.act, prob))


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("tokens,experts,top_k", [(2, 64, 8), (40, 16, 4), (300, 4, 2)])
def test_parts_and_replays_give_what_run_gives(tokens, experts, top_k, kind, dtype):
    layer, _, _, x, logits, shared, gate = make(kind, dtype, tokens, experts, top_k, 264, 96)
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


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("tokens", [3, 50, 300])
def test_a_token_that_is_not_finite_stays_to_itself(tokens, kind, dtype):
    layer, _, _, x, logits, _, _ = make(kind, dtype, tokens, 8, 2, 296, 136)
    logits = dev(logits)
    fine = layer.run(x, logits).clone()
    x[tokens // 2, 290] = torch.nan
    got = layer.run(x, logits)
    assert got[tokens // 2].isnan().all()
    keep = [i for i in range(tokens) if i != tokens // 2]
    assert torch.equal(got[keep], fine[keep])
    # an infinity at a row's end meets no padding of the next
    x[tokens // 2] = 0
    x[tokens // 2, 295] = torch.inf
    got = layer.run(x, logits)
    assert torch.equal(got[keep], fine[keep])


@pytest.mark.parametrize("kind,dtype", [("int8", BF16), ("half", BF16)])
@pytest.mark.parametrize("tokens,experts,top_k", [(2, 64, 8), (300, 4, 2)])
def test_activations_outside_fp16(tokens, experts, top_k, kind, dtype):
    case = make(kind, dtype, tokens, experts, top_k, 256, 96, size=300.0)
    check_run(*case, {})
    assert (case[0].act.abs() > 65520).float().mean() > 0.05


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_rows_in_the_layers_own_buffer(kind, dtype):
    """The activations' buffer seen as rows: a call that is given them reads all of them before it writes."""
    tokens, hidden, inner, top_k = 4, 64, 64, 2
    layer, gate_up, _, x, logits, _, _ = make(kind, dtype, tokens, 8, top_k, hidden, inner)
    ids, _ = layer.route(dev(logits))
    layer.place(ids)
    layer.up(x)
    held = layer.act[:tokens].clone()
    order, _ = slots_of(host(ids))
    check(layer.up(layer.act[:tokens]), *gate_up.products(held, host(ids).reshape(-1)[order], order // top_k, swiglu), dtype)


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_rows_in_the_layers_own_buffer_within_a_graph(kind, dtype):
    tokens, hidden, inner, top_k = 4, 64, 64, 2
    layer, gate_up, _, x, logits, _, _ = make(kind, dtype, tokens, 8, top_k, hidden, inner)
    ids, _ = layer.route(dev(logits))
    layer.place(ids)
    rows = layer.act[:tokens]
    layer.up(rows.copy_(x))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = layer.up(rows)
    order, _ = slots_of(host(ids))
    for seed in range(3):
        fresh = rows_of(np.random.default_rng(seed), tokens, hidden, dtype)
        rows.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        check(got, *gate_up.products(fresh, host(ids).reshape(-1)[order], order // top_k, swiglu), dtype)


@pytest.mark.parametrize("kind,dtype", KINDS)
def test_a_stream_that_the_caller_names(kind, dtype):
    """All of a call, the copy of rows that lie in the layer's own buffer as well, is behind what that stream has to do."""
    tokens, hidden, inner, top_k = 4, 64, 64, 2
    layer, gate_up, _, x, logits, _, _ = make(kind, dtype, tokens, 8, top_k, hidden, inner)
    ids, _ = layer.route(dev(logits))
    layer.place(ids)
    side = torch.cuda.Stream()
    rows = layer.act[:tokens]
    rows.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)
        rows.copy_(x)
    got = layer.up(rows, stream=side.cuda_stream)
    side.synchronize()
    order, _ = slots_of(host(ids))
    check(got, *gate_up.products(x, host(ids).reshape(-1)[order], order // top_k, swiglu), dtype)


@pytest.mark.parametrize("block_m", [16, 64, 128])
@pytest.mark.parametrize("kind,dtype", KINDS)
def test_banks_beyond_4_gib(kind, dtype, block_m):
    """Ten experts of half a GiB each and one of 300 rows; the last expert's results."""
    g = torch.Generator(device=DEV).manual_seed(2)
    experts, n, k, slots = 10, 8192, 65536 if kind == "int8" else 32768, 300
    values = torch.randint(-15, 16, (experts, 512, n // 16, 8, 16, 16 if kind == "int8" else 8), dtype=torch.int8, device=DEV, generator=g)
    tiles = values if kind == "int8" else values.to(dtype)
    x = torch.randint(-15, 16, (slots, k), dtype=torch.int8, device=DEV, generator=g)
    x[:, 0] = 127  # (scale 1, codes the values themselves)
    units = torch.zeros((-(-slots // block_m), 4), dtype=torch.int32, device=DEV)
    for i in range(len(units)):
        units[i, :3] = torch.tensor([9, i * block_m, min(block_m, slots - i * block_m)])
    out = torch.empty((slots, n), device=DEV)
    shape = dict(rows=slots, E=experts, N=n, K=k, tiles=len(units), block_m=block_m, output_dtype="float32")
    common = dict(Out=out, TileCount=torch.tensor([len(units)], dtype=torch.int32, device=DEV), TileUnits=units, W=tiles)
    if kind == "int8":
        q, s = int8.quantize(x.half())
        assert (s == 1).all()
        kernel("int8_token_grouped", **shape)(A=q, AS=s, WS=torch.ones((experts, n), device=DEV), **common)
    else:
        kernel("half_grouped", dtype=int8.dtype_name(dtype), **shape)(A=x.to(dtype), **common)
    for tile in (0, n // 16 - 1):
        w = values[9, :, tile].movedim(2, 0).reshape(16, k).double()
        assert torch.equal(out[:, tile * 16:tile * 16 + 16].double(), x.double() @ w.T)  # (whole numbers below 2^24, and so are all sums on the way)


@pytest.mark.parametrize("kind,dtype", KINDS)
@pytest.mark.parametrize("output", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("block_m", [16, 64, 128])
def test_grouped_writes_its_rows_and_columns_only(kind, dtype, output, block_m):
    """Units of odd lengths, one of them empty, rows and channels behind the ends untouched."""
    rng = np.random.default_rng(3)
    experts, n, k = 5, 70, 200
    types = {"float16": F16, "bfloat16": BF16, "float32": torch.float32}
    bank = Bank(rng, kind, dtype, experts, n, k)
    units = [(4, 0, min(13, block_m)), (0, 13, min(16, block_m)), (2, 29, 1), (2, 30, 0)]
    slots = 30
    x = rows_of(rng, slots, k, dtype).to(DEV)
    out = torch.full((slots + 4, n), 91.0, dtype=types[output], device=DEV)
    units_given, count = torch.zeros((len(units) + 2, 4), dtype=torch.int32, device=DEV), torch.tensor([len(units)], dtype=torch.int32, device=DEV)
    units_given[:len(units), :3] = torch.tensor(units, dtype=torch.int32)
    shape = dict(rows=slots, E=experts, N=n, K=k, tiles=len(units) + 2, block_m=block_m, output_dtype=output)
    tiles = byte_tiles.tiles(bank.given[0])
    common = dict(Out=out, TileCount=count, TileUnits=units_given, W=tiles)
    if kind == "int8":
        q, s = int8.quantize(x)
        kernel("int8_token_grouped", **shape)(A=q, AS=s, WS=byte_tiles.channels(bank.given[1]), **common)
    else:
        kernel("half_grouped", dtype=int8.dtype_name(dtype), **shape)(A=x, **common)
    chosen = np.empty(slots, int)
    for e, first, rows in units:
        chosen[first:first + rows] = e
    check(out[:slots], *bank.products(x, chosen, np.arange(slots)), types[output])
    assert (out[slots:] == 91).all()


def test_refusals():
    for kind, dtype in KINDS:
        layer, _, _, x, logits, shared, gate = make(kind, dtype, 4, 8, 2, 64, 32)
        assert layer.tile_count.tolist() == [0] and (layer.slot_map == -1).all()
        for call in (lambda: layer.up(x), lambda: layer.down(layer.act, layer.prob)):
            with pytest.raises(RuntimeError, match="place"):
                call()
        other = BF16 if dtype == F16 else F16
        logits = dev(logits)
        _, prob = layer.route(logits)
        layer.place(layer.ids)
        for call in (lambda: layer.up(x.to(other)), lambda: layer.up(x[:3]), lambda: layer.down(layer.act.to(other), prob), lambda: layer.down(layer.act, prob, shared.to(other), gate),
                     lambda: layer.down(layer.act, prob, shared), lambda: layer.run(x.float(), logits), lambda: layer.place(layer.ids.long())):
            with pytest.raises(ValueError):
                call()
    # 16-bit rows that no 16-byte load can start at
    layer, _, _, x, logits, _, _ = make("half", BF16, 4, 8, 2, 64, 32)
    layer.route(dev(logits))
    layer.place(layer.ids)
    moved = torch.empty(x.numel() + 1, dtype=BF16, device=DEV)[1:].view(x.shape).copy_(x)
    with pytest.raises(lib.OrxError) as error:
        layer.up(moved)
    assert error.value.code == lib.ORX_ERR_BAD_ARGUMENT and "aligned" in str(error.value)


@pytest.mark.parametrize("dtype,smallest", [(F16, 2.0**-24), (BF16, 2.0**-133)])
@pytest.mark.parametrize("block_m", [16, 64, 128])
@pytest.mark.parametrize("of_rows", [False, True])
def test_subnormal_values_count(of_rows, block_m, dtype, smallest):
    """Whole multiples of the type's smallest value, below its smallest normal one, times whole numbers (bf16: of 2^110): the sums are whole multiples of fp32's, exact."""
    g = torch.Generator(device=DEV).manual_seed(5)
    experts, n, k, slots = 3, 72, 264, 150
    small, large = ((slots, k), (experts, n, k)) if of_rows else ((experts, n, k), (slots, k))
    small = (torch.randint(-7, 8, small, device=DEV, generator=g).double() * smallest).to(dtype)
    large = (torch.randint(-7, 8, large, device=DEV, generator=g).double() * (1.0 if dtype == F16 else 2.0**110)).to(dtype)
    assert 0 < small.abs().max() < torch.finfo(dtype).smallest_normal
    x, w = (small, large) if of_rows else (large, small)
    units = torch.tensor([[i % experts, first, min(block_m, slots - first), 0] for i, first in enumerate(range(0, slots, block_m))], dtype=torch.int32, device=DEV)
    out = torch.empty((slots, n), device=DEV)
    kernel("half_grouped", rows=slots, E=experts, N=n, K=k, tiles=len(units), block_m=block_m, dtype=int8.dtype_name(dtype), output_dtype="float32")(
        A=x, Out=out, TileCount=torch.tensor([len(units)], dtype=torch.int32, device=DEV), TileUnits=units, W=byte_tiles.tiles(w))
    for e, first, rows, _ in units.tolist():
        at = slice(first, first + rows)
        want = x[at].double() @ w[e].double().t().contiguous()
        assert want.any() and torch.equal(out[at].double(), want)
