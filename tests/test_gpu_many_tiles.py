"""Int8 linears and expert products whose workgroups take several tiles, or several blocks of channels, one behind the other: every row and channel against 64 bits.

What a launch does at the border of two tiles (scales, tokens and weights of the next tile under way, sums that start again, results that leave under the next requests) only happens where there are
more tiles than workgroups; each test asserts that from the started grid.

Tolerances: those of test_gpu_int8.py, derived there.  16-bit products have values k / 32 with whole |k| <= 15, so their sums are whole multiples of 2^-10 below 2^24 of them at K <= 65536: exact in fp32
in any order, and only SwiGLU and the output round."""
import numpy as np
import pytest
import torch

from orinfer_amd import byte_tiles, int8, programs
from tests.gpu_util import kernel
from tests.started_util import started
from tests.test_gpu_expert_layers import check_run, make
from tests.test_gpu_int8 import HALF, TYPES

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16 = torch.float16, torch.bfloat16
NAMES = {dtype: name for name, dtype in TYPES.items()}
# (threads, dynamic LDS) of the dense products: rows and channels of a tile
FORMS = {(512, 16384): (16, 32), (256, 32768): (64, 32), (256, 71936): (64, 64), (256, 161792): (64, 128), (256, 158720): (96, 128), (512, 143872): (128, 128), (256, 77824): (128, 256),
         (512, 146432): (256, 256)}


def generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def whole(g, most, *shape):
    return torch.randint(-most, most + 1, shape, dtype=torch.int8, device=DEV, generator=g)


def weights(g, *shape):
    return whole(g, 127, *shape), (torch.rand(shape[:-1], generator=g, device=DEV) * 0.9 + 0.1) / 64


def rows_of(g, rows, k, dtype, side):
    size = torch.exp2(torch.randint(-6, 6, (rows, 1), generator=g, device=DEV).float())
    return ((torch.randn((rows, k), generator=g, device=DEV) + side) * size / 16).to(dtype)


def product(codes, scales, zeros, w, w_scale, bias=None):
    """In 64 bits, and the bound of its roundings: test_gpu_int8.product on the GPU."""
    sums = (codes.double() - (0 if zeros is None else zeros.double()[:, None])) @ w.double().t().contiguous()
    want = sums * w_scale.double() * scales.double()[:, None]
    bound = 3 * 2.0**-24 * 1.0001 * want.abs()
    if bias is not None:
        want = want + bias.double()
        bound = bound + 2.0**-24 * 1.0001 * (want.abs() + bound)
    return want, bound


def swiglu(want, bound):
    half = want.shape[1] // 2
    gate, up, eg, eu = want[:, :half], want[:, half:], bound[:, :half], bound[:, half:]
    silu = gate * torch.sigmoid(gate)
    return silu * up, 1.1 * eg * (up.abs() + eu) + silu.abs() * eu + 8 * 2.0**-24 * (silu * up).abs()


def check(got, want, bound):
    dtype, got = got.dtype, got.double()
    allowed = bound + want.abs() * HALF[dtype] * 1.0001 + (2.0**-25 if dtype == F16 else 0)
    fine = ((got - want).abs() <= allowed) | (got == want)
    if dtype == F16:
        fine |= got.isinf() & (got.sign() == want.sign()) & (want.abs() + bound >= 65520)
    assert fine.all(), (torch.nonzero(~fine)[:4].tolist(), int((~fine).sum()))


# ---- experts -------------------------------------------------------------------------------------------------------------------------------------
def listed_units(rng, count, block_m, experts):
    """Units of all lengths, none of the same expert as its neighbour more often than chance has it: (expert, first slot, slots), in an order that is not that of the slots."""
    lengths = np.minimum(rng.choice([block_m, block_m, block_m, block_m // 2, block_m // 2 + 1, 1, 0, 17, block_m - 1], count), block_m)
    first = np.concatenate([[0], np.cumsum(lengths)[:-1]])
    units = np.stack([rng.integers(0, experts, count), first, lengths, np.zeros(count, int)], 1).astype(np.int32)
    return units[rng.permutation(count)], int(lengths.sum())


@pytest.mark.parametrize("kind,dtype", [("int8", F16), ("int8", BF16), ("half", F16), ("half", BF16)])
@pytest.mark.parametrize("block_m", [64, 128])
@pytest.mark.parametrize("width", [208, 496, 752, 1504])  # bytes of a row: 2, 4, 6 and 12 steps
@pytest.mark.parametrize("count,n,gather,epilogue,output", [(24, 21994, True, "swiglu", None), (150, 2701, False, "none", "float32"), (150, 2698, True, "swiglu", "float32"), (40, 9003, True, "none", None)])
def test_units_that_follow_one_another(kind, dtype, block_m, width, count, n, gather, epilogue, output):
    experts, paired = 12, epilogue == "swiglu"
    g, rng = generator(width + count), np.random.default_rng(width + count + block_m)
    k = (width - 5 if kind == "int8" else width // 2)
    units, slots = listed_units(rng, count, block_m, experts)
    rows = 333 if gather else slots
    token = torch.from_numpy(rng.integers(0, rows, slots).astype(np.int32)).to(DEV)
    shape = dict(rows=slots, E=experts, N=n, K=k, tiles=count + 3, block_m=block_m, gather=gather, epilogue=epilogue, output_dtype=output or NAMES[dtype])
    given = torch.zeros((count + 3, 4), dtype=torch.int32, device=DEV)
    given[:count] = torch.from_numpy(units)
    out = torch.full((slots + 2, n // 2 if paired else n), 91.0, dtype=TYPES[shape["output_dtype"]], device=DEV)
    call = dict(Out=out, TileCount=torch.tensor([count], dtype=torch.int32, device=DEV), TileUnits=given, **({"SlotToken": token} if gather else {}))
    if kind == "int8":
        w, scale = weights(g, experts, n, k)
        codes = torch.zeros((rows, int8.padded(k)), dtype=torch.int8, device=DEV)
        codes[:, :k] = whole(g, 127, rows, k)
        row_scale = torch.rand(rows, generator=g, device=DEV) / 64 + 2.0**-10
        run, call = kernel("int8_token_grouped", **shape), dict(call, A=codes, AS=row_scale, W=byte_tiles.tiles(w, paired), WS=byte_tiles.channels(scale, paired))
    else:
        w, x = whole(g, 15, experts, n, k).to(dtype) / 32, whole(g, 15, rows, k).to(dtype) / 32
        run, call = kernel("half_grouped", dtype=NAMES[dtype], **shape), dict(call, A=x, W=byte_tiles.tiles(w, paired))
    # (128 or 256 channels to a tile, of which there are whole fours of 16)
    tiles = count * -(-call["W"].shape[-4] * 16 // (128 if block_m == 64 else 256))
    (workgroups, *_), = started(run)
    assert workgroups in (512, 1024) and tiles > 2 * workgroups
    run(**call)
    first = out.clone()
    for e in range(experts):
        at = torch.cat([torch.arange(f, f + length, device=DEV) for unit_expert, f, length, _ in units.tolist() if unit_expert == e] or [torch.arange(0, device=DEV)])
        if len(at) == 0:
            continue
        row = token[at].long() if gather else at
        if kind == "int8":
            pair = product(codes[row, :k], row_scale[row], None, w[e], scale[e])
        else:
            want = x[row].double() @ w[e].double().t().contiguous()
            pair = want, torch.zeros_like(want)
        check(first[at], *(swiglu(*pair) if paired else pair))
    assert (first[slots:] == 91).all()
    out.fill_(91)
    run(**call)
    assert torch.equal(out, first)


@pytest.mark.parametrize("kind,dtype", [("int8", F16), ("int8", BF16), ("half", F16), ("half", BF16)])
@pytest.mark.parametrize("block_m", [64, 128])
@pytest.mark.parametrize("hidden,inner", [(200, 1400), (2600, 136)])
def test_layers_of_long_prompts(kind, dtype, block_m, hidden, inner):
    """Lists as the routes' launch makes them: experts of very different numbers of rows, first or second products of more tiles than workgroups."""
    tokens, experts, top_k = 4000, 64, 2
    layer, gate_up, down, x, logits, shared, gate = make(kind, dtype, tokens, experts, top_k, hidden, inner, block_m=block_m)
    logits = logits + np.linspace(-3, 3, experts, dtype=np.float32)
    check_run(layer, gate_up, down, x, logits, shared, gate, {})
    (workgroups, *_), = started(layer.k_up if inner > hidden else layer.k_down)
    channels = (layer.w1 if inner > hidden else layer.w2).shape[-4] * 16
    assert int(layer.tile_count) * -(-channels // (128 if block_m == 64 else 256)) > workgroups


@pytest.mark.parametrize("kind,dtype", [("int8", BF16), ("half", F16)])
def test_experts_of_2_to_4_gib(kind, dtype):
    """Bytes of an expert's weights that 31 bits do not count."""
    g = generator(3)
    experts, k, slots = 2, 65536, 130
    n = 49088 if kind == "int8" else 24512
    values = whole(g, 15, experts, k * (1 if kind == "int8" else 2) // 128, -(-n // 64) * 4, 8, 16, 16 if kind == "int8" else 8)
    tiles = values if kind == "int8" else values.to(dtype)
    x = whole(g, 15, slots, k)
    x[:, 0] = 127  # (scale 1, codes the values themselves)
    for block_m in (64, 128):
        starts = range(0, slots, block_m)
        units = torch.tensor([[i % 2, first, min(block_m, slots - first), 0] for i, first in enumerate(starts)], dtype=torch.int32, device=DEV)
        out = torch.empty((slots, n), device=DEV)
        shape = dict(rows=slots, E=experts, N=n, K=k, tiles=len(units), block_m=block_m, output_dtype="float32")
        call = dict(Out=out, TileCount=torch.tensor([len(units)], dtype=torch.int32, device=DEV), TileUnits=units, W=tiles)
        if kind == "int8":
            q, s = int8.quantize(x.half())
            kernel("int8_token_grouped", **shape)(A=q, AS=s, WS=torch.ones((experts, -(-n // 64) * 64), device=DEV), **call)
        else:
            kernel("half_grouped", dtype=NAMES[dtype], **shape)(A=x.to(dtype), **call)
        for i, first in enumerate(starts):
            for tile in (0, n // 32, n // 16 - 1):
                w = values[i % 2, :, tile].movedim(2, 0).reshape(16, k).double()
                rows = slice(first, min(first + block_m, slots))
                assert torch.equal(out[rows, tile * 16:tile * 16 + 16].double(), x[rows].double() @ w.t().contiguous())  # (whole numbers below 2^24, and so are all sums on the way)


# ---- linears -------------------------------------------------------------------------------------------------------------------------------------
def linear_case(rows, n, k, dtype, zero_points, biased, epilogue="none", dtype_out=None):
    g = generator(rows * n + k)
    x = rows_of(g, rows, k, dtype, 0.7 * zero_points)
    w, scale = weights(g, n, k)
    bias = torch.randn(n, generator=g, device=DEV) if biased else None
    codes, scales, *zeros = int8.quantize(x, zero_points)
    want = product(codes, scales, zeros[0] if zeros else None, w, scale, bias)
    return x, w, scale, bias, swiglu(*want) if epilogue == "swiglu" else want


@pytest.mark.parametrize("zero_points,biased,dtype", [(False, False, F16), (True, True, BF16), (False, True, BF16), (True, False, F16)])
@pytest.mark.parametrize("epilogue", ["none", "swiglu"])
@pytest.mark.parametrize("rows,n,k,tile", [
    (1183, 2050, 200, (64, 64)), (1959, 2050, 500, (64, 64)), (2735, 1102, 200, (64, 128)), (407, 9002, 500, (64, 128)), (407, 9002, 700, (64, 128)), (3899, 2050, 200, (96, 128)), (213, 16998, 700, (96, 128)),
    (2929, 2050, 200, (128, 128)), (213, 23990, 500, (128, 128)), (213, 32990, 700, (128, 128)), (3050, 7998, 200, (128, 256)), (3050, 7998, 500, (128, 256)), (2500, 7998, 700, (128, 256)),
    (795, 23990, 1280, (128, 256)), (1183, 32990, 500, (256, 256)), (2735, 32990, 200, (256, 256))])
def test_tiles_of_linears_that_follow_one_another(rows, n, k, tile, epilogue, zero_points, biased, dtype):
    x, w, scale, bias, want = linear_case(rows, n, k, dtype, zero_points, biased, epilogue)
    linear = programs.Int8Linear(w, scale, rows, bias=bias, zero_points=zero_points, dtype=dtype, epilogue=epilogue)
    (workgroups, threads, lds), = started(linear.projection, rows)
    assert FORMS[threads, lds] == tile and -(-rows // tile[0]) * -(-linear.weight.shape[-4] * 16 // tile[1]) > workgroups
    got = linear.run(x)
    check(got, *want)
    first = got.clone()
    assert torch.equal(linear.run(x), first)


FEW = [(1, 9013, 2560), (2, 17005, 2560), (5, 17005, 1111), (8, 17005, 2560), (8, 24601, 4096), (4, 17005, 5000), (2, 9013, 9000), (1, 9013, 17408), (1, 33100, 520), (2, 17100, 1000), (6, 33100, 264),
       (8, 17100, 1024)]


@pytest.mark.parametrize("zero_points,biased,dtype", [(False, False, F16), (True, True, BF16), (False, True, BF16), (True, False, F16)])
@pytest.mark.parametrize("epilogue", ["none", "swiglu"])
@pytest.mark.parametrize("rows,n,k", FEW)
def test_blocks_of_channels_that_follow_one_another(rows, n, k, epilogue, zero_points, biased, dtype):
    """Few rows, quantised by the product: a workgroup does so once for all of its channels."""
    n = 2 * n if epilogue == "swiglu" else n
    x, w, scale, bias, want = linear_case(rows, n, k, dtype, zero_points, biased, epilogue)
    linear = programs.Int8Linear(w, scale, 8, bias=bias, zero_points=zero_points, dtype=dtype, epilogue=epilogue)
    alone = kernel("int8_token_projection", M=rows, N=n, K=k, input_dtype=NAMES[dtype], dynamic_rows=True, zero_points=zero_points, bias=biased, epilogue=epilogue, output_dtype=NAMES[dtype])
    (workgroups, threads, _), = started(alone, rows)
    assert threads == (256 if k <= 1024 else 512) and linear.weight.shape[-4] // (2 if epilogue == "swiglu" else 1) > workgroups
    out = torch.full((rows + 1, want[0].shape[1]), 91.0, dtype=dtype, device=DEV)
    alone(A=x, Out=out, W=linear.weight, m=rows, **linear.channel)
    check(out[:rows], *want)
    assert (out[rows] == 91).all()
    check(linear.run(x), *want)


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("epilogue", ["none", "swiglu"])
@pytest.mark.parametrize("rows,n,k", [(8, 300, 2560), (7, 66, 3001), (5, 130, 4096), (4, 66, 5000), (3, 130, 8192), (2, 66, 9000), (2, 130, 16384), (1, 66, 17408), (1, 130, 32768)])
def test_long_rows_that_the_product_quantises(rows, n, k, epilogue, dtype, zero_points):
    x, w, scale, bias, want = linear_case(rows, n, k, dtype, zero_points, True, epilogue)
    linear = programs.Int8Linear(w, scale, rows, bias=bias, zero_points=zero_points, dtype=dtype, epilogue=epilogue)
    shape = dict(N=n, K=k, dynamic_rows=True, zero_points=zero_points, bias=True, epilogue=epilogue, output_dtype=NAMES[dtype])
    out = torch.full((rows + 1, want[0].shape[1]), 91.0, dtype=dtype, device=DEV)
    kernel("int8_token_projection", M=rows, input_dtype=NAMES[dtype], **shape)(A=x, Out=out, W=linear.weight, m=rows, **linear.channel)
    check(out[:rows], *want)
    assert (out[rows] == 91).all()
    check(linear.run(x), *want)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("tokens,experts,top_k,hidden,inner,few", [(1, 16, 2, 4096, 40, "few_up"), (1, 16, 2, 2568, 72, "few_up"), (2, 16, 2, 40, 2568, "few_down"), (1, 8, 2, 64, 4096, "few_down"),
                                                                   (12, 2, 1, 3001, 17, "few_up"), (12, 2, 1, 40, 3001, "few_down"), (12, 2, 1, 520, 24, "few_up")])
def test_experts_that_quantise_long_rows_and_more_than_eight(tokens, experts, top_k, hidden, inner, few, dtype):
    layer, gate_up, down, x, logits, shared, gate = make("int8", dtype, tokens, experts, top_k, hidden, inner)
    assert getattr(layer, few) is not None
    if tokens == 12:
        logits[:, 0] += 3.0
        logits[:2, 0] = -50.0  # ten or more tokens to one expert, others to the other
        logits[2:, 0] = 50.0
    check_run(layer, gate_up, down, x, logits, shared, gate, {})
    assert tokens != 12 or int(layer.counts.max()) == 10


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("rows,n,k,tile", [
    (7, 300, 2560, (16, 32)), (500, 258, 4096, (64, 32)), (400, 514, 300, (64, 64)), (1024, 1058, 129, (64, 128)), (1024, 2050, 520, (96, 128)), (1500, 2050, 520, (128, 128)), (2048, 2050, 1111, (128, 256)),
    (2040, 5004, 2560, (256, 256))])
def test_linears_with_swiglu_to_32_bits(rows, n, k, tile, zero_points):
    x, w, scale, bias, want = linear_case(rows, n, k, torch.float32, zero_points, True, "swiglu")
    q = torch.empty((-(-rows // 16), int8.steps(k), 2048), dtype=torch.int8, device=DEV)
    s, z = torch.empty(rows, device=DEV), torch.empty(rows, dtype=torch.int32, device=DEV)
    zeros = ({"Z": z}, {"AZ": z, "WSum": byte_tiles.channels(w.sum(1, dtype=torch.int32), paired=True)}) if zero_points else ({}, {})
    kernel("int8_token_quantization", K=k, input_dtype="float32", layout="tiles", zero_points=zero_points)(Q=q, S=s, X=x, rows=rows, **zeros[0])
    project = kernel("int8_token_projection", M=rows, N=n, K=k, zero_points=zero_points, bias=True, epilogue="swiglu", output_dtype="float32")
    (_, threads, lds), = started(project)
    assert FORMS[threads, lds] == tile
    out = torch.full((rows + 1, n // 2), 91.0, device=DEV)
    channel = dict(WS=byte_tiles.channels(scale, paired=True), Bias=byte_tiles.channels(bias, paired=True))
    project(A=q, AS=s, Out=out, W=byte_tiles.tiles(w, paired=True), **channel, **zeros[1])
    check(out[:rows], *want)
    assert (out[rows] == 91).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rows,k", [(1, 300), (8, 520), (5, 2560), (2, 9000)])
def test_few_rows_with_swiglu_to_32_bits(rows, k, dtype):
    x, w, scale, bias, want = linear_case(rows, 130, k, dtype, True, True, "swiglu")
    out = torch.full((rows + 1, 65), 91.0, device=DEV)
    channel = dict(WS=byte_tiles.channels(scale, paired=True), Bias=byte_tiles.channels(bias, paired=True), WSum=byte_tiles.channels(w.sum(1, dtype=torch.int32), paired=True))
    kernel("int8_token_projection", M=rows, N=130, K=k, input_dtype=NAMES[dtype], zero_points=True, bias=True, epilogue="swiglu", output_dtype="float32")(
        A=x, Out=out, W=byte_tiles.tiles(w, paired=True), **channel)
    check(out[:rows], *want)
    assert (out[rows] == 91).all()


@pytest.mark.parametrize("kind,dtype", [("int8", BF16), ("half", F16), ("half", BF16)])
@pytest.mark.parametrize("width", [208, 1504])
def test_units_of_16_with_swiglu_to_32_bits(kind, dtype, width):
    g, rng = generator(width), np.random.default_rng(width)
    experts, n, k = 5, 90, width if kind == "int8" else width // 2
    units, slots = listed_units(rng, 20, 16, experts)
    units = torch.from_numpy(units).to(DEV)
    out = torch.full((slots + 1, n // 2), 91.0, device=DEV)
    shape = dict(rows=slots, E=experts, N=n, K=k, tiles=len(units), block_m=16, epilogue="swiglu", output_dtype="float32")
    call = dict(Out=out, TileCount=torch.tensor([len(units)], dtype=torch.int32, device=DEV), TileUnits=units)
    if kind == "int8":
        w, scale = weights(g, experts, n, k)
        q, s = int8.quantize(rows_of(g, slots, k, dtype, 0))
        kernel("int8_token_grouped", **shape)(A=q, AS=s, W=byte_tiles.tiles(w, True), WS=byte_tiles.channels(scale, True), **call)
    else:
        w, x = whole(g, 15, experts, n, k).to(dtype) / 32, whole(g, 15, slots, k).to(dtype) / 32
        kernel("half_grouped", dtype=NAMES[dtype], **shape)(A=x, W=byte_tiles.tiles(w, True), **call)
    for e, first, length, _ in units.tolist():
        at = slice(first, first + length)
        if kind == "int8":
            pair = product(q[at], s[at], None, w[e], scale[e])
        else:
            want = x[at].double() @ w[e].double().t().contiguous()
            pair = want, torch.zeros_like(want)
        check(out[at], *swiglu(*pair))
    assert (out[slots] == 91).all()


def test_a_matrix_of_2_to_4_gib():
    """Rows by tiles times weights whose bytes 31 bits do not count: the largest matrix that the kernel with weights in registers takes."""
    g = generator(4)
    n, k, rows = 65472, 65536, 300
    tiles = whole(g, 127, k // 128, n // 16, 8, 16, 16)
    scale = torch.rand(n, device=DEV, generator=g) / 2**20
    x = whole(g, 127, rows, k)
    x[:, 0] = 127  # (scale 1, codes the values themselves)
    q, s = torch.empty((-(-rows // 16), k // 128, 2048), dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV)
    kernel("int8_token_quantization", K=k, input_dtype="float32", layout="tiles")(Q=q, S=s, X=x.float(), rows=rows)
    project = kernel("int8_token_projection", M=rows, N=n, K=k, output_dtype="float32")
    (workgroups, threads, lds), = started(project)
    assert FORMS[threads, lds] == (128, 256) and 3 * (n // 256) > workgroups
    out = torch.empty((rows, n), device=DEV)
    project(A=q, AS=s, Out=out, W=tiles, WS=scale)
    for tile in (0, 1, n // 32, n // 16 - 1):
        w = tiles[:, tile].movedim(2, 0).reshape(16, k).double()
        want = (x.double() @ w.t().contiguous()) * scale[tile * 16:tile * 16 + 16].double()
        check(out[:, tile * 16:tile * 16 + 16], want, 3 * 2.0**-24 * 1.0001 * want.abs())
