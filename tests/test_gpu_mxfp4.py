"""MXFP4 rows, linears and experts against the 64-bit oracle.

Tolerances, derived: codes, exponents and dequantised values are equal.  A product's sum of K terms is exact within a block of 32 (multiples of 1/4 up to 36, 13 bits), blocks are
added in fp32: at most K / 32 + 8 additions (splits over waves among them) of a relative 2^-23 of the sum of magnitudes S (the matrix unit's rounding mode is not documented), then
the output's half step 2^-11 (fp16), 2^-8 (bf16), 2^-24 (fp32) of the value, 2^-25 where fp16 is subnormal.  SwiGLU: |d silu| <= 1.1 |d gate|, |silu(g)| <= |g|, and 8 * 2^-24 of the value for
exp, quotient and product."""
import numpy as np
import pytest
import torch

from oracle import mxfp4 as orc
from orinfer_amd import lib, mxfp4, programs
from tests.gpu_util import dev, host, kernel
from tests.test_mxfp4 import TILES

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
HALF = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}


def weights(rng, *shape, low=118, high=124):
    n, k = shape[-2:]
    return (rng.integers(0, 256, (*shape[:-1], k // 2), dtype=np.uint8), rng.integers(low, high, (*shape[:-1], k // 32), dtype=np.uint8))


def rows_of(rng, rows, k, dtype):
    x = rng.standard_normal((rows, k)) * np.exp2(rng.integers(-6, 6, (rows, 1)))
    x.reshape(-1)[rng.integers(0, x.size, max(1, x.size // 500))] *= 20
    return torch.from_numpy(x.astype(np.float32)).to(dtype)


def product(a, w):
    """want and the bound of the fp32 sums"""
    k = a.shape[1]
    return a @ w.T, (np.abs(a) @ np.abs(w).T) * (k / 32 + 8) * 2.0**-23


def check(got, want, bound, dtype):
    got = got.detach().cpu().double().numpy()
    off = np.abs(got - want)
    allowed = bound + np.abs(want) * HALF[dtype] * 1.0001 + (2.0**-25 if dtype == torch.float16 else 0)
    fine = off <= allowed
    if dtype == torch.float16:  # rounding to nearest gives infinity from 65504 plus half a step of 32 on
        fine |= np.isinf(got) & (np.sign(got) == np.sign(want)) & (np.abs(want) + bound >= 65520)
    assert fine.all(), (off.max(), np.unravel_index((off - allowed).argmax(), off.shape))


# ---- quantisation ------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("rows,k,pad", [(1, 1, 32), (1, 32, 32), (3, 33, 256), (5, 100, 32), (7, 2560, 256), (64, 264, 32), (130, 1000, 256), (33, 4096, 32)])
@pytest.mark.parametrize("scale", ["floor", "ceil"])
def test_quantisation_is_the_oracles(name, rows, k, pad, scale):
    x = rows_of(np.random.default_rng(rows * k), rows, k, TYPES[name])
    codes, exponents = orc.quantise(x.double().numpy(), ceil=scale == "ceil", pad=pad)
    # surplus rows behind the last stay as they were
    q = torch.full((rows + 1, codes.shape[1]), 171, dtype=torch.uint8, device=DEV)
    s = torch.full((rows + 1, exponents.shape[1]), 171, dtype=torch.uint8, device=DEV)
    kernel("mxfp4_quantization", K=k, input_dtype=name, scale=scale, pad=pad)(Q=q, S=s, X=x.to(DEV), rows=rows)
    written = k + -k % pad  # of rows at an odd multiple of 256 what lies behind is left as it was
    np.testing.assert_array_equal(host(s[:rows, :written // 32]), exponents[:, :written // 32])
    np.testing.assert_array_equal(host(q[:rows, :written // 2]), codes[:, :written // 2])
    assert (q[:rows, written // 2:] == 171).all() and (s[:rows, written // 32:] == 171).all()
    assert (q[rows] == 171).all() and (s[rows] == 171).all()
    for out in TYPES.values():
        got = mxfp4.dequantize(q[:rows], s[:rows], k, out, pad=pad)
        want = torch.from_numpy(orc.values(codes, exponents)[:, :k]).to(out)
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("rows,k", [(1, 32), (1, 7), (5, 300), (16, 256), (17, 2560), (100, 1000), (33, 4096)])
def test_quantisation_by_tiles(name, rows, k):
    x = rows_of(np.random.default_rng(rows * k), rows, k, TYPES[name])
    codes, exponents = orc.quantise(np.pad(x.double().numpy(), ((0, -rows % 16), (0, -k % 256))))
    want = mxfp4.tiles(torch.from_numpy(codes), torch.from_numpy(exponents))
    tiles, steps = -(-rows // 16), -(-k // 256)
    q, s = torch.full((tiles * steps * 2048 + 16,), 171, dtype=torch.uint8, device=DEV), torch.full((tiles * steps * 128 + 16,), 171, dtype=torch.uint8, device=DEV)
    kernel("mxfp4_quantization", K=k, input_dtype=name, layout="tiles")(Q=q, S=s, X=x.to(DEV), rows=rows)
    assert torch.equal(q[:-16].cpu(), want[0].flatten()) and torch.equal(s[:-16].cpu(), want[1].flatten())
    assert (q[-16:] == 171).all() and (s[-16:] == 171).all()


@pytest.mark.parametrize("name", ["float16", "bfloat16"])
@pytest.mark.parametrize("offset", [1, 4])
def test_quantisation_of_rows_that_are_not_16_byte_aligned(name, offset):
    x = rows_of(np.random.default_rng(offset), 9, 96, TYPES[name])
    moved = torch.empty(9 * 96 + offset, dtype=TYPES[name], device=DEV)[offset:].view(9, 96).copy_(x)
    codes, exponents = mxfp4.quantize(moved)
    want = orc.quantise(x.double().numpy())
    np.testing.assert_array_equal(host(codes), want[0])
    np.testing.assert_array_equal(host(exponents), want[1])
    back = torch.zeros(9 * 96 + offset, dtype=TYPES[name], device=DEV)
    kernel("mxfp4_dequantization", K=96, output_dtype=name)(Q=codes, S=exponents, Y=back[offset:], rows=9)
    assert torch.equal(back[offset:].view(9, 96).cpu(), torch.from_numpy(orc.values(*want)).to(TYPES[name])) and not back[:offset].any()


def test_every_fp16_value_by_itself_and_in_company():
    every = np.arange(65536, dtype=np.uint16).view(np.float16)
    alone = np.zeros((65536, 32), np.float16)
    alone[:, 5] = every
    beside = alone.copy()
    beside[:, 9] = 1.0
    for x in (alone, beside):
        for ceil in (False, True):
            with np.errstate(invalid="ignore"):
                codes, exponents = orc.quantise(x.astype(np.float64), ceil=ceil)
            got = mxfp4.quantize(torch.from_numpy(x).to(DEV), scale="ceil" if ceil else "floor")
            np.testing.assert_array_equal(host(got[1]), exponents)
            np.testing.assert_array_equal(host(got[0]), codes)


def test_fp32_extremes_zeros_infinities_and_nan():
    x = np.zeros((8, 64), np.float32)
    x[1, 3], x[1, 40] = 1e-45, -1e-38          # the smallest power there is
    x[2, 3], x[2, 40] = 3.4e38, -3.0e38
    x[3, 3], x[3, 40] = np.inf, 1.0            # the first block is NaN, the second is not
    x[4, 3], x[4, 40] = np.nan, -2.0
    x[5, :] = -0.0
    x[6, :32], x[6, 32:] = 5.9e-39, 2.0**-126
    codes, exponents = orc.quantise(x.astype(np.float64))
    got = mxfp4.quantize(torch.from_numpy(x).to(DEV))
    np.testing.assert_array_equal(host(got[1]), exponents)
    np.testing.assert_array_equal(host(got[0]), codes)
    back = host(mxfp4.dequantize(*got, 64, torch.float32))
    assert np.isnan(back[3, :32]).all() and np.isnan(back[4, :32]).all() and not np.isnan(back[3:5, 32:]).any()


# ---- linears -----------------------------------------------------------------------------------------------------------------------------------
def linear_case(rows, n, k, dtype=torch.float16, epilogue="none", seed=0, capacity=None):
    rng = np.random.default_rng(rows * 1000003 + n * 1009 + k + seed)
    codes, exponents = weights(rng, n, k)
    x = rows_of(rng, rows, k, dtype)
    linear = programs.Mxfp4Linear(dev(codes), dev(exponents), capacity or rows, dtype=dtype, epilogue=epilogue)
    a, w = orc.values(*orc.quantise(x.double().numpy())), orc.values(codes, exponents)
    if epilogue == "none":
        return linear, x.to(DEV), *product(a, w)
    (gate, dg), (up, du) = product(a, w[:n // 2]), product(a, w[n // 2:])
    want = orc.silu(gate) * up
    return linear, x.to(DEV), want, 1.1 * dg * (np.abs(up) + du) + np.abs(gate) * du + 8 * 2.0**-24 * np.abs(want)


@pytest.mark.parametrize("rows", [1, 2, 3, 8, 15, 16, 17, 31, 32, 33, 64, 65, 100, 129, 200, 257, 300, 520])
@pytest.mark.parametrize("n,k", [(48, 64), (100, 416), (257, 1024), (1000, 2560)])
def test_linear(rows, n, k):
    linear, x, want, bound = linear_case(rows, n, k, capacity=rows + 1)
    linear.out.fill_(-7)
    got = linear.run(x)
    check(got, want, bound, torch.float16)
    assert (linear.out[rows:] == -7).all()


@pytest.mark.parametrize("rows", [1, 5, 33, 130, 600])
@pytest.mark.parametrize("n,k", [(64, 96), (330, 800), (2048, 1536)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_linear_with_swiglu(rows, n, k, dtype):
    linear, x, want, bound = linear_case(rows, n, k, dtype, "swiglu")
    assert linear.run(x).shape == (rows, n // 2)
    check(linear.run(x), want, bound, dtype)


@pytest.mark.parametrize("rows,n,k", [(1, 9728, 2560), (4, 17408, 5120), (40, 5120, 17408), (1000, 640, 4096), (2049, 520, 768), (513, 4096, 512), (2300, 2200, 544),
                                      (2049, 4097, 288)])
def test_linear_of_large_shapes(rows, n, k):
    linear, x, want, bound = linear_case(rows, n, k, torch.bfloat16)
    check(linear.run(x), want, bound, torch.bfloat16)


@pytest.mark.parametrize("rows,n", [(1, 33), (70, 97), (300, 258)])
def test_linear_with_fp32_output_at_an_odd_address(rows, n):
    rng = np.random.default_rng(n)
    codes, exponents = weights(rng, n, 320)
    x = rows_of(rng, rows, 320, torch.float32)
    q, s = torch.empty(-(-rows // 16) * 2 * 2048, dtype=torch.uint8, device=DEV), torch.empty(-(-rows // 16) * 2 * 128, dtype=torch.uint8, device=DEV)
    kernel("mxfp4_quantization", K=320, input_dtype="float32", layout="tiles")(Q=q, S=s, X=x.to(DEV), rows=rows)
    w, ws = mxfp4.tiles(dev(codes), dev(exponents))
    out = torch.full((rows * n + 9,), -7.0, device=DEV)
    kernel("mxfp4_projection", M=rows, N=n, K=320, output_dtype="float32")(A=q, AS=s, Out=out[1:], W=w, WS=ws)
    want, bound = product(orc.values(*orc.quantise(x.double().numpy())), orc.values(codes, exponents))
    check(out[1:1 + rows * n].view(rows, n), want, bound, torch.float32)
    assert out[0] == -7 and (out[1 + rows * n:] == -7).all()


@pytest.mark.parametrize("epilogue", ["none", "swiglu"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,n,k", [shape for shape, _, _ in TILES])
def test_tiles_of_every_kind(rows, n, k, dtype, epilogue):
    """The last rows and channels of a tile, results at an odd address, nothing behind them."""
    rng = np.random.default_rng(n)
    codes, exponents = weights(rng, n, k)
    x = rows_of(rng, rows, k, torch.float16)
    q, s = (torch.empty(-(-rows // 16) * -(-k // 256) * size, dtype=torch.uint8, device=DEV) for size in (2048, 128))
    kernel("mxfp4_quantization", K=k, layout="tiles")(Q=q, S=s, X=x.to(DEV), rows=rows)
    w, ws = mxfp4.tiles(dev(codes), dev(exponents), paired=epilogue == "swiglu")
    columns = n // 2 if epilogue == "swiglu" else n
    out = torch.full((rows * columns + 9,), -7.0, dtype=dtype, device=DEV)
    kernel("mxfp4_projection", M=rows, N=n, K=k, output_dtype=mxfp4.dtype_name(dtype), epilogue=epilogue)(A=q, AS=s, Out=out[1:], W=w, WS=ws)
    a, b = orc.values(*orc.quantise(x.double().numpy())), orc.values(codes, exponents)
    if epilogue == "none":
        want, bound = product(a, b)
    else:
        (gate, dg), (up, du) = product(a, b[:columns]), product(a, b[columns:])
        want = orc.silu(gate) * up
        bound = 1.1 * dg * (np.abs(up) + du) + np.abs(gate) * du + 8 * 2.0**-24 * np.abs(want)
    check(out[1:1 + rows * columns].view(rows, columns), want, bound, dtype)
    assert out[0] == -7 and (out[1 + rows * columns:] == -7).all()


@pytest.mark.parametrize("epilogue", ["none", "swiglu"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 2, 7, 16])
@pytest.mark.parametrize("n,k", [(32, 32), (94, 608), (700, 2304), (9000, 512)])
def test_rows_that_the_projection_quantises(rows, n, k, dtype, epilogue):
    """16-bit rows at an address of their own alignment give what the quantiser and the projection give."""
    linear, x, want, bound = linear_case(rows, n, k, dtype, epilogue)
    moved = torch.empty(rows * k + 1, dtype=dtype, device=DEV)[1:].view(rows, k).copy_(x)
    out = torch.full((rows * want.shape[1] + 3,), -7, dtype=dtype, device=DEV)
    kernel("mxfp4_projection", M=16, N=n, K=k, dynamic_rows=True, input_dtype=mxfp4.dtype_name(dtype), output_dtype=mxfp4.dtype_name(dtype), epilogue=epilogue)(
        A=moved, Out=out[1:], W=linear.weight, WS=linear.powers, m=rows)
    got = out[1:1 + want.size].view(want.shape)
    check(got, want, bound, dtype)
    assert out[0] == -7 and (out[1 + want.size:] == -7).all()


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_a_block_of_nan_stays_in_its_row_and_weights_of_nan_in_their_channel(rows):
    rng = np.random.default_rng(rows)
    codes, exponents = weights(rng, 80, 512)
    exponents[17, 3] = 255
    x = rows_of(rng, rows, 512, torch.float16)
    x[rows // 2, 100] = float("inf")
    got = programs.Mxfp4Linear(dev(codes), dev(exponents), rows).run(x.to(DEV)).cpu()
    nan = torch.zeros_like(got, dtype=torch.bool)
    nan[rows // 2], nan[:, 17] = True, True
    assert torch.equal(got.isnan(), nan)


def test_linear_of_no_rows_and_refusals():
    linear, x, _, _ = linear_case(4, 64, 96)
    assert linear.run(x[:0]).shape == (0, 64)
    for bad in (torch.cat([x, x]), x.float(), x[:, :64], x.t(), x[:, ::2], x.cpu(), x[0]):
        with pytest.raises(ValueError):
            linear.run(bad)
    codes, exponents = dev(np.zeros((4, 32), np.uint8)), dev(np.zeros((4, 2), np.uint8))
    for args, named in (((codes, exponents, 0), {}), ((codes, exponents, 4), dict(dtype=torch.float32)), ((codes[0], exponents[0], 4), {}),
                        ((codes[:3], exponents[:3], 4), dict(epilogue="swiglu"))):
        with pytest.raises(ValueError):
            programs.Mxfp4Linear(*args, **named)


@pytest.mark.parametrize("rows", [1, 3, 40, 300])
def test_linear_on_another_stream_and_replayed_from_a_graph(rows):
    linear, x, want, bound = linear_case(rows, 528, 1056)
    eager = linear.run(x).clone()
    check(eager, want, bound, torch.float16)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = linear.run(x)
    for step in range(3):
        x.copy_(x.flip(0) if rows > 1 else -x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, linear.run(x))
        torch.cuda.synchronize()


def test_two_linears_on_two_streams_at_once():
    cases = [linear_case(rows, 700, 1184, seed=seed) for seed, rows in enumerate((300, 17, 2, 40))]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        for (linear, x, _, _), stream in zip(cases, streams):
            with torch.cuda.stream(stream):
                linear.run(x)
    torch.cuda.synchronize()
    for linear, x, want, bound in cases:
        check(linear.out, want, bound, torch.float16)


def sampled(rows):
    return np.unique(np.concatenate([np.arange(3), np.arange(rows // 2, rows // 2 + 3), np.arange(rows - 5, rows)]))


def test_quantisation_of_more_than_4_gib():
    rows, k = 2**20 + 3, 2304
    x = torch.randn((rows // 8 + 1, k), device=DEV).to(torch.bfloat16).repeat(8, 1)[:rows]
    at = torch.from_numpy(sampled(rows)).to(DEV)
    x[-5:] *= 3
    codes, exponents = mxfp4.quantize(x)
    want_codes, want_exponents = orc.quantise(x[at].double().cpu().numpy())
    np.testing.assert_array_equal(host(codes[at]), want_codes)
    np.testing.assert_array_equal(host(exponents[at]), want_exponents)
    back = mxfp4.dequantize(codes, exponents, k, torch.bfloat16)
    np.testing.assert_array_equal(host(back[at].float()), orc.values(want_codes, want_exponents))


def test_linear_with_more_than_4_gib_of_results():
    rows, n, k = 2**20 + 3, 2100, 64
    rng = np.random.default_rng(4)
    codes, exponents = weights(rng, n, k)
    x = torch.randn((rows, k), device=DEV).half()
    linear = programs.Mxfp4Linear(dev(codes), dev(exponents), rows)
    at = sampled(rows)
    want, bound = product(orc.values(*orc.quantise(x[torch.from_numpy(at).to(DEV)].double().cpu().numpy())), orc.values(codes, exponents))
    check(linear.run(x)[torch.from_numpy(at).to(DEV)], want, bound, torch.float16)


# ---- experts -----------------------------------------------------------------------------------------------------------------------------------
def moe_case(tokens, experts, top_k, hidden, inner, seed=0, skew=0.0, **options):
    rng = np.random.default_rng(seed + tokens * 131 + experts)
    gate_up, down = weights(rng, experts, 2 * inner, hidden), weights(rng, experts, hidden, inner)
    layer = programs.Mxfp4MoeLayer(tokens, experts, top_k, hidden, inner, *map(dev, gate_up), *map(dev, down), **options)
    x = rows_of(rng, tokens, hidden, torch.float16)
    logits = (rng.standard_normal((tokens, experts)) - skew * np.log(np.arange(1, experts + 1))).astype(np.float32)
    return layer, gate_up, down, x, logits, rng


def slots_of(ids):
    order = np.argsort(ids.reshape(-1), kind="stable")
    slot = np.empty_like(order)
    slot[order] = np.arange(order.size)
    return order, slot.reshape(ids.shape)


SHAPES = [(1, 8, 2, 64, 32), (3, 16, 4, 256, 96), (5, 128, 8, 512, 64), (40, 8, 2, 320, 160), (64, 60, 6, 288, 128), (256, 32, 4, 512, 256), (300, 4, 2, 256, 544),
          (700, 8, 3, 512, 256), (1100, 2, 1, 256, 128), (2, 8, 2, 9728, 64), (2, 8, 3, 64, 9728)]


@pytest.mark.parametrize("tokens,experts,top_k,hidden,inner", SHAPES)
@pytest.mark.parametrize("block_m", [None, 16, 64, 128, 256])
def test_experts(tokens, experts, top_k, hidden, inner, block_m):
    layer, gate_up, down, x, logits, rng = moe_case(tokens, experts, top_k, hidden, inner, skew=1.1, block_m=block_m)
    layer.act.fill_(-7)
    ids, prob = layer.route(dev(logits))
    want_ids, want_prob = orc.routes(logits, top_k)
    np.testing.assert_array_equal(host(ids), want_ids)
    np.testing.assert_allclose(host(prob), want_prob, rtol=2e-6)
    order, slot = slots_of(want_ids)
    np.testing.assert_array_equal(host(layer.place(ids)), slot)
    act = layer.up(x.to(DEV))
    a = orc.values(*orc.quantise(x.double().numpy()))[order // top_k]
    chosen = want_ids.reshape(-1)[order]
    want, bound = np.empty((order.size, inner)), np.empty((order.size, inner))
    for e in np.unique(chosen):
        at = chosen == e
        w = orc.values(gate_up[0][e], gate_up[1][e])
        (gate, dg), (up, du) = product(a[at], w[:inner]), product(a[at], w[inner:])
        want[at] = orc.silu(gate) * up
        bound[at] = 1.1 * dg * (np.abs(up) + du) + np.abs(gate) * du + 8 * 2.0**-24 * np.abs(want[at])
    check(act, want, bound, torch.float16)
    # the second products from rows of our own
    rows = torch.from_numpy(rng.standard_normal((order.size, inner)).astype(np.float16))
    out = layer.down(rows.to(DEV), prob)
    b = orc.values(*orc.quantise(rows.double().numpy()))
    y, dy = np.empty((order.size, hidden)), np.empty((order.size, hidden))
    for e in np.unique(chosen):
        at = chosen == e
        y[at], dy[at] = product(b[at], orc.values(down[0][e], down[1][e]))
    p = host(prob).astype(np.float64)[:, :, None]
    want, each = (y[slot] * p).sum(1), (np.abs(y[slot]) * p).sum(1)
    # each product is rounded to fp16, then top_k products and sums in fp32
    check(out, want, (dy[slot] * p).sum(1) + each * (2.0**-11 + 2 * top_k * 2.0**-24) + 2.0**-25, torch.float16)


@pytest.mark.parametrize("tokens,experts,top_k,block_m", [(8, 64, 8, None), (1, 3, 3, None), (40, 64, 8, None), (40, 64, 8, 64), (90, 5, 4, 128), (300, 7, 2, 256)])
def test_every_route_to_one_expert(tokens, experts, top_k, block_m):
    """A token may name an expert more than once: its slots are in the order of its routes, the others have none."""
    hidden, inner = 288, 96
    layer, gate_up, down, x, _, rng = moe_case(tokens, experts, top_k, hidden, inner, block_m=block_m)
    ids, e = torch.full((tokens, top_k), experts - 1, dtype=torch.int32, device=DEV), experts - 1
    np.testing.assert_array_equal(host(layer.place(ids)), np.arange(tokens * top_k).reshape(tokens, top_k))
    a, w = orc.values(*orc.quantise(x.double().numpy())), orc.values(gate_up[0][e], gate_up[1][e])
    (gate, dg), (up, du) = product(a, w[:inner]), product(a, w[inner:])
    want = orc.silu(gate) * up
    bound = 1.1 * dg * (np.abs(up) + du) + np.abs(gate) * du + 8 * 2.0**-24 * np.abs(want)
    check(layer.up(x.to(DEV)), want.repeat(top_k, 0), bound.repeat(top_k, 0), torch.float16)
    rows = torch.from_numpy(rng.standard_normal((tokens * top_k, inner)).astype(np.float16))
    prob = rng.random((tokens, top_k)).astype(np.float32)
    y, dy = product(orc.values(*orc.quantise(rows.double().numpy())), orc.values(down[0][e], down[1][e]))
    y, dy, p = y.reshape(tokens, top_k, hidden), dy.reshape(tokens, top_k, hidden), prob.astype(np.float64)[:, :, None]
    check(layer.down(rows.to(DEV), dev(prob)), (y * p).sum(1), (dy * p).sum(1) + (np.abs(y) * p).sum(1) * (2.0**-11 + 2 * top_k * 2.0**-24) + 2.0**-25, torch.float16)


def test_experts_with_more_than_4_gib_of_rows():
    tokens, experts, top_k, hidden, inner = 2**18 + 1, 5, 4, 2112, 64
    rng = np.random.default_rng(11)
    gate_up, down = weights(rng, experts, 2 * inner, hidden), weights(rng, experts, hidden, inner)
    layer = programs.Mxfp4MoeLayer(tokens, experts, top_k, hidden, inner, *map(dev, gate_up), *map(dev, down))
    ids = torch.rand((tokens, experts), device=DEV).argsort(1)[:, :top_k].int().contiguous()
    slot = layer.place(ids).long()
    prob = torch.rand((tokens, top_k), device=DEV)
    act = torch.randn((tokens * top_k, inner), device=DEV).half()
    out = layer.down(act, prob)
    at = torch.from_numpy(sampled(tokens)).to(DEV)
    rows, chosen, p = act[slot[at]].double().cpu().numpy(), host(ids[at]), host(prob[at]).astype(np.float64)[:, :, None]
    y, dy = np.empty((*chosen.shape, hidden)), np.empty((*chosen.shape, hidden))
    for i, e in np.ndindex(*chosen.shape):
        y[i, e], dy[i, e] = (r[0] for r in product(orc.values(*orc.quantise(rows[i, e][None])), orc.values(down[0][chosen[i, e]], down[1][chosen[i, e]])))
    check(out[at], (y * p).sum(1), (dy * p).sum(1) + (np.abs(y) * p).sum(1) * (2.0**-11 + 2 * top_k * 2.0**-24) + 2.0**-25, torch.float16)


def same(a, b):
    """Bit for bit (rows that overflow fp16 end as NaN, which no comparison of values finds equal)."""
    assert torch.equal(a.view(torch.int16), b.view(torch.int16))


def test_a_layer_as_it_is_used_captured_and_replayed():
    layer, gate_up, down, x, logits, rng = moe_case(48, 64, 6, 512, 160, scoring="sigmoid", bias=np.linspace(-0.1, 0.1, 64), groups=8, top_groups=3, scale=2.5)
    x, logits = x.to(DEV), dev(logits)
    shared, gate = rows_of(rng, 48, 512, torch.float16).to(DEV), torch.randn(48, device=DEV).half()
    stream = torch.cuda.Stream()
    eager = layer.run(x, logits, shared, gate).clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = layer.run(x, logits, shared, gate)
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize()
        same(out, layer.run(x, logits, shared, gate) if step else eager)
        torch.cuda.synchronize()
        logits.copy_(logits.roll(1, 1))
        x.neg_()
        torch.cuda.synchronize()
        eager = layer.run(x, logits, shared, gate).clone()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        same(out, eager)
    # the parts make the same
    ids, prob = layer.route(logits)
    layer.place(ids)
    same(layer.down(layer.up(x), prob, shared, gate), eager)


def test_experts_refuse_what_does_not_fit():
    layer, gate_up, down, x, logits, _ = moe_case(4, 8, 2, 64, 32)
    x, logits = x.to(DEV), dev(logits)
    ids, prob = layer.route(logits)
    for call in (lambda: layer.route(logits[:3]), lambda: layer.route(logits.half()), lambda: layer.place(ids.long()), lambda: layer.up(x[:, :32]), lambda: layer.up(x[:3]),
                 lambda: layer.down(layer.act[:1], prob), lambda: layer.down(layer.act, prob, shared=x), lambda: layer.run(x.cpu(), logits)):
        with pytest.raises(ValueError):
            call()
    args = [4, 8, 2, 64, 32, *map(dev, gate_up), *map(dev, down)]
    with pytest.raises(ValueError):
        programs.Mxfp4MoeLayer(*args, bias=np.zeros(7))
    with pytest.raises(ValueError):
        programs.Mxfp4MoeLayer(*args[:5], *args[7:], *args[5:7])
    with pytest.raises(lib.OrxError):
        programs.Mxfp4MoeLayer(*args, groups=3)
