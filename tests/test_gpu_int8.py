"""Rows of 8-bit integers and linears with them against the 64-bit oracle.

Tolerances, derived: codes, scales and zero points are equal.  A product's sum is exact in 32 bits; then one rounding of 2^-24 each for its conversion, the channel's scale, the row's scale and the
bias (of the value in front of it), and the output's half step 2^-11 (fp16), 2^-8 (bf16), 2^-24 (fp32) of the value, 2^-25 where fp16 is subnormal.  SwiGLU: |d silu| <= 1.1 |d gate|,
|silu(g)| <= |g|, and 8 * 2^-24 of the value for exp, quotient and product."""
import numpy as np
import pytest
import torch

from oracle import int8 as orc
from orinfer_amd import byte_tiles, int8, lib, programs
from tests.gpu_util import kernel

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
HALF = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}


def rows_of(rng, rows, k, dtype, side=0.0):
    x = (rng.standard_normal((rows, k)) + side) * np.exp2(rng.integers(-6, 6, (rows, 1)))
    x.reshape(-1)[rng.integers(0, x.size, max(1, x.size // 500))] *= 20
    return torch.from_numpy(x.astype(np.float32)).to(dtype)


def weights_of(rng, *shape):
    w = rng.integers(-127, 128, shape, dtype=np.int8)
    return w, (rng.random(shape[:-1]) * 0.9 + 0.1).astype(np.float32) / 64


def check(got, want, bound, dtype):
    got = got.detach().cpu().double().numpy()
    with np.errstate(invalid="ignore"):
        off = np.abs(got - want)
    allowed = bound + np.abs(want) * HALF[dtype] * 1.0001 + (2.0**-25 if dtype == torch.float16 else 0)
    fine = (off <= allowed) | (got == want) | (np.isnan(got) & np.isnan(want))  # (fp16 activations may be infinite: infinities and NaN are where 64 bits have them)
    if dtype == torch.float16:  # rounding to nearest gives infinity from 65504 plus half a step of 32 on
        fine |= np.isinf(got) & (np.sign(got) == np.sign(want)) & (np.abs(want) + bound >= 65520)
    assert fine.all(), (off.max(), np.unravel_index((off - allowed).argmax(), off.shape))


def product(codes, scales, zeros, w, w_scale, bias=None):
    """want, and the bound of its roundings"""
    whole = (codes.astype(np.int64) - zeros[:, None].astype(np.int64)).astype(np.float64) @ w.T.astype(np.float64)  # (exact: below 2^53)
    want = whole * w_scale.astype(np.float64) * scales[:, None]
    bound = 3 * 2.0**-24 * 1.0001 * np.abs(want)
    if bias is not None:
        want = want + bias.astype(np.float64)
        bound = bound + 2.0**-24 * 1.0001 * (np.abs(want) + bound)
    return want, bound


def swiglu(want, bound):
    half = want.shape[1] // 2
    (gate, up), (eg, eu) = (want[:, :half], want[:, half:]), (bound[:, :half], bound[:, half:])
    silu = orc.silu(gate)
    return silu * up, 1.1 * eg * (np.abs(up) + eu) + np.abs(silu) * eu + 8 * 2.0**-24 * np.abs(silu * up)


# ---- quantisation ------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 8), (3, 33), (5, 100), (7, 2560), (64, 264), (130, 1000), (33, 4096), (9, 2049), (6, 8200), (5, 17408), (2, 40001), (4100, 500), (4097, 7),
                                    (1025, 1100), (1024, 4096), (1026, 5120), (1030, 9000), (16390, 304), (8201, 1304), (4099, 1504), (1601, 5000)])
def test_quantisation_is_the_oracles(rows, k, name, zero_points):
    x = rows_of(np.random.default_rng(rows * k), rows, k, TYPES[name], side=1.0 * zero_points)
    codes, scales, zeros = orc.quantise(x.double().numpy(), zero_points)
    # surplus rows behind the last stay as they were
    q = torch.full((rows + 1, int8.padded(k)), 91, dtype=torch.int8, device=DEV)
    s, z = torch.full((rows + 1,), 7.5, device=DEV), torch.full((rows + 1,), 91, dtype=torch.int32, device=DEV)
    kernel("int8_token_quantization", K=k, input_dtype=name, zero_points=zero_points)(Q=q, S=s, X=x.to(DEV), rows=rows, **({"Z": z} if zero_points else {}))
    written = -(-k // 256) * 256
    np.testing.assert_array_equal(q[:rows, :k].cpu().numpy(), codes)
    np.testing.assert_array_equal(s[:rows].cpu().double().numpy(), scales)
    if zero_points:
        np.testing.assert_array_equal(z[:rows].cpu().numpy(), zeros)
    else:
        assert (q[:rows, k:written] == 0).all()
    assert (q[:rows, written:] == 91).all() and (q[rows] == 91).all() and s[rows] == 7.5 and z[rows] == 91
    again = int8.quantize(x.to(DEV), zero_points)
    assert torch.equal(again[0], q[:rows, :k]) and torch.equal(again[1], s[:rows]) and (not zero_points or torch.equal(again[2], z[:rows]))


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("rows,k", [(1, 128), (1, 7), (5, 300), (16, 256), (17, 2560), (100, 1000), (33, 4096), (4099, 200), (1030, 1500), (1025, 5000), (19, 9000), (16390, 304), (8201, 1304), (1042, 1504), (1601, 5000), (4103, 2568), (2050, 1501)])
def test_quantisation_by_tiles(rows, k, name, zero_points):
    x = rows_of(np.random.default_rng(rows * k), rows, k, TYPES[name], side=1.0 * zero_points).to(DEV)
    want = int8.quantize(x, zero_points)
    tiles, steps = -(-rows // 16), int8.steps(k)
    q = torch.full((tiles * steps * 2048 + 16,), 91, dtype=torch.int8, device=DEV)
    s, z = torch.full((rows + 1,), 7.5, device=DEV), torch.full((rows + 1,), 91, dtype=torch.int32, device=DEV)
    kernel("int8_token_quantization", K=k, input_dtype=name, zero_points=zero_points, layout="tiles")(Q=q, S=s, X=x, rows=rows, **({"Z": z} if zero_points else {}))
    got = q[:-16].view(tiles, steps, 8, 16, 16).permute(0, 3, 1, 2, 4).reshape(tiles * 16, steps * 128)
    assert torch.equal(got[:rows, :k], want[0]) and torch.equal(s[:rows], want[1]) and s[rows] == 7.5 and z[rows] == 91 and (q[-16:] == 91).all()
    assert (got[rows:] == 91).all()  # rows that are not there stay as they were
    assert torch.equal(z[:rows], want[2]) if zero_points else (got[:rows, k:] == 0).all()


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("name", list(TYPES))
def test_values_at_and_beside_the_borders_of_codes(name, zero_points):
    """Scales whose quotients lie at k + 1/2 or next to it: the largest value decides the scale, the others are its halves and their neighbours."""
    dtype, levels = TYPES[name], 255 if zero_points else 127
    largest = torch.tensor([127.0, 254.0, 63.5, 1.0, 0.3, 255.0, 510.0, 3e-5, 300.0, 7.0]).to(dtype)
    x = torch.zeros((len(largest), 1600), dtype=dtype)
    for row, top in enumerate(largest.double().tolist()):
        scale = float(np.float32(top) / np.float32(levels))
        ties = torch.tensor([(j + 0.5) * scale * (-1) ** j for j in range(0, levels - 1)], dtype=torch.float64)
        near = ties.float().to(dtype)
        values = torch.cat([near, near.nextafter(torch.zeros_like(near)), near.nextafter(torch.full_like(near, torch.inf)), -near])
        if zero_points:
            values = values.abs().clamp(max=top)
        values = values[values.abs() <= top]
        x[row, 1:1 + len(values)] = values
        x[row, 0] = top
    codes, scales, zeros = orc.quantise(x.double().numpy(), zero_points)
    got = int8.quantize(x.to(DEV), zero_points)
    np.testing.assert_array_equal(got[1].cpu().double().numpy(), scales)
    np.testing.assert_array_equal(got[0].cpu().numpy(), codes)
    if zero_points:
        np.testing.assert_array_equal(got[2].cpu().numpy(), zeros)


@pytest.mark.parametrize("name", list(TYPES))
def test_rows_of_zeros_small_values_infinities_and_nan(name):
    dtype = TYPES[name]
    tiny = torch.finfo(dtype).tiny
    x = torch.zeros((8, 200), dtype=dtype)
    x[1] = tiny
    x[2, 5] = torch.inf
    x[3, 199] = torch.nan
    x[4, 7] = -torch.inf
    x[5] = torch.finfo(dtype).max
    x[6, ::2] = -torch.finfo(dtype).max
    x[7, 3] = torch.finfo(dtype).smallest_normal / 4
    for zero_points in (False, True):
        codes, scales, zeros = orc.quantise(x.double().numpy(), zero_points)
        got = int8.quantize(x.to(DEV), zero_points)
        np.testing.assert_array_equal(got[1].cpu().double().numpy(), scales)
        np.testing.assert_array_equal(got[0].cpu().numpy(), codes)
        assert np.isnan(scales[2:5]).all() and np.isfinite(scales[[0, 1, 5, 6, 7]]).all()
        if zero_points:
            np.testing.assert_array_equal(got[2].cpu().numpy(), zeros)
    if name != "float16":  # a range that leaves fp32
        x = torch.full((1, 9), torch.finfo(dtype).max, dtype=dtype)
        x[0, 0] *= -1
        codes, scales, zeros = int8.quantize(x.to(DEV), zero_points=True)
        assert scales.isnan().all() and (codes == 0).all() and (zeros == 0).all()


def test_shapes_of_quantize():
    x = torch.randn((2, 3, 5, 70), device=DEV, dtype=torch.bfloat16)
    codes, scales, zeros = int8.quantize(x.transpose(0, 2), zero_points=True)
    assert codes.shape == (5, 3, 2, 70) and scales.shape == zeros.shape == (5, 3, 2)
    flat = int8.quantize(x.transpose(0, 2).reshape(-1, 70), zero_points=True)
    assert torch.equal(flat[0].reshape(codes.shape), codes) and torch.equal(flat[1].view(5, 3, 2), scales)
    empty = int8.quantize(x[:0])
    assert empty[0].shape == (0, 3, 5, 70) and empty[1].shape == (0, 3, 5)


# ---- linears -----------------------------------------------------------------------------------------------------------------------------------
LINEARS = [(1, 16, 128), (1, 9, 7), (1, 1, 1), (6, 1, 300), (7, 300, 2560), (8, 130, 2048), (8, 70, 4100), (1, 300, 2560), (2, 33, 5000), (3, 48, 640), (4, 31, 4097), (5, 96, 1000), (16, 128, 1024), (17, 40, 129), (31, 260, 2560), (33, 513, 512), (64, 100, 1111),
           (65, 300, 300), (130, 520, 1280), (200, 1030, 384), (300, 264, 2048), (513, 700, 257),
           (1024, 256, 64), (1030, 520, 300), (2500, 1100, 640), (500, 258, 4096), (1024, 1058, 129), (1024, 2050, 520), (2048, 2050, 520), (2048, 4098, 2560), (1500, 2050, 520), (2048, 2050, 1111), (2048, 5000, 2560)]


@pytest.mark.parametrize("zero_points,biased", [(False, False), (True, True), (True, False), (False, True)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,n,k", LINEARS)
def test_linear(rows, n, k, dtype, zero_points, biased):
    rng = np.random.default_rng(rows * n + k)
    x = rows_of(rng, rows, k, dtype, side=0.7 * zero_points)
    w, scale = weights_of(rng, n, k)
    bias = rng.standard_normal(n).astype(np.float32) * 30 if biased else None
    linear = programs.Int8Linear(torch.from_numpy(w), torch.from_numpy(scale), rows, bias=bias, zero_points=zero_points, dtype=dtype)
    got = linear.run(x.to(DEV))
    want, bound = product(*orc.quantise(x.double().numpy(), zero_points), w, scale, bias)
    assert got.shape == (rows, n) and got.dtype == dtype
    check(got, want, bound, dtype)


@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("rows,n,k", [(1, 32, 128), (1, 34, 2000), (3, 300, 1111), (20, 66, 512), (64, 1000, 256), (150, 258, 640), (400, 514, 300), (1500, 1058, 520), (500, 258, 4096), (1024, 1058, 129), (1024, 2050, 520), (2048, 2050, 520), (2040, 4106, 2560), (1500, 2050, 520), (2048, 2050, 1111), (2040, 5004, 2560)])
def test_linear_with_swiglu(rows, n, k, zero_points):
    rng = np.random.default_rng(rows * n + k)
    x = rows_of(rng, rows, k, torch.bfloat16)
    w, scale = weights_of(rng, n, k)
    bias = rng.standard_normal(n).astype(np.float32)
    linear = programs.Int8Linear(torch.from_numpy(w), torch.from_numpy(scale), rows, bias=bias, zero_points=zero_points, dtype=torch.bfloat16, epilogue="swiglu")
    want, bound = swiglu(*product(*orc.quantise(x.double().numpy(), zero_points), w, scale, bias))
    got = linear.run(x.to(DEV))
    assert got.shape == (rows, n // 2)
    check(got, want, bound, torch.bfloat16)


def test_extreme_codes_add_exactly():
    """All codes at their ends over the longest K: the bracket comes close to 2^31."""
    k = int8.MOST_K
    w = np.full((5, k), -128, np.int8)
    w[1] = 127
    w[2, ::2] = 127
    scale = np.full(5, 2.0**-20, np.float32)
    x = torch.full((3, k), 1.0, dtype=torch.bfloat16)
    x[1, 1::2] = -1
    x[2] = -1
    for zero_points in (False, True):
        linear = programs.Int8Linear(torch.from_numpy(w), torch.from_numpy(scale), 3, zero_points=zero_points, dtype=torch.bfloat16)
        want, bound = product(*orc.quantise(x.double().numpy(), zero_points), w, scale)
        check(linear.run(x.to(DEV)), want, bound, torch.bfloat16)


@pytest.mark.parametrize("rows", [1, 3, 40, 300])
def test_rows_that_are_not_finite_stay_to_themselves(rows):
    rng = np.random.default_rng(rows)
    x = rows_of(rng, rows, 300, torch.bfloat16)
    bad = x.clone()
    bad[rows // 2, 7] = torch.inf
    w, scale = weights_of(rng, 100, 300)
    linear = programs.Int8Linear(torch.from_numpy(w), torch.from_numpy(scale), rows, dtype=torch.bfloat16)
    fine = linear.run(x.to(DEV)).clone()
    got = linear.run(bad.to(DEV))
    assert got[rows // 2].isnan().all()
    keep = [i for i in range(rows) if i != rows // 2]
    assert torch.equal(got[keep], fine[keep])


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("rows,n,k", [(1, 33, 256), (6, 130, 384), (70, 50, 129), (260, 530, 128), (1100, 300, 300), (30, 130, 2560), (490, 250, 4096), (1020, 1050, 129), (1020, 2042, 520), (2045, 2042, 520), (2045, 4106, 2560), (500, 258, 4096), (2045, 2050, 1111), (2045, 5002, 2560)])
def test_projection_writes_its_rows_and_columns_only(rows, n, k, name):
    rng = np.random.default_rng(n)
    x = rows_of(rng, rows, k, torch.float32)
    w, scale = weights_of(rng, n, k)
    q = torch.empty((-(-rows // 16), int8.steps(k), 2048), dtype=torch.int8, device=DEV)
    s = torch.empty(rows, device=DEV)
    kernel("int8_token_quantization", K=k, input_dtype="float32", layout="tiles")(Q=q, S=s, X=x.to(DEV), rows=rows)
    project = kernel("int8_token_projection", M=rows + 3, N=n, K=k, dynamic_rows=True, output_dtype=name)
    out = torch.full((rows + 3, n), 91.0, dtype=TYPES[name], device=DEV)
    tiles, channels = byte_tiles.tiles(torch.from_numpy(w)).to(DEV), byte_tiles.channels(torch.from_numpy(scale)).to(DEV)
    project(A=q, AS=s, Out=out, W=tiles, WS=channels, m=rows)
    codes, scales, zeros = orc.quantise(x.double().numpy())
    check(out[:rows], *product(codes, scales, zeros, w, scale), TYPES[name])
    assert (out[rows:] == 91).all()


def test_fewer_rows_than_the_capacity_and_a_result_given_back():
    rng = np.random.default_rng(5)
    w, scale = weights_of(rng, 256, 256)
    linear = programs.Int8Linear(torch.from_numpy(w), torch.from_numpy(scale / 16), 300, dtype=torch.bfloat16)
    for rows in (1, 2, 4, 5, 17, 40, 300):
        x = rows_of(rng, rows, 256, torch.bfloat16).to(DEV)
        first = linear.run(x)
        assert first.shape == (rows, 256)
        held = first.clone()
        want, bound = product(*orc.quantise(held.cpu().double().numpy()), w, scale / 16)
        check(linear.run(first), want, bound, torch.bfloat16)  # its own last result
    assert linear.run(torch.empty((0, 256), dtype=torch.bfloat16, device=DEV)).shape == (0, 256)


def test_captured_and_replayed():
    rng = np.random.default_rng(6)
    w, scale = weights_of(rng, 300, 520)
    linear = programs.Int8Linear(torch.from_numpy(w), torch.from_numpy(scale), 64, dtype=torch.float16, zero_points=True)
    for rows in (1, 33):
        x = rows_of(rng, rows, 520, torch.float16).to(DEV)
        linear.run(x)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = linear.run(x)
        for seed in range(3):
            fresh = rows_of(np.random.default_rng(seed), rows, 520, torch.float16)
            x.copy_(fresh)
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            check(out, *product(*orc.quantise(fresh.double().numpy(), True), w, scale), torch.float16)


def test_two_streams_with_objects_of_their_own():
    rng = np.random.default_rng(8)
    w, scale = weights_of(rng, 500, 700)
    streams = [torch.cuda.Stream() for _ in range(2)]
    linears = [programs.Int8Linear(torch.from_numpy(w), torch.from_numpy(scale), 100, dtype=torch.float16) for _ in range(2)]
    xs = [rows_of(rng, 100, 700, torch.float16).to(DEV) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for linear, x, stream in zip(linears, xs, streams):
            with torch.cuda.stream(stream):
                out = linear.run(x)
    torch.cuda.synchronize()
    for linear, x in zip(linears, xs):
        check(linear.out, *product(*orc.quantise(x.cpu().double().numpy()), w, scale), torch.float16)


def test_matrices_and_rows_beyond_4_gib():
    """Bytes of weights, of rows and of results that 32 bits do not count.  (Codes are random, the weights' laid out already: each tile has its own multiple, told by its channels' results.)"""
    g = torch.Generator(device=DEV).manual_seed(1)
    n, k = 66000, 65536  # 4.3 GB of weights
    tiles = torch.randint(-127, 128, (k // 128, -(-n // 64) * 4, 8, 16, 16), dtype=torch.int8, device=DEV, generator=g)
    scale = torch.rand(-(-n // 64) * 64, device=DEV, generator=g) / 2**20
    last = list(range(65984, 66000))
    for rows in (1, 30, 60, 200, 300, 500):  # (a launch of every kind that the sizes allow)
        x = torch.randint(-127, 128, (rows, k), device=DEV, generator=g)
        x[:, 0] = 127  # (scale 1, codes the values themselves)
        q, s = torch.empty((-(-rows // 16), k // 128, 2048), dtype=torch.int8, device=DEV), torch.empty(rows, device=DEV)
        kernel("int8_token_quantization", K=k, input_dtype="float32", layout="tiles")(Q=q, S=s, X=x.float(), rows=rows)
        out = torch.empty((rows, n), device=DEV)
        kernel("int8_token_projection", M=rows, N=n, K=k, output_dtype="float32")(A=q, AS=s, Out=out, W=tiles, WS=scale)
        for tile in (0, last[0] // 16):
            w = tiles[:, tile].movedim(2, 0).reshape(16, k).double()  # (16 channels, K in order: steps, pieces, bytes)
            want = (x.double() @ w.T) * scale[tile * 16:tile * 16 + 16].double()
            assert ((out[:, tile * 16:tile * 16 + 16].double() - want).abs() <= 3 * 2.0**-24 * 1.0001 * want.abs()).all(), (rows, tile)
    del tiles, out
    rows, n, k = 140000, 40, 65000  # 9 GB of codes
    x = torch.randint(-127, 128, (rows, k), dtype=torch.int8, device=DEV, generator=g).half()
    x[:, 0] = 127
    w = torch.randint(-127, 128, (n, k), dtype=torch.int8, device=DEV, generator=g)
    linear = programs.Int8Linear(w, torch.full((n,), 2.0**-14), rows, dtype=torch.float16)
    out = linear.run(x)
    want = x[-300:].double() @ w.double().T / 2.0**14
    assert ((out[-300:].double() - want).abs() <= (2.0**-11 + 2.0**-20) * want.abs() + 2.0**-25).all()
    del x, linear, out
    rows, n, k = 1 << 20, 4200, 64  # 8.8 GB of results
    x = torch.randint(-127, 128, (rows, k), dtype=torch.int8, device=DEV, generator=g).half()
    x[:, 0] = 127
    w = torch.randint(-127, 128, (n, k), dtype=torch.int8, device=DEV, generator=g)
    out = programs.Int8Linear(w, torch.full((n,), 2.0**-10), rows, dtype=torch.float16).run(x)
    want = x[-300:].double() @ w.double().T / 2.0**10
    assert ((out[-300:].double() - want).abs() <= (2.0**-11 + 2.0**-20) * want.abs() + 2.0**-25).all()


def test_refusals_of_tensors():
    w, scale = torch.zeros((32, 64), dtype=torch.int8), torch.ones(32)
    linear = programs.Int8Linear(w, scale, 4)
    for bad in (torch.zeros((5, 64), dtype=torch.float16, device=DEV), torch.zeros((1, 63), dtype=torch.float16, device=DEV), torch.zeros((1, 64), device=DEV), torch.zeros((1, 64), dtype=torch.float16),
                torch.zeros((2, 128), dtype=torch.float16, device=DEV)[:, ::2]):
        with pytest.raises(ValueError):
            linear.run(bad)
    with pytest.raises(ValueError):
        int8.quantize(torch.zeros((2, 0), device=DEV))
    with pytest.raises(ValueError):
        int8.quantize(torch.zeros((2, 4), dtype=torch.float64, device=DEV))


@pytest.mark.parametrize("layout", ["rows", "tiles"])
@pytest.mark.parametrize("zero_points", [False, True])
@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("rows,k", [(3, 33), (40, 300), (1030, 1100), (2050, 1501), (1601, 5000), (9, 9001)])
def test_behind_k_stands_the_code_of_0(rows, k, name, zero_points, layout):
    """... up to a multiple of 256: the row's zero point, or 0 without zero points and in rows that are not finite."""
    x = rows_of(np.random.default_rng(rows + k), rows, k, TYPES[name], side=1.0 * zero_points)
    x[rows // 2, k // 2] = torch.inf
    steps = int8.steps(k)
    q = torch.full((-(-rows // 16) * 16 * (steps | 1) * 128,), 91, dtype=torch.int8, device=DEV)
    s, z = torch.empty(rows, device=DEV), torch.zeros(rows, dtype=torch.int32, device=DEV)
    kernel("int8_token_quantization", K=k, input_dtype=name, zero_points=zero_points, layout=layout)(Q=q, S=s, X=x.to(DEV), rows=rows, **({"Z": z} if zero_points else {}))
    if layout == "tiles":
        tiles = -(-rows // 16)
        got = q[:tiles * steps * 2048].view(tiles, steps, 8, 16, 16).permute(0, 3, 1, 2, 4).reshape(tiles * 16, steps * 128)[:rows]
    else:
        got = q.view(-1, (steps | 1) * 128)[:rows, :steps * 128]
    assert torch.equal(got[:, k:].int(), z[:, None].expand(rows, steps * 128 - k)) and (got[rows // 2] == 0).all() and s[rows // 2].isnan()
    if zero_points:
        assert (z != 0).any()
