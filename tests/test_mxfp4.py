"""MXFP4 without a GPU: the oracle's format, the layout of the products' weights, variants and refusals of the symbols, argument lists."""
import numpy as np
import pytest
import torch

from oracle import mxfp4 as orc
from orinfer_amd import lib, mxfp4
from tests.started_util import reported, started


def test_oracle_rounds_to_nearest_even_codes_and_saturates():
    x = np.zeros((1, 32))
    x[0, :12] = [4, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7.9, -0.3, -5.1]
    codes, exponents = orc.quantise(x)
    assert exponents[0, 0] == 127  # 7.9 has the power of 4, two exponents above 1
    got = orc.values(codes, exponents)[0, :12]
    np.testing.assert_array_equal(got, [4, 0, 1, 1, 2, 2, 4, 4, 6, 6, -0.5, -6])
    codes, exponents = orc.quantise(x, ceil=True)
    assert exponents[0, 0] == 128 and orc.values(codes, exponents)[0, 9] == 8
    for largest, byte in ((6.0, 127), (6.0001, 128), (8.0, 128)):
        assert orc.quantise(np.full((1, 32), largest), ceil=True)[1][0, 0] == byte
    assert orc.quantise(np.zeros((1, 32)))[1][0, 0] == 0 and orc.quantise(np.full((1, 3), np.inf))[1][0, 0] == 255


@pytest.mark.parametrize("n,k,paired", [(16, 256, False), (40, 96, False), (33, 544, False), (32, 256, True), (24, 64, True), (70, 288, True)])
def test_tiles_hold_every_block_and_power_where_a_lane_reads_it(n, k, paired):
    rng = np.random.default_rng(n * k)
    codes = torch.from_numpy(rng.integers(0, 256, (2, n, k // 2), dtype=np.uint8))
    exponents = torch.from_numpy(rng.integers(0, 256, (2, n, k // 32), dtype=np.uint8))
    w, ws = mxfp4.tiles(codes, exponents, paired=paired)
    half = n // 2 if paired else n
    tiles, steps = -(-half // 16) * (2 if paired else 1), -(-k // 256)
    assert w.shape == (2, tiles, steps, 8, 16, 16) and ws.shape == (2, tiles, steps, 16, 2, 4)
    assert w.is_contiguous() and ws.is_contiguous()
    seen = torch.zeros((2, n, k // 32), dtype=torch.int32)
    for tile in range(tiles):
        for r in range(16):
            row = (tile // 2 * 16 + r) if paired else tile * 16 + r
            live = row < half
            row += half if paired and tile % 2 else 0
            for step in range(steps):
                for b in range(8):
                    block = step * 8 + b
                    if live and block < k // 32:
                        assert torch.equal(w[:, tile, step, b, r], codes[:, row, block * 16:block * 16 + 16])
                        assert torch.equal(ws[:, tile, step, r, b & 1, b >> 1], exponents[:, row, block])
                        seen[:, row, block] += 1
                    else:
                        assert not w[:, tile, step, b, r].any() and not ws[:, tile, step, r, b & 1, b >> 1].any()
    assert (seen == 1).all()


def test_tiles_refuse_what_does_not_go_together():
    good = torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((4, 2), dtype=torch.uint8)
    mxfp4.tiles(*good)
    for codes, exponents, paired in ((good[0].int(), good[1], False), (good[0], good[1][:, :1], False), (good[0][:, :31], good[1], False),
                                     (good[0][:3], good[1][:3], True), (good[0][:0], good[1][:0], False), (good[0][:, :24], good[1], False)):
        with pytest.raises(ValueError):
            mxfp4.tiles(codes, exponents, paired=paired)


def test_arguments_in_launch_order():
    assert lib.Kernel("mxfp4_quantization", K=100).arg_names == ["Q", "S", "X", "rows"]
    assert lib.Kernel("mxfp4_dequantization", K=100).arg_names == ["Q", "S", "Y", "rows"]
    shape = dict(N=96, K=320)
    assert lib.Kernel("mxfp4_projection", M=3, **shape).arg_names == ["A", "AS", "Out", "W", "WS"]
    assert lib.Kernel("mxfp4_projection", M=3, dynamic_rows=True, **shape).arg_names == ["A", "AS", "Out", "W", "WS", "m"]
    assert lib.Kernel("mxfp4_projection", M=3, input_dtype="bfloat16", **shape).arg_names == ["A", "Out", "W", "WS"]
    grouped = dict(rows=12, E=4, tiles=8, **shape)
    assert lib.Kernel("mxfp4_grouped", **grouped).arg_names == ["A", "AS", "Out", "TileCount", "TileUnits", "W", "WS"]
    assert lib.Kernel("mxfp4_grouped", gather=True, **grouped).arg_names == ["A", "AS", "Out", "SlotToken", "TileCount", "TileUnits", "W", "WS"]
    assert lib.Kernel("mxfp4_grouped", gather=True, input_dtype="float16", **grouped).arg_names == ["A", "Out", "SlotToken", "TileCount", "TileUnits", "W", "WS"]
    router = dict(M=3, E=64, top_k=4)
    assert lib.Kernel("router_topk", scoring="sigmoid", **router).arg_names == ["IDs", "Logits", "Prob"]
    assert lib.Kernel("router_topk", bias=True, dynamic_rows=True, **router).arg_names == ["Bias", "IDs", "Logits", "Prob", "m"]
    assert lib.Kernel("router_topk?M=3&E=64&top_k=4&scoring=sigmoid&scale=2.5").arg_names == ["IDs", "Logits", "Prob"]


GROUPED = dict(rows=12, E=4, N=96, K=320, tiles=8)
ROUTER = dict(M=3, E=64, top_k=4)


@pytest.mark.parametrize("symbol,variant", [
    ("mxfp4_quantization", dict(K=0)), ("mxfp4_quantization", dict(K=64, pad=64)), ("mxfp4_quantization", dict(K=64, scale="round")),
    ("mxfp4_quantization", dict(K=64, input_dtype="int8")), ("mxfp4_quantization", dict(K=64, M=0)), ("mxfp4_quantization", dict(K=1 << 25)),
    ("mxfp4_quantization", dict(K=64, layout="columns")), ("mxfp4_quantization", dict(K=64, layout="tiles", pad=256)),
    ("mxfp4_projection", dict(M=17, N=96, K=320, input_dtype="float16")), ("mxfp4_projection", dict(M=16, N=96, K=1 << 16, input_dtype="float16")),
    ("mxfp4_projection", dict(M=1, N=96, K=320, input_dtype="float32")), ("mxfp4_grouped", dict(GROUPED, block_m=64, input_dtype="float16")), ("mxfp4_grouped", dict(GROUPED, block_m=32)),
    ("mxfp4_grouped", dict(GROUPED, input_dtype="bfloat16")), ("mxfp4_dequantization", dict(K=64, output_dtype="e4m3")), ("mxfp4_dequantization", dict(K=64, scale="ceil")),
    ("mxfp4_projection", dict(M=1, N=96, K=100)), ("mxfp4_projection", dict(M=0, N=96, K=320)), ("mxfp4_projection", dict(M=1, N=0, K=320)),
    ("mxfp4_projection", dict(M=1, N=97, K=320, epilogue="swiglu")), ("mxfp4_projection", dict(M=1, N=96, K=320, epilogue="gelu")),
    ("mxfp4_projection", dict(M=1, N=96, K=320, output_dtype="int8")), ("mxfp4_projection", dict(M=1, N=96, K=320, packed_k=128)),
    ("mxfp4_grouped", dict(GROUPED, block_m=24)), ("mxfp4_grouped", dict(GROUPED, E=0)), ("mxfp4_grouped", dict(GROUPED, tiles=0)),
    ("mxfp4_grouped", dict(GROUPED, K=40)),
    ("router_topk", dict(ROUTER, scoring="relu")), ("router_topk", dict(ROUTER, groups=3)), ("router_topk", dict(ROUTER, groups=8, top_groups=9)),
    ("router_topk", dict(ROUTER, groups=8, top_groups=0)), ("router_topk", dict(ROUTER, top_k=9, groups=8, top_groups=1)),
    ("router_topk", dict(ROUTER, groups=8, group_best=3)), ("router_topk", dict(ROUTER, scale=0)), ("router_topk", dict(ROUTER, scale=-1.5)),
    ("router_topk", dict(ROUTER, scale="much")), ("router_topk", dict(ROUTER, scale=True)), ("router_topk", dict(ROUTER, bias=1)),
    ("router_topk", dict(ROUTER, scoring="sigmoid", quantize_hidden=64)), ("router_topk", dict(ROUTER, scoring="sigmoid", metadata=True)),
    ("router_topk", dict(M=3, E=128, top_k=4, groups=128, top_groups=4)), ("router_topk_warp", dict(M=3, E=64, top_k=4, scoring="sigmoid")),
])
def test_variants_that_are_not_served_are_refused(symbol, variant):
    with pytest.raises(lib.OrxError) as error:
        lib.Kernel(symbol, **variant)
    assert error.value.code == lib.ORX_ERR_BAD_VARIANT and symbol.removesuffix("_warp") in str(error.value) or "variant field" in str(error.value) or "dtype" in str(error.value)


def test_rows_outside_the_capacity_and_bad_pointers_are_refused_before_anything_is_enqueued():
    linear = lib.Kernel("mxfp4_projection", M=4, N=96, K=320, dynamic_rows=True)
    good = dict(A=4096, AS=4096, Out=4096, W=4096, WS=4096, m=4)
    for change, code in ((dict(m=5), lib.ORX_ERR_ROWS), (dict(m=0), lib.ORX_ERR_ROWS), (dict(A=4104), lib.ORX_ERR_BAD_ARGUMENT), (dict(W=0), lib.ORX_ERR_BAD_ARGUMENT),
                         (dict(Out=4097), lib.ORX_ERR_BAD_ARGUMENT)):
        with pytest.raises(lib.OrxError) as error:
            linear(stream=0, **dict(good, **change))
        assert error.value.code == code
    quantise = lib.Kernel("mxfp4_quantization", K=64)
    for change, code in ((dict(rows=0), lib.ORX_ERR_ROWS), (dict(X=4097), lib.ORX_ERR_BAD_ARGUMENT), (dict(Q=4098), lib.ORX_ERR_BAD_ARGUMENT),
                         (dict(S=0), lib.ORX_ERR_BAD_ARGUMENT), (dict(rows=1 << 25), lib.ORX_ERR_ROWS)):
        with pytest.raises(lib.OrxError) as error:
            quantise(stream=0, **dict(dict(Q=4096, S=4096, X=4096, rows=2), **change))
        assert error.value.code == code
    # the largest rows of the longest K still fit a launch
    longest = lib.Kernel("mxfp4_quantization", K=1 << 24)
    assert longest.geometry(0)[0][0] < 1 << 24


def test_records_name_the_kernel_that_runs():
    for kernel in (lib.Kernel("mxfp4_projection", M=200, N=96, K=320, dynamic_rows=True), lib.Kernel("mxfp4_grouped", **GROUPED),
                   lib.Kernel("mxfp4_quantization", K=64, M=300), lib.Kernel("router_topk", **ROUTER, scoring="sigmoid")):
        rows = (1, 17, 64, 65, 200) if kernel.symbol == "mxfp4_projection" else (0,)
        for r in rows:
            assert reported(kernel, r) in started(kernel, r)


# a shape for every kind of tile: 64 x 128 as a whole and in halves of an odd number of steps, 128 x 128 likewise and of an even number, 256 x 256, halves of a step each
TILES = [((160, 17400, 512), 256, 52224), ((440, 4090, 2080), 512, 104448), ((256, 17402, 512), 256, 69632), ((700, 4096, 3232), 512, 139264), ((680, 4002, 1536), 512, 139264),
         ((2049, 4098, 512), 512, 139264), ((200, 8100, 512), 512, 104448)]


def test_a_projection_takes_larger_tiles_where_there_are_more():
    """Threads and LDS of the kernel by rows (without a device 256 CUs are taken)."""
    linear = lib.Kernel("mxfp4_projection", M=8192, N=4096, K=4096, dynamic_rows=True)
    assert [started(linear, rows)[0][1:] for rows in (32, 64, 300, 512, 2048, 8192)] == [(512, 32768), (512, 32768), (256, 32768), (512, 104448), (256, 69632), (512, 139264)]
    assert all(len(started(linear, rows)) == 1 for rows in (1, 64, 65, 8192))
    for (rows, n, k), threads, lds in TILES:
        assert started(lib.Kernel("mxfp4_projection", M=rows, N=n, K=k), 0)[0][1:] == (threads, lds), (rows, n, k)
    for block_m, lds in ((16, 8192), (64, 52224), (128, 69632), (256, 139264)):
        assert started(lib.Kernel("mxfp4_grouped", **GROUPED, block_m=block_m))[0][2] == lds


def test_oracle_routes_by_hand():
    logits = np.log([[0.1, 0.4, 0.2, 0.3]])
    ids, weights = orc.routes(logits, 2)
    assert ids.tolist() == [[1, 3]] and np.allclose(weights, [[4 / 7, 3 / 7]])
    ids, weights = orc.routes(logits, 2, bias=[0, -1, 0, 0], renormalize=False, scale=2.0)
    assert ids.tolist() == [[3, 2]] and np.allclose(weights, [[0.6, 0.4]])
    ids, _ = orc.routes(logits, 2, groups=2, top_groups=1)  # 0.5 against 0.5 up to rounding: groups by their best alone
    ids, _ = orc.routes(logits, 2, groups=2, top_groups=1, group_best=1)
    assert ids.tolist() == [[1, 0]]
    ids, weights = orc.routes(logits, 3, bias=[0, -np.inf, -np.inf, 0])
    assert ids.tolist() == [[3, 0, 1]] and weights[0, 2] == 0
