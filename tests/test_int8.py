"""Int8 linears and expert layers, and 16-bit expert layers, without a GPU: the oracle's rules, the layout of the products' weights, variants and refusals of the symbols, argument lists, devices."""
import numpy as np
import pytest
import torch

from oracle import int8 as orc
from orinfer_amd import byte_tiles, int8, lib, programs
from tests.started_util import reported, started
from tests.test_mxfp4_layer import gpus, launches  # noqa: F401  (fixture)


def test_oracle_rounds_quotients_to_even_and_takes_zero_points():
    codes, scales, zeros = orc.quantise([[127.0, 0.5, 1.5, 2.5, -2.5, -126.5, 3.4]])
    assert scales[0] == 1 and zeros[0] == 0 and codes[0].tolist() == [127, 0, 2, 2, -2, -126, 3]
    codes, scales, zeros = orc.quantise([[-51.0, 204.0, 0.0, 0.5, 1.5]], zero_points=True)
    assert scales[0] == 1 and zeros[0] == -77 and codes[0].tolist() == [-128, 127, -77, -77, -75]
    np.testing.assert_array_equal(orc.values(codes, scales, zeros), [[-51, 204, 0, 0, 2]])
    codes, scales, zeros = orc.quantise([[3.0, 5.0], [-3.0, -5.0]], zero_points=True)  # rows of one sign keep 0
    assert zeros.tolist() == [-128, 127] and codes.tolist() == [[25, 127], [-26, -128]]
    codes, scales, _ = orc.quantise([[0.0, 0.0], [np.inf, 1.0], [1e-35, 0.0]])
    assert scales[0] == scales[2] == 2.0**-100 and np.isnan(scales[1]) and not codes.any()


@pytest.mark.parametrize("n,k,paired,dtype", [(16, 128, False, torch.int8), (40, 96, False, torch.int8), (33, 301, False, torch.int8), (32, 256, True, torch.int8), (24, 64, True, torch.bfloat16),
                                              (70, 100, True, torch.float16), (5, 1, False, torch.bfloat16)])
def test_tiles_hold_every_byte_where_a_lane_reads_it(n, k, paired, dtype):
    rng = np.random.default_rng(n * k)
    size = torch.empty(0, dtype=dtype).element_size()
    raw = torch.from_numpy(rng.integers(0, 256, (2, n, k * size), dtype=np.uint8))
    w = byte_tiles.tiles(raw.view(dtype), paired=paired)
    half = n // 2 if paired else n
    tiles, steps = -(-n // 64) * 4, -(-k * size // 256) * 2
    assert w.shape == (2, steps, tiles, 8, 16, 16) and w.is_contiguous() and w.dtype == torch.uint8
    wide = torch.nn.functional.pad(raw, (0, steps * 128 - k * size)).view(2, n, steps, 8, 16)
    values = torch.arange(1.0, n + 1)
    channels = byte_tiles.channels(values, paired=paired)
    assert channels.shape == (tiles, 16) and channels.is_contiguous()
    for tile in range(tiles):
        for r in range(16):
            row = (tile // 2 * 16 + r) if paired else tile * 16 + r
            live = row < half
            row += half if paired and tile % 2 else 0
            assert torch.equal(w[:, :, tile, :, r], wide[:, row] if live else torch.zeros_like(wide[:, 0]))
            assert channels[tile, r] == (values[row] if live else 0)


def test_tiles_refuse_what_they_do_not_lay_out():
    for weight, paired in ((torch.zeros((4, 32)), False), (torch.zeros((4, 32), dtype=torch.uint8), False), (torch.zeros(4, dtype=torch.int8), False), (torch.zeros((3, 32), dtype=torch.int8), True),
                           (torch.zeros((0, 32), dtype=torch.int8), False), (torch.zeros((4, 0), dtype=torch.int8), False)):
        with pytest.raises(ValueError):
            byte_tiles.tiles(weight, paired=paired)
    with pytest.raises(ValueError):
        byte_tiles.channels(torch.zeros(3), paired=True)


def test_arguments_in_launch_order():
    assert lib.Kernel("int8_token_quantization", K=100).arg_names == ["Q", "S", "X", "rows"]
    assert lib.Kernel("int8_token_quantization", K=100, zero_points=True).arg_names == ["Q", "S", "X", "Z", "rows"]
    shape = dict(N=96, K=320)
    assert lib.Kernel("int8_token_projection", M=3, **shape).arg_names == ["A", "AS", "Out", "W", "WS"]
    full = dict(dynamic_rows=True, zero_points=True, bias=True)
    assert lib.Kernel("int8_token_projection", M=3, **full, **shape).arg_names == ["A", "AS", "AZ", "Bias", "Out", "W", "WS", "WSum", "m"]
    assert lib.Kernel("int8_token_projection", M=3, input_dtype="bfloat16", **full, **shape).arg_names == ["A", "Bias", "Out", "W", "WS", "WSum", "m"]
    grouped = dict(rows=12, E=4, tiles=8, **shape)
    assert lib.Kernel("int8_token_grouped", **grouped).arg_names == ["A", "AS", "Out", "TileCount", "TileUnits", "W", "WS"]
    assert lib.Kernel("int8_token_grouped", gather=True, input_dtype="float16", **grouped).arg_names == ["A", "Out", "SlotToken", "TileCount", "TileUnits", "W", "WS"]
    assert lib.Kernel("half_grouped", **grouped).arg_names == ["A", "Out", "TileCount", "TileUnits", "W"]
    assert lib.Kernel("half_grouped", gather=True, dtype="bfloat16", **grouped).arg_names == ["A", "Out", "SlotToken", "TileCount", "TileUnits", "W"]


GROUPED = dict(rows=12, E=4, N=96, K=320, tiles=8)


@pytest.mark.parametrize("symbol,variant", [
    ("int8_token_quantization", dict(K=0)), ("int8_token_quantization", dict(K=64, input_dtype="int8")), ("int8_token_quantization", dict(K=64, M=0)), ("int8_token_quantization", dict(K=1 << 25)),
    ("int8_token_quantization", dict(K=64, zero_points=1)), ("int8_token_quantization", dict(K=64, pad=128)), ("int8_token_quantization", dict(K=64, layout="columns")),
    ("int8_token_projection", dict(M=17, N=96, K=320, input_dtype="float16")), ("int8_token_projection", dict(M=1, N=96, K=1 << 16, input_dtype="float16")),
    ("int8_token_projection", dict(M=16, N=96, K=8192, input_dtype="bfloat16")), ("int8_token_projection", dict(M=1, N=96, K=320, input_dtype="float32")),
    ("int8_token_projection", dict(M=0, N=96, K=320)), ("int8_token_projection", dict(M=1, N=0, K=320)), ("int8_token_projection", dict(M=1, N=96, K=65537)),
    ("int8_token_projection", dict(M=1, N=97, K=320, epilogue="swiglu")), ("int8_token_projection", dict(M=1, N=96, K=320, epilogue="gelu")),
    ("int8_token_projection", dict(M=1, N=96, K=320, output_dtype="int8")), ("int8_token_projection", dict(M=1, N=96, K=320, packed_k=128)), ("int8_token_projection", dict(M=1, N=96, K=320, bias=3)),
    ("int8_token_grouped", dict(GROUPED, block_m=24)), ("int8_token_grouped", dict(GROUPED, E=0)), ("int8_token_grouped", dict(GROUPED, tiles=0)), ("int8_token_grouped", dict(GROUPED, rows=0)),
    ("int8_token_grouped", dict(GROUPED, block_m=64, input_dtype="float16")), ("int8_token_grouped", dict(GROUPED, K=8192, input_dtype="float16")), ("int8_token_grouped", dict(GROUPED, zero_points=True)),
    ("half_grouped", dict(GROUPED, K=324)), ("half_grouped", dict(GROUPED, dtype="int8")), ("half_grouped", dict(GROUPED, dtype="float32")), ("half_grouped", dict(GROUPED, input_dtype="float16")),
])
def test_variants_that_are_not_served_are_refused(symbol, variant):
    with pytest.raises(lib.OrxError) as error:
        lib.Kernel(symbol, **variant)
    assert error.value.code == lib.ORX_ERR_BAD_VARIANT
    text = str(error.value)
    assert symbol in text or any(key in text for key in variant)


def test_rows_outside_the_capacity_and_bad_pointers_are_refused_before_anything_is_enqueued():
    linear = lib.Kernel("int8_token_projection", M=4, N=96, K=320, dynamic_rows=True, zero_points=True, bias=True)
    good = dict(A=4096, AS=4096, AZ=4096, Bias=4096, Out=4096, W=4096, WS=4096, WSum=4096, m=4)
    for change, code in ((dict(m=5), lib.ORX_ERR_ROWS), (dict(m=0), lib.ORX_ERR_ROWS), (dict(A=4104), lib.ORX_ERR_BAD_ARGUMENT), (dict(W=0), lib.ORX_ERR_BAD_ARGUMENT),
                         (dict(Out=4097), lib.ORX_ERR_BAD_ARGUMENT), (dict(WSum=4100), lib.ORX_ERR_BAD_ARGUMENT), (dict(AZ=0), lib.ORX_ERR_BAD_ARGUMENT), (dict(AS=4098), lib.ORX_ERR_BAD_ARGUMENT)):
        with pytest.raises(lib.OrxError) as error:
            linear(stream=0, **dict(good, **change))
        assert error.value.code == code
    halves = lib.Kernel("half_grouped", **GROUPED)
    for change in (dict(A=4104), dict(Out=4097), dict(TileUnits=4104), dict(TileCount=0)):
        with pytest.raises(lib.OrxError) as error:
            halves(stream=0, **dict(dict(A=4096, Out=4096, TileCount=4096, TileUnits=4096, W=4096), **change))
        assert error.value.code == lib.ORX_ERR_BAD_ARGUMENT
    quantise = lib.Kernel("int8_token_quantization", K=64)
    for change, code in ((dict(rows=0), lib.ORX_ERR_ROWS), (dict(X=4097), lib.ORX_ERR_BAD_ARGUMENT), (dict(Q=4100), lib.ORX_ERR_BAD_ARGUMENT),
                         (dict(S=0), lib.ORX_ERR_BAD_ARGUMENT), (dict(rows=1 << 25), lib.ORX_ERR_ROWS)):
        with pytest.raises(lib.OrxError) as error:
            quantise(stream=0, **dict(dict(Q=4096, S=4096, X=4096, rows=2), **change))
        assert error.value.code == code


def test_records_name_the_kernel_that_runs():
    for kernel in (lib.Kernel("int8_token_projection", M=9000, N=96, K=320, dynamic_rows=True), lib.Kernel("int8_token_grouped", **GROUPED), lib.Kernel("half_grouped", **GROUPED),
                   lib.Kernel("int8_token_quantization", K=64, M=300), lib.Kernel("int8_token_quantization", K=40000, M=9000)):
        for r in (1, 17, 64, 65, 200, 9000) if kernel.symbol == "int8_token_projection" else (0,):
            assert reported(kernel, r) in started(kernel, r)


@pytest.mark.parametrize("rows,n,k,kind", [
    (1, 130, 2560, "16 rows"), (16, 7168, 5120, "16 rows"), (500, 258, 4096, "64 rows"), (64, 5120, 17408, "64 rows"), (1, 66, 129, "64 x 64"), (128, 7168, 5120, "64 x 64"),
    (1024, 1058, 129, "64 x 128"), (32, 17408, 5120, "64 x 128"), (1024, 2050, 520, "96 x 128"), (333, 7168, 5120, "96 x 128"), (1500, 2050, 520, "128 x 128"), (500, 7168, 5120, "128 x 128"),
    (2048, 2050, 1111, "128 x 256"), (1024, 7168, 5120, "128 x 256"), (2048, 5000, 2560, "256 x 256"), (8192, 4096, 4096, "256 x 256"), (300, 65472, 65536, "128 x 256"),
    (500, 66000, 65536, "256 x 256")])
def test_which_kernel_the_rows_of_a_linear_start(rows, n, k, kind):
    """(as many rows as a test on the GPU has for each; a matrix of 4 GiB is not for the kernel that counts its bytes in 32 bits)"""
    lds = {(512, 16384): "16 rows", (256, 32768): "64 rows", (256, 71936): "64 x 64", (256, 161792): "64 x 128", (256, 158720): "96 x 128", (512, 143872): "128 x 128", (256, 77824): "128 x 256", (512, 146432): "256 x 256"}
    (_, threads, shared), = started(lib.Kernel("int8_token_projection", M=rows, N=n, K=k))
    assert lds.get((threads, shared), (threads, shared)) == kind


def linear_of(device, n=64, k=96, capacity=5, scale_device=None, **options):
    return programs.Int8Linear(torch.empty((n, k), dtype=torch.int8, device=device), torch.empty(n, device=scale_device or device), capacity, **options)


def int8_bank(device, *shape):
    return torch.empty(shape, dtype=torch.int8, device=device), torch.empty(shape[:-1], device=device)


def half_bank(device, *shape):
    return (torch.empty(shape, dtype=torch.bfloat16, device=device),)


LAYERS = [(programs.Int8MoeLayer, int8_bank), (programs.HalfMoeLayer, half_bank)]


def layer_of(make, bank, device, other=None, **options):
    return make(3, 4, 2, 96, 64, *bank(device, 4, 128, 96), *bank(other or device, 4, 96, 64), **options)


@pytest.mark.parametrize("device,stays", [("cuda:1", "cuda:1"), ("cuda:0", "cuda:0"), ("cpu", "cuda:0")])
def test_weights_stay_on_their_gpu(gpus, device, stays):  # noqa: F811
    held = [linear_of(device, zero_points=True, bias=torch.zeros(64, device=device))] + [layer_of(*kind, device, bias=[0.0] * 4) for kind in LAYERS]
    for one in held:
        assert str(one.device) == stays
        assert {str(t.device) for t in vars(one).values() if isinstance(t, torch.Tensor)} == {stays}
    assert {str(t.device) for t in held[0].channel.values()} == {stays}


def test_weights_of_several_gpus_are_refused(gpus):  # noqa: F811
    with pytest.raises(ValueError, match="several GPUs"):
        linear_of("cuda:0", scale_device="cuda:1")
    for kind in LAYERS:
        with pytest.raises(ValueError, match="several GPUs"):
            layer_of(*kind, "cuda:0", "cuda:1")
    assert str(linear_of("cuda:1", scale_device="cpu").device) == "cuda:1"  # what is on the host joins the other


def test_shapes_and_types_that_do_not_fit_are_refused(gpus):  # noqa: F811
    w, s = int8_bank("cuda:0", 64, 96)
    for arguments, options in (((w.float(), s, 5), {}), ((w[0], s, 5), {}), ((w, s[:63], 5), {}), ((w, s, 0), {}), ((w, s, (1 << 24) + 1), {}), ((w, s, 5), dict(dtype=torch.float32)),
                               ((w, s, 5), dict(bias=torch.empty(63, device="cuda:0"))), ((w[:63], s[:63], 5), dict(epilogue="swiglu"))):
        with pytest.raises(ValueError):
            programs.Int8Linear(*arguments, **options)
    with pytest.raises(lib.OrxError):
        programs.Int8Linear(*int8_bank("cuda:0", 16, 65537), 1)
    gate_up, down = int8_bank("cuda:0", 4, 128, 96), int8_bank("cuda:0", 4, 96, 64)
    for a, b, options in ((gate_up, (down[0][:3], down[1]), {}), ((gate_up[0][:, :126], gate_up[1]), down, {}), ((gate_up[0], gate_up[1][:, :5]), down, {}), (gate_up, (down[0].half(), down[1]), {}),
                          ((gate_up[0].half(), gate_up[1]), (down[0].half(), down[1]), {}), (gate_up, down, dict(dtype=torch.float32)), (gate_up, down, dict(bias=[0.0] * 3))):
        with pytest.raises(ValueError):
            programs.Int8MoeLayer(3, 4, 2, 96, 64, *a, *b, **options)
    for dtypes in ((torch.float32, torch.float32), (torch.float16, torch.bfloat16), (torch.int8, torch.int8)):
        with pytest.raises(ValueError):
            programs.HalfMoeLayer(3, 4, 2, 96, 64, gate_up[0].to(dtypes[0]), down[0].to(dtypes[1]))
    with pytest.raises(lib.OrxError) as error:  # rows of 100 values end within a 16-byte piece
        programs.HalfMoeLayer(3, 4, 2, 100, 64, *half_bank("cuda:0", 4, 128, 100), *half_bank("cuda:0", 4, 100, 64))
    assert error.value.code == lib.ORX_ERR_BAD_VARIANT and "multiple of 8" in str(error.value)
    for kind in LAYERS:
        for options in (dict(block_m=32), dict(scoring="relu"), dict(group_best=3)):
            with pytest.raises(lib.OrxError) as error:
                layer_of(*kind, "cuda:0", **options)
            assert error.value.code == lib.ORX_ERR_BAD_VARIANT
    with pytest.raises(ValueError):
        int8.quantize(torch.zeros((2, 3)))


@pytest.mark.parametrize("capacity,k", [(7_000_000, 5120), (1 << 24, 2080), (1 << 24, 1), (131_056, 65536)])
def test_a_linear_serves_its_capacity(gpus, capacity, k):  # noqa: F811
    """Every launch of as many rows as the object was made for is one that can be made."""
    linear = linear_of("cuda:0", 16, k, capacity)
    for kernel in (linear.quantizer, linear.projection):
        (groups, *_), (threads, *_), _ = kernel.geometry(capacity)
        assert 0 < groups * threads < 1 << 32


def test_rows_in_the_buffer_that_a_launch_writes_are_quantised_before_it():
    """Where every workgroup reads all rows, none may write over them."""
    buffer = torch.zeros(10 * 64, dtype=torch.float16)
    out = buffer[2 * 64:8 * 64].view(6, 64)
    for first, rows, apart in ((0, 2, True), (8, 2, True), (2, 1, False), (2, 4, False), (7, 1, False), (1, 2, False), (7, 3, False), (0, 4, False)):
        made = object.__new__(programs.Int8Linear)
        vars(made).update(few_rows=4, few="kernel", quantizer="kernel", projection="kernel", out=out, weight=None, channel={}, a_q=None, a_s=None, zero_points=False)
        x = buffer[first * 64:(first + rows) * 64].view(rows, 64)
        assert launches(made, "_run", x, rows) == (["few"] if apart else ["quantizer", "projection"]), (first, rows)
    for x, want in ((out, ["k_quantise_tokens", "k_up"]), (buffer[:128].view(2, 64), ["few_up"])):
        layer = object.__new__(programs.Int8MoeLayer)
        vars(layer).update(tokens=len(x), few_up="kernel", k_quantise_tokens="kernel", k_up="kernel", act=out, a_q=None, a_s=None, slot_token=None, tile_count=None, tile_units=None, w1=None, s1=None)
        assert launches(layer, "_up", x) == want
