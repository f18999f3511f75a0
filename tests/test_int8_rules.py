"""Which launches int8 linears and layers of experts choose, by rules on sizes, without a GPU."""
import pytest
import torch

from orinfer_amd import lib, programs
from tests.test_int8 import LAYERS
from tests.test_mxfp4_layer import gpus  # noqa: F401  (fixture)


def few_rows(n, k, capacity=64, **options):
    linear = programs.Int8Linear(torch.empty((n, k), dtype=torch.int8, device="cuda:0"), torch.empty(n, device="cuda:0"), capacity, **options)
    assert linear.few is not None
    return linear.few_rows


@pytest.mark.parametrize("k,plain,zeros,gated", [(1000, 8, 8, 8), (2560, 8, 8, 8), (2561, 8, 4, 4), (4096, 8, 4, 4), (4097, 4, 4, 2), (5120, 4, 4, 2), (8192, 4, 4, 2), (8193, 2, 2, 2), (17408, 1, 1, 1)])
def test_rows_that_one_launch_quantises_and_multiplies(gpus, k, plain, zeros, gated):  # noqa: F811
    """(more of them are faster in two launches, or do not fit)"""
    assert few_rows(64, k) == plain and few_rows(64, k, zero_points=True) == zeros
    assert few_rows(64, k, epilogue="swiglu") == few_rows(64, k, epilogue="swiglu", zero_points=True) == gated


@pytest.mark.parametrize("k,rows", [(512, [1, 2, 3, 4, 5, 6, 7, 8]), (4097, [1, 2, 3, 4, 4, 4, 4, 4])])
def test_a_linear_made_for_few_rows_takes_all_of_them_in_one_launch(gpus, k, rows):  # noqa: F811
    assert [few_rows(64, k, capacity) for capacity in range(1, 9)] == rows


@pytest.mark.parametrize("experts,hidden,inner,first,second", [
    (128, 2048, 512, 8, 48), (128, 3264, 224, 8, 48), (60, 1024, 768, 10, 68), (16, 4096, 1536, 13, 91), (32, 4096, 512, 9, 64), (8, 1024, 1024, 64, 426), (8, 256, 128, 384, 2560)])
def test_rows_to_a_unit(experts, hidden, inner, first, second):
    """The fewer tiles both products have, the more routes to an expert are faster in short units."""
    def unit(routes):
        return programs._unit_rows(routes, experts, hidden, inner, 1 << 20)

    assert [unit(bound * experts + more) for bound in (first, second) for more in (-1, 0)] == [16, 64, 64, 128]


@pytest.mark.parametrize("kind", LAYERS)
def test_a_layer_takes_the_rule_for_its_own_bank(gpus, kind):  # noqa: F811
    make, bank = kind

    def unit(routes, **options):
        return make(routes, 8, 1, 1024, 128, *bank("cuda:0", 8, 256, 1024), *bank("cuda:0", 8, 1024, 128), **options).block_m

    assert [unit(8 * bound + more) for bound in (153, 1024) for more in (-1, 0)] == [16, 64, 64, 128]  # (80 tiles)
    assert unit(8, block_m=64) == 64


def test_matrices_of_4_gib_go_in_units_of_16():
    assert [programs._unit_rows(100000, 16, 4096, 1536, size) for size in ((1 << 32) - 1, 1 << 32)] == [128, 16]


@pytest.mark.parametrize("rows,most", [(1, 32768), (2, 16384), (3, 8192), (4, 8192), (5, 4096), (8, 4096), (16, 4096), (17, 0)])
@pytest.mark.parametrize("epilogue", ["none", "swiglu"])
def test_the_longest_rows_that_a_projection_quantises(rows, most, epilogue):
    for k in (most, most + 1):
        shape = dict(M=rows, N=64, K=k or 1, input_dtype="bfloat16", epilogue=epilogue, zero_points=True)
        if k == most and most:
            assert lib.Kernel("int8_token_projection", **shape).arg_names == ["A", "Out", "W", "WS", "WSum"]
        else:
            with pytest.raises(lib.OrxError) as error:
                lib.Kernel("int8_token_projection", **shape)
            assert error.value.code == lib.ORX_ERR_BAD_VARIANT
    grouped = dict(rows=12, E=4, N=64, tiles=8, input_dtype="float16", epilogue=epilogue)
    assert lib.Kernel("int8_token_grouped", K=4096, **grouped).arg_names[0] == "A"
    with pytest.raises(lib.OrxError):
        lib.Kernel("int8_token_grouped", K=4097, **grouped)


@pytest.mark.parametrize("kind", LAYERS)
def test_a_layer_without_experts_is_refused(gpus, kind):  # noqa: F811
    make, bank = kind
    with pytest.raises(ValueError, match="expert"):
        make(3, 0, 2, 96, 64, *bank("cuda:0", 0, 128, 96), *bank("cuda:0", 0, 96, 64))
