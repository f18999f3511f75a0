"""Which launches int8 linears and layers of experts choose, by rules on sizes, without a GPU."""
import pytest
import torch

from orinfer_amd import programs
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
