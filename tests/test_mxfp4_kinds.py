"""MXFP4 without a GPU: codes of refusals, which kernel a projection's rows start, the oracle's groups by hand."""
import numpy as np
import pytest

from oracle import mxfp4 as orc
from orinfer_amd import lib
from tests import test_mxfp4
from tests.started_util import started

REFUSED = test_mxfp4.test_variants_that_are_not_served_are_refused.pytestmark[0].args[1]


@pytest.mark.parametrize("symbol,variant", REFUSED)
def test_a_refusal_has_its_code_and_says_what_it_is_about(symbol, variant):
    with pytest.raises(lib.OrxError) as error:
        lib.Kernel(symbol, **variant)
    assert error.value.code == lib.ORX_ERR_BAD_VARIANT
    text = str(error.value)
    assert symbol in text or any(key in text for key in variant)


# rows x channels of a tile and halves of K, of test_mxfp4.TILES in order
KINDS = [(64, 128, 1), (64, 128, 2), (128, 128, 1), (128, 128, 2), (128, 128, 2), (256, 256, 1), (64, 128, 2)]


@pytest.mark.parametrize("epilogue", ["none", "swiglu"])
def test_tiles_of_every_kind_are_told_apart(epilogue):
    """Tiles of 256 x 256 and of 128 x 128 in halves have as many threads and as much LDS; not as many workgroups."""
    cus, to_a_cu = 256, {64: 3, 128: 2, 256: 1}
    for ((rows, n, k), _, _), (tile_rows, channels, halves) in zip(test_mxfp4.TILES, KINDS, strict=True):
        def workgroups(tile_rows, channels, halves):
            sixteens = 2 * -(-n // 32) if epilogue == "swiglu" else -(-n // 16)
            tiles = -(-rows // tile_rows) * -(-sixteens // (channels // 16))
            return tiles if halves == 2 else min(tiles, cus * to_a_cu[tile_rows])

        (got, *_), = started(lib.Kernel("mxfp4_projection", M=rows, N=n, K=k, epilogue=epilogue), 0)
        assert got == workgroups(tile_rows, channels, halves), (rows, n, k)
        if halves == 2:
            assert got <= cus and k > 256  # a workgroup to a tile, a step at least to a half
        if (tile_rows, halves) in ((256, 1), (128, 2)):
            assert got != workgroups(*((128, 128, 2) if tile_rows == 256 else (256, 256, 1))), (rows, n, k)
    assert set(KINDS) == {(64, 128, 1), (64, 128, 2), (128, 128, 1), (128, 128, 2), (256, 256, 1)}
    steps = [-(-k // 256) % 2 for ((_, _, k), _, _), (_, _, halves) in zip(test_mxfp4.TILES, KINDS) if halves == 2]
    assert {0, 1} == set(steps)  # the middle step that both halves have, and none


def test_oracle_groups_by_hand():
    logits = np.log([[0.05, 0.35, 0.28, 0.32]])
    ids, weights = orc.routes(logits, 2, groups=2, top_groups=1)  # 0.40 against 0.60
    assert ids.tolist() == [[3, 2]] and np.allclose(weights, [[0.32 / 0.6, 0.28 / 0.6]])
    ids, _ = orc.routes(logits, 2, groups=2, top_groups=1, group_best=1)  # 0.35 against 0.32
    assert ids.tolist() == [[1, 0]]
    ids, weights = orc.routes(logits, 2, groups=2, top_groups=1, bias=[0.25, 0, 0, 0], renormalize=False)  # 0.65 against 0.60; weights without the bias
    assert ids.tolist() == [[1, 0]] and np.allclose(weights, [[0.35, 0.05]])
    ids, _ = orc.routes(logits, 3, groups=4, top_groups=3)
    assert ids.tolist() == [[1, 3, 2]]
