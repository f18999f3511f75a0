"""What the MXFP4 layers ask for, without a GPU."""
import pytest

from orinfer_amd import lib

COMBINE = dict(M=4, H=256, top_k=2)


def test_weighted_sums_take_fp16_or_fp32_rows():
    plain = lib.Kernel("moe_combine", **COMBINE)
    wide = lib.Kernel("moe_combine", **COMBINE, expert_dtype="float32")
    assert wide.arg_names == plain.arg_names and wide.geometry() == plain.geometry()
    with pytest.raises(lib.OrxError) as error:
        lib.Kernel("moe_combine", **COMBINE, expert_dtype="bfloat16")
    assert error.value.code == lib.ORX_ERR_BAD_VARIANT and "expert_dtype" in str(error.value)
    named = dict(Expert=4096, Output=4096, Prob=4096, Shared=0, SharedGate=0, SlotMap=4096)
    for kernel, address in ((plain, 4097), (wide, 4098)):  # rows are aligned as their type
        with pytest.raises(lib.OrxError) as error:
            kernel(stream=0, **dict(named, Expert=address))
        assert error.value.code == lib.ORX_ERR_BAD_ARGUMENT
