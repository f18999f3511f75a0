"""The MXFP4 kernels built here: what touches a sum waits for it."""
from tests import test_codegen
from tests.test_codegen import built  # noqa: F401  (fixture)


def test_sums_of_scaled_multiplies_are_awaited(built, monkeypatch):  # noqa: F811
    """The compiler itself keeps 12 wait states between v_mfma_scale_f32_32x32x64 of 4-bit codes and another access to its sum, 8 behind the 16 x 16 x 128 form; where two ways
    lead from a multiply to the use it has been seen to count the longer one only."""
    for family, count, states in (("mx_tiles_kernel", 32, 12), ("mx_rows_kernel", 14, 8)):
        monkeypatch.setattr(test_codegen, "RESULT_WAIT", states)
        chosen = {name: code for name, code in built.items() if family in name}
        assert len(chosen) >= count
        for name, (code, targets) in chosen.items():
            assert not (problems := test_codegen.faults(code, targets)), (name, sorted(problems)[:5])
