"""The kernels of products by byte tiles built here: what touches a sum waits for it."""
from tests import test_codegen
from tests.test_codegen import built  # noqa: F401  (fixture)


def test_sums_of_multiplies_are_awaited(built, monkeypatch):  # noqa: F811
    """The multiplies of the kernel whose weights go straight to registers are statements that the compiler does not look into.  It keeps 8 wait states itself between a multiply of 16 x 16
    and another access to its sum, of 64 8-bit integers and of 32 16-bit values alike."""
    monkeypatch.setattr(test_codegen, "RESULT_WAIT", 8)
    for family, count in (("byte_wide_kernel", 28), ("byte_tiles_kernel", 16), ("byte_rows_kernel", 40)):
        chosen = {name: code for name, code in built.items() if family in name}
        assert len(chosen) >= count, (family, len(chosen))
        for name, (code, targets) in chosen.items():
            assert not (problems := test_codegen.faults(code, targets)), (name, sorted(problems)[:5])


def test_sums_stay_where_they_are_between_multiplies(built):  # noqa: F811
    """(a copy of a sum would be taken in front of the multiply's end, or cost as many registers again)"""
    for name, (code, _) in built.items():
        if "byte_wide_kernel" not in name:
            continue
        for _, ins in code:
            assert not ins.name.startswith(("v_accvgpr", "v_swap")), (name, ins.text)
            if ins.multiply:
                operands = ins.text.partition(" ")[2].split(", ")
                assert operands[0] == operands[3], (name, ins.text)


def test_nothing_is_reloaded_while_the_next_weights_are_on_their_way(built):  # noqa: F811
    """A reload from scratch waits for every load in front of it: from the first multiply on the kernel of few rows has the next weights under way."""
    for name, (code, _) in built.items():
        if "byte_rows_kernel" not in name:
            continue
        first = next(i for i, (_, ins) in enumerate(code) if ins.multiply)
        late = [ins.text for _, ins in code[first:] if ins.name.startswith("scratch_")]
        assert not late, (name, late[:5])
