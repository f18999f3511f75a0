"""What the MXFP4 layers ask for, without a GPU."""
import contextlib

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from orinfer_amd import lib, programs

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


@pytest.fixture
def gpus(monkeypatch):
    """Tensors of shapes alone on GPUs that are not there; GPU 0 is current."""
    monkeypatch.setattr(torch.cuda, "device", lambda _: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(lib.Kernel, "workspace", lambda self: None)
    with FakeTensorMode():
        yield


def weights(device, *shape):
    n, k = shape[-2:]
    return [torch.empty((*shape[:-1], k // piece), dtype=torch.uint8, device=device) for piece in (2, 32)]


@pytest.mark.parametrize("device,stays", [("cuda:1", "cuda:1"), ("cuda:0", "cuda:0"), ("cpu", "cuda:0")])
def test_weights_stay_on_their_gpu(gpus, device, stays):
    linear = programs.Mxfp4Linear(*weights(device, 64, 96), 5)
    layer = programs.Mxfp4MoeLayer(3, 4, 2, 96, 64, *weights(device, 4, 128, 96), *weights(device, 4, 96, 64), bias=[0.0] * 4)
    for held in (linear, layer):
        assert str(held.device) == stays
        assert {str(t.device) for t in vars(held).values() if isinstance(t, torch.Tensor)} == {stays}


def test_weights_of_several_gpus_are_refused(gpus):
    here, there = weights("cuda:0", 64, 96), weights("cuda:1", 64, 96)
    with pytest.raises(ValueError, match="several GPUs"):
        programs.Mxfp4Linear(here[0], there[1], 5)
    with pytest.raises(ValueError, match="several GPUs"):
        programs.Mxfp4MoeLayer(3, 4, 2, 96, 64, *weights("cuda:0", 4, 128, 96), *weights("cuda:1", 4, 96, 64))
    assert str(programs.Mxfp4Linear(there[0], weights("cpu", 64, 96)[1], 5).device) == "cuda:1"  # what is on the host joins the other


@pytest.mark.parametrize("capacity,k", [(7_000_000, 5120), (1 << 24, 2080), (1 << 24, 32), (131_056, 1 << 20)])
def test_a_linear_serves_its_capacity(gpus, capacity, k):
    """Every launch of as many rows as the object was made for is one that can be made."""
    linear = programs.Mxfp4Linear(*weights("cuda:0", 16, k), capacity)
    for kernel in (linear.quantizer, linear.projection):
        (groups, *_), (threads, *_), _ = kernel.geometry(capacity)
        assert 0 < groups * threads < 1 << 32
    assert linear.quantizer.geometry(capacity)[0][0] * 512 >= -(-capacity // 16) * k  # a workgroup takes 16 rows x 512 of K at most


def test_rows_that_no_launch_takes_are_refused_where_the_object_is_made(gpus):
    for make in (lambda: programs.Mxfp4Linear(*weights("cuda:0", 16, 1 << 20), 131_057),
                 lambda: programs.Mxfp4MoeLayer(5_000_000, 2, 1, 8192, 32, *weights("cuda:0", 2, 64, 8192), *weights("cuda:0", 2, 8192, 32))):
        with pytest.raises(lib.OrxError) as error:
            make()
        assert error.value.code == lib.ORX_ERR_BAD_VARIANT and "M must be" in str(error.value)


def launches(made, method, *args):
    """Which of an object's kernels a call launches, in order."""
    seen = []
    for name in [name for name, value in vars(made).items() if value == "kernel"]:
        setattr(made, name, lambda name=name, **_: seen.append(name))
    getattr(made, method)(*args, 0)
    return seen


def test_rows_in_the_buffer_that_a_launch_writes_are_quantised_before_it():
    """Where every workgroup reads all rows, none may write over them."""
    def linear(x, rows):
        made = object.__new__(programs.Mxfp4Linear)
        vars(made).update(few_rows=4, few="kernel", quantizer="kernel", projection="kernel", out=out, weight=None, powers=None, a_q=None, a_s=None)
        return launches(made, "_run", x, rows)

    buffer = torch.zeros(10 * 64, dtype=torch.float16)
    out = buffer[2 * 64:8 * 64].view(6, 64)
    for first, rows, apart in ((0, 2, True), (8, 2, True), (2, 1, False), (2, 4, False), (7, 1, False), (1, 2, False), (7, 3, False), (0, 4, False)):
        x = buffer[first * 64:(first + rows) * 64].view(rows, 64)
        assert linear(x, rows) == (["few"] if apart else ["quantizer", "projection"]), (first, rows)
    assert linear(torch.zeros(5, 64).half(), 5) == ["quantizer", "projection"]

    for x, want in ((out, ["k_quantise_tokens", "k_up"]), (buffer[:128].view(2, 64), ["few_up"])):
        layer = object.__new__(programs.Mxfp4MoeLayer)
        vars(layer).update(tokens=len(x), few_up="kernel", k_quantise_tokens="kernel", k_up="kernel", act=out, a_q=None, a_s=None, slot_token=None, tile_count=None, tile_units=None, w1=None, p1=None)
        assert launches(layer, "_up", x) == want


def test_layers_are_of_fp16_or_bf16(gpus):
    arguments = [3, 4, 2, 96, 64, *weights("cuda:0", 4, 128, 96), *weights("cuda:0", 4, 96, 64)]
    for dtype in (torch.float16, torch.bfloat16):
        layer = programs.Mxfp4MoeLayer(*arguments, dtype=dtype)
        assert layer.act.dtype == layer.out.dtype == dtype and layer.down_out.dtype == torch.float32
    with pytest.raises(ValueError):
        programs.Mxfp4MoeLayer(*arguments, dtype=torch.float32)


def test_weighted_sums_are_fp16_or_bf16():
    plain, brain = (lib.Kernel("moe_combine", **COMBINE, expert_dtype="float32", output_dtype=name) for name in ("float16", "bfloat16"))
    assert brain.arg_names == plain.arg_names and brain.geometry() == plain.geometry()
    for bad in (dict(output_dtype="bfloat16"), dict(output_dtype="float32"), dict(expert_dtype="float32", output_dtype="float32")):
        with pytest.raises(lib.OrxError) as error:
            lib.Kernel("moe_combine", **COMBINE, **bad)
        assert error.value.code == lib.ORX_ERR_BAD_VARIANT and "output_dtype" in str(error.value)


@pytest.mark.parametrize("options", [dict(group_best=3), dict(group_best=0), dict(groups=2, group_best=3), dict(top_groups=2), dict(scoring="relu"), dict(scale=0.0), dict(block_m=32)])
def test_layers_refuse_routing_that_is_not_served(gpus, options):
    with pytest.raises(lib.OrxError) as error:
        programs.Mxfp4MoeLayer(3, 4, 2, 96, 64, *weights("cuda:0", 4, 128, 96), *weights("cuda:0", 4, 96, 64), **options)
    assert error.value.code == lib.ORX_ERR_BAD_VARIANT


def test_experts_have_no_rows_before_they_have_places(gpus):
    """Lists that no launch has written would send the products anywhere."""
    layer = programs.Mxfp4MoeLayer(3, 4, 2, 96, 64, *weights("cuda:0", 4, 128, 96), *weights("cuda:0", 4, 96, 64))
    x = torch.empty((3, 96), dtype=torch.float16, device="cuda:0")
    for call in (lambda: layer.up(x), lambda: layer.down(layer.act, layer.prob)):
        with pytest.raises(RuntimeError, match="place"):
            call()
