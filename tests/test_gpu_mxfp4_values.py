"""Every value: codes and powers of all bf16 and fp32 magnitudes, what every code stands for under every power, in every type."""
import numpy as np
import pytest
import torch

from oracle import mxfp4 as orc
from orinfer_amd import mxfp4
from tests.gpu_util import host

pytestmark = pytest.mark.gpu
DEV = "cuda"


def bf16_as_fp32(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


@pytest.mark.parametrize("scale", ["floor", "ceil"])
@pytest.mark.parametrize("company", [None, 1.0, 2.0**-126, 2.0**-133, 3.0e38])
def test_every_bf16_value_by_itself_and_in_company(company, scale):
    """Subnormal, largest, infinite and NaN values among them; beside them a value that sets the power or does not."""
    x = np.zeros((65536, 32), np.float32)
    x[:, 5] = bf16_as_fp32(np.arange(65536, dtype=np.uint32))
    if company is not None:
        x[:, 9] = company
    device = torch.from_numpy(x).to(torch.bfloat16)
    assert torch.equal(device[:, 5].view(torch.int16) & 0x7F80, torch.from_numpy(np.arange(65536, dtype=np.uint16).view(np.int16)) & 0x7F80)  # (a NaN's other bits may change)
    with np.errstate(invalid="ignore"):
        codes, exponents = orc.quantise(device.double().numpy(), ceil=scale == "ceil")
    got = mxfp4.quantize(device.to(DEV), scale=scale)
    np.testing.assert_array_equal(host(got[1]), exponents)
    np.testing.assert_array_equal(host(got[0]), codes)


@pytest.mark.parametrize("scale", ["floor", "ceil"])
def test_fp32_values_of_every_exponent(scale):
    """Magnitudes of every exponent, subnormal ones among them, beside values of other exponents, and both neighbours of every border of the codes."""
    rng = np.random.default_rng(32)
    bits = rng.integers(0, 2**32, (8192, 64), dtype=np.uint32)
    at = np.arange(8192) % 256  # a row's exponents lie within 40 of one another, some rows are subnormal as a whole
    exponent = np.clip(at[:, None] - rng.integers(0, 40, bits.shape), 0, 254).astype(np.uint32)
    bits = (bits & 0x807FFFFF) | (exponent << 23)
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0], np.float32)
    beside = np.concatenate([borders, np.nextafter(borders, np.float32(0)), np.nextafter(borders, np.float32(9))])
    with np.errstate(over="ignore"):
        bits[::2, 1:1 + len(beside)] = (np.ldexp(beside[None], np.minimum(at[::2, None] - 131, 124))).astype(np.float32).view(np.uint32)
        bits[::2, 0] = np.ldexp(np.float32(4), np.minimum(at[::2] - 131, 124)).astype(np.float32).view(np.uint32)
    x = bits.view(np.float32)
    codes, exponents = orc.quantise(x.astype(np.float64), ceil=scale == "ceil")
    got = mxfp4.quantize(torch.from_numpy(x).to(DEV), scale=scale)
    np.testing.assert_array_equal(host(got[1]), exponents)
    np.testing.assert_array_equal(host(got[0]), codes)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_every_code_under_every_power(dtype):
    """Equal to the 64-bit value rounded once: infinite above the type's range, subnormal below it, NaN under byte 255."""
    codes = np.tile(np.arange(0, 256, 17, dtype=np.uint8), (256, 1))  # sixteen codes, each twice: a block
    exponents = np.arange(256, dtype=np.uint8)[:, None]
    want = torch.from_numpy(orc.values(codes, exponents)).to(dtype)
    got = mxfp4.dequantize(torch.from_numpy(codes).to(DEV), torch.from_numpy(exponents).to(DEV), 32, dtype).cpu()
    nan = torch.isnan(want)
    assert torch.equal(nan, torch.isnan(got)) and nan[255].all() and not nan[:255].any()
    as_bits = torch.int32 if dtype == torch.float32 else torch.int16
    assert torch.equal(got[~nan].view(as_bits), want[~nan].view(as_bits))
