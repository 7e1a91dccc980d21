"""The activations of checkpointed tensors in fp32 to a few units of its last bit, and 16-bit results down to their type's least number.

Tolerances count half steps of fp32 (UNIT, relative to the value).  The hardware's power of two and reciprocal are off by one step, two
UNIT, the sums and products of a formula by one UNIT each, and a result below the normal numbers by half the least number."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import copy_numpy_to_gpu, from_storage, to_storage
from row_operations import FORMATS, UNIT, decode, download, rounding, upload, value_and_slope, within
from thor_amd import physical as ph
from thor_amd.dtypes import DataType

pytestmark = pytest.mark.gpu
LEAST = 2.0**-149
SWISH, GELU = ph.ActivationKind.swish, ph.ActivationKind.gelu


@pytest.fixture(scope="module")
def stream(gpu):
    return ph.Stream(0)


def grid():
    """From beyond the deepest tail to beyond where both functions are x, dense where they bend; rows end inside a chunk."""
    x = np.concatenate([np.linspace(-112, 112, 40001), np.linspace(-15, 15, 60001), -np.logspace(-30, 2, 3000), [0.0, -0.0, -3e38, 3e38]])
    return np.pad(x, (0, -len(x) % 259)).astype(np.float32).reshape(-1, 259)


def forward(kind, x, dtype, stream, format=DataType.int8):
    tx, x64 = upload(x, dtype, stream)
    plan = ph.CheckpointedActivation(kind, format).stamp(tx, stream)
    plan.run()
    return download(plan.get_output_tensor(), stream), x64


def backward(kind, dtype, stream, format=DataType.int8):
    """(dx with and without the multiplier, dz, x) for an error and a multiplier of ones, at every finite code of scales from 2^-30 on: any for int8, powers of two for the
    others."""
    if format == DataType.int8:
        codes = np.concatenate([[-127], np.arange(-127, 128), [1, -1, 127]]).astype(np.int8)
        scales = np.concatenate([np.linspace(0.002, 0.9, 390), 2.0**-np.arange(3.0, 33.0, 3.0)])
        one = np.int8(1)
    else:
        codes = np.arange(256, dtype=np.uint8)
        codes = codes[np.isfinite(from_storage(codes, format))]
        scales = 2.0**np.arange(-30.0, -1.0 if format == DataType.fp8_e4m3 else -9.0)
        one = to_storage(np.ones(1, np.float32), format)[0]
    codes = codes[None].repeat(len(scales), 0)
    scales = scales.astype(np.float32)[:, None].repeat(-(-codes.shape[1] // 128), 1)
    kept = ph.ActivationCheckpoint(copy_numpy_to_gpu(codes, stream, format), copy_numpy_to_gpu(scales, stream, DataType.fp32))
    ones = ph.ActivationCheckpoint(copy_numpy_to_gpu(np.full_like(codes, one), stream, format), copy_numpy_to_gpu(np.ones_like(scales), stream, DataType.fp32))
    tdy, _ = upload(np.ones(codes.shape), dtype, stream)
    plan = ph.CheckpointedActivationBackward(kind).stamp(tdy, kept, stream, multiplier_checkpoint=ones)
    plan.run()
    alone = ph.CheckpointedActivationBackward(kind).stamp(tdy, kept, stream)
    alone.run()
    return (np.stack([download(p.get_input_gradient_tensor(), stream) for p in (plan, alone)]), download(plan.get_multiplier_gradient_tensor(), stream),
            decode(codes, scales, format).astype(np.float64))


def terms(kind, x):
    """The two terms of the slope, each as a magnitude: s and |x s (1 - s)|, or Phi and |x| phi."""
    if kind == SWISH:
        s, rest = np.exp(-np.logaddexp(0, -x)), np.exp(-np.logaddexp(0, x))
        return s + np.abs(x) * s * rest
    f, slope, _, _ = value_and_slope(kind, x)
    phi = np.where(x == 0, 0.5, f / np.where(x == 0, 1.0, x))
    return phi + np.abs(slope - phi)


def test_swish_in_fp32(stream):
    """x s: the power 2, its argument's last rounding 0.2, e r 1, 1 + e 1, the reciprocal 2, the product with x 1: 7.2 UNIT, taken as 8.
    The slope s + x s (1 - s): 6.2 of s, and 13.4 and a rounding of the other term: 16 of both."""
    got, x = forward(SWISH, grid(), DataType.fp32, stream)
    f = value_and_slope(SWISH, x)[0]
    within(got, f, 8 * UNIT * np.abs(f) + LEAST, "f")
    dx, dz, x = backward(SWISH, DataType.fp32, stream)
    f, slope, _, _ = value_and_slope(SWISH, x)
    within(dx, np.stack([slope, slope]), 16 * UNIT * terms(SWISH, x) + LEAST, "slope")
    within(dz, f, 8 * UNIT * np.abs(f) + LEAST, "f backward")


@pytest.mark.parametrize("kind", [SWISH, GELU], ids=lambda k: k.name)
@pytest.mark.parametrize("dtype", [DataType.bf16, DataType.fp16], ids=lambda d: d.name)
def test_results_of_16_bits_down_to_the_least(stream, dtype, kind):
    """One rounding to the type, and before it what fp32 exponents of up to 190 lose: half of 2^-16 times ln 2 for the exponent's own
    rounding, twice for gelu's square, 1.1e-5, and the units of the formula: 2e-5 in all."""
    got, x = forward(kind, np.clip(grid(), -60000, 60000), dtype, stream)
    f = value_and_slope(kind, x)[0]
    off = 2e-5 * np.abs(f)
    within(got, f, off + rounding(np.abs(f) + off, dtype), "f")
    dx, dz, x = backward(kind, dtype, stream)
    f, slope, _, _ = value_and_slope(kind, x)
    off = 2e-5 * terms(kind, x)
    within(dx, np.stack([slope, slope]), off + rounding(np.abs(slope) + off, dtype), "slope")
    off = 2e-5 * np.abs(f)
    within(dz, f, off + rounding(np.abs(f) + off, dtype), "f backward")


@pytest.mark.parametrize("format", FORMATS, ids=lambda f: f.name)
def test_gelu_in_fp32(stream, format):
    """x Phi(x): 2.2 the power, 1.3 the reciprocal that the tail's factor follows 2.7 times, 2.6 its polynomial and 1 its last product,
    two more products: 9.1 UNIT, taken as 10.  Above zero that is what is taken from x.  The slope's two terms have one more product, and
    above zero the difference from one a rounding: 12 of both."""
    got, x = forward(GELU, grid(), DataType.fp32, stream, format)
    f = value_and_slope(GELU, x)[0]
    within(got, f, 10 * UNIT * np.abs(f) + LEAST, "f")
    dx, dz, x = backward(GELU, DataType.fp32, stream, format)
    f, slope, _, _ = value_and_slope(GELU, x)
    within(dx, np.stack([slope, slope]), 12 * UNIT * terms(GELU, x) + LEAST, "slope")
    within(dz, f, 10 * UNIT * np.abs(f) + LEAST, "f backward")


@pytest.mark.parametrize("kind", list(ph.ActivationKind), ids=lambda k: k.name)
@pytest.mark.parametrize("dtype", [DataType.fp32, DataType.bf16], ids=lambda d: d.name)
@pytest.mark.parametrize("format", FORMATS, ids=lambda f: f.name)
def test_errors_times_multipliers_that_overflow(stream, format, dtype, kind):
    """Where the slope is zero the gradient is, though error times multiplier is over fp32's range; where it is one, the gradient is too."""
    cols = 261  # chunks and a tail
    x = np.where(np.arange(cols) % 2 == 0, -200.0, 200.0)[None].repeat(2, 0)
    save, gate = (ph.CheckpointSave(format).stamp(upload(v, DataType.fp32, stream)[0], stream) for v in (x, np.full((2, cols), 2.0**70)))
    tdy, dy = upload(np.array([[2.0**70], [2.0**-70]]).repeat(cols, 1), dtype, stream)
    plan = ph.CheckpointedActivationBackward(kind).stamp(tdy, save.get_checkpoint(), stream, multiplier_checkpoint=gate.get_checkpoint())
    for p in (save, gate, plan):
        p.run()
    got = download(plan.get_input_gradient_tensor(), stream)
    assert not got[:, ::2].any() and (got[0, 1::2] == np.inf).all() and np.abs(got[1, 1::2] - 1.0).max() <= rounding(1.0, dtype) + 6 * UNIT


@pytest.mark.parametrize("kind", [SWISH, GELU], ids=lambda k: k.name)
def test_values_of_16_bits_near_ties(stream, kind):
    """fp16 results below 2^-14 are multiples of 2^-24, and a value near a tie between two shows what it was before its rounding: within
    the units that value_and_slope() counts, over twenty million products of an fp16 input and a multiplier that brings it there."""
    x = np.arange(1 << 16, dtype=np.uint16).view(np.float16).astype(np.float32)
    x = x[np.isfinite(x) & (np.abs(x) <= 2) & (np.abs(x) >= 2.0**-5)][None]
    rows, cols = 1500, x.shape[1]
    tx, x64 = upload(x, DataType.fp16, stream)
    least = np.abs(value_and_slope(kind, x64)[0])
    tz, z = upload(2.0**np.random.default_rng(0).uniform(-17, -14, (rows, cols)) / least, DataType.fp16, stream)
    plan = ph.CheckpointedActivation(kind, DataType.int8).stamp(tx.alias_view([rows, cols], [0, 1]), stream, multiplier=tz)
    plan.run()
    f, _, f_off, _ = value_and_slope(kind, x64)
    off = z * f_off + 2 * UNIT * np.abs(f * z)
    within(download(plan.get_output_tensor(), stream), f * z, off + rounding(np.abs(f * z) + off, DataType.fp16), "f z")
