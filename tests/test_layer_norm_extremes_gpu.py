"""Layer norm where its sums are long, its values large or its mean far from zero, against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import copy_gpu_to_numpy
from row_operations import (CHAIN, UNIT, decode, download, half_step_of_code, layer_norm, layer_norm_gradient_tolerances, layer_norm_gradients, rounding,
                            upload, within)
from thor_amd import physical as ph
from thor_amd.dtypes import DataType

pytestmark = pytest.mark.gpu
EPSILON = 1e-5


@pytest.fixture(scope="module")
def stream(gpu):
    return ph.Stream(0)


def gradients_of(plan, stream):
    return (download(plan.get_input_gradient_tensor(), stream), download(plan.get_weight_gradient_tensor(), stream),
            download(plan.get_bias_gradient_tensor(), stream))


@pytest.mark.parametrize("rows,cols,dtype", [(3, 5, DataType.fp32), (4, 130, DataType.bf16), (5, 700, DataType.fp32), (9, 4099, DataType.bf16), (3, 17001, DataType.fp32),
                                             (600, 5, DataType.bf16), (600, 130, DataType.fp32), (700, 700, DataType.bf16), (530, 9001, DataType.bf16)])
def test_gradients_of_constant_rows_far_from_zero(stream, rows, cols, dtype):
    """A row that is its mean has h = 0 however large it is: lanes that have no element of it add nothing to its sums, 0 - mean times rstd
    neither."""
    rng = np.random.default_rng([rows, cols])
    x = rng.standard_normal((rows, cols))
    x[1] = 2.0**122  # times rstd it is over fp32's range
    tx, x = upload(x, dtype, stream)
    tdy, dy = upload(0.05 * rng.standard_normal((rows, cols)), dtype, stream)
    tw, w = upload(1 + 0.2 * rng.standard_normal(cols), DataType.fp32, stream)
    tmean, mean = upload(x.mean(1, keepdims=True), DataType.fp32, stream)
    trstd, rstd = upload(1 / np.sqrt(x.var(1, keepdims=True) + EPSILON), DataType.fp32, stream)
    h = (x - mean) * rstd
    assert not h[1].any() and 2.0**122 * rstd[1, 0] > 2.0**128
    want = layer_norm_gradients(dy, h, rstd, w)
    off = layer_norm_gradient_tolerances(dy, h, 2 * UNIT * np.abs(h), rstd, w, dtype, DataType.fp32)
    plans = [ph.LayerNormBackward(asked, asked).stamp(tdy, tx, trstd, stream, mean=tmean, weight=tw) for asked in (True, False)]
    for plan in plans:
        plan.run()
    for got, value, o, what in zip(gradients_of(plans[0], stream), want, off, ("dx", "dweight", "dbias")):
        within(got, value, o, what)
    within(download(plans[1].get_input_gradient_tensor(), stream), want[0], off[0], "dx alone")


# every form of the forward pass: teams of 16 to 1024 lanes, rows with and without a tail, of whole chunks, whole blocks and full ones,
# of any length; rows in turn
MEANS = [(3, 7, DataType.fp32), (40, 128, DataType.bf16), (5, 200, DataType.fp32), (9, 512, DataType.fp16), (4, 1000, DataType.fp32), (3, 2048, DataType.bf16),
         (3, 2569, DataType.fp32), (5, 4096, DataType.fp32), (3, 6664, DataType.fp16), (2, 8192, DataType.fp32), (3, 11008, DataType.bf16), (2, 16384, DataType.fp32),
         (3, 16387, DataType.fp32), (2, 40000, DataType.fp32), (9000, 60, DataType.fp32), (2600, 1537, DataType.fp32)]


@pytest.mark.parametrize("rows,cols,dtype", MEANS, ids=[f"{r}x{c}-{d.name}" for r, c, d in MEANS])
def test_means_that_are_large_against_the_deviation(stream, rows, cols, dtype):
    """h and rstd have the precision of differences from the mean: CHAIN roundings of these, however large the mean is.  The differences are
    from the mean as its sum's CHAIN roundings leave it, which is where the tolerance's second part is from.  16-bit rows up to some
    length keep the mean as it is: their h moves by its roundings, and the variance by their square."""
    rng = np.random.default_rng([rows, cols, 1])
    x = rng.standard_normal((rows, cols)) + np.where(np.arange(rows) % 3 == 0, 1.0, np.where(np.arange(rows) % 3 == 1, -300.0, 6e4 / 8))[:, None]
    if dtype == DataType.fp32:
        x[-1] += 65536.0
    tx, x = upload(x, dtype, stream)
    tw, w = upload(1 + 0.2 * rng.standard_normal(cols), DataType.fp32, stream)
    tb, b = upload(0.1 * rng.standard_normal(cols), DataType.fp32, stream)
    plan = ph.LayerNorm(EPSILON, DataType.fp8_e4m3).stamp(tx, stream, weight=tw, bias=tb)
    plan.run()
    y, mean, rstd, h = layer_norm(x, w, b, EPSILON)
    from_near = CHAIN * UNIT * np.abs(x).mean(1, keepdims=True)  # how far the value that differences are taken from may be off the mean
    refined = dtype == DataType.fp32 or cols > (6144 if dtype == DataType.fp16 else 16384)
    mean_off = CHAIN * UNIT * (np.abs(x - mean).mean(1, keepdims=True) + from_near) if refined else from_near
    rstd_off = rstd * (CHAIN * UNIT * (1 + (from_near * rstd)**2) + (0.0 if refined else (from_near * rstd)**2))
    h_off = rstd * mean_off + np.abs(h) * (rstd_off / rstd + 4 * UNIT) + 2 * UNIT * rstd * from_near
    y_off = np.abs(w) * h_off + 4 * UNIT * (np.abs(h * w) + np.abs(b))
    within(download(plan.get_mean_tensor(), stream), mean, mean_off + rounding(mean, DataType.fp32), "mean")
    within(download(plan.get_reciprocal_deviation_tensor(), stream), rstd, rstd_off, "rstd")
    within(download(plan.get_output_tensor(), stream), y, y_off + rounding(np.abs(y) + y_off, dtype), "y")
    scales = copy_gpu_to_numpy(plan.get_checkpoint().scales, stream)
    kept = decode(copy_gpu_to_numpy(plan.get_checkpoint().codes, stream), scales, DataType.fp8_e4m3).astype(np.float64)
    within(kept, h, h_off + half_step_of_code(np.abs(h) + h_off, scales, DataType.fp8_e4m3), "restored")


@pytest.mark.parametrize("dtype,cols", [(DataType.fp16, 37), (DataType.fp16, 4096), (DataType.bf16, 6144), (DataType.fp16, 6143), (DataType.fp16, 8191), (DataType.bf16, 16384),
                                        (DataType.fp16, 12003), (DataType.fp32, 130), (DataType.fp32, 4099), (DataType.fp32, 16384), (DataType.fp16, 20001),
                                        (DataType.fp32, 50003)])
def test_constant_rows_are_zero_before_the_bias(stream, dtype, cols):
    """Exactly where the sums are exact, in bf16, and in fp16 up to 6144 columns.  Elsewhere a mean that is off by a last bit is refined: what is left
    of x - mean is CHAIN roundings of a difference that is CHAIN roundings of x, and rstd is at most 1 / sqrt(epsilon)."""
    values = np.array([2047.0, -1.0009765625, 37.28125, 0.333251953125, 60000.0 if dtype == DataType.fp16 else 123456.0])
    tx, x = upload(np.repeat(values[:, None], cols, 1), dtype, stream)
    plan = ph.LayerNorm(EPSILON).stamp(tx, stream)
    plan.run()
    y = download(plan.get_output_tensor(), stream)
    if dtype == DataType.bf16 or (dtype == DataType.fp16 and cols <= 6144):
        assert not y.any() and np.array_equal(download(plan.get_mean_tensor(), stream), x[:, :1])
    within(y, np.zeros_like(x), np.broadcast_to((CHAIN * UNIT)**2 * np.abs(x) / np.sqrt(EPSILON), x.shape), "y")


@pytest.mark.parametrize("cols", [100, 1000, 9001, 16387])
def test_the_mean_of_a_row_with_an_infinity(stream, cols):
    """It is that infinity, or no number where there are both; the row's results are no numbers."""
    x = np.random.default_rng(cols).standard_normal((4, cols)).astype(np.float32)
    x[1, cols // 2], x[2, cols - 1], x[3, 0], x[3, 5] = np.inf, -np.inf, np.inf, -np.inf
    tx, _ = upload(x, DataType.fp32, stream)
    plan = ph.LayerNorm(EPSILON).stamp(tx, stream)
    plan.run()
    mean = download(plan.get_mean_tensor(), stream)[:, 0]
    assert np.isfinite(mean[0]) and mean[1] == np.inf and mean[2] == -np.inf and np.isnan(mean[3])
    assert np.isnan(download(plan.get_output_tensor(), stream)[1:]).all()


@pytest.mark.parametrize("cols", [60, 1000, 9002, 16386, 40004])
def test_squares_that_overflow(stream, cols):
    """Differences of 2^100 have squares over fp32's range: rstd is zero and the output the bias, in rows of every length."""
    x = np.where(np.arange(cols) % 2 == 0, 1.0, -1.0)[None].repeat(3, 0).astype(np.float32)
    x[1] *= np.float32(2.0**100)
    tx, _ = upload(x, DataType.fp32, stream)
    tb, b = upload(np.random.default_rng(cols).standard_normal(cols), DataType.fp32, stream)
    plan = ph.LayerNorm(EPSILON).stamp(tx, stream, bias=tb)
    plan.run()
    mean, rstd = download(plan.get_mean_tensor(), stream)[:, 0], download(plan.get_reciprocal_deviation_tensor(), stream)[:, 0]
    assert not mean.any() and rstd[1] == 0 and np.isfinite(rstd).all()
    assert np.array_equal(download(plan.get_output_tensor(), stream)[1], b)


@pytest.mark.parametrize("rows,cols", [(1 << 23, 4), (1 << 19, 2052), (7 << 14, 16400)])
def test_parameter_gradients_over_many_rows(stream, rows, cols):
    """A sum over rows has CHAIN roundings at most, however many rows there are.  The rows are one value, of which an addition to a sum
    between 512 and 1024 loses 0.49 of a last bit every time: a chain of 1024 rows would be off by 240 roundings."""
    value = np.float32(1 + 0.49 * 2.0**-14)
    one, _ = upload(np.ones((1, cols)), DataType.fp32, stream)
    error, _ = upload(np.full((1, cols), value), DataType.fp32, stream)
    mean, _ = upload(np.zeros((rows, 1)), DataType.fp32, stream)
    rstd, _ = upload(np.ones((rows, 1)), DataType.fp32, stream)
    everywhere = lambda t: t.alias_view([rows, cols], [0, 1])  # noqa: E731
    plan = ph.LayerNormBackward().stamp(everywhere(error), everywhere(one), rstd, stream, mean=mean)
    plan.run()
    want = np.full(cols, rows * np.float64(value))
    for got in (plan.get_weight_gradient_tensor(), plan.get_bias_gradient_tensor()):
        within(download(got, stream), want, (CHAIN + 1) * UNIT * want, "sum over rows")
