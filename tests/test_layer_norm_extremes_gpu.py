"""Layer norm where its sums are long, its values large or its mean far from zero, against the definition in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from helpers import copy_gpu_to_numpy
from row_operations import UNIT, download, layer_norm_gradient_tolerances, layer_norm_gradients, upload, within
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
