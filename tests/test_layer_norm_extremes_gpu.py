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
