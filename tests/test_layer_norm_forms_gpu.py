"""Layer norm's kernels for many rows: every team, with tails, whole chunks and full rows, from the input and from codes, with fewer rows in
use than there are, more than one share of the parameter gradients per block, and results that hold something else before every run."""
from __future__ import annotations

import numpy as np
import pytest

import test_layer_norm_gpu as base
from helpers import copy_gpu_to_numpy, from_storage
from row_operations import (CHAIN, UNIT, decode, download, layer_norm, layer_norm_gradient_tolerances, layer_norm_gradients, layer_norm_tolerances, offsets_tensor,
                            upload, within)
from thor_amd import physical as ph
from thor_amd.dtypes import DataType

pytestmark = pytest.mark.gpu
EPSILON = 1e-5
E4M3, E5M2, INT8 = DataType.fp8_e4m3, DataType.fp8_e5m2, DataType.int8


@pytest.fixture(scope="module")
def stream(gpu):
    return ph.Stream(0)


# fp32 from codes: teams of 32 to 1024 lanes with a tail and of whole chunks, full ones of six and twelve wavefronts, rows of any length
# with several shares and with one that is the result; 16 bits: 1024 lanes with a tail and full, and teams that only fp32 had
STEPS = [(2000, 40, DataType.fp32, INT8), (900, 131, DataType.fp32, E4M3), (700, 1001, DataType.fp32, E4M3), (700, 1004, DataType.fp32, E5M2), (600, 2051, DataType.fp32, INT8),
         (600, 2564, DataType.fp32, E5M2), (600, 5121, DataType.fp32, INT8), (600, 5124, DataType.fp32, E4M3), (520, 6144, DataType.fp32, E4M3),
         (520, 9001, DataType.fp32, E4M3), (520, 9004, DataType.fp32, INT8), (515, 12001, DataType.fp32, E4M3), (515, 12288, DataType.fp32, E5M2),
         (513, 16380, DataType.fp32, E5M2), (513, 16383, DataType.fp32, E4M3), (513, 16384, DataType.fp32, INT8), (513, 16387, DataType.fp32, E4M3),
         (520, 17000, DataType.fp32, INT8), (514, 70001, DataType.fp32, E4M3), (520, 14337, DataType.bf16, E4M3), (520, 16383, DataType.fp16, INT8),
         (513, 16384, DataType.bf16, E5M2), (700, 1001, DataType.bf16, INT8), (520, 20001, DataType.bf16, E4M3)]


@pytest.mark.parametrize("rows,cols,dtype,format", STEPS, ids=[f"{r}x{c}-{d.name}-{f.name}" for r, c, d, f in STEPS])
def test_steps_through_a_checkpoint(stream, rows, cols, dtype, format):
    base.test_step_through_a_checkpoint(stream, rows, cols, dtype, format)


@pytest.mark.parametrize("rows,cols,dtype", [(520, 16383, DataType.fp32), (513, 16384, DataType.fp32), (520, 14337, DataType.bf16), (514, 70001, DataType.fp32),
                                             (900, 131, DataType.fp16), (600, 2564, DataType.fp32)], ids=str)
def test_backward_from_the_input(stream, rows, cols, dtype):
    base.test_backward_from_the_input(stream, rows, cols, dtype)


# a length of each kind of team, and how many of the rows are in use: none, one, fewer than the blocks take at once, all but one
USED = [(rows, cols, dtype, used) for rows, cols, dtype in ((5000, 60, DataType.bf16), (5000, 61, DataType.fp32), (1500, 700, DataType.fp16), (1100, 2501, DataType.bf16),
                                                          (700, 5124, DataType.fp32), (600, 9001, DataType.fp32), (600, 16384, DataType.bf16), (520, 17001, DataType.bf16))
        for used in (0, 1, 100, rows - 1)]


@pytest.mark.parametrize("rows,cols,dtype,used", USED, ids=[f"{r}x{c}-{d.name}-{u}" for r, c, d, u in USED])
def test_many_rows_of_which_fewer_are_in_use(stream, rows, cols, dtype, used):
    """The rows behind hold NaN.  The plans run with all rows in use first, so that the workspace and the gradients hold NaN too; then the
    offsets change."""
    x, dy, w, _ = base.data(rows, cols, 20)
    x[used:], dy[used:] = np.nan, np.nan
    tx, x = upload(x, dtype, stream)
    tdy, dy = upload(dy, dtype, stream)
    tw, w = upload(w, DataType.fp32, stream)
    offsets = offsets_tensor([0, rows // 2, rows], stream)
    forward = ph.LayerNorm(EPSILON, INT8).stamp(tx, stream, weight=tw, segment_offsets=offsets)
    rstd_tensor = forward.get_reciprocal_deviation_tensor()
    from_input = ph.LayerNormBackward().stamp(tdy, tx, rstd_tensor, stream, mean=forward.get_mean_tensor(), weight=tw, segment_offsets=offsets)
    from_codes = ph.LayerNormBackward().stamp(tdy, forward.get_checkpoint(), rstd_tensor, stream, weight=tw, segment_offsets=offsets)
    assert from_input.get_workspace_size_in_bytes() > 0 and from_codes.get_workspace_size_in_bytes() > 0
    plans = (forward, from_input, from_codes)
    for plan in plans:
        plan.run()
    if used < rows - 1:
        assert np.isnan(base.gradients_of(from_input, stream)[1]).all() and np.isnan(base.gradients_of(from_codes, stream)[2]).all()
    per_row = [forward.get_output_tensor(), forward.get_mean_tensor(), rstd_tensor, forward.get_checkpoint().codes, forward.get_checkpoint().scales,
               from_input.get_input_gradient_tensor(), from_codes.get_input_gradient_tensor()]
    for t in per_row:
        t.memset_async(0x5A, stream)
    offsets.copy_from_async(offsets_tensor([0, used, used], stream), stream)
    for plan in plans:
        plan.run()
    for t in per_row:
        assert (copy_gpu_to_numpy(t, stream).view(np.uint8).reshape(rows, -1)[used:] == 0x5A).all()
    if used == 0:
        for plan in (from_input, from_codes):
            assert not base.gradients_of(plan, stream)[1].any() and not base.gradients_of(plan, stream)[2].any()
        return
    x, dy = x[:used], dy[:used]
    y, mean, _, _ = layer_norm(x, w, 0.0, EPSILON)
    y_off, mean_off, _, _ = layer_norm_tolerances(x, w, np.zeros(cols), EPSILON, dtype)
    within(download(forward.get_output_tensor(), stream)[:used], y, y_off, "y")
    within(download(forward.get_mean_tensor(), stream)[:used], mean, mean_off, "mean")
    rstd = download(rstd_tensor, stream)[:used]
    codes, scales = (copy_gpu_to_numpy(t, stream)[:used] for t in (forward.get_checkpoint().codes, forward.get_checkpoint().scales))
    for plan, h, h_off in ((from_input, (x - download(forward.get_mean_tensor(), stream)[:used]) * rstd, 2 * UNIT),
                           (from_codes, decode(codes, scales, INT8).astype(np.float64), UNIT)):
        off = layer_norm_gradient_tolerances(dy, h, h_off * np.abs(h), rstd, w, dtype, DataType.fp32)
        got = base.gradients_of(plan, stream)
        for g, want, o, what in zip((got[0][:used], *got[1:]), layer_norm_gradients(dy, h, rstd, w), off, ("dx", "dweight", "dbias")):
            within(g, want, o, what)


# rows enough for several shares per block (over 128 rows for every team): teams of 16, 32, 64, 128 and 512 lanes, with and without a tail
SHARES = [(2_200_000, 7, DataType.bf16), (1_200_000, 4, DataType.fp32), (600_000, 301, DataType.bf16), (300_000, 1001, DataType.fp16), (140_000, 2048, DataType.bf16),
          (34_000, 8191, DataType.bf16)]


@pytest.mark.parametrize("used", [None, 777])
@pytest.mark.parametrize("rows,cols,dtype", SHARES, ids=[f"{r}x{c}-{d.name}" for r, c, d in SHARES])
def test_more_than_one_share_per_block(stream, rows, cols, dtype, used):
    """Every row of input and error is the same one, mean and rstd are each row's own: the gradients of the parameters follow from sums of
    these."""
    rng = np.random.default_rng([rows, cols])
    tx, x = upload(rng.standard_normal((1, cols)), dtype, stream)
    tdy, dy = upload(rng.standard_normal((1, cols)), dtype, stream)
    tw, w = upload(1 + 0.2 * rng.standard_normal(cols), DataType.fp32, stream)
    tmean, mean = upload(0.5 * rng.standard_normal((rows, 1)), DataType.fp32, stream)
    trstd, rstd = upload(rng.uniform(0.5, 1.5, (rows, 1)), DataType.fp32, stream)
    everywhere = lambda t: t.alias_view([rows, cols], [0, 1])  # noqa: E731
    offsets = offsets_tensor([0, used], stream) if used else None
    plan = ph.LayerNormBackward().stamp(everywhere(tdy), everywhere(tx), trstd, stream, mean=tmean, weight=tw, segment_offsets=offsets)
    plan.get_input_gradient_tensor().memset_async(0x5A, stream)
    plan.run()
    count = used or rows
    mean, rstd = mean[:count], rstd[:count]
    most = np.abs(dy) * (np.abs(x) * rstd.sum() + (np.abs(mean) * rstd).sum())  # at least the sum of the products' magnitudes
    dw, db = dy * (x * rstd.sum() - (mean * rstd).sum()), count * dy
    got = [download(t, stream)[None] for t in (plan.get_weight_gradient_tensor(), plan.get_bias_gradient_tensor())]
    within(got[0], dw, (CHAIN + 4) * UNIT * most, "dweight")
    within(got[1], db, (CHAIN + 1) * UNIT * np.abs(db), "dbias")
    at = np.r_[0:3, count - 3:count]
    view = plan.get_input_gradient_tensor()
    for r in at:
        g = copy_gpu_to_numpy(view.alias_view([1, cols], [cols, 1], int(r) * cols), stream)
        h = (x - mean[r]) * rstd[r]
        want = layer_norm_gradients(dy, h, rstd[r:r + 1], w)[0]
        off = layer_norm_gradient_tolerances(dy, h, 2 * UNIT * (np.abs(x) + np.abs(mean[r])) * rstd[r], rstd[r:r + 1], w, dtype, DataType.fp32)[0]
        within(from_storage(g, dtype).astype(np.float64), want, off, f"dx of row {r}")
    if used:
        rest = copy_gpu_to_numpy(view.alias_view([2, cols], [cols, 1], used * cols), stream)
        assert (rest.view(np.uint8) == 0x5A).all()


def test_results_that_hold_something_else_before_every_run(stream):
    """On the plan's stream, on another and on two at once: every run writes all of its results, on the stream that it was given."""
    rows, cols = 3000, 1030
    rng = np.random.default_rng(31)
    tx, _ = upload(rng.standard_normal((rows, cols)), DataType.bf16, stream)
    tw, _ = upload(rng.standard_normal(cols), DataType.fp32, stream)
    errors = [upload(rng.standard_normal((rows, cols)), DataType.bf16, stream)[0] for _ in range(2)]
    norms = [ph.LayerNorm(EPSILON, E4M3).stamp(tx, stream, weight=tw) for _ in range(2)]
    norms[0].run()
    backs = [ph.LayerNormBackward().stamp(e, norms[0].get_checkpoint(), norms[0].get_reciprocal_deviation_tensor(), stream, weight=tw) for e in errors]
    stream.synchronize()
    of_norm = [[n.get_output_tensor(), n.get_mean_tensor(), n.get_reciprocal_deviation_tensor(), n.get_checkpoint().codes, n.get_checkpoint().scales] for n in norms]
    of_back = [[b.get_input_gradient_tensor(), b.get_weight_gradient_tensor(), b.get_bias_gradient_tensor()] for b in backs]
    bits = lambda tensors: [copy_gpu_to_numpy(t, stream).tobytes() for t in tensors]  # noqa: E731
    want_norm, want_back = bits(of_norm[0]), []
    for b, tensors in zip(backs, of_back):
        b.run()
        want_back.append(bits(tensors))
    others = [ph.Stream(0), ph.Stream(0)]
    # the forward plan that no backward plan reads from, on one stream after the other
    for on in (stream, *others):
        for t in of_norm[1]:
            t.memset_async(0x5A, on)
        norms[1].run_on(on)
        on.synchronize()
        assert bits(of_norm[1]) == want_norm
    for _ in range(5):
        for b, tensors, on in zip(backs, of_back, others):
            for t in tensors:
                t.memset_async(0x5A, on)
            b.run_on(on)
        for on in others:
            on.synchronize()
        assert [bits(t) for t in of_back] == want_back
    for b, tensors, on in zip(backs, of_back, reversed(others)):
        for t in tensors:
            t.memset_async(0x5A, on)
        b.run_on(on)
        on.synchronize()
    assert [bits(t) for t in of_back] == want_back
