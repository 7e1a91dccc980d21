"""More of what the row operators refuse without a GPU: checkpoints that Python allocates."""
from __future__ import annotations

import pytest

from thor_amd import physical as ph
from thor_amd.dtypes import DataType


@pytest.mark.parametrize("dtype", [d for d in DataType if d not in (DataType.fp8_e4m3, DataType.fp8_e5m2, DataType.int8)], ids=lambda d: d.name)
def test_checkpoints_of_other_types(dtype):
    """As ActivationCheckpoint::allocate: before any tensor is made of it."""
    with pytest.raises(ValueError, match="supports checkpoints in fp8_e4m3, fp8_e5m2 and int8"):
        ph.ActivationCheckpoint.allocate([4, 130], dtype)


def test_a_checkpoint_without_axes():
    with pytest.raises(ValueError, match="requires at least one axis"):
        ph.ActivationCheckpoint.allocate([], DataType.int8)


def test_a_checkpoint_without_elements():
    with pytest.raises(ValueError, match="must be non-zero"):
        ph.ActivationCheckpoint.allocate([4, 0], DataType.int8)
