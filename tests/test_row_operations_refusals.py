"""More of what the row operators refuse without a GPU: checkpoints that Python allocates, and epsilons in the device interface."""
from __future__ import annotations

import ctypes
import math

import pytest

from thor_amd import _lib
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


class Rows(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("outer", ctypes.c_int64), ("inner", ctypes.c_int64)]


class LayerNormCall(ctypes.Structure):
    """thorhip_layer_norm."""
    _fields_ = [("dtype", ctypes.c_int), ("parameter_dtype", ctypes.c_int), ("checkpoint_dtype", ctypes.c_int), ("extent_is_64", ctypes.c_int),
                ("rows", ctypes.c_uint32), ("columns", ctypes.c_uint32), ("inner_rows", ctypes.c_uint32), ("epsilon", ctypes.c_float), ("input", Rows), ("output", Rows),
                ("weight", ctypes.c_void_p), ("bias", ctypes.c_void_p), ("mean", ctypes.c_void_p), ("rstd", ctypes.c_void_p), ("codes", ctypes.c_void_p),
                ("scales", ctypes.c_void_p), ("extent", ctypes.c_void_p)]


@pytest.mark.parametrize("epsilon", [0.0, -1e-5, 1e-40, math.inf, math.nan])
def test_epsilons_of_the_device_interface(epsilon):
    """A row of one value has the root of epsilon alone, which has to be a normal number; refused before anything is looked at."""
    call = LayerNormCall(int(DataType.fp32), int(DataType.fp32), 0, 0, 1, 4, 0, epsilon)
    assert _lib.load().thorhip_layer_norm_forward(ctypes.byref(call), None, 0, None, 0) == -1
    assert b"thorhip_layer_norm_forward: epsilon" in _lib.load().thorhip_last_error()
    call.epsilon = 1e-5
    assert _lib.load().thorhip_layer_norm_forward(ctypes.byref(call), None, 0, None, 0) == -1
    assert b"NULL tensor" in _lib.load().thorhip_last_error()
