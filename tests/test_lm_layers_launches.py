"""What the library's own launchers do not launch they say, on the CPU: nothing is enqueued."""
import ctypes
import subprocess

import pytest

from mlir_edsl_hip import _native
from mlir_edsl_hip.build import LIB_PATH

INVALID_VALUE = 1  # hipErrorInvalidValue


def exported(name):
    """The mangled name of a C++ function of the library."""
    symbols = subprocess.run(["nm", "-D", "--defined-only", LIB_PATH], capture_output=True, text=True, check=True).stdout
    (found,) = [s.split()[-1] for s in symbols.splitlines() if name in s]
    return getattr(_native.lib(), found)


@pytest.mark.parametrize("rows16,cols16", [(1, 3), (1, 5), (2, 0), (3, 4), (4, 4), (4, 8), (0, 1), (5, 1)])
def test_streamed_8_bit_layers_of_other_widths(rows16, cols16):
    launch = exported("launch_i8_skinny")
    launch.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_void_p]
    launch.restype = ctypes.c_int
    args = ctypes.create_string_buffer(512)  # of no rows and columns
    assert launch(args, rows16, cols16, None) == INVALID_VALUE


@pytest.mark.parametrize("kind,direct,big", [(0, 0, 0), (0, 1, 0), (1, 1, 1), (2, 1, 1)])
def test_two_products_of_tiles_that_take_one(kind, direct, big):
    """f32, and the largest tiles: the second operand's pointer, the third of the arguments, is given."""
    launch = exported(f"launch_grouped_weightsILi{kind}E")
    launch.argtypes = [ctypes.c_void_p, ctypes.c_bool, ctypes.c_bool, ctypes.c_void_p]
    launch.restype = ctypes.c_int
    args = ctypes.create_string_buffer(512)
    ctypes.c_void_p.from_buffer(args, 2 * ctypes.sizeof(ctypes.c_void_p)).value = 0x1000
    assert launch(args, direct, big, None) == INVALID_VALUE
