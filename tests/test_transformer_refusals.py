"""CPU tests of what the transformer ops refuse at their limits: outputs that
other workgroups' reads would race with, and sizes past the kernels' reach."""
import ctypes

import pytest

from tensorflow_musa_extension_amd import _lib
from test_transformer_abi import A, B, F, GAP, INV, Q, T, UNI, call, norm, size

ROWS = 300


@pytest.mark.parametrize("c", [1, 8])
@pytest.mark.parametrize("at", [0, 4])
def test_rstd_is_no_input(c, at):
    """Only y and sum may take x's or residual's memory: another row's
    workgroup may still have to read what rstd would be written over.  With
    one column they have the same size too."""
    x, g = T(0, (ROWS, c)), T(1, (c,))
    y, s, r = T(2, (ROWS, c)), T(5, (ROWS, c)), T(4, (ROWS, c))
    over = T(0, (ROWS,), ptr=A + at)
    code, msg = norm(x=x, g=g, y=y, rstd=over)
    assert (code, msg) == (INV, "MusaAddRmsNorm: rstd overlaps x")
    over = T(4, (ROWS,), ptr=A + 4 * GAP + at)
    code, msg = norm(x=x, r=r, g=g, y=y, s=s, rstd=over)
    assert (code, msg) == (INV, "MusaAddRmsNorm: rstd overlaps residual")
    code, msg = call("TFMA_MusaAddRmsNormQuantized", None, x, r, g, 1e-5, T(2, (ROWS, c), Q), over, s)
    assert (code, msg) == (INV, "MusaAddRmsNormQuantized: scale overlaps residual")
    code, msg = norm(x=x, g=g, y=y, rstd=T(2, (ROWS,)))
    assert (code, msg) == (INV, "MusaAddRmsNorm: y and rstd overlap")


@pytest.mark.parametrize("rows,c", [(ROWS, 8), (1, 8), (1, 1)])
@pytest.mark.parametrize("which", ["y_backprop", "sum", "sum_backprop"])
def test_gamma_backprop_is_no_input(rows, c, which):
    a = {"y_backprop": T(0, (rows, c)), "sum": T(1, (rows, c)), "sum_backprop": T(6, (rows, c))}
    over = T(0, (c,), ptr=a[which].data)
    code, msg = call("TFMA_MusaAddRmsNormGrad", None, a["y_backprop"], a["sum"], T(2, (c,)),
                     T(3, (rows,)), a["sum_backprop"], T(4, (rows, c)), over,
                     ctypes.c_void_p(A + 9 * GAP), 1 << 30)
    assert (code, msg) == (INV, f"MusaAddRmsNormGrad: gamma_backprop overlaps {which}")


@pytest.mark.parametrize("k", [(1 << 23) + 16, 17825792, 1 << 25, (1 << 30) - 16])
def test_8_bit_rows_past_the_tiles_offsets(k):
    """Rows whose 256 of a tile pass 2^31 bytes."""
    x, w = T(0, (1, k), Q), T(20, (128, k), Q)
    want = ("MusaLinearQuantized: the inner dimension of 8-bit operands must be at most 8388608, "
            f"got {k}")
    code, msg = call("TFMA_MusaLinearQuantized", None, x, T(60, (1,)), w, T(61, (128,)), None, None,
                     b"", T(62, (1, 128), B), ctypes.c_void_p(A + 70 * GAP), 1 << 30)
    assert (code, msg) == (UNI, want)
    code, msg, _ = size("TFMA_MusaLinearWorkspaceBytes", x, w, 1)
    assert (code, msg) == (UNI, want.replace("Quantized", ""))


def test_8_bit_rows_as_long_as_the_tiles_offsets():
    code, _, need = size("TFMA_MusaLinearWorkspaceBytes", T(0, (64, 1 << 23), Q),
                         T(20, (128, 1 << 23), Q), 1)
    assert code == _lib.OK and need > 0
