"""The dense operators through the C ABI: results that share memory with an input are refused (the kernels read their inputs
again after others have begun to write).  No GPU needed: every call here lacks a pointer that is looked for afterwards, so
what passes the check under test is refused by the next one, and nothing is ever launched on the made-up addresses."""
import ctypes as C

import pytest

from cbm4gnn_amd import _lib

CBM_ERR_NULL, CBM_ERR_SHAPE = 1, 3
BASE, OTHER = 1 << 40, 1 << 44
BYTES = {0: 4, 1: 2, 2: 2}


def batch(rows):
    return C.byref(_lib.CbmNormBatch(samples=1, max_len=rows, rows=rows, piece_rows=64))


def forward(x, y, rows, ch, ldx, ldy, dtype):
    assert rows >= 1 << 20                                  # in pieces, which need the workspace that is missing
    return _lib.hip_lib().cbm_group_norm_forward(batch(rows), x, y, None, None, None, None, None, ch, 1, ldx, ldy, 1e-5, 0, dtype, None)


def backward(x, dy, dx, rows, ch, ldx, ldg, ldd, dtype):
    return _lib.hip_lib().cbm_group_norm_backward(batch(rows), x, dy, dx, None, None, OTHER, OTHER, None, None, None, ch, 1, ldx, ldg, ldd,
                                                  0, dtype, None)


def scores_backward(z, grad, rows, classes, ld, ldg, dtype):
    return _lib.hip_lib().cbm_label_scores_backward(z, OTHER, None, None, None, OTHER, None, None, grad, rows, classes, 0, ld, ldg, -100,
                                                    dtype, None)


def statuses(d, rows, ch, ld, ld_out, dtype):
    """Of every call, with the result d bytes after the input."""
    out = [backward(BASE, OTHER, BASE + d, rows, ch, ld, ch, ld_out, dtype), backward(OTHER, BASE, BASE + d, rows, ch, ch, ld, ld_out, dtype),
           scores_backward(BASE, BASE + d, rows, ch, ld, ld_out, dtype)]
    return out + ([forward(BASE, BASE + d, rows, ch, ld, ld_out, dtype)] if rows >= 1 << 20 else [])


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("rows,ch", [(1, 4), (5, 258), (9000, 517), (300, 64), (1 << 20, 258), (1 << 20, 64)])
def test_results_over_inputs(rows, ch, dtype):
    e = BYTES[dtype]
    end = rows * ch * e
    for d in (0, e, (ch - 1) * e, (rows - 1) * ch * e, end - 1):
        for sign in (1, -1):
            assert set(statuses(sign * d, rows, ch, ch, ch, dtype)) == {CBM_ERR_SHAPE}, d
    for d in (end, -end):
        assert set(statuses(d, rows, ch, ch, ch, dtype)) == {CBM_ERR_NULL}, d
    assert set(statuses(0, rows, ch, ch + 3, ch, dtype)) == set(statuses(-end + 1, rows, ch, ch + 3, ch, dtype)) == {CBM_ERR_SHAPE}
    assert set(statuses(-end, rows, ch, ch + 3, ch, dtype)) == {CBM_ERR_NULL}
    for ld in (2 * ch, 2 * ch + 5):                         # columns of one buffer
        for d in ((ch - 1) * e, (1 - ch) * e):
            assert set(statuses(d, rows, ch, ld, ld, dtype)) == {CBM_ERR_SHAPE}
        for d in (ch * e, -ch * e, (ld - ch) * e, ld * rows * e):
            assert set(statuses(d, rows, ch, ld, ld, dtype)) == {CBM_ERR_NULL}
        if rows > 1:
            assert set(statuses((ld - ch + 1) * e, rows, ch, ld, ld, dtype)) == {CBM_ERR_SHAPE}       # the next row
            assert set(statuses(ld * (rows - 1) * e, rows, ch, ld, ld, dtype)) == {CBM_ERR_SHAPE}     # the last one


def test_against_every_byte():
    """Small matrices of one stride, every distance, against the bytes themselves."""
    for rows, ch, ld in ((1, 3, 3), (2, 3, 3), (3, 2, 5), (4, 1, 4), (3, 3, 4)):
        at = {(r * ld + c) * 4 + b for r in range(rows) for c in range(ch) for b in range(4)}
        for d in range(-(rows * ld + 2) * 4, (rows * ld + 2) * 4 + 1):
            meet = any(p + d in at for p in at)
            assert scores_backward(BASE, BASE + d, rows, ch, ld, ld, 0) == (CBM_ERR_SHAPE if meet else CBM_ERR_NULL), (rows, ch, ld, d)
