"""Attention of chunks over the 8-bit paged cache: tiles of 128 and of 256 rows (fp16), with the oracle of
test_paged_q8.py (GPU).  Which of them a call takes is asserted, so that another rule for the choice cannot
leave one of them without a test.

Tolerance of fp16 rows.  The weights of V are sums of two fp16 numbers: off by at most 2^-22 of
themselves, 4 units of FP32's 2^-24, where test_paged.ref_attn's e32 counts 20 at least of the same sum of
sizes; so 1.2 e32.  The largest weight is held as 2^7 or more, and below fp16's normal numbers the second part
is a multiple of 2^-24: off by 2^-25, 2^-32 of the largest, as likely up as down in each position.
"""

import ctypes

import numpy as np
import pytest

from test_paged import ref_attn
from test_paged_q8 import PagedQ8


class AttnArgs(ctypes.Structure):
    """cf_paged_q8_args_t (kernels.h)."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k", "v", "o", "table", "seq_lens", "q_start")] + \
               [(n, ctypes.c_int64) for n in ("q_stride", "page_stride", "row_stride", "head_stride")] + \
               [(n, ctypes.c_int32) for n in ("B", "T", "H_q", "H_kv", "d", "page_size", "num_pages", "max_pages", "max_new",
                                              "max_len")] + \
               [("scale", ctypes.c_float), ("elem", ctypes.c_int32), ("workspace", ctypes.c_void_p), ("uncut", ctypes.c_int32),
                ("k_scales", ctypes.c_void_p), ("v_scales", ctypes.c_void_p), ("block", ctypes.c_int32)]


def tile_rows(native, c, max_new=0, max_len=0):
    """Rows of the tiles that a call on fp16 rows takes where its tiles may be cut: its workspace, which
    holds records of whole tiles, beside that of the same call on FP32 rows, whose tiles have 128."""
    native.cf_paged_attn_q8_bytes.restype = ctypes.c_size_t
    full = c.width * c.P
    size = []
    for elem in (1, 0):                                  # CF_ELEM_F16, CF_ELEM_F32
        a = AttnArgs(q_stride=c.H * c.d, page_stride=c.P * c.H_kv * c.d, row_stride=c.H_kv * c.d, head_stride=c.d, B=c.B, T=c.T,
                     H_q=c.H, H_kv=c.H_kv, d=c.d, page_size=c.P, num_pages=c.n_pages, max_pages=c.width,
                     max_new=min(max_new, c.T) or c.T, max_len=min(max_len, full) or full, scale=c.scale, elem=elem, block=c.block)
        size.append(native.cf_paged_attn_q8_bytes(ctypes.byref(a)))
    assert size[0] > 0 and size[1] > 0, "tiles that are not cut tell nothing"
    return 256 if size[0] > 1.5 * size[1] else 128


def check_tight(c, got):
    """c.check with the tolerance of weights in two parts."""
    want, e32, _ = ref_attn(c.q, c.kp, c.vp, c.table, c.lens, c.start, c.scale)
    outside = np.isnan(want).all((1, 2))
    assert (got[outside] == 7.0).all(), "rows of no sequence were written"
    v = np.abs(c.vp[np.isfinite(c.vp)]).max()
    tol = 1.2 * e32 + 2.0 ** -11 * np.abs(want) + 2.0 ** -25 + 4 * np.sqrt(c.lens.max()) * 2.0 ** -32 * v
    off = np.abs(got.astype(np.float64) - want)
    bad = ~(off <= tol) & ~outside[:, None, None]
    assert not bad.any(), "%d values off, first at %s by %s, allowed %s" % (
        bad.sum(), np.argwhere(bad)[0], off[bad][0], tol[bad][0])


@pytest.mark.gpu
@pytest.mark.parametrize("H,H_kv,d,new,past,rows", [
    (8, 2, 128, [90, 1, 17], [700, 300, 0], 128), (4, 4, 64, [130, 40], [600, 90], 128),
    (32, 8, 128, [300, 1, 40], [2500, 900, 0], 256), (32, 8, 64, [300, 1, 40], [2500, 900, 0], 256)])
def test_weights_are_not_rounded_to_fp16(gpu, H, H_kv, d, new, past, rows):
    """Chunks and what stands beside them: results are off by their own rounding and FP32's, no more."""
    c = PagedQ8(new, past, H, H_kv, d, 16, True, seed=51)
    assert tile_rows(gpu, c, max(new)) == rows
    check_tight(c, c.run(max_new=max(new)))
