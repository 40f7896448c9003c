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

import cudaforge_amd as cf
from helpers import dev
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


# Fewer rows than fill the chip over a long context, whose ranges are cut, and more over a short one; rows of chunks
# that end inside a wave's share, single rows, none.
BIG = [(32, 8, 128, [200, 1, 58, 0, 3], [2300, 900, 0, 40, 2044]), (64, 16, 64, [131, 1, 5], [2200, 31, 700]),
       (64, 8, 64, [513, 1, 300], [60, 900, 0]), (32, 8, 128, [1540, 20], [5, 560])]


@pytest.mark.gpu
@pytest.mark.parametrize("H,H_kv,d,new,past", BIG)
def test_tiles_of_256_rows(gpu, H, H_kv, d, new, past):
    """Hints that are right, absent and wrong; Q as a part of a projection, K and V of a page in one tensor."""
    c = PagedQ8(new, past, H, H_kv, d, 16, True, seed=52)
    assert tile_rows(gpu, c, max(new)) == 256 and tile_rows(gpu, c, 0) == 256
    check_tight(c, c.run(max_new=max(new)))
    check_tight(c, c.run(max_len=1))                     # in one range; which tiles goes by the rows alone
    wide = np.full((c.T, (H + 2 * H_kv) * d), 9.0, c.dt)
    wide[:, :H * d] = c.q.reshape(c.T, -1)
    both = np.full((c.n_pages, 16, 2, H_kv, d), 0x7f, np.uint8)
    both[:, :, 0], both[:, :, 1] = c.codes
    kv = dev(both)
    bufs = [dev(wide), kv, kv.ptr + H_kv * d] + c.bufs()[3:]
    check_tight(c, c.run(bufs, q_stride=(H + 2 * H_kv) * d, page_stride=32 * H_kv * d, row_stride=2 * H_kv * d))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_tiles_of_256_rows_with_missing_pages(gpu, d):
    c = PagedQ8([260, 2, 30], [2300, 500, 100], 32, 8, d, 16, True, seed=53)
    c.table[0, [0, 5, 6, 100, 159]] = [-1, c.n_pages, 2 ** 31 - 1, -2 ** 31, -3]
    c.table[0, 20:60] = -1                               # whole blocks and, cut, whole ranges
    c.table[2, :] = -1
    assert tile_rows(gpu, c) == 256
    for hint in (0, 1):
        got = c.run(max_len=hint)
        check_tight(c, got)
        assert (got[262:292] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_tiles_of_256_rows_with_nan(gpu, d):
    """NaN V among the cached, in a new token, and of a whole block's power; a K in one head; rows that do not
    see them keep theirs."""
    new, past = [260, 40], [2300, 500]
    c = PagedQ8(new, past, 32, 8, d, 16, True, seed=54)
    at = lambda b, pos: (c.table[b, pos // 16], pos % 16)
    nan = np.zeros(c.q.shape, bool)
    r = [np.arange(c.start[b], c.start[b + 1]) for b in range(2)]
    c.codes[1][at(0, 77)][:, 3] = 0x7f                   # seen by all
    nan[r[0], :, 3] = True
    for k in (70, 130, 259):                             # in different waves' rows and tiles
        c.codes[1][at(0, past[0] + k)][:, 5 + k % 7] = 0xff
        nan[r[0][k:], :, 5 + k % 7] = True
    c.powers[1][c.table[1, 3], 0, 2] = 255               # a block of V in KV head 2
    nan[r[1], 8:12] = True
    c.codes[0][at(0, past[0] + 200)][6, 9] = 0x7f        # a K in KV head 6
    nan[r[0][200:], 24:28] = True
    assert tile_rows(gpu, c) == 256
    clean = PagedQ8(new, past, 32, 8, d, 16, True, seed=54)
    for hint in (0, 1):
        got = c.run(max_len=hint)
        assert (np.isnan(got) == nan).all()
        base = clean.run(max_len=hint)
        got[nan] = base[nan]
        check_tight(clean, got)


@pytest.mark.gpu
def test_tiles_of_256_rows_without_a_workspace(gpu):
    c = PagedQ8([260, 1, 20], [2300, 900, 3], 32, 8, 128, 16, True, seed=55)
    assert tile_rows(gpu, c) == 256
    st = cf.Stream()
    o = dev(np.full(c.q.shape, 7.0, c.dt))
    bufs = c.bufs()
    gpu.gpu_inject_alloc_failures(1000)
    try:
        rc = cf.call_op(c.op, bufs, [o], c.params(), st)
    finally:
        gpu.gpu_inject_alloc_failures(0)
    assert rc == 0
    st.synchronize()
    check_tight(c, o.download())
