"""mha_paged_attn_{f16,f32}_cuda at the edges of what its arrays may hold, against the 64-bit oracle and
the tolerances of test_paged.py (GPU)."""

import ctypes
from ctypes import c_void_p

import numpy as np
import pytest

import cudaforge_amd as cf
from helpers import dev
from test_paged import I32, Paged, ref_attn

SHAPES = [(8, 2, 64, 16), (8, 2, 128, 32), (16, 1, 64, 16), (5, 5, 33, 7)]     # the last: the plain kernel


def fill(c, seed=99):
    """Finite values where Paged leaves NaN: every position of every page."""
    rng = np.random.default_rng(seed)
    for x in (c.kp, c.vp):
        x[np.isnan(x)] = rng.standard_normal(int(np.isnan(x).sum())).astype(c.dt)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,P", SHAPES)
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 2], [40, 1, 33]])
def test_lengths_past_the_table(gpu, f16, H, H_kv, d, P, new):
    """A length past its table's row is the row's: its rows are the last positions of it."""
    c = Paged(new, [90, 300, 20], H, H_kv, d, P, f16, seed=23)
    fill(c)
    rng = np.random.default_rng(5)
    held = c.table >= 0
    c.table[~held] = rng.integers(0, c.n_pages, int((~held).sum()))           # pages of others: shared
    full = c.width * P
    for past in (full + 1, 2 ** 30, 2 ** 31 - 1):
        c.lens[:] = [past, full, min(past, full + 7)]
        got = c.run(max_new=max(new))
        assert not np.isnan(ref_attn(c.q, c.kp, c.vp, c.table, c.lens, c.start, c.scale)[0][:c.start[-1]]).any()
        c.check(got)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,P", SHAPES)
@pytest.mark.parametrize("wide", [False, True])
def test_offsets_past_the_rows(gpu, f16, H, H_kv, d, P, wide):
    """Offsets below 0 and behind the last row are clamped: a sequence has the rows between."""
    c = Paged([4, 40 if wide else 4, 3, 2], [90, 150, 60, 33], H, H_kv, d, P, f16, seed=25, pad=0)
    fill(c)
    for start in ([-4, 4, c.T - 5, 10 ** 6, 2 ** 31 - 1], [-2 ** 31, -7, 5, c.T, c.T + 9], [0, 0, c.T, c.T, c.T],
                  [3, 4, 6, 6, c.T - 2]):
        c.start = np.array(start, I32)
        c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,P", SHAPES)
@pytest.mark.parametrize("n", [4, 40])
def test_offsets_out_of_order(gpu, f16, H, H_kv, d, P, n):
    """Offsets that fall: the sequence that ends before it starts has no rows, the next one has the
    rows from its offset on.  Rows of one sequence only are that sequence's, rows of none are left."""
    c = Paged([n, 3, n, 2], [90, 40, 60, 33], H, H_kv, d, P, f16, seed=27)
    fill(c)
    a, b = c.start[1], c.start[1] - 2
    c.start = np.array([0, a, b, b + n, b + n + 2], I32)                      # rows b .. a - 1: two sequences'
    got = c.run(max_new=n)
    want, e32, e16 = ref_attn(c.q, c.kp, c.vp, c.table, c.lens, c.start, c.scale)
    first = c.start.copy()
    first[2:] = [a] * 3                                                       # the first sequence alone
    other = ref_attn(c.q, c.kp, c.vp, c.table, c.lens, first, c.scale)[0]
    tol = e16 + 2.0 ** -11 * np.abs(want) + 2.0 ** -25 if f16 else e32 + 2.0 ** -24 * np.abs(want)
    alone = np.r_[0:b, a:b + n + 2]
    assert (np.abs(got[alone] - want[alone]) <= tol[alone]).all()
    both = got[b:a].astype(np.float64)
    near = lambda x: np.abs(both - x) <= 4 * tol[b:a] + 2.0 ** -9 * np.abs(x)
    assert (near(want[b:a]) | near(other[b:a])).all()
    assert (got[b + n + 2:] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,P", SHAPES)
@pytest.mark.parametrize("n", [1, 9, 100])
@pytest.mark.parametrize("far", [9.0, 14.0, 17.6, 20.0])
def test_many_small_weights_beside_a_large_one(gpu, f16, H, H_kv, d, P, n, far):
    """One position scores `far` above some ten thousand equal ones: each of them weighs e^-far of it,
    below what fp16 holds beside 1 (2^-25 = e^-17.3), all together as much as the tolerance many times."""
    c = Paged([n], [12000 - n], H, H_kv, d, P, f16, seed=31, pad=0)
    rng = np.random.default_rng(3)
    c.q[:] = 1
    c.kp[:] = 0
    c.vp[:] = (1 + rng.random(c.vp.shape) / 4).astype(c.dt)
    c.kp[c.table[0, 0], 0] = far / (c.scale * d)
    c.vp[c.table[0, 0], 0] = 0
    for hint in (0, 1):                                  # the positions shared out, and in one range
        c.check(c.run(max_new=n, max_len=hint))


ODD_CASES = [
    (8, 2, 64, 16, [12, 2, 8], [100, 30, 7]), (8, 2, 128, 16, [4, 4, 4], [2500, 60, 1500]), (32, 8, 128, 16, [1] * 5, [4000, 300, 90, 2222, 17]),
    (12, 12, 64, 16, [1, 1], [700, 333]), (12, 12, 64, 16, [9] * 12, [300] * 12), (8, 4, 128, 32, [150, 40, 90, 1], [33, 9, 200, 600]),
    (4, 4, 64, 16, [130, 2], [4000, 3000]), (128, 64, 64, 16, [400], [64]), (4, 2, 40, 5, [7, 3], [20, 9]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,P,new,past", ODD_CASES)
def test_infinite_and_nan_v_among_the_cached(gpu, f16, H, H_kv, d, P, new, past):
    """Infinite and NaN V of cached positions, which every row sees, in dims of their own; in three of
    these and one more a new token has another that only rows from it on see."""
    c = Paged(new, past, H, H_kv, d, P, f16, seed=33)
    clean = c.vp.copy()
    inf, nan = np.inf, np.nan
    at = lambda b, pos: (c.table[b, pos // P], pos % P)
    want = np.zeros(c.q.shape)                           # inf, -inf or NaN; 0: as without them
    for b, (n, p) in enumerate(zip(new, past)):
        r = np.arange(c.start[b], c.start[b + 1])
        for dim, pos, x in ((3, p // 2, nan), (5, 0, inf), (d - 1, p - 1, -inf), (7, p // 3, inf), (7, p // 2, -inf), (20, p // 4, inf)):
            c.vp[at(b, pos)][:, dim] = x
            want[r, :, dim] = nan if want[r[0], 0, dim] == -x else x
        h = n // 2
        new_at = at(b, p + h)
        c.vp[new_at][:, 5], c.vp[new_at][:, 20], c.vp[new_at][:, 3], c.vp[new_at][:, 11] = -inf, inf, inf, nan
        want[r[h:], :, 5], want[r[h:], :, 11] = nan, nan
    odd = want != 0
    dirty = c.vp
    for hint in (0, 1):
        c.vp = dirty
        got = c.run(max_new=max(new), max_len=hint)
        assert np.array_equal(got[odd].astype(np.float64), want[odd], equal_nan=True)
        c.vp = clean
        plain = c.run(max_new=max(new), max_len=hint)
        got[odd] = plain[odd]
        c.check(got)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new,past", [([1, 1, 1], [5000, 40, 1700]), ([70, 1, 30], [3000, 900, 10])])
def test_without_memory_for_a_workspace(gpu, f16, new, past):
    """No buffer to be had, or a recording on a stream that has none: the tiles are not cut, and the call
    succeeds.  What the stream had before is used again afterwards."""
    c = Paged(new, past, 8, 2, 128, 16, f16, seed=35)
    bufs = [dev(x) for x in (c.q, c.kp, c.vp, c.table, c.lens, c.start)]
    st = cf.Stream()
    o = dev(np.full(c.q.shape, 7.0, c.dt))
    gpu.gpu_inject_alloc_failures(1000)
    try:
        rc = cf.call_op(c.op, bufs, [o], c.params(max_new=max(new)), st)
    finally:
        gpu.gpu_inject_alloc_failures(0)
    assert rc == 0
    st.synchronize()
    c.check(o.download())

    st = cf.Stream()
    o = dev(np.full(c.q.shape, 7.0, c.dt))
    ex = c_void_p()
    held = gpu.gpu_workspace_size()
    assert gpu.gpu_capture_begin(st.handle) == 0
    rc = cf.call_op(c.op, bufs, [o], c.params(max_new=max(new)), st)
    assert gpu.gpu_capture_end(st.handle, ctypes.byref(ex)) == 0
    assert rc == 0 and gpu.gpu_workspace_size() == held
    for drop in (0, 500, 0):
        lens = c.lens.copy()
        c.lens = np.maximum(lens - drop, new).astype(I32)
        bufs[4].upload(c.lens)
        assert gpu.gpu_graph_launch(ex, st.handle) == 0
        st.synchronize()
        c.check(o.download())
        c.lens = lens
        c.check(c.run(max_new=max(new)))                 # eager, with a buffer
    gpu.gpu_graph_exec_destroy(ex)


@pytest.mark.gpu
@pytest.mark.parametrize("H,H_kv,d,P", SHAPES)
@pytest.mark.parametrize("n", [1, 9, 100])
def test_large_fp32_values(gpu, H, H_kv, d, P, n):
    """V of up to 2^120: weights of at most 1 of 150 positions leave their sum below FP32's 2^128."""
    c = Paged([n], [150 - n], H, H_kv, d, P, False, seed=37)
    c.vp[:] *= np.float32(2.0 ** 118)
    for std in (0, 1, 5):
        x = Paged([n], [150 - n], H, H_kv, d, P, False, seed=37, k_std=std)
        x.vp = c.vp
        for hint in (0, 1):
            x.check(x.run(max_new=n, max_len=hint))
