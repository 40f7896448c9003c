"""qk_norm_rope_{f16,f32}_cuda on many rows: results that are stored past the caches (more than 64 MiB of them), and
more rows than one launch takes (GPU).  Rows repeat, so that the oracle of test_qk_norm.py sees each once or
a sample of them."""

import numpy as np
import pytest

import cudaforge_amd as cf
from helpers import dev
from test_qk_norm import F32, Rows, frequencies, ref_rows

PAST_BYTES = 64 << 20


def take(c, rows):
    """The same call's rows `rows`, for check()."""
    s = object.__new__(Rows)
    s.__dict__ = dict(c.__dict__, T=len(rows), x=[x[rows] for x in c.x], y=[y[rows] for y in c.y], pos=c.pos[rows])
    return s


def large(T, *args, pads=(0, 0, 0, 0), **kw):
    """Rows(T, ..) of which 1009 are random and the others repeat them, at positions of their own."""
    c = Rows(1009, *args, pads=pads, **kw)
    c.x = [x[np.arange(T) % 1009] for x in c.x]
    c.y = [np.full((T, y.shape[1]), 7.0, y.dtype) for y in c.y]
    c.T, c.pos = T, np.random.default_rng(T).integers(0, 100000, T).astype(np.int32)
    c.pos[np.arange(3, T, 97)] = -1
    c.pos[[0, T - 2, T - 1]] = [5, -1, 77]
    return c


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("norm", [0, 1, 2])
@pytest.mark.parametrize("halves,r,pads", [(1, 128, (0, 0, 0, 0)), (0, 64, (64, 192, 128, 32))])
@pytest.mark.parametrize("in_place", [False, True])
def test_results_past_the_caches(gpu, f16, norm, halves, r, pads, in_place):
    T = 8195 if f16 else 4099
    c = large(T, 32, 8, 128, f16, r, halves, norm, pads=pads, seed=5)
    assert T * 40 * 128 * (2 if f16 else 4) > PAST_BYTES
    got = c.run(in_place)
    rows = np.unique(np.concatenate((np.arange(9), np.arange(T - 9, T), np.random.default_rng(1).integers(0, T, 200), [100, 197])))
    take(c, rows).check([g[rows] for g in got], in_place)
    left = c.pos < 0                                     # every row of a negative position, and what lies between
    for i in range(2):
        before, w = (c.x if in_place else c.y)[i], c.heads[i] * c.d
        assert (got[i][left] == before[left]).all() and (got[i][:, w:] == before[:, w:]).all()
    again = [g.copy() for g in got]
    c.pos = c.pos[np.arange(T) % 1009]                   # rows that repeat in position too: the same bits
    got = c.run(in_place)
    for g in got:
        assert (g[1009:].view(np.uint8) == g[np.arange(1009, T) % 1009].view(np.uint8)).all()
    take(c, rows).check([g[rows] for g in got], in_place)
    assert any((a != g).any() for a, g in zip(again, got))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_q_and_k_in_place_in_one_projection(gpu, f16):
    """Q and K as parts of one large (T, (H_q + 2 H_kv) d) array, in place; V stays as it is."""
    T, H, H_kv, d = (8195 if f16 else 4099), 32, 8, 128
    c = large(T, H, H_kv, d, f16, 0, 1, 1, seed=6)
    w, es = (H + 2 * H_kv) * d, (2 if f16 else 4)
    qkv = np.concatenate((c.x[0], c.x[1], np.full((T, H_kv * d), 3.0, c.dt)), 1)
    buf = dev(qkv)
    p = cf.QkNormRopeParams(num_tokens=T, num_heads=H, num_kv_heads=H_kv, head_dim=d, halves=1, norm=1, eps=c.eps,
                            rope_base=c.base, q_stride=w, k_stride=w, q_out_stride=w, k_out_stride=w)
    k = buf.ptr + H * d * es
    ins = [buf, k, dev(c.pos), dev(c.gain[0]), dev(c.gain[1]), None, None]
    assert cf.call_op("qk_norm_rope_%s_cuda" % ("f16" if f16 else "f32"), ins, [buf, k], p) == 0
    got = buf.download()
    assert (got[:, (H + H_kv) * d:] == 3.0).all()
    rows = np.unique(np.concatenate((np.arange(9), np.arange(T - 9, T), np.random.default_rng(1).integers(0, T, 200))))
    take(c, rows).check([got[rows][:, :H * d], got[rows][:, H * d:(H + H_kv) * d]], True)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d", [16, 10])
def test_more_rows_than_a_launch_takes(gpu, f16, d):
    """2^24 rows are a launch's of either kernel (d = 10 takes the plain one), or its first round; rows and positions
    repeat after 1009, and so do the results."""
    T, n = 2 ** 24 + 1013, 1009
    c = Rows(n, 1, 0, d, f16, 0, 1, 1, seed=7)
    at = np.arange(T) % n
    x = dev(c.x[0][at])
    p = cf.QkNormRopeParams(num_tokens=T, num_heads=1, head_dim=d, halves=1, norm=1, eps=c.eps, rope_base=c.base)
    ins = [x, None, dev(c.pos[at]), dev(c.gain[0]), None, None, None]
    assert cf.call_op("qk_norm_rope_%s_cuda" % ("f16" if f16 else "f32"), ins, [x, None], p) == 0
    got = x.download()
    x.free()
    want, err = ref_rows(c.x[0].reshape(n, 1, d), c.pos, c.gain[0], None, 1, c.eps, d, 1, frequencies(d, float(F32(c.base))), 1.0)
    tol = err + (2.0 ** -11 * np.abs(want) + 2.0 ** -25 if f16 else 2.0 ** -24 * np.abs(want) + 2.0 ** -140)
    turned = c.pos >= 0
    assert (np.abs(got[:n].reshape(want.shape) - want) <= tol)[turned].all()
    assert (got[:n][~turned] == c.x[0][~turned]).all()
    for i in range(n, T, n):
        assert (got[i:i + n] == got[:min(n, T - i)]).all()
