"""Attention over the 8-bit paged cache where V are NaN or past the range of the type that the matrix cores
take, with the oracle and the tolerances of test_paged_q8.py (GPU)."""

import numpy as np
import pytest

from test_paged import ref_attn
from test_paged_q8 import PagedQ8


def allowed(c):
    """The oracle's result and what a call may be off by."""
    want, e32, e16 = ref_attn(c.q, c.kp, c.vp, c.table, c.lens, c.start, c.scale)
    return want, e16 + 2.0 ** -11 * np.abs(want) + 2.0 ** -25 if c.f16 else e32 + 2.0 ** -24 * np.abs(want)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,n,past", [(4, 2, 64, 3, 62), (8, 2, 128, 3, 2046), (4, 2, 64, 40, 30), (8, 2, 128, 40, 2010),
                                             (4, 2, 24, 3, 62)])
@pytest.mark.parametrize("nan", [False, True])
def test_hidden_v_past_the_types_range(gpu, f16, H, H_kv, d, n, past, nan):
    """The last token's block of V is past the largest number of the products' type in one head, and a NaN
    stands among the cached V: rows before that block have NaN where that one is, and nothing else of
    either."""
    c = PagedQ8([n], [past], H, H_kv, d, 16, f16, seed=61)
    last = past + n - 1
    c.powers[1][c.table[0, last // 16], 0, 1] = 150 if f16 else 253
    if nan:
        c.codes[1][c.table[0, 1], 5, :, 3] = 0x7f
    c.refresh()
    first = last // 16 * 16 - past                       # the block's first new token
    assert 0 < first < n
    with np.errstate(invalid="ignore", over="ignore"):
        want, tol = allowed(c)
    want, tol = want[:first], tol[:first]
    for hint in (0, 1):                                  # the positions shared out, and in one range
        got = c.run(max_new=n, max_len=hint)[:first].astype(np.float64)
        assert (np.isnan(got) == np.isnan(want)).all()
        assert np.isnan(want[:, :, 3]).all() == nan and not np.isnan(np.delete(want, 3, 2)).any()
        assert (np.isnan(want) | (np.abs(got - want) <= tol)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,n,past", [(4, 2, 24, 1, 200), (5, 5, 33, 12, 300), (4, 2, 64, 1, 200), (8, 2, 128, 12, 2000),
                                             (4, 2, 64, 90, 700)])
@pytest.mark.parametrize("hidden", [False, True])
def test_a_seen_nan_counts_whatever_it_weighs(gpu, f16, H, H_kv, d, n, past, hidden):
    """One position scores 200 above all others, whose weights are 0 in FP32: a NaN V among them is NaN in the
    rows that see it on every path, also where a later token's NaN makes rows be computed again."""
    c = PagedQ8([n], [past], H, H_kv, d, 16, f16, seed=63, pad=0)
    c.q[:] = 1
    c.codes[0][:] = 0
    c.powers[0][:] = 127
    c.codes[0][c.table[0, 0], 0] = 0x38                  # 1
    c.powers[0][c.table[0, 0]] = 127 + 3                 # 8: a score of scale * 8 d
    c.scale = float(np.float32(200.0 / (8 * d)))
    at = lambda pos: (c.table[0, pos // 16], pos % 16)
    c.codes[1][at(past // 2)][:, 3] = 0x7f
    if hidden:
        c.codes[1][at(past + n - 1)][:, 5] = 0xff
    c.refresh()
    nan = np.zeros(c.q.shape, bool)
    nan[:, :, 3] = True
    nan[n - 1, :, 5] = hidden
    want = np.repeat(c.vp[c.table[0, 0], 0], H // H_kv, 0)[None]
    for hint in (0, 1):
        got = c.run(max_new=n, max_len=hint).astype(np.float64)
        assert (np.isnan(got) == nan).all()
        # The first position's V: p = 1 and l = 1, or all of it at one scale; six roundings at most.
        assert (nan | (np.abs(got - want) <= (2.0 ** -11 + 2.0 ** -24 if f16 else 6.01 * 2.0 ** -24) * np.abs(want))).all()
