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
