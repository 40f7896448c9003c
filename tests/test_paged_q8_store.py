"""The 8-bit store where rows that are not stored stand among those of a block, bit by bit against
test_paged_q8.py's oracle (GPU)."""

import numpy as np
import pytest

from test_paged_q8 import Store


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,d,P,block", [(8, 128, 16, 16), (3, 64, 128, 64), (2, 128, 96, 48), (3, 33, 32, 8), (2, 256, 16, 16)])
def test_skipped_rows_inside_a_block(gpu, f16, H, d, P, block):
    """A block's rows with rows of invalid slots between them, NaN and infinite and huge, in order and not."""
    s = Store(f16, H, d, P, block, 24 * 64 // P, seed=71)
    n, none = s.n_pages * P, [-1, -2 ** 31, s.n_pages * P, 2 ** 31 - 1]

    def call(slots):
        k, v = s.rows(len(slots)), s.rows(len(slots), 30.0)
        out = [i for i, x in enumerate(slots) if not 0 <= x < n]
        for x in (k, v):                                 # what is not stored counts for no power
            x[out[0::3]] = np.nan
            x[out[1::3]] = np.inf
            x[out[2::3]] = 60000.0
        s.call(k, v, slots)

    call([5 % block, -1, 7 % block])
    call([block + 1, -1, -1, block, -1, 2 * block - 1, n, 2 * block])
    # A block's first and last row 63 rows apart, with nothing stored between.
    call([3 * block] + [-1] * 62 + [4 * block - 1])
    # Calls of every block, its rows in any order, some left out, at every place in groups of 64 rows; what
    # was stored before goes on.
    for take in (block, max(block // 2, 1), 2):
        slots = []
        for b in s.rng.permutation(n // block):
            own = list(b * block + s.rng.permutation(block)[:take])
            for _ in range(int(s.rng.integers(0, min(65 - len(own), 9)))):
                own.insert(int(s.rng.integers(0, len(own) + 1)), none[int(s.rng.integers(0, 4))])
            slots += own + [-1] * int(s.rng.integers(0, 3)) * 40 * int(b % 5 == 0)
        call(slots)
