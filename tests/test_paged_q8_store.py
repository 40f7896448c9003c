"""The 8-bit store where rows that are not stored stand among those of a block, and on more rows than one launch
takes, bit by bit against test_paged_q8.py's oracle (GPU)."""

import numpy as np
import pytest

import cudaforge_amd as cf
from helpers import dev
from test_paged_q8 import Store, encode, power_for


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


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d,block", [(2, 1), (16, 1), (16, 4)])
def test_more_rows_than_a_launch_takes(gpu, f16, d, block):
    """2^23 rows are a launch's.  Blocks of rows that repeat after 997 go to slots in another order: every code
    and every power, and nothing behind the last."""
    n, t = 2 ** 23 // block + 5, "f16" if f16 else "f32"
    rng = np.random.default_rng(73)
    base = (rng.standard_normal((997, block, d)) * np.exp2(rng.integers(-9, 9, (997, block, 1)))).astype(np.float16 if f16 else np.float32)
    power = power_for(np.abs(base.astype(np.float64)).max((1, 2)))
    code = encode(base.astype(np.float64) * 2.0 ** (127.0 - power)[:, None, None])
    at, to = np.arange(n) % 997, rng.permutation(n)
    slots = (to[:, None] * block + np.arange(block)).astype(np.int32)
    ins = [dev(base[at]), dev(base[::-1][at]), dev(slots)]
    pages = [dev(np.full((n + 3, block, 1, d), 0x55, np.uint8)) for _ in range(2)]
    powers = [dev(np.full((n + 3, 1, 1), 9, np.uint8)) for _ in range(2)]
    p = cf.KvPageStoreQ8Params(num_tokens=n * block, num_kv_heads=1, head_dim=d, page_size=block, num_pages=n + 3, block_size=block)
    assert cf.call_op("kv_page_store_q8_%s_cuda" % t, ins, pages + powers, p) == 0
    for x, y, c, e in zip(pages, powers, (code, code[::-1]), (power, power[::-1])):
        x, y = x.download().reshape(n + 3, block, d), y.download().reshape(-1)
        assert (y[to] == e[at]).all() and (y[n:] == 9).all()
        assert (x[to] == c[at]).all() and (x[n:] == 0x55).all()
