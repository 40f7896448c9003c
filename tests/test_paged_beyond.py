"""Attention over paged caches with more sequences than half of 31 bits count: the plain kernels find a
row's sequence among all of them (GPU).  The middle of two such numbers is past 31 bits where it is taken
as half of their sum."""

import numpy as np
import pytest

import cudaforge_amd as cf
from helpers import dev


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
def test_a_row_behind_2_to_the_30_sequences(gpu, q8):
    """All sequences but the last four are empty; theirs are rows 0 .. 3, over one position each, whose V is
    the result."""
    B, H, d, P, n_pages = (1 << 30) + 10, 2, 8, 16, 8
    rng = np.random.default_rng(2)
    rows = 4
    start, lens, table = (cf.DeviceBuffer(4 * n) for n in (B + 1, B, B))      # 4.3 GB each
    for x in (start, lens, table):
        x.fill_zero()

    def put(buf, at, values):
        v = np.ascontiguousarray(values, np.int32)
        assert gpu.gpu_memcpy_h2d(buf.ptr + 4 * at, v.ctypes.data, v.nbytes, None) == 0
        assert gpu.gpu_stream_synchronize(None) == 0

    page = np.array([3, 0, 7, 5])
    put(start, B - rows, np.arange(rows + 1))
    put(lens, B - rows, np.ones(rows))
    put(table, B - rows, page)
    q = dev(rng.standard_normal((rows, H, d)).astype(np.float16))
    o = cf.DeviceBuffer(2 * rows * H * d, np.float16, (rows, H, d))
    common = dict(batch_size=B, num_tokens=rows, num_heads=H, num_kv_heads=H, head_dim=d, scale=0.5, page_size=P,
                  num_pages=n_pages, max_pages=1)
    if q8:
        codes = [rng.integers(0, 100, (n_pages, P, H, d)).astype(np.uint8) for _ in range(2)]
        powers = [dev(np.full((n_pages, 1, H), 127, np.uint8)) for _ in range(2)]
        c = codes[1][page, 0].astype(int)
        want = np.where(c > 7, (8 + c % 8) * 2.0 ** (c // 8 - 10.0), c * 2.0 ** -9)
        ins = [q, dev(codes[0]), dev(codes[1]), table, lens, start] + powers
        assert cf.call_op("mha_paged_attn_q8_f16_cuda", ins, [o], cf.MhaPagedQ8Params(**common)) == 0
    else:
        kv = [rng.standard_normal((n_pages, P, H, d)).astype(np.float16) for _ in range(2)]
        want = kv[1][page, 0].astype(np.float64)
        ins = [q, dev(kv[0]), dev(kv[1]), table, lens, start]
        assert cf.call_op("mha_paged_attn_f16_cuda", ins, [o], cf.MhaPagedParams(**common)) == 0
    got = o.download()
    for x in (start, lens, table):
        x.free()
    # p = 1 and l = 1: the value itself.
    assert (got == want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("q8", [False, True])
def test_more_rows_than_a_round_takes(gpu, q8):
    """2^24 rows of a head are a round of the plain kernels' workgroups; each of these is a sequence of one
    position."""
    T, H, d, P, n_pages = 2 ** 22 + 3, 4, 4, 16, 1000
    rng = np.random.default_rng(3)
    page = (np.arange(T) * 7 % n_pages).astype(np.int32)
    q = dev(np.ones((T, H, d), np.float16))
    o = cf.DeviceBuffer(2 * T * H * d, np.float16, (T, H, d))
    index = [dev(page.reshape(T, 1)), dev(np.ones(T, np.int32)), dev(np.arange(T + 1, dtype=np.int32))]
    common = dict(batch_size=T, num_tokens=T, num_heads=H, num_kv_heads=2, head_dim=d, scale=0.5, page_size=P,
                  num_pages=n_pages, max_pages=1)
    if q8:
        c = rng.integers(0, 100, (n_pages, P, 2, d))
        v = np.where(c > 7, (8 + c % 8) * 2.0 ** (c // 8 - 10.0), c * 2.0 ** -9)
        codes, powers = dev(c.astype(np.uint8)), dev(np.full((n_pages, 1, 2), 127, np.uint8))
        assert cf.call_op("mha_paged_attn_q8_f16_cuda", [q, codes, codes] + index + [powers, powers], [o],
                          cf.MhaPagedQ8Params(**common)) == 0
    else:
        v = rng.standard_normal((n_pages, P, 2, d)).astype(np.float16)
        kv = dev(v)
        assert cf.call_op("mha_paged_attn_f16_cuda", [q, kv, kv] + index, [o], cf.MhaPagedParams(**common)) == 0
    want = np.repeat(v[:, 0], 2, 1).astype(np.float16)
    assert (o.download() == want[page]).all()
