"""The paged operators with more sequences and rows than a launch or a plan takes in one piece (GPU).
Sequences of one position, whose attention is that position's V, and rows stored as they are, so
that results are known without a sum."""

import numpy as np
import pytest

import cudaforge_amd as cf
from helpers import dev

I32 = np.int32
BEYOND = 2 ** 23 + 5                # a launch has at most 2^23 workgroups


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("B,H,H_kv,d", [(32768, 4, 1, 64), (32769, 4, 1, 64), (300000, 8, 2, 128), (BEYOND, 1, 1, 64)])
def test_attention_of_very_many_sequences(gpu, f16, B, H, H_kv, d):
    P, n_pages, rng = 16, 50, np.random.default_rng(B)
    dt = np.float16 if f16 else np.float32
    row = rng.standard_normal((1000, H, d)).astype(dt)
    q = row[np.arange(B) % 1000]
    k, v = (rng.standard_normal((n_pages, P, H_kv, d)).astype(dt) for _ in range(2))
    page = rng.integers(-1, n_pages, B).astype(I32)             # -1: a sequence that sees nothing
    lens = np.ones(B, I32)
    p = cf.MhaPagedParams(batch_size=B, num_tokens=B, num_heads=H, num_kv_heads=H_kv, head_dim=d, scale=0.125, page_size=P,
                          num_pages=n_pages, max_pages=1, max_new=1, max_len=1)
    o = cf.DeviceBuffer(q.nbytes, dt, q.shape)
    assert cf.call_op("mha_paged_attn_%s_cuda" % ("f16" if f16 else "f32"),
                      [dev(q), dev(k), dev(v), dev(page.reshape(B, 1)), dev(lens), dev(np.arange(B + 1, dtype=I32))], [o], p) == 0
    got = o.download()
    want = np.concatenate((v[:, 0], np.zeros((1, H_kv, d), dt)))[page]
    want = np.repeat(want, H // H_kv, 1).astype(np.float64)
    # O = (p v) (1 / l) with l = p, whatever p is: three roundings of at most 2^-24, of which fp16's one
    # rounding at the end, of at least 2^-11 v or none, leaves nothing (v is an fp16 number itself).
    assert (np.abs(got - want) <= (0.0 if f16 else 3.01 * 2.0 ** -24) * np.abs(want)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_store_of_very_many_rows(gpu, f16):
    T, P, d, rng = BEYOND, 8, 2, np.random.default_rng(1)
    dt = np.float16 if f16 else np.float32
    n_pages = -(-T // P) + 1
    x = rng.standard_normal((T, 1, d), np.float32).astype(dt)
    slots = rng.permutation(T).astype(I32)
    pages = [dev(np.zeros((n_pages, P, 1, d), dt)) for _ in range(2)]
    p = cf.KvPageStoreParams(num_tokens=T, num_kv_heads=1, head_dim=d, page_size=P, num_pages=n_pages)
    assert cf.call_op("kv_page_store_%s_cuda" % ("f16" if f16 else "f32"), [dev(x), dev(x[::-1]), dev(slots)], pages, p) == 0
    for got, want in zip(pages, (x, x[::-1])):
        got = got.download().reshape(-1, 1, d)
        assert np.array_equal(got[slots], want) and not got[T:].any()


@pytest.mark.gpu
def test_map_of_very_many_sequences(gpu):
    B, P, width, rng = BEYOND, 4, 2, np.random.default_rng(2)
    cached = rng.integers(0, 5, B).astype(I32)
    new = rng.integers(0, 5, B).astype(I32)
    new[rng.random(B) < 0.1] = -1
    fits = new >= 0
    n = np.maximum(new, 0)
    held = (cached + P - 1) // P
    need = np.where(fits, (cached + n + P - 1) // P - held, 0)
    back = np.where(fits, 0, held)
    total, spare = int(need.sum()), 7
    n_pages = int(held.sum()) + total + spare
    pages = rng.permutation(n_pages).astype(I32)
    table = np.full((B, width), -1, I32)
    table[held == 1, 0] = pages[total + spare:]
    ring = np.full(n_pages, -1, I32)
    ring[:total + spare] = pages[:total + spare]
    T = int(n.sum()) + 3
    bufs = [dev(x) for x in (cached, new, np.array([0, total + spare, 0], I32), table, ring)]
    lens, start, pos, slots = (cf.DeviceBuffer(4 * k, I32) for k in (B, B + 1, T, T))
    p = cf.KvPageMapParams(batch_size=B, num_tokens=T, page_size=P, num_pages=n_pages, max_pages=width, ring_size=n_pages)
    assert cf.call_op("kv_page_map_i32_cuda", bufs[:3], [bufs[3], bufs[4], lens, start, pos, slots, bufs[2]], p) == 0
    first = np.cumsum(need) - need
    want_table = table.copy()
    for j in range(2):                                          # need is 0, 1 or 2 pages
        at = np.nonzero(need > j)[0]
        want_table[at, held[at] + j] = pages[first[at] + j]
    want_start = np.concatenate(([0], np.cumsum(n)))
    assert np.array_equal(bufs[3].download(), want_table)
    assert np.array_equal(lens.download(), np.where(fits, cached + n, 0))
    assert np.array_equal(start.download(), want_start)
    b = np.repeat(np.arange(B), n)
    at = cached[b] + np.arange(T - 3) - want_start[b]
    assert np.array_equal(pos.download(), np.concatenate((at, [-1] * 3)))
    assert np.array_equal(slots.download(), np.concatenate((want_table[b, at // P] * P + at % P, [-1] * 3)))
    returned = table[(back == 1), 0]
    assert list(bufs[2].download()) == [total, spare + len(returned), 0]
    assert np.array_equal(bufs[4].download()[total:total + spare + len(returned)], np.concatenate((pages[total:total + spare], returned)))
