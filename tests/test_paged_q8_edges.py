"""The 8-bit paged cache at the edges of what its arrays may hold, with the oracle and the tolerances of
test_paged_q8.py (GPU)."""

import ctypes
from ctypes import c_void_p

import numpy as np
import pytest

import cudaforge_amd as cf
from helpers import dev
from test_paged import I32, ref_attn
from test_paged_q8 import U8, VALUE, PagedQ8, Store, quantise, same_codes, values

SHAPES = [(8, 2, 64, 16, 16), (8, 2, 128, 32, 32), (16, 1, 64, 64, 16), (5, 5, 33, 14, 7)]     # the last: the plain kernel


def fill(c, seed=99):
    """Finite codes and ordinary powers where PagedQ8 leaves NaN."""
    rng = np.random.default_rng(seed)
    for codes, powers in zip(c.codes, c.powers):
        free = codes & 127 == 127
        codes[free] = rng.integers(0, 100, int(free.sum())).astype(U8)
        odd = (powers > 140) | (powers < 100)
        powers[odd] = rng.integers(110, 124, int(odd.sum())).astype(U8)
    c.refresh()


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,P,block", SHAPES)
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 2], [40, 1, 33]])
def test_lengths_past_the_table(gpu, f16, H, H_kv, d, P, block, new):
    """A length past its table's row is the row's: its rows are the last positions of it."""
    c = PagedQ8(new, [90, 300, 20], H, H_kv, d, P, f16, block=block, seed=23)
    fill(c)
    rng = np.random.default_rng(5)
    held = c.table >= 0
    c.table[~held] = rng.integers(0, c.n_pages, int((~held).sum()))           # pages of others: shared
    full = c.width * P
    for past in (full + 1, 2 ** 31 - 1):
        c.lens[:] = [past, full, min(past, full + 7)]
        c.check(c.run(max_new=max(new)))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,P,block", SHAPES)
@pytest.mark.parametrize("wide", [False, True])
def test_offsets_past_the_rows(gpu, f16, H, H_kv, d, P, block, wide):
    """Offsets below 0 and behind the last row are clamped: a sequence has the rows between."""
    c = PagedQ8([4, 40 if wide else 4, 3, 2], [90, 150, 60, 33], H, H_kv, d, P, f16, block=block, seed=25, pad=0)
    fill(c)
    for start in ([-4, 4, c.T - 5, 10 ** 6, 2 ** 31 - 1], [-2 ** 31, -7, 5, c.T, c.T + 9], [0, 0, c.T, c.T, c.T],
                  [3, 4, 6, 6, c.T - 2]):
        c.start = np.array(start, I32)
        c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,P,block", SHAPES)
def test_hints_that_are_wrong(gpu, f16, H, H_kv, d, P, block):
    """max_new and max_len choose kernels; what they say need not hold."""
    c = PagedQ8([50, 1, 7], [900, 2500, 3], H, H_kv, d, P, f16, block=block, seed=7)
    for new in (0, 1, 60):
        for length in (0, 1, 700, 5000):
            c.check(c.run(max_new=new, max_len=length))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d", [64, 128, 24])
@pytest.mark.parametrize("scale", [0.0, -0.1, 3.0, 1e-3])
def test_scales(gpu, f16, d, scale):
    for n in (1, 30):
        c = PagedQ8([n, n], [100, 10], 4, 2, d, 16, f16, seed=9, scale=scale)
        c.check(c.run(max_new=n))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,P,block", SHAPES)
@pytest.mark.parametrize("n", [1, 9, 100])
@pytest.mark.parametrize("far", [9.0, 14.0, 17.6, 20.0])
def test_many_small_weights_beside_a_large_one(gpu, f16, H, H_kv, d, P, block, n, far):
    """One position scores `far` above some ten thousand equal ones: each of them weighs e^-far of it,
    all together as much as the tolerance many times."""
    c = PagedQ8([n], [12000 - n], H, H_kv, d, P, f16, block=block, seed=31, pad=0)
    rng = np.random.default_rng(3)
    c.q[:] = 1
    k, v = np.zeros(c.kp.shape), 1 + rng.random(c.vp.shape) / 4
    k[c.table[0, 0], 0] = far / (c.scale * d)
    v[c.table[0, 0], 0] = 0
    (c.codes[0], c.powers[0]), (c.codes[1], c.powers[1]) = (quantise(x, block) for x in (k, v))
    c.refresh()
    for hint in (0, 1):                                  # the positions shared out, and in one range
        c.check(c.run(max_new=n, max_len=hint))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,P,new,past", [
    (8, 2, 64, 16, [12, 2, 8], [100, 30, 7]), (32, 8, 128, 16, [1] * 5, [4000, 300, 90, 2222, 17]), (12, 12, 64, 32, [1, 1], [700, 333]),
    (8, 4, 128, 32, [150, 40, 90, 1], [33, 9, 200, 600]), (4, 4, 64, 16, [130, 2], [4000, 3000]), (16, 4, 128, 16, [400], [64])])
def test_nan_v_among_the_cached(gpu, f16, H, H_kv, d, P, new, past):
    """NaN codes of cached positions, which every row sees, in dims of their own, and of a new one that only
    rows from it on see; a cached block of power 255 in one head of one sequence."""
    c = PagedQ8(new, past, H, H_kv, d, P, f16, seed=33)
    clean = [x.copy() for x in c.codes + c.powers]
    at = lambda b, pos: (c.table[b, pos // P], pos % P)
    want = np.zeros(c.q.shape, bool)
    for b, (n, p) in enumerate(zip(new, past)):
        r = np.arange(c.start[b], c.start[b + 1])
        for dim, pos in ((3, p // 2), (d - 1, p - 1)):
            c.codes[1][at(b, pos)][:, dim] = 0x7f
            want[r, :, dim] = True
        h = n // 2
        c.codes[1][at(b, p + h)][:, 11] = 0xff
        want[r[h:], :, 11] = True
    G = H // H_kv
    page, row = at(0, past[0] // 3)
    c.powers[1][page, row // 16, H_kv - 1] = 255
    want[c.start[0]:c.start[1], (H_kv - 1) * G:] = True
    dirty = c.codes + c.powers
    for hint in (0, 1):
        c.codes, c.powers = dirty[:2], dirty[2:]
        got = c.run(max_new=max(new), max_len=hint)
        assert (np.isnan(got) == want).all()
        c.codes, c.powers = clean[:2], clean[2:]
        c.refresh()
        plain = c.run(max_new=max(new), max_len=hint)
        got[want] = plain[want]
        c.check(got)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("n", [1, 12, 150])
@pytest.mark.parametrize("d", [64, 128, 20])
def test_nan_keys(gpu, f16, n, d):
    """A block of K of power 255: every element of the rows that see it is NaN, and no other."""
    c = PagedQ8([n, n], [64, 64], 4, 2, d, 16, f16, seed=34)
    c.powers[0][c.table[0, 2], 0, 1] = 255
    new_block = (64 + n - 1) // 16                       # of the last new token
    c.powers[0][c.table[1, new_block], 0, 0] = 255
    c.refresh()
    got = c.run(max_new=n)
    nan = np.zeros(c.q.shape, bool)
    nan[:n, 2:] = True
    first = max(new_block * 16 - 64, 0)                  # the block's first new token
    nan[n + first:2 * n, :2] = True
    assert (np.isnan(got) == nan).all()


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new,past", [([1, 1, 1], [5000, 40, 1700]), ([70, 1, 30], [3000, 900, 10])])
def test_without_memory_for_a_workspace(gpu, f16, new, past):
    """No buffer to be had, or a recording on a stream that has none: the tiles are not cut, and the call
    succeeds.  What the stream had before is used again afterwards."""
    c = PagedQ8(new, past, 8, 2, 128, 16, f16, seed=35)
    bufs = c.bufs()
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
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new,past", [([1, 1, 1, 1], [3000, 40, 1700, 900]), ([130, 1, 60], [1500, 700, 10])])
def test_a_recording_at_other_lengths(gpu, f16, new, past):
    """One recording, replayed with shorter and longer contexts and other tables, beside eager calls of the
    same stream; the same call twice gives the same bits."""
    c = PagedQ8(new, past, 8, 2, 128, 16, f16, seed=36)
    st = cf.Stream()
    bufs, o = c.bufs(), dev(np.full(c.q.shape, 7.0, c.dt))
    call = lambda: cf.call_op(c.op, bufs, [o], c.params(max_new=max(new)), st)
    assert call() == 0                                   # sizes the workspace
    st.synchronize()
    ex = c_void_p()
    assert gpu.gpu_capture_begin(st.handle) == 0
    rc = call()
    assert gpu.gpu_capture_end(st.handle, ctypes.byref(ex)) == 0 and rc == 0
    full = c.lens.copy()
    for i, drop in enumerate((0, 600, 39, 2, 0)):
        c.lens = np.maximum(full - drop, new).astype(I32)
        bufs[4].upload(c.lens)
        assert gpu.gpu_graph_launch(ex, st.handle) == 0
        st.synchronize()
        got = o.download()
        c.check(got)
        assert call() == 0
        st.synchronize()
        assert (o.download().view(np.uint8) == got.view(np.uint8)).all()
    gpu.gpu_graph_exec_destroy(ex)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_pages_beyond_32_bits(gpu, f16):
    """Pages 2^30 bytes apart, the last of them 5 to 6 GB into the buffers: stored there, attended from
    there, by the matrix cores and by the plain kernel (a stride off the 16-byte grid)."""
    H, H_kv, d, P, n_pages = 8, 2, 64, 16, 6
    t = "f16" if f16 else "f32"
    c = PagedQ8([1, 20], [30, 10], H, H_kv, d, P, f16, seed=19, pad=0, spare=0)
    assert c.n_pages <= n_pages - 1
    at = np.concatenate([c.table[b, np.arange(c.lens[b]) // P] * P + np.arange(c.lens[b]) % P for b in range(2)])
    k, v = (x.reshape(-1, H_kv, d)[at].astype(c.dt) for x in (c.kp, c.vp))
    for extra in (0, 1):
        step = (1 << 30) + extra
        caches = [cf.DeviceBuffer(n_pages * step) for _ in range(2)]
        powers = [dev(np.zeros((n_pages, 1, H_kv), U8)) for _ in range(2)]
        far = [5, 4, 3, 2][:c.n_pages]                   # pages from the far end
        table = np.where(c.table >= 0, np.take(np.array(far + [0], I32), np.maximum(c.table, 0)), -1).astype(I32)
        slots = np.concatenate([[table[b, j // P] * P + j % P for j in range(c.lens[b])] for b in range(2)]).astype(I32)
        p = cf.KvPageStoreQ8Params(num_tokens=len(slots), num_kv_heads=H_kv, head_dim=d, page_size=P, num_pages=n_pages,
                                   page_stride=step)
        assert cf.call_op("kv_page_store_q8_%s_cuda" % t, [dev(k), dev(v), dev(slots)], caches + powers, p) == 0
        # The values were codes before: they are stored as they are, at the same or another power.
        p = cf.MhaPagedQ8Params(batch_size=2, num_tokens=c.T, num_heads=H, num_kv_heads=H_kv, head_dim=d, scale=c.scale,
                                page_size=P, num_pages=n_pages, max_pages=c.width, page_stride=step)
        o = dev(np.full(c.q.shape, 7.0, c.dt))
        assert cf.call_op(c.op, [dev(c.q)] + caches + [dev(table), dev(c.lens), dev(c.start)] + powers, [o], p) == 0
        c.check(o.download())
        for x in caches:
            x.free()


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("B,H,H_kv,d", [(32768, 4, 1, 64), (32769, 4, 1, 64), (70, 12, 12, 64), (200, 8, 2, 128)])
def test_many_sequences(gpu, f16, B, H, H_kv, d):
    """Sequences of one position, whose attention is that position's V, up to more than the tiles take."""
    P, n_pages, rng = 16, 50, np.random.default_rng(B)
    dt = np.float16 if f16 else np.float32
    q = rng.standard_normal((1000, H, d)).astype(dt)[np.arange(B) % 1000]
    (k, kp), (v, vp) = (quantise(rng.standard_normal((n_pages, P, H_kv, d)), 16) for _ in range(2))
    page = rng.integers(-1, n_pages, B).astype(I32)             # -1: a sequence that sees nothing
    p = cf.MhaPagedQ8Params(batch_size=B, num_tokens=B, num_heads=H, num_kv_heads=H_kv, head_dim=d, scale=0.125, page_size=P,
                            num_pages=n_pages, max_pages=1, max_new=1, max_len=1)
    o = cf.DeviceBuffer(q.nbytes, dt, q.shape)
    ins = [dev(x) for x in (q, k, v, page.reshape(B, 1), np.ones(B, I32), np.arange(B + 1, dtype=I32), kp, vp)]
    assert cf.call_op("mha_paged_attn_q8_%s_cuda" % ("f16" if f16 else "f32"), ins, [o], p) == 0
    want = np.concatenate((values(v, vp)[:, 0], np.zeros((1, H_kv, d))))[page]
    want = np.repeat(want, H // H_kv, 1)
    # O = (p v) (1 / l) with l = p: the parts of p are p exactly, three sums of parts of p v and two roundings.
    tol = 2.0 ** -11 + 2.0 ** -24 if f16 else 6.01 * 2.0 ** -24
    assert (np.abs(o.download() - want) <= tol * np.abs(want)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_many_uneven_sequences(gpu, f16):
    """More sequences than a wave has lanes, short and long ones, chunks among them."""
    rng = np.random.default_rng(8)
    for new in ([1] * 90, [1 if i % 17 else 40 for i in range(90)]):
        past = [int(x) for x in rng.integers(0, 90, 90)]
        past[3], past[77] = 2300, 1500
        c = PagedQ8(new, past, 4, 2, 64, 16, f16, seed=41)
        c.check(c.run(max_new=max(new)))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv", [(32, 32), (16, 2)])
@pytest.mark.parametrize("B", [7, 64])
def test_more_units_than_go_in_one_round(gpu, f16, H, H_kv, B):
    """Up to 64 sequences of every kind, whose ranges the tiles take by their length: chunks of one tile and of
    several, single rows, empty ones, equal lengths."""
    new = [300, 1, 40, 0, 129, 1, 257] + [1, 1, 20, 0, 1, 33, 1] * 8 + [64]
    past = [500, 900, 0, 300, 1500, 0, 2] + [200, 63, 64, 5, 200, 31, 700] * 8 + [0]
    c = PagedQ8(new[:B], past[:B], H, H_kv, 64, 32, f16, seed=43)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_store_again_changes_nothing(gpu, f16):
    """The same rows to the same slots once more: a power that has grown stays, and so do all bits."""
    s = Store(f16, 4, 64, 32, 16, 20, seed=21)
    k, v = s.rows(70), s.rows(70, 30.0)
    slots = np.arange(70) + 5
    for _ in range(2):
        s.call(k, v, slots)
    before = [b.download().copy() for b in s.bufs]
    s.call(k, v, slots)
    assert all((a == b.download()).all() for a, b in zip(before, s.bufs))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d", [64, 24])
def test_store_powers_that_are_not_ordinary(gpu, f16, d):
    """Blocks whose power is 0, 254 or 255 are gone on with: 255 stays, 254 leaves only zeros and the type's
    largest values, 0 grows."""
    s = Store(f16, 2, d, 16, 16, 3, seed=22)
    for i, p in enumerate((0, 254, 255)):
        for x in s.powers:
            x[i] = p
        for c in s.cells:
            c[16 * i:16 * i + 16] &= 0x77
    for buf, x in zip(s.bufs, s.raw + s.powers):
        pass
    for raw, c in zip(s.raw, s.cells):
        raw[s.index()] = c
    for buf, x in zip(s.bufs, s.raw + s.powers):
        buf.upload(x)
    s.call(s.rows(6), s.rows(6, 100.0), [3, 4, 19, 20, 35, 36])
    for p in s.powers:
        assert (p[1] == 254).all() and (p[2] == 255).all() and (p[0] > 100).all()


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_store_of_very_many_rows(gpu, f16):
    """More rows than 2^23 workgroups of one launch would take one by one; a block per row."""
    T, P, d = 2 ** 23 + 5, 8, 2
    dt = np.float16 if f16 else np.float32
    n_pages = -(-T // P) + 1
    rng = np.random.default_rng(1)
    x = VALUE[rng.integers(1, 0x7e, T * d)].astype(dt).reshape(T, 1, d)
    slots = rng.permutation(T).astype(I32)
    pages = [dev(np.zeros((n_pages, P, 1, d), U8)) for _ in range(2)]
    powers = [dev(np.zeros((n_pages, P, 1), U8)) for _ in range(2)]
    p = cf.KvPageStoreQ8Params(num_tokens=T, num_kv_heads=1, head_dim=d, page_size=P, num_pages=n_pages, block_size=1)
    assert cf.call_op("kv_page_store_q8_%s_cuda" % ("f16" if f16 else "f32"), [dev(x), dev(x[::-1]), dev(slots)], pages + powers, p) == 0
    for codes, power, want in zip(pages, powers, (x, x[::-1])):
        codes, power = codes.download().reshape(-1, d), power.download().reshape(-1)
        got = VALUE[codes[slots]] * 2.0 ** (power[slots, None] - 127.0)
        # Rows of one block whose smaller value leaves the normal range of the larger one's power are rounded.
        off = np.abs(got - want[:, 0])
        assert (off <= 2.0 ** (power[slots, None] - 127.0 - 10)).all() and not codes[T:].any()
    assert same_codes(codes, codes)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("n", [3, 40])
def test_v_beyond_fp16_stays_where_it_is_seen(gpu, f16, n):
    """A new token whose V is past fp16's largest: rows before it are not touched."""
    c = PagedQ8([n], [50], 4, 2, 64, 16, f16, seed=43)
    slot = int(c.table[0, (50 + n - 1) // 16]) * 16 + (50 + n - 1) % 16
    c.powers[1].reshape(-1, 2)[slot // 16] = 150         # the last token's block
    c.refresh()
    got = c.run(max_new=n)
    want, e32, e16 = ref_attn(c.q, c.kp, c.vp, c.table, c.lens, c.start, c.scale)
    first = (50 + n - 1) // 16 * 16 - 50                 # the block's first new token
    before = np.arange(max(first, 0))
    tol = e16 + 2.0 ** -11 * np.abs(want) + 2.0 ** -25 if f16 else e32 + 2.0 ** -24 * np.abs(want)
    assert (np.abs(got[before] - want[before]) <= tol[before]).all()
    if not f16:
        c.check(got)
