"""The paged KV cache: kv_page_map_i32_cuda, kv_page_store_{f16,f32}_cuda and
mha_paged_attn_{f16,f32}_cuda against plain implementations in 64 bits (GPU), what they
refuse (CPU), and a run of the three together.

Tolerances.  A value is rounded to its type once, by at most eps/2 = 2^-11 (fp16) or 2^-24
(fp32) of itself.  In attention, with A = sum p |v| / sum p and r = sqrt(sum p^2 v^2) / sum p:
  - FP32 sums over n positions and d dims: roundings of at most 2^-24 of a partial sum, as
    likely up as down.  4 sqrt(n) 2^-24 A is about 7 standard deviations of n of them; a score
    is off by 2 sqrt(d) 2^-24 of the sum of its terms' sizes (s), which moves p by as much
    relative to itself; 16 more for the exponential, the scale and the division.
  - fp16 holds p for the products with V: off by a share of at most 2^-11 each, uniform, so
    the sum is off by 2^-11 r / sqrt(3) in the standard deviation; 4 2^-11 r is 7 of them.
    Below 2^-14 p is a multiple of 2^-24 instead.
"""

import ctypes
import math
from ctypes import c_void_p

import numpy as np
import pytest

import cudaforge_amd as cf
from helpers import dev

I32 = np.int32


# ------------------------------------------------------------------ the operators, in 64 bits ---

def ref_map(cached, new, table, ring, head, avail, T, P, num_pages):
    """kv_page_map_i32_cuda request by request (include/paged_ops.h)."""
    table, ring, old = table.copy(), ring.copy(), ring.copy()
    R, width = len(ring), table.shape[1]
    ceil = lambda x: -(-x // P)
    page = lambda x: int(x) if 0 <= x < num_pages else -1
    seq_lens, start, pos, slots = [], [0], [], []
    asked = taken = back = refused = 0
    for b, (c, n) in enumerate(zip(cached, new)):
        c, n = min(max(int(c), 0), width * P), int(n)
        have = ceil(c)
        if n < 0:
            for j in range(have):
                ring[(head + avail + back + j) % R] = table[b, j]
            back += have
            seq_lens.append(0)
            start.append(start[-1])
            continue
        fits = c + n <= width * P
        need = ceil(c + n) - have if fits else 0
        ok = fits and (need == 0 or asked + need <= avail)
        for j in range(need if fits else width - have):
            table[b, have + j] = page(old[(head + asked + j) % R]) if ok else -1
        asked += need
        taken += need if ok else 0
        refused += not ok
        for i in range(c, c + n):
            pg = page(table[b, i // P]) if ok else -1
            pos.append(i)
            slots.append(pg * P + i % P if pg >= 0 else -1)
        seq_lens.append(c + n)
        start.append(start[-1] + n)
    pad = T - len(pos)
    pos, slots = (np.array((x + [-1] * max(pad, 0))[:T], I32) for x in (pos, slots))
    return dict(table=table, ring=ring, seq_lens=np.array(seq_lens, I32), q_start=np.array(start, I32), positions=pos,
                slots=slots, counters=np.array([(head + taken) % R, min(avail - taken + back, R), refused], I32))


def ref_turn(x, pos, base):
    """Pairs (2i, 2i + 1) of x (T, H, d) turned by pos * base^(-2i / d), in 64 bits."""
    d = x.shape[-1]
    a = pos.astype(np.float64)[:, None] * float(np.float32(base)) ** (-2.0 * np.arange(d // 2) / d)
    z = (x[..., 0::2] + 1j * x[..., 1::2]) * np.exp(1j * a)[:, None, :]
    y = np.empty(x.shape)
    y[..., 0::2], y[..., 1::2] = z.real, z.imag
    return y


def ref_attn(q, kp, vp, table, lens, start, scale):
    """mha_paged_attn on dense (pages, P, H_kv, d) arrays: O and what it may be off by in FP32
    and fp16 arithmetic (both without the rounding of the result); rows outside are NaN."""
    T, H, d = q.shape
    n_pages, P, H_kv, _ = kp.shape
    out, e32, e16 = (np.full(q.shape, np.nan) for _ in range(3))
    u = 2.0 ** -24
    for b in range(len(lens)):
        r0, r1 = (min(max(int(x), 0), T) for x in start[b:b + 2])
        n, L = r1 - r0, min(max(int(lens[b]), 0), table.shape[1] * P)
        if n <= 0:
            continue
        j = np.arange(L)
        pg = table[b, j // P] if L else np.zeros(0, int)
        ok = (pg >= 0) & (pg < n_pages)
        j, at = j[ok], pg[ok].astype(np.int64) * P + (j % P)[ok]
        seen = j[None, :] <= (L - n + np.arange(n))[:, None]
        for h in range(H):
            k = kp.reshape(-1, H_kv, d)[at, h // (H // H_kv)].astype(np.float64)
            v = vp.reshape(-1, H_kv, d)[at, h // (H // H_kv)].astype(np.float64)
            qh = q[r0:r1, h].astype(np.float64)
            s = np.where(seen, qh @ k.T * scale, -np.inf)
            m = np.maximum(s.max(1, initial=-1e300, keepdims=True), -1e300)
            p = np.exp(s - m)
            tot = p.sum(1, keepdims=True)
            some = tot[:, 0] > 0
            p = np.divide(p, tot, out=np.zeros_like(p), where=tot > 0)
            o = p @ v
            A = p @ np.abs(v)
            size = np.where(seen, np.abs(qh) @ np.abs(k).T * abs(scale), 0.0).max(1, initial=0.0)[:, None]
            nn = math.sqrt(max(len(j), 1))
            off = A * u * (4 * nn + 2 * math.sqrt(d) * size + 16)
            low = 4 * nn * 2.0 ** -25 * np.abs(v).max(0, initial=0.0)[None, :]
            out[r0:r1, h] = np.where(some[:, None], o, 0.0)
            e32[r0:r1, h] = off
            e16[r0:r1, h] = off + 4 * 2.0 ** -11 * np.sqrt((p * p) @ (v * v)) + low
    return out, e32, e16


# ------------------------------------------------------------------ building a case ---

class Paged:
    """Sequences of `past` + `new` positions on pages handed out at random.  Every position no
    sequence holds is NaN in both caches."""

    def __init__(self, new, past, H, H_kv, d, P, f16, seed=1, pad=3, spare=3, scale=None, width=None, k_std=1.0):
        rng = np.random.default_rng(seed)
        dt = np.float16 if f16 else np.float32
        self.new, self.past = new, past
        self.H, self.H_kv, self.d, self.P, self.f16, self.dt = H, H_kv, d, P, f16, dt
        self.B = len(new)
        self.lens = np.array([n + c for n, c in zip(new, past)], I32)
        self.start = np.concatenate(([0], np.cumsum(new))).astype(I32)
        self.T = int(self.start[-1]) + pad
        held = [-(-int(x) // P) for x in self.lens]
        self.n_pages = sum(held) + spare
        self.width = width or max(max(held), 1)
        pages = rng.permutation(self.n_pages)
        self.table = np.full((self.B, self.width), -1, I32)
        self.kp = np.full((self.n_pages, P, H_kv, d), np.nan, dt)
        self.vp = np.full((self.n_pages, P, H_kv, d), np.nan, dt)
        at = 0
        for b, h in enumerate(held):
            self.table[b, :h] = pages[at:at + h]
            at += h
            for j in range(h):
                rows = min(P, int(self.lens[b]) - j * P)
                pg = self.table[b, j]
                self.kp[pg, :rows] = (rng.standard_normal((rows, H_kv, d)) * k_std).astype(dt)
                self.vp[pg, :rows] = rng.standard_normal((rows, H_kv, d)).astype(dt)
        self.q = rng.standard_normal((self.T, H, d)).astype(dt)
        self.scale = float(np.float32(1.0 / math.sqrt(d) if scale is None else scale))

    def params(self, **kw):
        return cf.MhaPagedParams(batch_size=self.B, num_tokens=self.T, num_heads=self.H, num_kv_heads=self.H_kv,
                                 head_dim=self.d, scale=self.scale, page_size=self.P, num_pages=self.n_pages,
                                 max_pages=self.width, **kw)

    @property
    def op(self):
        return "mha_paged_attn_f16_cuda" if self.f16 else "mha_paged_attn_f32_cuda"

    def run(self, bufs=None, stream=None, **kw):
        bufs = bufs or [dev(x) for x in (self.q, self.kp, self.vp, self.table, self.lens, self.start)]
        o = dev(np.full(self.q.shape, 7.0, self.dt))
        assert cf.call_op(self.op, bufs, [o], self.params(**kw), stream) == 0
        if stream is not None:
            stream.synchronize()
        return o.download()

    def check(self, got):
        want, e32, e16 = ref_attn(self.q, self.kp, self.vp, self.table, self.lens, self.start, self.scale)
        outside = np.isnan(want).all((1, 2))
        assert (got[outside] == 7.0).all(), "rows of no sequence were written"
        got = got.astype(np.float64)
        tol = e16 + 2.0 ** -11 * np.abs(want) + 2.0 ** -25 if self.f16 else e32 + 2.0 ** -24 * np.abs(want)
        bad = ~(np.abs(got - want) <= tol) & ~outside[:, None, None]
        assert not bad.any(), "%d values off, first at %s: %s for %s, allowed %s" % (
            bad.sum(), np.argwhere(bad)[0], got[bad][0], want[bad][0], tol[bad][0])


# ------------------------------------------------------------------ refusals (CPU) ---

DUMMY = ctypes.create_string_buffer(256)
DP = ctypes.addressof(DUMMY)


def _call(native, name, ins, outs, params):
    a, b = (c_void_p * max(len(ins), 1))(*ins), (c_void_p * max(len(outs), 1))(*outs)
    p = ctypes.cast(ctypes.pointer(params), c_void_p) if params is not None else None
    return native.operator_find(name.encode()).contents.func(a, b, p, None)


def test_paged_registry_and_layouts(native):
    for n, t in (("kv_page_map_i32_cuda", b"i32"), ("kv_page_store_f16_cuda", b"f16"), ("kv_page_store_f32_cuda", b"f32"),
                 ("mha_paged_attn_f16_cuda", b"f16"), ("mha_paged_attn_f32_cuda", b"f32")):
        assert native.operator_find(n.encode()).contents.data_type == t
    assert ctypes.sizeof(cf.KvPageMapParams) == 48
    assert ctypes.sizeof(cf.KvPageStoreParams) == 104
    assert ctypes.sizeof(cf.MhaPagedParams) == 120


MAP_OK = dict(batch_size=2, num_tokens=8, page_size=16, num_pages=64, max_pages=8, ring_size=64)


@pytest.mark.parametrize("change", [
    dict(batch_size=0), dict(batch_size=-1), dict(num_tokens=-1), dict(page_size=0), dict(num_pages=0), dict(max_pages=0),
    dict(ring_size=0), dict(ring_size=(1 << 30) + 1), dict(num_pages=1 << 28), dict(max_pages=1 << 28),
    dict(batch_size=1 << 28), dict(num_tokens=1 << 31),
])
def test_map_refuses_parameters(native, change):
    assert _call(native, "kv_page_map_i32_cuda", [DP] * 3, [DP] * 7, cf.KvPageMapParams(**dict(MAP_OK, **change))) == -1


@pytest.mark.parametrize("n_in,n_out", [(i, None) for i in range(3)] + [(None, o) for o in range(7)])
def test_map_refuses_missing_arrays(native, n_in, n_out):
    ins, outs = [DP] * 3, [DP] * 7
    if n_in is not None:
        ins[n_in] = None
    else:
        outs[n_out] = None
    assert _call(native, "kv_page_map_i32_cuda", ins, outs, cf.KvPageMapParams(**MAP_OK)) == -1
    assert _call(native, "kv_page_map_i32_cuda", [DP] * 3, [DP] * 7, None) == -1


STORE_OK = dict(num_tokens=4, num_heads=8, num_kv_heads=2, head_dim=64, page_size=16, num_pages=8, rope_base=10000.0)


@pytest.mark.parametrize("change", [
    dict(num_tokens=-1), dict(num_kv_heads=0), dict(head_dim=0), dict(head_dim=63), dict(head_dim=258), dict(page_size=0),
    dict(num_pages=0), dict(num_pages=1 << 28), dict(rope_base=-1.0), dict(rope_base=math.nan), dict(rope_base=math.inf),
    dict(num_heads=0), dict(q_stride=-8), dict(kv_stride=-8), dict(q_out_stride=-8), dict(page_stride=-8),
    dict(row_stride=-8), dict(head_stride=-8),
])
@pytest.mark.parametrize("op", ["kv_page_store_f16_cuda", "kv_page_store_f32_cuda"])
def test_store_refuses_parameters(native, op, change):
    assert _call(native, op, [DP] * 5, [DP] * 3, cf.KvPageStoreParams(**dict(STORE_OK, **change))) == -1


def test_store_refuses_missing_arrays(native):
    op, p = "kv_page_store_f16_cuda", cf.KvPageStoreParams(**STORE_OK)
    for i in range(4):
        assert _call(native, op, [None if j == i else DP for j in range(5)], [DP] * 3, p) == -1
    for o in range(2):
        assert _call(native, op, [DP] * 5, [None if j == o else DP for j in range(3)], p) == -1
    assert _call(native, op, [DP] * 4 + [None], [DP] * 3, p) == -1            # a place for Q, but no Q
    assert _call(native, op, [DP] * 5, [DP, DP, None], p) == -1               # and the reverse
    assert _call(native, op, [DP] * 5, [DP] * 3, None) == -1
    assert _call(native, op, [DP] * 5, [DP] * 3, cf.KvPageStoreParams(**dict(STORE_OK, num_tokens=0))) == 0


ATTN_OK = dict(batch_size=2, num_tokens=4, num_heads=8, num_kv_heads=2, head_dim=64, scale=0.125, page_size=16, num_pages=8,
               max_pages=4)


@pytest.mark.parametrize("change", [
    dict(batch_size=-1), dict(num_tokens=-1), dict(num_heads=0), dict(num_kv_heads=3), dict(head_dim=0), dict(head_dim=513),
    dict(page_size=0), dict(num_pages=0), dict(max_pages=0), dict(num_pages=1 << 28), dict(max_pages=1 << 28),
    dict(max_new=-1), dict(q_stride=-8), dict(page_stride=-8), dict(row_stride=-8), dict(head_stride=-8),
    dict(num_heads=65536, num_kv_heads=65536), dict(num_tokens=1 << 31),
])
@pytest.mark.parametrize("op", ["mha_paged_attn_f16_cuda", "mha_paged_attn_f32_cuda"])
def test_attn_refuses_parameters(native, op, change):
    assert _call(native, op, [DP] * 6, [DP], cf.MhaPagedParams(**dict(ATTN_OK, **change))) == -1


def test_attn_refuses_missing_arrays(native):
    op, p = "mha_paged_attn_f16_cuda", cf.MhaPagedParams(**ATTN_OK)
    for i in range(6):
        assert _call(native, op, [None if j == i else DP for j in range(6)], [DP], p) == -1
    assert _call(native, op, [DP] * 6, [None], p) == -1
    assert _call(native, op, [DP] * 6, [DP], None) == -1
    for zero in ("batch_size", "num_tokens"):                                  # nothing to do
        assert _call(native, op, [DP] * 6, [DP], cf.MhaPagedParams(**dict(ATTN_OK, **{zero: 0}))) == 0


@pytest.mark.parametrize("op", ["mha_paged_attn_f16_cuda", "mha_paged_attn_f32_cuda"])
@pytest.mark.parametrize("same", [0, 1, 2])
def test_attn_refuses_a_result_over_an_input(native, op, same):
    ins = [DP + 16 * i for i in range(6)]
    assert _call(native, op, ins, [ins[same]], cf.MhaPagedParams(**ATTN_OK)) == -1


def test_references_agree_on_a_plain_case():
    """The oracle of attention against a softmax written out for one row, and its error bounds
    against a planted mistake: one of 200 positions left out is seen."""
    c = Paged([3], [197], 4, 2, 64, 16, True, pad=0)
    out, e32, e16 = ref_attn(c.q, c.kp, c.vp, c.table, c.lens, c.start, c.scale)
    at = c.table[0, np.arange(199) // 16] * 16 + np.arange(199) % 16
    k, v = (x.reshape(-1, 2, 64)[at, 1].astype(np.float64) for x in (c.kp, c.vp))
    s = k @ c.q[1, 3].astype(np.float64) * c.scale
    w = np.exp(s) / np.exp(s).sum()
    assert np.allclose(out[1, 3], w @ v, rtol=1e-12, atol=1e-13)
    w[77] = 0.0
    off = np.abs(w @ v / w.sum() - out[1, 3])
    assert (off > e16[1, 3] + 2.0 ** -11 * np.abs(out[1, 3])).any()


# ------------------------------------------------------------------ the map (GPU) ---

def run_map(cached, new, table, ring, head, avail, T, P, num_pages, in_place=False, stream=None):
    B = len(cached)
    c, n, cnt = dev(np.asarray(cached, I32)), dev(np.asarray(new, I32)), dev(np.array([head, avail, 0], I32))
    t, r = dev(table), dev(ring)
    sl = c if in_place else dev(np.full(B, 77, I32))
    after = cnt if in_place else dev(np.full(3, 77, I32))
    qs, pos, slots = (dev(np.full(k, 77, I32)) for k in (B + 1, max(T, 1), max(T, 1)))
    p = cf.KvPageMapParams(batch_size=B, num_tokens=T, page_size=P, num_pages=num_pages, max_pages=table.shape[1],
                           ring_size=len(ring))
    assert cf.call_op("kv_page_map_i32_cuda", [c, n, cnt], [t, r, sl, qs, pos, slots, after], p, stream) == 0
    if stream is not None:
        stream.synchronize()
    return dict(table=t.download(), ring=r.download(), seq_lens=sl.download(), q_start=qs.download(),
                positions=pos.download()[:T], slots=slots.download()[:T], counters=after.download())


def map_case(seed, B, P, width, chunk, ends, short=0, pad=5):
    """Random requests; `short`: so many pages fewer than they ask for are free."""
    rng = np.random.default_rng(seed)
    cap = width * P
    cached = rng.integers(0, cap + 1, B)
    cached[rng.random(B) < 0.3] = 0
    new = np.minimum(rng.integers(0, chunk + 1, B), cap - cached)
    new[rng.random(B) < ends] = -1
    held = -(-cached // P)
    need = np.where(new >= 0, -(-(cached + np.maximum(new, 0)) // P) - held, 0).sum()
    avail = max(int(need) - short, 0) + (7 if short == 0 else 0)
    num_pages = int(held.sum()) + avail + 1
    pages = rng.permutation(num_pages).astype(I32)
    table = np.full((B, width), -1, I32)
    at = avail
    for b in range(B):
        table[b, :held[b]] = pages[at:at + held[b]]
        at += held[b]
    ring = np.full(num_pages + 3, -5, I32)
    head = int(rng.integers(0, len(ring)))
    ring[(head + np.arange(avail)) % len(ring)] = pages[:avail]
    T = int(np.maximum(new, 0).sum()) + pad
    return [cached, new, table, ring, head, avail, T, P, num_pages]


def same(got, want):
    for k in want:
        assert np.array_equal(got[k], want[k]), k


@pytest.mark.gpu
@pytest.mark.parametrize("B,P,width,chunk,ends", [
    (1, 16, 4, 1, 0.0), (1, 1, 5000, 4200, 0.0), (3, 7, 40, 90, 0.0), (16, 16, 256, 1, 0.0), (63, 16, 20, 40, 0.2),
    (65, 32, 9, 17, 0.3), (1024, 16, 4, 3, 0.1), (1023, 16, 30, 200, 0.1), (1025, 16, 4, 2, 0.1), (3000, 32, 32, 43, 0.05),
    (2, 16, 4000, 30000, 0.0),
])
def test_map(gpu, B, P, width, chunk, ends):
    for short in (0, 3):
        c = map_case(B + P, B, P, width, chunk, ends, short)
        want = ref_map(c[0], c[1], c[2], c[3], c[4], c[5], c[6], c[7], c[8])
        same(run_map(*c), want)
        same(run_map(*c, in_place=True), want)


@pytest.mark.gpu
@pytest.mark.parametrize("many", [False, True])     # one launch and two
def test_map_edges(gpu, many):
    """Past the end of the table, no free page at all, no tokens, ended with nothing held, rows
    that T cuts off, places of the ring that hold no page, counters and lengths out of range."""
    P, width, num_pages = 16, 3, 40
    cached = [40, 0, 48, 16, 0, 15, -4, 33] + [0] * (1100 if many else 0)
    new = [9, 0, 1, 1, -1, 1, 2, -9] + [0] * (1100 if many else 0)
    table = np.full((len(cached), width), -1, I32)
    table[0], table[2], table[3, 0], table[5, 0], table[7] = [1, 2, 3], [4, 5, 6], 7, 99, [8, 9, 10]
    ring = np.array([11, -3, 12, 1000, 13, 14, 15, 16, 17], I32)
    for head, avail, T in ((7, 5, 14), (4, 0, 14), (1, 2, 5), (-7, 100, 20), (2 ** 31 - 1, -1, 14)):
        n = [max(x, 0) for x in new] if avail > 5 else new      # the ring has no room for more than it can hold
        same(run_map(cached, n, table, ring, head, avail, T, P, num_pages),
             ref_map(cached, n, table, ring, max(head, 0) % 9, min(max(avail, 0), 9), T, P, num_pages))


@pytest.mark.gpu
@pytest.mark.parametrize("many", [False, True])
def test_map_of_lengths_whose_sum_passes_32_bits(gpu, many):
    """Nothing out of range is touched: entries of the table stay pages or -1, slots stay below the
    last page's end."""
    P, width, num_pages, T = 16, 4, 64, 50
    big = 2 ** 31 - 1
    new = [5, big, big, 3, big, 20] + [1] * (1100 if many else 0)
    cached = [0] * len(new)
    table, ring = np.full((len(new), width), -1, I32), np.arange(num_pages, dtype=I32)
    got = run_map(cached, new, table, ring, 0, num_pages, T, P, num_pages)
    assert (got["table"] >= -1).all() and (got["table"] < num_pages).all()
    assert (got["slots"] >= -1).all() and (got["slots"] < num_pages * P).all()


# ------------------------------------------------------------------ the store (GPU) ---

@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("T,H,H_kv,d,P,rope,form", [
    (1, 12, 12, 64, 16, True, "dense"), (37, 32, 8, 128, 16, True, "dense"), (300, 4, 1, 80, 7, True, "dense"),
    (65, 6, 2, 256, 64, True, "dense"), (33, 3, 3, 6, 5, True, "dense"), (29, 5, 5, 33, 16, False, "dense"),
    (129, 16, 4, 128, 16, False, "dense"), (50, 8, 2, 64, 16, True, "qkv"), (50, 8, 2, 64, 16, False, "heads"),
    (31, 8, 2, 64, 16, True, "odd"), (31, 8, 2, 64, 16, False, "odd"), (40, 8, 2, 128, 32, True, "in_place"),
    (40, 8, 2, 128, 32, True, "no_q"),
])
def test_store(gpu, f16, T, H, H_kv, d, P, rope, form):
    rng = np.random.default_rng(T + d)
    dt = np.float16 if f16 else np.float32
    n_pages, base = -(-2 * T // P) + 1, 10000.0
    mk = lambda *s: rng.standard_normal(s).astype(dt)
    q, k, v = mk(T, H, d), mk(T, H_kv, d), mk(T, H_kv, d)
    pos = rng.integers(0, 1 << 20, T).astype(I32)
    pos[0] = 0
    slots = rng.permutation(n_pages * P)[:T].astype(I32)
    if T > 5:
        slots[3], slots[4], pos[5] = -1, n_pages * P, -1
    kp, vp = mk(n_pages, P, H_kv, d), mk(n_pages, P, H_kv, d)
    name = "kv_page_store_%s_cuda" % ("f16" if f16 else "f32")
    kw, es, off = {}, np.dtype(dt).itemsize, 0
    if form == "qkv":                                   # one row-concatenated projection
        rows = dev(np.concatenate([x.reshape(T, -1) for x in (q, k, v)], 1))
        ins = [rows.ptr + H * d * es, rows.ptr + (H + H_kv) * d * es, None, None, rows.ptr]
        kw = dict(q_stride=(H + 2 * H_kv) * d, kv_stride=(H + 2 * H_kv) * d)
    elif form == "odd":                                 # nothing on a 16-byte boundary
        off = 1
        bufs = [dev(np.concatenate(([np.nan], x.ravel())).astype(dt)) for x in (k, v, q)]
        ins = [bufs[0].ptr + es, bufs[1].ptr + es, None, None, bufs[2].ptr + es]
    else:
        bufs = [dev(x) for x in (k, v, q)]
        ins = [bufs[0], bufs[1], None, None, bufs[2]]
    ins[2], ins[3] = dev(slots), dev(pos)
    pages = (lambda x: x.transpose(0, 2, 1, 3)) if form == "heads" else (lambda x: x)   # (pages, H_kv, P, d)
    if form == "heads":
        kw = dict(row_stride=d, head_stride=P * d)
    dk, dv = dev(np.ascontiguousarray(pages(kp))), dev(np.ascontiguousarray(pages(vp)))
    qo = bufs[2] if form == "in_place" else dev(np.full((T, H, d), 7.0, dt))
    outs = [dk, dv, qo]
    if form == "no_q":
        ins[4], outs[2] = None, None
    if not rope:
        ins, outs = ins[:3], outs[:2]
    p = cf.KvPageStoreParams(num_tokens=T, num_heads=H, num_kv_heads=H_kv, head_dim=d, page_size=P, num_pages=n_pages,
                             rope_base=base if rope else 0.0, **kw)
    assert cf.call_op(name, ins, outs, p) == 0
    ok = (slots >= 0) & (slots < n_pages * P)
    want_k, want_v = kp.astype(np.float64).reshape(-1, H_kv, d), vp.reshape(-1, H_kv, d).copy()
    tk = ref_turn(k.astype(np.float64), pos, base) if rope else k.astype(np.float64)
    want_k[slots[ok]], want_v[slots[ok]] = tk[ok], v[ok]
    got_k, got_v = (pages(x.download()).reshape(-1, H_kv, d) for x in (dk, dv))
    assert np.array_equal(got_v, want_v)
    # A turned pair: cos and sin off by 2^-23 (the angle in turns is rounded to FP32: 2^-25 of a
    # turn at most, times 2 pi, and their own), two products and a sum, one rounding to the type.
    half = 2.0 ** (-11 if f16 else -24)
    room = lambda x, y: 6 * 2.0 ** -24 * np.hypot(x[..., 0::2], x[..., 1::2]).repeat(2, -1) + half * np.abs(y) + 2.0 ** -25 * f16
    if rope:
        t = room(k.astype(np.float64), tk)
        assert (np.abs(got_k[slots[ok]] - tk[ok]) <= t[ok]).all()
        kept = np.ones(len(want_k), bool)
        kept[slots[ok]] = False
        assert np.array_equal(got_k[kept], want_k[kept])
    else:
        assert np.array_equal(got_k, want_k)
    if rope and form != "no_q":
        tq = ref_turn(q.astype(np.float64), pos, base)
        got = qo.download()
        turned = pos >= 0
        assert (np.abs(got - tq) <= room(q.astype(np.float64), tq))[turned].all()
        assert np.array_equal(got[~turned], (q if form == "in_place" else np.full_like(q, 7.0))[~turned])


# ------------------------------------------------------------------ attention (GPU) ---

HEADS = [(12, 12, 64), (8, 2, 128), (32, 8, 128), (8, 1, 64), (4, 4, 128), (16, 1, 64), (6, 2, 80), (5, 5, 33)]


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d", HEADS)
@pytest.mark.parametrize("new,past", [
    ([1], [0]), ([1], [256]), ([1, 1, 1, 1, 1], [0, 15, 16, 63, 700]), ([3, 0, 1, 4], [100, 5, 0, 1000]), ([64], [0]),
    ([17, 1, 130], [31, 200, 3]), ([65, 33], [500, 0]),
])
def test_attention(gpu, f16, H, H_kv, d, new, past):
    for P in (16, 32) if d in (64, 128) else (16, 5):
        c = Paged(new, past, H, H_kv, d, P, f16, seed=H + d + sum(past))
        c.check(c.run())
        c.check(c.run(max_new=max(new)))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("P", [1, 3, 16, 48, 64, 128, 256])
def test_attention_page_sizes(gpu, f16, P):
    c = Paged([1, 40, 2], [300, 77, 513], 8, 2, 64, P, f16)
    c.check(c.run(max_new=40))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d", [(32, 8, 128), (12, 12, 64), (6, 3, 40)])
def test_attention_split_over_long_contexts(gpu, f16, H, H_kv, d):
    """Few rows over long caches, where the positions of a row are shared out and joined."""
    for new in ([1, 1, 1], [5, 1, 2], [40, 1, 1]):
        c = Paged(new, [6000, 3, 1500], H, H_kv, d, 16, f16, seed=7)
        c.check(c.run(max_new=max(new)))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new", [[1, 1, 1, 1], [20, 1, 70, 3]])
def test_attention_many_sequences_and_sharp_scores(gpu, f16, new):
    """More sequences than a wave has lanes; scores of tens, so that the running maximum moves."""
    past = [(37 * i * i) % 400 for i in range(140)]
    c = Paged((new * 35), past, 8, 2, 64, 16, f16, seed=3, k_std=6.0)
    c.check(c.run(max_new=max(new)))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,P", [(8, 2, 64, 16), (8, 2, 128, 32), (5, 5, 33, 7)])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_empty_rows_and_bad_pages(gpu, f16, H, H_kv, d, P, wide):
    """Pages that are none (-1, past the end) hold no position, also all of a sequence's; lengths
    below the row count, zero, negative and past the table; offsets that leave a sequence out."""
    new = [4, 1, 3, 2, 30 if wide else 2, 1, 2]
    c = Paged(new, [90, 40, 60, 3, 200, 0, 10], H, H_kv, d, P, f16, seed=5)
    t = c.table
    t[0, 1], t[0, -1 if t[0, -1] >= 0 else 0] = -1, 2 ** 31 - 1
    t[1, :] = -2
    t[4, 0] = c.n_pages
    c.lens[2], c.lens[3], c.lens[5] = 2, 0, -5
    # What a page in use holds past its sequence's length is NaN; so is all of a lost page.
    c.check(c.run(max_new=max(new)))
    c.lens[4] = 2 ** 31 - 1                     # clamped to the table, whose end is -1
    t[4, -(-230 // P) - (0 if wide else 2):] = -1
    full = c.table.shape[1] * P
    ref = c.lens.copy()
    ref[4] = full
    got = c.run(max_new=max(new))
    c.lens = ref
    ok = ~np.isnan(ref_attn(c.q, c.kp, c.vp, c.table, c.lens, c.start, c.scale)[0]).any()
    if ok:
        c.check(got)
    c.start[3], c.start[4] = 1000, -3           # offsets out of order: no fault, rows in range
    c.run(max_new=max(new))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new", [[1, 1], [70, 5]])
def test_attention_strides(gpu, f16, new):
    """Q out of a row-concatenated projection; K and V interleaved per page, heads outermost; rows
    a little longer than they need be, and a base off the 16-byte grid."""
    H, H_kv, d, P = 8, 2, 64, 16
    c = Paged(new, [130, 40], H, H_kv, d, P, f16)
    es = np.dtype(c.dt).itemsize
    want = c.run()
    c.check(want)
    tail = [dev(x) for x in (c.table, c.lens, c.start)]
    rows = np.full((c.T, (H + 2 * H_kv) * d), np.nan, c.dt)
    rows[:, :H * d] = c.q.reshape(c.T, -1)
    both = np.stack([c.kp.transpose(0, 2, 1, 3), c.vp.transpose(0, 2, 1, 3)], 1)      # (pages, 2, H_kv, P, d)
    kv = dev(np.ascontiguousarray(both))
    got = c.run([dev(rows), kv.ptr, kv.ptr + H_kv * P * d * es] + tail, q_stride=(H + 2 * H_kv) * d,
                page_stride=2 * H_kv * P * d, row_stride=d, head_stride=P * d)
    assert np.array_equal(got[:c.start[-1]], want[:c.start[-1]])
    for shift, row in ((0, H_kv * d + 8), (1, H_kv * d + 1)):
        wide = np.full((2, c.n_pages, P, row), np.nan, c.dt)
        wide[0, ..., :H_kv * d], wide[1, ..., :H_kv * d] = c.kp.reshape(c.n_pages, P, -1), c.vp.reshape(c.n_pages, P, -1)
        kv = dev(np.concatenate((np.full(shift, np.nan, c.dt), wide.ravel())))
        got = c.run([dev(c.q), kv.ptr + shift * es, kv.ptr + (shift + wide[0].size) * es] + tail, page_stride=P * row,
                    row_stride=row)
        c.check(got)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_attention_scales(gpu, f16, scale):
    c = Paged([1, 33], [100, 20], 4, 2, 64, 16, f16, scale=scale)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,new,past", [
    (48, 16, 64, [300, 250, 400, 290], [100, 0, 700, 64]),      # fp16: tiles of 256 rows, not cut
    (64, 16, 128, [300, 200, 350], [100, 1700, 40]),
    (128, 64, 64, [384], [2500]),                               # ... and cut
    (8, 8, 64, [200] * 3 + [1] * 70 + [90], [0, 900, 5000] + [11 * i for i in range(70)] + [2000]),
])
def test_attention_wide_tiles(gpu, f16, H, H_kv, d, new, past):
    c = Paged(new, past, H, H_kv, d, 16, f16, seed=9)
    c.check(c.run(max_new=max(new)))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new,past", [([1, 1, 1], [5000, 20, 1300]), ([200, 1, 30], [3000, 2500, 10]), ([2] * 40, [1100] * 40)])
def test_attention_with_hints_that_are_too_small(gpu, f16, new, past):
    """max_new and max_len choose kernels; what passes them is computed all the same."""
    for H, H_kv, d in ((8, 2, 128), (16, 16, 64)):
        c = Paged(new, past, H, H_kv, d, 16, f16, seed=11)
        for max_new, max_len in ((1, 0), (1, 64), (max(new), 1), (17, 600), (2 ** 40, 2 ** 40)):
            c.check(c.run(max_new=max_new, max_len=max_len))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,P,new,past", [
    (8, 2, 64, 16, [12, 2, 8], [100, 30, 0]), (8, 2, 128, 16, [4, 4, 4], [2500, 60, 1500]), (12, 12, 64, 16, [9] * 12, [300] * 12),
    (8, 4, 128, 32, [150, 40, 90], [33, 0, 200]), (4, 4, 64, 16, [130, 2], [4000, 3000]), (128, 64, 64, 16, [400], [64]),
    (4, 2, 40, 5, [7, 3], [20, 9]),
])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_attention_ignores_what_a_row_does_not_see(gpu, f16, H, H_kv, d, P, new, past, bad):
    """K and V of one new position of every sequence are infinite or NaN: the rows before it are
    what they are without, those from it on are not finite in that dim of V."""
    c = Paged(new, past, H, H_kv, d, P, f16, seed=13)
    at = [n // 2 for n in new]                      # row of each sequence whose position it is
    places = [(c.table[b, (past[b] + i) // P], (past[b] + i) % P) for b, i in enumerate(at)]
    kept = [(c.kp[x].copy(), c.vp[x].copy()) for x in places]
    for x in places:
        c.vp[x][:, 3] = bad
    got = c.run(max_new=max(new))
    for b, i in enumerate(at):
        seeing = got[c.start[b] + i:c.start[b + 1], :, 3]
        assert np.isnan(seeing).all() if np.isnan(bad) else (seeing == np.inf).all()
    for x in places:
        c.kp[x] = bad
    with_k = c.run(max_new=max(new))
    for x, (k, v) in zip(places, kept):
        c.kp[x], c.vp[x] = k, v
    clean = c.run(max_new=max(new))
    c.check(clean)
    for o, dims in ((got, np.arange(d) != 3), (with_k, np.zeros(d, bool))):
        mixed = clean.copy()                        # what cannot be compared is the clean result's
        for b, i in enumerate(at):
            rows = slice(c.start[b], c.start[b] + i)
            mixed[rows] = o[rows]
            rows = slice(c.start[b] + i, c.start[b + 1])
            mixed[rows][..., dims] = o[rows][..., dims]
        c.check(mixed)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new", [[1] * 3, [60, 1, 200]])
def test_attention_cut_and_captured(gpu, f16, new):
    """A captured call whose tiles are cut, replayed at other lengths with eager work in between."""
    c = Paged(new, [4000, 9, 2500], 16, 4, 128, 16, f16, seed=21)
    s = cf.Stream()
    bufs = [dev(x) for x in (c.q, c.kp, c.vp, c.table, c.lens, c.start)]
    o, full = dev(np.full(c.q.shape, 7.0, c.dt)), c.lens.copy()
    call = lambda out: cf.call_op(c.op, bufs, [out], c.params(max_new=max(new)), s)
    assert call(o) == 0
    s.synchronize()
    assert gpu.gpu_capture_begin(s.handle) == 0
    assert call(o) == 0
    graph = ctypes.c_void_p()
    assert gpu.gpu_capture_end(s.handle, ctypes.byref(graph)) == 0
    for drop in (0, 700, 64, 2300, 0):
        c.lens = np.maximum(full - drop, new).astype(I32)
        bufs[4].upload(c.lens)
        assert gpu.gpu_graph_launch(graph, s.handle) == 0
        s.synchronize()
        got = o.download()
        c.check(got)
        eager = dev(np.full(c.q.shape, 7.0, c.dt))
        assert call(eager) == 0
        s.synchronize()
        assert np.array_equal(eager.download(), got)
    gpu.gpu_graph_exec_destroy(graph)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("new", [[1] * 300, [1] * 259 + [40]])
def test_attention_of_many_sequences(gpu, f16, new):
    """More sequences than are looked at together, the last group of them not full, some empty."""
    past = [(53 * i) % 200 for i in range(len(new))]
    new = [0 if i % 17 == 5 else n for i, n in enumerate(new)]
    for H, H_kv, d in ((8, 2, 128), (3, 3, 64)):
        c = Paged(new, past, H, H_kv, d, 16, f16, seed=15)
        c.check(c.run(max_new=max(new)))
        c.check(c.run(max_new=max(new), max_len=max(n + p for n, p in zip(new, past))))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d", [(64, 1, 128), (48, 1, 64), (40, 2, 64)])
def test_attention_of_many_heads_per_group(gpu, f16, H, H_kv, d):
    """One token's heads alone are more than a narrow tile."""
    for new, past in (([1, 1], [700, 0]), ([3, 0, 2], [90, 5, 2000])):
        c = Paged(new, past, H, H_kv, d, 16, f16, seed=17)
        c.check(c.run(max_new=max(new)))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_pages_beyond_32_bits(gpu, f16):
    """Pages 2^30 bytes apart, the last of them 5 to 6 GB into the buffers: stored there, attended from
    there, by the matrix cores and by the plain kernel (a stride off the 16-byte grid)."""
    H, H_kv, d, P, n_pages = 8, 2, 64, 16, 6
    es = 2 if f16 else 4
    t = "f16" if f16 else "f32"
    c = Paged([1, 20], [30, 10], H, H_kv, d, P, f16, seed=19, pad=0, spare=0)
    assert c.n_pages <= n_pages - 1
    k, v = (np.concatenate([x[c.table[b, j // P], j % P][None] for b in range(2) for j in range(c.lens[b])])
            for x in (c.kp, c.vp))
    for extra in (0, 1):
        step = (1 << 30) // es + extra
        caches = [cf.DeviceBuffer(n_pages * (step * es)) for _ in range(2)]
        far = [5, 4, 3, 2][:c.n_pages]                   # pages from the far end
        table = np.where(c.table >= 0, np.take(np.array(far + [0], I32), np.maximum(c.table, 0)), -1).astype(I32)
        slots = np.concatenate([[table[b, j // P] * P + j % P for j in range(c.lens[b])] for b in range(2)]).astype(I32)
        p = cf.KvPageStoreParams(num_tokens=len(slots), num_heads=0, num_kv_heads=H_kv, head_dim=d, page_size=P,
                                 num_pages=n_pages, page_stride=step)
        assert cf.call_op("kv_page_store_%s_cuda" % t, [dev(k), dev(v), dev(slots)], caches, p) == 0
        c2 = cf.MhaPagedParams(batch_size=2, num_tokens=c.T, num_heads=H, num_kv_heads=H_kv, head_dim=d, scale=c.scale,
                               page_size=P, num_pages=n_pages, max_pages=c.width, page_stride=step)
        o = dev(np.full(c.q.shape, 7.0, c.dt))
        assert cf.call_op(c.op, [dev(c.q)] + caches + [dev(table), dev(c.lens), dev(c.start)], [o], c2) == 0
        c.check(o.download())
        for x in caches:
            x.free()


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_attention_of_a_contiguous_decode_cache(gpu, f16):
    """The cache of MHA_Decode as pages: the same attention as mha_decode_attn."""
    B, H, H_kv, d, cap, P = 5, 32, 8, 128, 512, 32
    rng = np.random.default_rng(4)
    dt = np.float16 if f16 else np.float32
    q, k, v = (rng.standard_normal(s).astype(dt) for s in ((B, H, d), (B, cap, H_kv, d), (B, cap, H_kv, d)))
    last = np.array([511, 0, 100, 31, 300], I32)
    o = dev(np.zeros_like(q))
    scale = float(np.float32(1.0 / math.sqrt(d)))
    assert cf.call_op("mha_decode_attn_%s_cuda" % ("f16" if f16 else "f32"), [dev(q), dev(k), dev(v), dev(last)], [o],
                      cf.MhaDecodeParams(B, H * d, H, H_kv, d, scale, -1, cap)) == 0
    c = Paged([1] * B, [0] * B, H, H_kv, d, P, f16, pad=0)
    c.q, c.kp, c.vp = q, k.reshape(-1, P, H_kv, d), v.reshape(-1, P, H_kv, d)
    c.n_pages, c.width, c.lens = B * cap // P, cap // P, last + 1
    c.table = np.arange(c.n_pages, dtype=I32).reshape(B, -1)
    got = c.run(max_new=1)
    c.check(got)
    c.check(o.download())


# ------------------------------------------------------------------ together (GPU) ---

class Step:
    """A server's device state: lengths, tables, ring and one layer's cache, and a step over it.
    The host keeps the tokens each sequence was given, in 64 bits after rotation."""

    def __init__(self, f16, B, T, H, H_kv, d, P, n_pages, width, seed=11):
        self.rng = np.random.default_rng(seed)
        self.f16, self.dt = f16, np.float16 if f16 else np.float32
        self.B, self.T, self.H, self.H_kv, self.d, self.P, self.n_pages, self.width = B, T, H, H_kv, d, P, n_pages, width
        self.table = dev(np.full((B, width), -1, I32))
        self.ring = dev(self.rng.permutation(n_pages).astype(I32))
        self.counters = dev(np.array([0, n_pages, 0], I32))
        self.lens, self.new = dev(np.zeros(B, I32)), dev(np.zeros(B, I32))
        self.start, self.pos, self.slots = (dev(np.zeros(k, I32)) for k in (B + 1, T, T))
        width_qkv = (H + 2 * H_kv) * d
        self.qkv, self.qr, self.o = (dev(np.zeros(s, self.dt)) for s in ((T, width_qkv), (T, H, d), (T, H, d)))
        self.kp, self.vp = (dev(np.full((n_pages, P, H_kv, d), np.nan, self.dt)) for _ in range(2))
        self.scale = float(np.float32(1.0 / math.sqrt(d)))
        self.held = [(np.zeros((0, H_kv, d)), np.zeros((0, H_kv, d))) for _ in range(B)]

    def launch(self, stream):
        t = "f16" if self.f16 else "f32"
        es, w = np.dtype(self.dt).itemsize, (self.H + 2 * self.H_kv) * self.d
        m = cf.KvPageMapParams(batch_size=self.B, num_tokens=self.T, page_size=self.P, num_pages=self.n_pages,
                               max_pages=self.width, ring_size=self.n_pages)
        s = cf.KvPageStoreParams(num_tokens=self.T, num_heads=self.H, num_kv_heads=self.H_kv, head_dim=self.d,
                                 page_size=self.P, num_pages=self.n_pages, rope_base=10000.0, q_stride=w, kv_stride=w)
        a = cf.MhaPagedParams(batch_size=self.B, num_tokens=self.T, num_heads=self.H, num_kv_heads=self.H_kv,
                              head_dim=self.d, scale=self.scale, page_size=self.P, num_pages=self.n_pages,
                              max_pages=self.width)
        q, k, v = self.qkv.ptr, self.qkv.ptr + self.H * self.d * es, self.qkv.ptr + (self.H + self.H_kv) * self.d * es
        assert cf.call_op("kv_page_map_i32_cuda", [self.lens, self.new, self.counters],
                          [self.table, self.ring, self.lens, self.start, self.pos, self.slots, self.counters], m, stream) == 0
        assert cf.call_op("kv_page_store_%s_cuda" % t, [k, v, self.slots, self.pos, q], [self.kp, self.vp, self.qr], s,
                          stream) == 0
        assert cf.call_op("mha_paged_attn_%s_cuda" % t, [self.qr, self.kp, self.vp, self.table, self.lens, self.start],
                          [self.o], a, stream) == 0

    def feed(self, new):
        """This step's tokens: uploads them and returns what attention should give, and its room."""
        qkv = self.rng.standard_normal((self.T, (self.H + 2 * self.H_kv) * self.d)).astype(self.dt)
        self.qkv.upload(qkv)
        self.new.upload(np.asarray(new, I32))
        H, H_kv, d = self.H, self.H_kv, self.d
        want, room = [], []
        row = 0
        for b, n in enumerate(new):
            if n < 0:
                self.held[b] = (np.zeros((0, H_kv, d)), np.zeros((0, H_kv, d)))
                continue
            x = qkv[row:row + n].astype(np.float64)
            row += n
            p = len(self.held[b][0]) + np.arange(n)
            q = ref_turn(x[:, :H * d].reshape(n, H, d), p, 10000.0).astype(self.dt).astype(np.float64)
            k = ref_turn(x[:, H * d:(H + H_kv) * d].reshape(n, H_kv, d), p, 10000.0).astype(self.dt).astype(np.float64)
            v = x[:, (H + H_kv) * d:].reshape(n, H_kv, d)
            K, V = (np.concatenate(z) for z in zip(self.held[b], (k, v)))
            self.held[b] = (K, V)
            if n == 0:
                continue
            L = len(K)
            o, e32, e16 = ref_attn(q, K.reshape(1, L, H_kv, d), V.reshape(1, L, H_kv, d), np.zeros((1, 1), int),
                                   np.array([L]), np.array([0, n]), self.scale)
            # q and k are rounded to the type from values that differ by FP32 roundings: now and
            # then to the other neighbour, a step of 2^-10 (fp16) of one of d terms of a score.
            step = 2.0 ** (-10 if self.f16 else -23)
            flip = 8 * step * np.abs(V).max() * self.scale
            want.append(o)
            room.append((e16 + 2.0 ** -11 * np.abs(o) + 2.0 ** -25 if self.f16 else e32 + 2.0 ** -24 * np.abs(o)) + flip)
        return (np.concatenate(want), np.concatenate(room)) if want else (None, None)


STEPS = [[20, 1, 33, 7], [1, 1, 1, 1], [1, 40, 1, -1], [1, 1, 1, 12], [1, 1, -1, 1], [1, 3, 0, 1], [2, -1, 50, 1]]


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("captured", [False, True])
def test_steps_of_a_server(gpu, f16, captured):
    """Prompts, decoding, a chunk continued, requests that end and new ones in their place, on pages
    handed round a small ring; eager, and one recording replayed with eager work in between."""
    st = cf.Stream()
    s = Step(f16, 4, 72, 8, 2, 64, 16, 14, 8)
    ex = c_void_p()
    if captured:
        s.feed([0] * 4)
        s.launch(st)                                   # sizes the workspace; adds no token
        st.synchronize()
        assert gpu.gpu_capture_begin(st.handle) == 0
        s.launch(st)
        assert gpu.gpu_capture_end(st.handle, ctypes.byref(ex)) == 0
    for new in STEPS:
        want, room = s.feed(new)
        if captured:
            assert gpu.gpu_graph_launch(ex, st.handle) == 0
        else:
            s.launch(st)
        st.synchronize()
        got = s.o.download()[:len(want)]
        assert s.counters.download()[2] == 0
        assert (np.abs(got - want) <= room).all(), new
        other = Paged([9, 1], [40, 700], 8, 2, 64, 16, f16)      # eager work on the default stream
        other.check(other.run())
    used = sum(-(-len(k) // 16) for k, _ in s.held)
    assert s.counters.download()[1] == 14 - used
    if captured:
        gpu.gpu_graph_exec_destroy(ex)


@pytest.mark.gpu
def test_two_streams_at_once(gpu):
    """The operators on two streams, each with its own workspace."""
    a, b = cf.Stream(), cf.Stream()
    x = Paged([1, 1, 1], [3000, 900, 2000], 32, 8, 128, 16, True, seed=1)
    y = Paged([1, 1], [2500, 4000], 32, 8, 128, 16, True, seed=2)
    bx = [dev(z) for z in (x.q, x.kp, x.vp, x.table, x.lens, x.start)]
    by = [dev(z) for z in (y.q, y.kp, y.vp, y.table, y.lens, y.start)]
    ox, oy = dev(np.full(x.q.shape, 7.0, x.dt)), dev(np.full(y.q.shape, 7.0, y.dt))
    for _ in range(20):
        assert cf.call_op(x.op, bx, [ox], x.params(max_new=1), a) == 0
        assert cf.call_op(y.op, by, [oy], y.params(max_new=1), b) == 0
    a.synchronize()
    b.synchronize()
    x.check(ox.download())
    y.check(oy.download())
