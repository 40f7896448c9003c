"""The paged KV cache in 8 bits: kv_page_store_q8_{f16,f32}_cuda bit by bit and
mha_paged_attn_q8_{f16,f32}_cuda against attention in 64 bits (GPU), and what they refuse (CPU).

What the store writes follows from its inputs exactly (a power of two, one rounding of each value,
one more of those that are rescaled), so codes and powers are compared bit by bit.  What attention
reads is exact too, so its tolerances are those of test_paged.py on the values that the codes stand
for: with fp16 rows the products' weights are rounded to fp16, with FP32 ones they and Q are held as
the sum of three bf16 numbers, 24 bits together.
"""

import ctypes
import math
from ctypes import c_void_p

import numpy as np
import pytest

import cudaforge_amd as cf
from helpers import dev
from test_paged import DP, I32, Paged, _call, ref_attn
from test_qk_norm import frequencies, ref_rows

U8 = np.uint8


# ------------------------------------------------------------------ the numbers, in 64 bits ---

def _values():
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (8 + m) * 2.0 ** (e - 10.0), m * 2.0 ** -9)
    v = np.where((e == 15) & (m == 7), np.nan, v)
    return np.where(c >= 128, -v, v)


VALUE = _values()
POWER = np.array([2.0 ** (i - 127) for i in range(255)] + [np.nan])
MOST = {np.dtype(np.float16): 61440.0, np.dtype(np.float32): 1.875 * 2.0 ** 127}


def encode(x):
    """The nearest codes of values of at most 448 in size, ties to even; NaN is 0x7f."""
    x = np.asarray(x, np.float64)
    a = np.where(np.isfinite(x), np.abs(x), 0.0)
    _, e = np.frexp(a)
    step = 2.0 ** (np.maximum(e - 1, -6) - 3.0)
    q = np.round(a / step) * step                       # numpy rounds ties to even
    code = np.searchsorted(VALUE[:127], q).astype(U8)
    assert (VALUE[code] == q).all()
    return np.where(np.isfinite(x), code | np.where(np.signbit(x), 128, 0), 127).astype(U8)


def power_for(most):
    """The least power of each largest size."""
    out = np.zeros(most.shape, int)
    for i, m in np.ndenumerate(most):
        p = 0
        if m > 0:
            p = max(math.frexp(m)[1] - 9 + 127, 0)
            while p > 0 and m <= 448 * 2.0 ** (p - 1 - 127):
                p -= 1
            while m > 448 * 2.0 ** (p - 127):
                p += 1
        out[i] = p
    return out


def ref_store(rows, slots, cells, powers, block):
    """kv_page_store_q8 of K or V: cells (n_slots, H, d) codes and powers (n_slots / block, H)."""
    cells, powers = cells.copy(), powers.copy()
    dt = rows.dtype
    rows = rows.astype(np.float64)
    finite = np.where(np.isfinite(rows), np.abs(rows), 0.0)
    ok = (slots >= 0) & (slots < len(cells))
    for b in np.unique(slots[ok] // block):
        at = np.flatnonzero(ok & (slots // block == b))
        need = power_for(finite[at].max((0, 2)))
        first = (slots[at] == b * block).any()
        now = need if first else np.maximum(powers[b].astype(int), need)
        others = np.setdiff1d(np.arange(b * block, (b + 1) * block), slots[at])
        if not first:
            for h in np.flatnonzero(now > powers[b]):
                x = VALUE[cells[others, h]]
                cells[others, h] = np.where(np.isnan(x), cells[others, h], encode(x * 2.0 ** (float(powers[b, h]) - now[h])))
        powers[b] = now
        two = 2.0 ** (127.0 - now)[None, :, None]
        limit = np.minimum(448.0, MOST[dt] * two)
        x = rows[at] * two
        cells[slots[at]] = encode(np.where(np.isfinite(x), np.clip(x, -limit, limit), np.nan))
    return cells, powers


def same_codes(got, want):
    """Bit by bit, but for the sign of a NaN."""
    return ((got == want) | ((got & 127 == 127) & (want & 127 == 127))).all()


def quantise(x, block):
    """Dense pages (n, P, H, d) as codes and powers, block by block; NaN where x is."""
    n, P, H, d = x.shape
    y = x.astype(np.float64).reshape(n, P // block, block, H, d)
    p = power_for(np.where(np.isfinite(y), np.abs(y), 0.0).max((2, 4)))
    c = encode(y * 2.0 ** (127.0 - p)[:, :, None, :, None])
    return c.reshape(x.shape), p.astype(U8)


def values(codes, powers):
    n, P, H, d = codes.shape
    block = P // powers.shape[1]
    return (VALUE[codes].reshape(n, P // block, block, H, d) * POWER[powers][:, :, None, :, None]).reshape(codes.shape)


class PagedQ8(Paged):
    """Paged with its caches in 8 bits: kp and vp are the values that the codes stand for.  What no
    sequence holds is NaN, and blocks of nothing else have the power 255 or any other."""

    def __init__(self, *args, block=16, scales=1.0, **kw):
        super().__init__(*args, **kw)
        self.block = block
        rng = np.random.default_rng(77)
        self.codes, self.powers = [], []
        for name in ("kp", "vp"):
            x = getattr(self, name).astype(np.float64)
            if scales != 1.0:                            # blocks of very different size
                f = np.exp2(np.round(rng.uniform(-scales, scales, (x.shape[0], x.shape[1] // block, 1, x.shape[2], 1))))
                x = (x.reshape(x.shape[0], -1, block, *x.shape[2:]) * f).reshape(x.shape)
            c, p = quantise(x, block)
            free = (c & 127 == 127).reshape(x.shape[0], -1, block, *x.shape[2:]).all((2, 4))
            p[free] = rng.choice([255, 254, 0, 127], int(free.sum()))
            self.codes.append(c)
            self.powers.append(p)
        self.refresh()

    def refresh(self):
        self.kp, self.vp = (values(c, p) for c, p in zip(self.codes, self.powers))

    @property
    def op(self):
        return "mha_paged_attn_q8_f16_cuda" if self.f16 else "mha_paged_attn_q8_f32_cuda"

    def params(self, **kw):
        return cf.MhaPagedQ8Params(batch_size=self.B, num_tokens=self.T, num_heads=self.H, num_kv_heads=self.H_kv,
                                   head_dim=self.d, scale=self.scale, page_size=self.P, num_pages=self.n_pages,
                                   max_pages=self.width, **dict(dict(block_size=self.block), **kw))

    def bufs(self):
        return [dev(x) for x in (self.q, *self.codes, self.table, self.lens, self.start, *self.powers)]

    def run(self, bufs=None, stream=None, **kw):
        return super().run(bufs or self.bufs(), stream, **kw)


# ------------------------------------------------------------------ refusals (CPU) ---

STORE_OK = dict(num_tokens=4, num_kv_heads=2, head_dim=64, page_size=32, num_pages=8, block_size=16)
STORES = ["kv_page_store_q8_f16_cuda", "kv_page_store_q8_f32_cuda"]
ATTN_OK = dict(batch_size=2, num_tokens=4, num_heads=8, num_kv_heads=2, head_dim=64, scale=0.125, page_size=32, num_pages=8,
               max_pages=4, block_size=16)
ATTNS = ["mha_paged_attn_q8_f16_cuda", "mha_paged_attn_q8_f32_cuda"]


def test_layouts(native):
    assert ctypes.sizeof(cf.KvPageStoreQ8Params) == 80
    assert ctypes.sizeof(cf.MhaPagedQ8Params) == 128
    for n in STORES + ATTNS:
        assert native.operator_find(n.encode()).contents.data_type == (b"f16" if "f16" in n else b"f32")


@pytest.mark.parametrize("change", [
    dict(num_tokens=-1), dict(num_tokens=1 << 31), dict(num_kv_heads=0), dict(num_kv_heads=65536), dict(head_dim=0),
    dict(head_dim=65536), dict(num_kv_heads=60000, head_dim=60000), dict(page_size=0), dict(num_pages=0),
    dict(num_pages=1 << 27), dict(block_size=-1), dict(block_size=5), dict(block_size=64), dict(page_size=128, block_size=128),
    dict(page_size=24, block_size=0), dict(kv_stride=-1), dict(page_stride=-1), dict(row_stride=-1), dict(head_stride=-1),
])
@pytest.mark.parametrize("op", STORES)
def test_store_refuses_parameters(native, op, change):
    assert _call(native, op, [DP] * 3, [DP] * 4, cf.KvPageStoreQ8Params(**dict(STORE_OK, **change))) == -1


@pytest.mark.parametrize("op", STORES)
def test_store_refuses_missing_arrays(native, op):
    p = cf.KvPageStoreQ8Params(**STORE_OK)
    for i in range(3):
        assert _call(native, op, [None if j == i else DP for j in range(3)], [DP] * 4, p) == -1
    for o in range(4):
        assert _call(native, op, [DP] * 3, [None if j == o else DP for j in range(4)], p) == -1
    assert _call(native, op, [DP] * 3, [DP] * 4, None) == -1
    assert _call(native, op, [DP] * 3, [DP] * 4, cf.KvPageStoreQ8Params(**dict(STORE_OK, num_tokens=0))) == 0


@pytest.mark.parametrize("op", STORES)
def test_store_refuses_arrays_given_twice(native, op):
    p, arrays = cf.KvPageStoreQ8Params(**STORE_OK), [DP + 64 * i for i in range(7)]
    for i in range(3, 7):
        for j in range(7):
            if i != j:
                names = [arrays[j] if k == i else x for k, x in enumerate(arrays)]
                assert _call(native, op, names[:3], names[3:], p) == -1


@pytest.mark.parametrize("change", [
    dict(batch_size=-1), dict(num_tokens=-1), dict(num_heads=0), dict(num_kv_heads=3), dict(head_dim=0), dict(head_dim=513),
    dict(page_size=0), dict(num_pages=0), dict(max_pages=0), dict(num_pages=1 << 27), dict(max_pages=1 << 27),
    dict(max_new=-1), dict(max_len=-1), dict(q_stride=-8), dict(page_stride=-8), dict(row_stride=-8), dict(head_stride=-8),
    dict(num_heads=65536, num_kv_heads=65536), dict(num_tokens=1 << 31), dict(block_size=-1), dict(block_size=5),
    dict(block_size=64), dict(page_size=24, block_size=0), dict(page_size=128, block_size=128),
])
@pytest.mark.parametrize("op", ATTNS)
def test_attn_refuses_parameters(native, op, change):
    ins = [DP + 8 * i for i in range(8)]
    assert _call(native, op, ins, [DP + 128], cf.MhaPagedQ8Params(**dict(ATTN_OK, **change))) == -1


@pytest.mark.parametrize("op", ATTNS)
def test_attn_refuses_missing_arrays(native, op):
    ins, p = [DP + 8 * i for i in range(8)], cf.MhaPagedQ8Params(**ATTN_OK)
    for i in range(8):
        assert _call(native, op, [None if j == i else x for j, x in enumerate(ins)], [DP + 128], p) == -1
    for same in (0, 1, 2, 6, 7):
        assert _call(native, op, ins, [ins[same]], p) == -1
    assert _call(native, op, ins, [None], p) == -1
    assert _call(native, op, ins, [DP + 128], None) == -1
    for zero in ("batch_size", "num_tokens"):
        assert _call(native, op, ins, [DP + 128], cf.MhaPagedQ8Params(**dict(ATTN_OK, **{zero: 0}))) == 0
        assert _call(native, op, ins, [DP + 128], cf.MhaPagedQ8Params(**dict(ATTN_OK, block_size=7, **{zero: 0}))) == -1


def test_the_numbers():
    """The oracle's codes at what decides a rounding, written out."""
    assert list(encode([1.0, 1.0625, 1.1875, 448.0, 447.0, 0.0, 2.0 ** -9, 2.0 ** -10, 1.01 * 2.0 ** -10, -1.0])) == \
        [0x38, 0x38, 0x3a, 0x7e, 0x7e, 0, 1, 0, 1, 0xb8]
    assert list(power_for(np.array([448.0, 448.1, 3.5, 3.51, 0.0, 65504.0, 2.0 ** -149]))) == [127, 128, 120, 121, 0, 135, 0]
    x = np.random.default_rng(1).standard_normal(4096) * 100
    assert (np.abs(VALUE[encode(x)] - x) <= np.maximum(np.abs(x) * 2.0 ** -4, 2.0 ** -10)).all()


# ------------------------------------------------------------------ the store (GPU) ---

class Store:
    """A cache in use, of random codes and powers, and calls on it."""

    def __init__(self, f16, H, d, P, block, n_pages, seed=1, pad=0, strides=None):
        self.rng = np.random.default_rng(seed)
        self.f16, self.dt = f16, np.float16 if f16 else np.float32
        self.H, self.d, self.P, self.block, self.n_pages, self.pad = H, d, P, block, n_pages, pad
        self.strides = strides or (0, 0, 0)
        n = n_pages * P
        self.cells = [self.rng.integers(0, 256, (n, H, d)).astype(U8) for _ in range(2)]
        self.powers = [self.rng.integers(110, 130, (n // block, H)).astype(U8) for _ in range(2)]
        page, row, head = self.at()
        self.raw = [np.full(page * n_pages, 0x55, U8) for _ in range(2)]
        for raw, c in zip(self.raw, self.cells):
            raw[self.index()] = c
        self.bufs = [dev(x) for x in self.raw + self.powers]

    def at(self):
        page, row, head = self.strides
        return page or self.P * self.H * self.d, row or self.H * self.d, head or self.d

    def index(self):
        """Byte of each (slot, head, value)."""
        page, row, head = self.at()
        s = np.arange(self.n_pages * self.P)
        return ((s // self.P * page + s % self.P * row)[:, None, None] + (np.arange(self.H) * head)[None, :, None] +
                np.arange(self.d)[None, None, :])

    def rows(self, T, std=1.0):
        w = self.H * self.d + self.pad
        x = self.rng.standard_normal((T, w)) * std * np.exp(self.rng.uniform(-2, 2, (T, 1)))
        return x.astype(self.dt)

    def call(self, k, v, slots, stream=None):
        """The operator and the oracle; both caches compared, what lies between cells too."""
        slots = np.asarray(slots, I32)
        page, row, head = self.strides
        p = cf.KvPageStoreQ8Params(num_tokens=len(slots), num_kv_heads=self.H, head_dim=self.d, page_size=self.P,
                                   num_pages=self.n_pages, block_size=self.block, kv_stride=self.H * self.d + self.pad,
                                   page_stride=page, row_stride=row, head_stride=head)
        name = "kv_page_store_q8_%s_cuda" % ("f16" if self.f16 else "f32")
        assert cf.call_op(name, [dev(k), dev(v), dev(slots)], self.bufs, p, stream) == 0
        if stream is not None:
            stream.synchronize()
        w = self.H * self.d
        for i, x in enumerate((k, v)):
            self.cells[i], self.powers[i] = ref_store(x[:, :w].reshape(-1, self.H, self.d), slots, self.cells[i],
                                                      self.powers[i], self.block)
            self.raw[i][self.index()] = self.cells[i]
            got = self.bufs[i].download().reshape(-1)
            assert (self.bufs[2 + i].download().reshape(self.powers[i].shape) == self.powers[i]).all(), "powers"
            assert same_codes(got, self.raw[i]), "codes"
            self.raw[i] = got.copy()                     # the signs of NaN as they are
            self.cells[i] = got[self.index()]


SHAPES = [(8, 128, 16, 16), (12, 64, 64, 32), (3, 64, 64, 64), (2, 128, 96, 48), (5, 33, 28, 7), (2, 256, 16, 16), (1, 80, 16, 4),
          (4, 8, 32, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,d,P,block", SHAPES)
def test_store_of_a_sequence(gpu, f16, H, d, P, block):
    """Prompt, single tokens, chunks that end inside blocks: each value against the oracle after each."""
    s = Store(f16, H, d, P, block, 40, seed=d)
    pages = s.rng.permutation(40)
    at = 0
    for n in (1, 1, 5, block, 1, 3 * block + 1, 70, 1, 1, 2):
        pos = at + np.arange(n)
        at += n
        assert at <= 40 * P
        s.call(s.rows(n), s.rows(n), pages[pos // P] * P + pos % P)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,d,P,block", [(8, 128, 16, 16), (2, 64, 128, 64), (3, 33, 32, 8)])
def test_store_of_many_rows(gpu, f16, H, d, P, block):
    """A step of many sequences, some of their rows not served, more rows than one workgroup's each."""
    s = Store(f16, H, d, P, block, 400 * 64 // P, seed=5)
    pages = s.rng.permutation(s.n_pages)
    slots, at = [], 0
    for n, past in ((1, 9), (300, 0), (1, 40), (517, 3), (1700, 15), (60, 64), (2, 5), (500, 1)):
        held = -(-(n + past) // P)
        pos = past + np.arange(n)
        own = pages[at + pos // P] * P + pos % P
        at += held
        slots += list(own if n != 60 else -np.ones(n, int))
    slots += [-1] * 7 + [s.n_pages * P, 2 ** 31 - 1, -2 ** 31]
    s.call(s.rows(len(slots)), s.rows(len(slots)), slots)
    s.call(s.rows(len(slots), 4.0), s.rows(len(slots), 0.1), slots)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d", [64, 36])
def test_store_rows_of_a_block_in_any_order(gpu, f16, d):
    s = Store(f16, 3, d, 32, 16, 8, seed=9)
    for take in (16, 9, 3):
        order = np.concatenate([b * 16 + s.rng.permutation(16)[:take] for b in s.rng.permutation(16)])
        s.call(s.rows(len(order)), s.rows(len(order)), order)
    s.call(s.rows(3), s.rows(3), [5, 3, 20])             # positions that were held are given again


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d", [64, 36])
def test_store_of_values_at_the_borders(gpu, f16, d):
    """Zeros, the type's largest and smallest, infinities and NaN, and blocks whose power grows by
    more than the codes have bits."""
    big, small = (65504.0, 2.0 ** -24) if f16 else (3.4028234e38, 2.0 ** -149)
    s = Store(f16, 2, d, 16, 16, 4, seed=10)
    rows = {name: s.rows(4) for name in ("zero", "big", "small", "inf", "nan", "mixed")}
    rows["zero"][:] = 0.0
    rows["big"][:, ::3] = big
    rows["big"][:, 1::3] = -big
    rows["small"][:] = small
    rows["inf"][:, ::2] = np.inf
    rows["inf"][:, 1::4] = -np.inf
    rows["nan"][:] = np.nan
    rows["mixed"][:, ::5] = np.inf
    rows["mixed"][:, 1::5] = big
    rows["mixed"][:, 2::5] = small
    for i, (a, b) in enumerate((("zero", "small"), ("small", "zero"), ("big", "nan"), ("inf", "mixed"), ("nan", "big"),
                                ("mixed", "inf"))):
        s.call(rows[a], rows[b], 16 * (i % 4) + np.arange(4))            # begins the block
        s.call(rows[b], rows[a], 16 * (i % 4) + 4 + np.arange(4))        # goes on with it
        s.call(s.rows(4), s.rows(4, 1000.0), 16 * (i % 4) + 8 + np.arange(4))
        assert np.isfinite(values(s.cells[0].reshape(4, 16, 2, d), s.powers[0].reshape(4, 1, 2))[i % 4, :4]).any() or a in ("nan",)
    for c, p in zip(s.cells, s.powers):                                   # what is read back fits the type
        v = values(c.reshape(4, 16, 2, d), p.reshape(4, 1, 2))
        v = v[:, :12]
        assert (np.isnan(v) | (np.abs(v) <= big)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_store_strides(gpu, f16):
    """Rows of a projection, pages of one tensor with K and V side by side, odd strides."""
    for d, pad, strides in ((64, 128, (16 * 3 * 64 * 2, 3 * 64 * 2, 128)), (64, 3, (16 * 200 + 5, 200, 66)), (33, 7, (0, 0, 0)),
                            (128, 0, (16 * 3 * 128 + 64, 3 * 128, 0)), (64, 1, (16, 64, 16 * 64))):
        if strides == (16, 64, 16 * 64):
            strides = (3 * 16 * 64, 64, 16 * 64)                          # heads outside positions
        s = Store(f16, 3, d, 16, 16, 6, seed=12, pad=pad, strides=strides)
        s.call(s.rows(40), s.rows(40), 5 + np.arange(40))
        s.call(s.rows(3), s.rows(3), 45 + np.arange(3))


# ------------------------------------------------------------------ attention (GPU) ---

KINDS = [(32, 8, 128, 16, 16), (8, 2, 64, 32, 16), (12, 12, 64, 64, 64), (16, 1, 128, 48, 48), (5, 5, 33, 28, 7), (4, 2, 128, 24, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,P,block", KINDS)
@pytest.mark.parametrize("new,past", [([1], [0]), ([1, 1, 1], [256, 0, 15]), ([3, 1, 4, 2], [90, 1500, 0, 700]),
                                      ([40, 1, 130], [0, 333, 17]), ([0, 5, 0], [3, 70, 0])])
def test_attention(gpu, f16, H, H_kv, d, P, block, new, past):
    c = PagedQ8(new, past, H, H_kv, d, P, f16, block=block, seed=d + len(new))
    c.check(c.run(max_new=max(new)))
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("new,past", [([1] * 5, [4000, 100, 2500, 1, 5000]), ([200], [1200]), ([300, 1, 7], [2000, 3000, 40]),
                                      ([64, 64], [64, 0])])
def test_attention_over_long_contexts(gpu, f16, d, new, past):
    c = PagedQ8(new, past, 8, 2, d, 16, f16, seed=3)
    c.check(c.run(max_new=max(new)))
    c.check(c.run(max_new=max(new), max_len=max(n + p for n, p in zip(new, past))))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d,n", [(64, 1), (128, 1), (64, 30), (128, 70), (40, 3)])
def test_attention_of_blocks_of_different_size(gpu, f16, d, n):
    """Powers from 2^-6 to 2^6 times each other, so that the largest block decides."""
    c = PagedQ8([n, n], [300, 37], 8, 2, d, 16, f16, seed=4, scales=6.0, k_std=0.05)
    c.check(c.run(max_new=n))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,P,block", KINDS[:2] + KINDS[4:])
@pytest.mark.parametrize("n", [1, 3, 50])
def test_attention_with_missing_pages(gpu, f16, H, H_kv, d, P, block, n):
    """Pages that are none, in the middle and at both ends; a sequence without any gives 0."""
    c = PagedQ8([n, n, n], [200, 180, 60], H, H_kv, d, P, f16, block=block, seed=6)
    c.table[0, [0, 3]] = [-1, c.n_pages]
    c.table[1, (180 + n - 1) // P] = 2 ** 31 - 1
    c.table[2, :] = -5
    got = c.run(max_new=n)
    c.check(got)
    assert (got[2 * n:3 * n] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("H,H_kv,d,P,block", [(8, 2, 64, 32, 16), (8, 2, 128, 16, 16), (4, 4, 36, 12, 6)])
@pytest.mark.parametrize("n", [2, 12, 90])
def test_nan_touches_only_rows_that_see_it(gpu, f16, H, H_kv, d, P, block, n):
    """NaN codes and NaN powers among the new positions' K and V and among the cached ones."""
    c = PagedQ8([n, n], [70, 100], H, H_kv, d, P, f16, block=block, seed=8)
    cells = [x.reshape(-1, H_kv, d) for x in c.codes]
    slot = lambda b, p: int(c.table[b, p // P]) * P + p % P
    cells[1][slot(0, 70 + n - 1), 0, 3] = 0xff                            # the last token's V
    cells[0][slot(0, 70 + n // 2), H_kv - 1, 5] = 0x7f                    # a K in the middle of the chunk
    cells[1][slot(1, 30), 0, 2] = 0x7f                                    # a cached V
    c.powers[1].reshape(-1, H_kv)[slot(1, 90) // block, H_kv - 1] = 255   # a cached block
    c.refresh()
    got = c.run(max_new=n).astype(np.float64)
    with np.errstate(invalid="ignore"):
        want, _, _ = ref_nan(c)
    assert (np.isnan(got[:c.start[-1]]) == np.isnan(want[:c.start[-1]])).all()
    clean = PagedQ8([n, n], [70, 100], H, H_kv, d, P, f16, block=block, seed=8)
    ok = ~np.isnan(want[:c.start[-1]])
    base = clean.run(max_new=n).astype(np.float64)[:c.start[-1]]
    want2, e32, e16 = ref_attn(clean.q, clean.kp, clean.vp, clean.table, clean.lens, clean.start, clean.scale)
    tol = 2 * ((e16 + 2.0 ** -11 * np.abs(want2) + 2.0 ** -25) if f16 else (e32 + 2.0 ** -24 * np.abs(want2)))
    assert (np.abs(got[:c.start[-1]] - base) <= tol[:c.start[-1]])[ok].all()


def ref_nan(c):
    """Where attention is NaN: a row that sees a NaN score all of it, one that sees a NaN V that dim."""
    out = np.zeros(c.q.shape)
    P, G = c.P, c.H // c.H_kv
    k, v = (x.reshape(-1, c.H_kv, c.d) for x in (c.kp, c.vp))
    for b in range(c.B):
        n, L = c.new[b], int(c.lens[b])
        at = c.table[b, np.arange(L) // P] * P + np.arange(L) % P
        for i in range(n):
            seen = at[:L - n + i + 1]
            for h in range(c.H):
                kn = np.isnan(k[seen, h // G]).any()
                out[c.start[b] + i, h] = np.where(kn | np.isnan(v[seen, h // G]).any(0), np.nan, 0.0)
    return out, None, None


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_powers_at_the_ends(gpu, f16):
    """Powers 0 and 1 (values next to nothing) beside ordinary ones, and a block of zeros with power 0."""
    for d, n in ((64, 1), (128, 20), (36, 2)):
        c = PagedQ8([n], [100], 4, 2, d, 16, f16, seed=13)
        P = c.P
        c.powers[0][c.table[0, 1]] = 0
        c.powers[1][c.table[0, 2]] = 1
        c.codes[1][c.table[0, 3]] = 0
        c.powers[1][c.table[0, 3]] = 0
        c.refresh()
        c.check(c.run(max_new=n))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d", [64, 128, 40])
def test_attention_strides(gpu, f16, d):
    """Q as part of a projection, K and V of a page side by side in one tensor."""
    H, H_kv, P, n = 8, 2, 16, 3
    for n in (3, 40):
        c = PagedQ8([n, 1], [100, 300], H, H_kv, d, P, f16, seed=14)
        wide = np.full((c.T, (H + 2 * H_kv) * d), 9.0, c.dt)
        wide[:, :H * d] = c.q.reshape(c.T, -1)
        both = np.full((c.n_pages, P, 2, H_kv, d), 0x7f, U8)
        both[:, :, 0], both[:, :, 1] = c.codes
        q, kv = dev(wide), dev(both)
        bufs = [q, kv, kv.ptr + H_kv * d] + c.bufs()[3:]
        p = c.params(max_new=n, q_stride=(H + 2 * H_kv) * d, page_stride=P * 2 * H_kv * d, row_stride=2 * H_kv * d)
        o = dev(np.full(c.q.shape, 7.0, c.dt))
        assert cf.call_op(c.op, bufs, [o], p) == 0
        c.check(o.download())


# ------------------------------------------------------------------ together (GPU) ---

class Step:
    """A server's device state with one layer's cache in 8 bits, and a step over it: pages, norms and
    rotation, store, attention.  Each operator is checked against its oracle on what the one before
    it left on the device."""

    def __init__(self, f16, B, T, H, H_kv, d, P, block, n_pages, width, seed=11):
        self.rng = np.random.default_rng(seed)
        self.f16, self.dt = f16, np.float16 if f16 else np.float32
        self.B, self.T, self.H, self.H_kv, self.d, self.P, self.block = B, T, H, H_kv, d, P, block
        self.n_pages, self.width = n_pages, width
        self.table = dev(np.full((B, width), -1, I32))
        self.ring = dev(self.rng.permutation(n_pages).astype(I32))
        self.counters = dev(np.array([0, n_pages, 0], I32))
        self.lens, self.new = dev(np.zeros(B, I32)), dev(np.zeros(B, I32))
        self.start, self.pos, self.slots = (dev(np.zeros(k, I32)) for k in (B + 1, T, T))
        self.qkv, self.o = dev(np.zeros((T, (H + 2 * H_kv) * d), self.dt)), dev(np.zeros((T, H, d), self.dt))
        self.q = dev(np.zeros((T, H, d), self.dt))
        self.gain = [dev((1 + 0.3 * self.rng.standard_normal(d)).astype(self.dt)) for _ in range(2)]
        self.pages = [dev(np.full((n_pages, P, H_kv, d), 0x7f, U8)) for _ in range(2)]
        self.powers = [dev(np.full((n_pages, P // block, H_kv), 255, U8)) for _ in range(2)]
        self.scale = float(np.float32(1.0 / math.sqrt(d)))
        self.cells = [x.download().reshape(-1, H_kv, d) for x in self.pages]
        self.held = [x.download().reshape(-1, H_kv) for x in self.powers]

    def launch(self, stream):
        t = "f16" if self.f16 else "f32"
        H, H_kv, d = self.H, self.H_kv, self.d
        es, w = np.dtype(self.dt).itemsize, (H + 2 * H_kv) * d
        m = cf.KvPageMapParams(batch_size=self.B, num_tokens=self.T, page_size=self.P, num_pages=self.n_pages,
                               max_pages=self.width, ring_size=self.n_pages)
        r = cf.QkNormRopeParams(num_tokens=self.T, num_heads=H, num_kv_heads=H_kv, head_dim=d, halves=1, norm=1, eps=1e-6,
                                rope_base=10000.0, q_stride=w, k_stride=w, k_out_stride=w)
        s = cf.KvPageStoreQ8Params(num_tokens=self.T, num_kv_heads=H_kv, head_dim=d, page_size=self.P, num_pages=self.n_pages,
                                   block_size=self.block, kv_stride=w)
        a = cf.MhaPagedQ8Params(batch_size=self.B, num_tokens=self.T, num_heads=H, num_kv_heads=H_kv, head_dim=d,
                                scale=self.scale, page_size=self.P, num_pages=self.n_pages, max_pages=self.width,
                                block_size=self.block)
        assert cf.call_op("kv_page_map_i32_cuda", [self.lens, self.new, self.counters],
                          [self.table, self.ring, self.lens, self.start, self.pos, self.slots, self.counters], m, stream) == 0
        # K in place, so that it stays beside V; Q to rows of its own.
        assert cf.call_op("qk_norm_rope_%s_cuda" % t, [self.qkv, self.qkv.ptr + H * d * es, self.pos] + self.gain + [None, None],
                          [self.q, self.qkv.ptr + H * d * es], r, stream) == 0
        assert cf.call_op("kv_page_store_q8_%s_cuda" % t, [self.qkv.ptr + H * d * es, self.qkv.ptr + (H + H_kv) * d * es, self.slots],
                          self.pages + self.powers, s, stream) == 0
        assert cf.call_op("mha_paged_attn_q8_%s_cuda" % t, [self.q] + self.pages + [self.table, self.lens, self.start] + self.powers,
                          [self.o], a, stream) == 0

    def feed(self, new):
        self.given = self.rng.standard_normal((self.T, (self.H + 2 * self.H_kv) * self.d)).astype(self.dt)
        self.qkv.upload(self.given)
        self.new.upload(np.asarray(new, I32))

    def check(self):
        H, H_kv, d = self.H, self.H_kv, self.d
        start, slots, pos = (x.download() for x in (self.start, self.slots, self.pos))
        n = int(start[-1])
        qkv, q = self.qkv.download(), self.q.download()
        before = self.given.reshape(self.T, -1, d)
        freq = frequencies(d, 10000.0)
        for x, y, g in ((before[:, :H], q, self.gain[0]), (before[:, H:H + H_kv], qkv[:, H * d:(H + H_kv) * d], self.gain[1])):
            want, err = ref_rows(x[:n], pos[:n], g.download(), None, 1, float(np.float32(1e-6)), d, 1, freq, 1.0)
            tol = err + (2.0 ** -11 * np.abs(want) + 2.0 ** -25 if self.f16 else 2.0 ** -24 * np.abs(want))
            assert (np.abs(y[:n].reshape(want.shape) - want) <= tol).all()
        k, v = qkv[:, H * d:(H + H_kv) * d].reshape(-1, H_kv, d), qkv[:, (H + H_kv) * d:].reshape(-1, H_kv, d)
        for i, x in enumerate((k, v)):
            self.cells[i], self.held[i] = ref_store(x, slots, self.cells[i], self.held[i], self.block)
            got = self.pages[i].download().reshape(self.cells[i].shape)
            assert (self.powers[i].download().reshape(self.held[i].shape) == self.held[i]).all()
            assert same_codes(got, self.cells[i])
            self.cells[i] = got
        if n == 0:
            return
        shape = (self.n_pages, self.P, H_kv, d)
        kv = [values(c.reshape(shape), p.reshape(self.n_pages, -1, H_kv)) for c, p in zip(self.cells, self.held)]
        want, e32, e16 = ref_attn(q, *kv, self.table.download(), self.lens.download(), start, self.scale)
        got = self.o.download()[:n].astype(np.float64)
        tol = e16 + 2.0 ** -11 * np.abs(want) + 2.0 ** -25 if self.f16 else e32 + 2.0 ** -24 * np.abs(want)
        assert (np.abs(got - want[:n]) <= tol[:n]).all()


STEPS = [[20, 1, 33, 7], [1, 1, 1, 1], [1, 40, 1, -1], [1, 1, 1, 12], [1, 1, -1, 1], [1, 3, 0, 1], [2, -1, 50, 1]]


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("captured", [False, True])
def test_steps_of_a_server(gpu, f16, captured):
    """Prompts, decoding, a chunk continued, requests that end and new ones in their pages, eager, and
    one recording replayed with eager work in between."""
    st = cf.Stream()
    s = Step(f16, 4, 72, 8, 2, 64, 32, 16, 9, 4)
    ex = c_void_p()
    if captured:
        s.feed([0] * 4)
        s.launch(st)                                   # sizes the workspace; adds no token
        st.synchronize()
        assert gpu.gpu_capture_begin(st.handle) == 0
        s.launch(st)
        assert gpu.gpu_capture_end(st.handle, ctypes.byref(ex)) == 0
    for new in STEPS:
        s.feed(new)
        if captured:
            assert gpu.gpu_graph_launch(ex, st.handle) == 0
        else:
            s.launch(st)
        st.synchronize()
        assert s.counters.download()[2] == 0
        s.check()
        other = PagedQ8([9, 1], [40, 700], 8, 2, 64, 16, f16)    # eager work on the default stream
        other.check(other.run())
    if captured:
        gpu.gpu_graph_exec_destroy(ex)


@pytest.mark.gpu
def test_two_streams_at_once(gpu):
    a, b = cf.Stream(), cf.Stream()
    x = PagedQ8([1, 1, 1], [3000, 900, 2000], 32, 8, 128, 16, True, seed=1)
    y = PagedQ8([1, 1], [2500, 4000], 32, 8, 128, 16, True, seed=2)
    bx, by = x.bufs(), y.bufs()
    ox, oy = dev(np.full(x.q.shape, 7.0, x.dt)), dev(np.full(y.q.shape, 7.0, y.dt))
    for _ in range(20):
        assert cf.call_op(x.op, bx, [ox], x.params(max_new=1), a) == 0
        assert cf.call_op(y.op, by, [oy], y.params(max_new=1), b) == 0
    a.synchronize()
    b.synchronize()
    x.check(ox.download())
    y.check(oy.download())
