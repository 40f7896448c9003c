"""qk_norm_rope_{f16,f32}_cuda: norms of Q and K and their rotation, against the formulas in 64 bits
(GPU), and what they refuse (CPU).

Tolerance, with u = 2^-24, n a normed value, S = scale |gain|, A the mean size of the head's
values: a sum over d <= 1024 values takes at most 16 additions per lane and 6 steps across lanes,
so a mean is off by at most 22 u A and a mean square by 24 u of itself (its squares rounded too),
a scale by half of that and 5 u for the division, the root and eps; x - mean, and three products
round once each.  So n is off by at most u (24 |n| + 24 S A) with norm 2, 24 u |n| with norm 1,
and with the bias by u of the sum.  cos and sin: the angle in half turns is rounded to FP32 once
(pi u) and sincospi is good to 2 ulp, 8 u together with the amplitude.  Turned: (|n0| + |n1|) 8 u
amplitude, two products and a sum 3 u of the same, and the pair's own errors.  The result rounds by
2^-11 (fp16; below 2^-14 by 2^-25) or 2^-24 of itself.
"""

import ctypes
import math
from ctypes import c_void_p

import numpy as np
import pytest

import cudaforge_amd as cf
from helpers import dev

U = 2.0 ** -24
F32 = np.float32


def frequencies(r, base, scaling=0, factor=1.0, original_len=1.0, low=1.0, high=4.0):
    """Radians per position of the r / 2 pairs, pair by pair (include/rope_ops.h)."""
    out = []
    for i in range(r // 2):
        f = base ** (-2.0 * i / r)
        if scaling == 1:
            f /= factor
        elif scaling == 2:
            t = original_len * f / (2 * math.pi)
            w = min(max((t - low) / (high - low), 0.0), 1.0)
            f = f * w + (1 - w) * f / factor
        elif scaling == 3:
            c = lambda t: r * math.log(original_len / (2 * math.pi * t)) / (2 * math.log(base))
            lo, hi = max(math.floor(c(high)), 0), min(math.ceil(c(low)), r - 1)
            g = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            f = f * (1 - g) + g * f / factor
        out.append(f)
    return np.array(out)


def ref_rows(x, pos, gain, bias, norm, eps, r, halves, freq, amp):
    """Rows (T, H, d) in 64 bits and what FP32 arithmetic may be off by; pos None: no rotation."""
    x = x.astype(np.float64)
    n, err = x, np.zeros_like(x)
    if norm:
        mean = x.mean(-1, keepdims=True) if norm == 2 else 0.0
        s = 1.0 / np.sqrt(((x - mean) ** 2).mean(-1, keepdims=True) + eps)
        g = 1.0 if gain is None else gain.astype(np.float64)
        n = (x - mean) * s * g
        err = U * (24 * np.abs(n) + (24 * s * np.abs(g) * np.abs(x).mean(-1, keepdims=True) if norm == 2 else 0.0))
        if norm == 2 and bias is not None:
            n = n + bias.astype(np.float64)
            err = err + U * np.abs(n)
    if pos is None:
        return n, err
    y, e = n.copy(), err.copy()
    a = pos.astype(np.float64)[:, None] * freq
    c, s = (f(a)[:, None, :] * amp for f in (np.cos, np.sin))
    i0 = np.arange(r // 2) if halves else 2 * np.arange(r // 2)
    i1 = i0 + (r // 2 if halves else 1)
    u, v = n[..., i0], n[..., i1]
    y[..., i0], y[..., i1] = u * c - v * s, u * s + v * c
    off = abs(amp) * (11 * U * (np.abs(u) + np.abs(v)) + err[..., i0] + err[..., i1])
    e[..., i0] = e[..., i1] = off
    return y, e


class Rows:
    """A call: rows of Q and K with strides, some of a negative position."""

    def __init__(self, T, H, H_kv, d, f16, r=0, halves=0, norm=1, base=10000.0, eps=1e-6, pads=(0, 0, 0, 0), seed=1,
                 gains=True, biases=True, far=100000, std=1.0, mean=0.0, **scaling):
        rng = np.random.default_rng(seed)
        self.dt = np.float16 if f16 else F32
        self.T, self.heads, self.d, self.norm, self.eps, self.base = T, (H, H_kv), d, norm, float(F32(eps)), base
        self.r, self.halves, self.f16, self.scaling = r or d, halves, f16, scaling
        self.step = [h * d + p for h, p in zip((H, H_kv, H, H_kv), pads)]
        self.pads = pads
        self.x = [(rng.standard_normal((T, s)) * std + mean).astype(self.dt) for s in self.step[:2]]
        self.y = [np.full((T, s), 7.0, self.dt) for s in self.step[2:]]
        self.gain = [(1 + 0.3 * rng.standard_normal(d)).astype(self.dt) if gains else None for _ in range(2)]
        self.bias = [(0.3 * rng.standard_normal(d)).astype(self.dt) if biases else None for _ in range(2)]
        self.pos = rng.integers(0, far, T).astype(np.int32)
        if T > 3:
            self.pos[[1, T - 1]] = -1
            self.pos[2] = 0
        amp = scaling.get("amplitude", 0.0)
        self.amp = float(F32(amp)) if amp else 1.0

    def params(self, in_place=False):
        out = self.step[:2] if in_place else self.step[2:]
        return cf.QkNormRopeParams(num_tokens=self.T, num_heads=self.heads[0], num_kv_heads=self.heads[1], head_dim=self.d,
                                   rotary_dim=self.r if self.r != self.d else 0, halves=self.halves, norm=self.norm,
                                   eps=self.eps, rope_base=self.base, q_stride=self.step[0], k_stride=self.step[1],
                                   q_out_stride=out[0], k_out_stride=out[1], **self.scaling)

    def run(self, in_place=False, stream=None, null_positions=False):
        x = [dev(a) for a in self.x]
        y = x if in_place else [dev(a) for a in self.y]
        ins = x + [None if null_positions else dev(self.pos)] + [None if a is None else dev(a) for a in self.gain + self.bias]
        op = "qk_norm_rope_%s_cuda" % ("f16" if self.f16 else "f32")
        assert cf.call_op(op, ins, y, self.params(in_place), stream) == 0
        if stream is not None:
            stream.synchronize()
        return [a.download() for a in y]

    def check(self, got, in_place=False):
        kw = {k: v for k, v in self.scaling.items() if k != "amplitude"}
        freq = frequencies(self.r, float(F32(self.base)), **kw) if self.base else None
        pos = self.pos if self.base else None
        for i in range(2):
            H = self.heads[i]
            w = H * self.d
            before = self.x[i] if in_place else self.y[i]
            left = (self.pos < 0) if self.base else np.zeros(self.T, bool)
            assert (got[i][left] == before[left]).all(), "rows of negative positions"
            assert (got[i][:, w:] == before[:, w:]).all(), "what lies between rows"
            want, err = ref_rows(self.x[i][:, :w].reshape(self.T, H, self.d), pos, self.gain[i], self.bias[i], self.norm,
                                 self.eps, self.r, self.halves, freq, self.amp)
            tol = err + (2.0 ** -11 * np.abs(want) + 2.0 ** -25 if self.f16 else U * np.abs(want) + 2.0 ** -140)
            off = np.abs(got[i][:, :w].reshape(want.shape).astype(np.float64) - want)
            bad = ~(off <= tol) & ~left[:, None, None]
            assert not bad.any(), (i, int(bad.sum()), np.argwhere(bad)[0], off[bad][0], tol[bad][0], want[bad][0])


# ------------------------------------------------------------------ refusals (CPU) ---

DUMMY = ctypes.create_string_buffer(4096)
DP = ctypes.addressof(DUMMY)
OK = dict(num_tokens=4, num_heads=8, num_kv_heads=2, head_dim=64, rotary_dim=32, halves=1, norm=1, eps=1e-6,
          rope_base=10000.0, scaling=2, factor=8.0, original_len=8192.0, low=1.0, high=4.0, amplitude=1.0)
OPS = ["qk_norm_rope_f16_cuda", "qk_norm_rope_f32_cuda"]


def _call(native, name, ins, outs, params):
    a, b = (c_void_p * len(ins))(*ins), (c_void_p * len(outs))(*outs)
    p = ctypes.cast(ctypes.pointer(params), c_void_p) if params is not None else None
    return native.operator_find(name.encode()).contents.func(a, b, p, None)


@pytest.mark.parametrize("change", [
    dict(num_tokens=-1), dict(num_tokens=1 << 31), dict(num_heads=-1), dict(num_kv_heads=-1), dict(num_heads=0, num_kv_heads=0),
    dict(num_heads=65536), dict(head_dim=0), dict(head_dim=1025), dict(rotary_dim=31), dict(rotary_dim=66), dict(rotary_dim=-2),
    dict(head_dim=512, rotary_dim=258), dict(head_dim=63, rotary_dim=0),
    dict(halves=2), dict(halves=-1), dict(norm=3), dict(norm=-1), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf),
    dict(rope_base=-1.0), dict(rope_base=math.nan), dict(rope_base=math.inf), dict(scaling=4), dict(scaling=-1),
    dict(factor=0.0), dict(factor=-2.0), dict(factor=math.inf), dict(original_len=0.0), dict(low=0.0), dict(low=4.0),
    dict(low=5.0), dict(high=math.inf), dict(scaling=3, rope_base=1.0), dict(scaling=3, rope_base=0.5),
    dict(amplitude=math.nan), dict(amplitude=math.inf), dict(q_stride=-8), dict(k_stride=-8), dict(q_out_stride=-8),
    dict(k_out_stride=-8),
])
@pytest.mark.parametrize("op", OPS)
def test_refuses_parameters(native, op, change):
    ins, outs = [DP + 64 * i for i in range(7)], [DP + 1024, DP + 2048]
    assert _call(native, op, ins, outs, cf.QkNormRopeParams(**dict(OK, **change))) == -1


@pytest.mark.parametrize("op", OPS)
def test_refuses_missing_arrays(native, op):
    ins, outs = [DP + 64 * i for i in range(7)], [DP + 1024, DP + 2048]
    p = cf.QkNormRopeParams(**OK)
    for i in range(3):
        assert _call(native, op, [None if j == i else x for j, x in enumerate(ins)], outs, p) == -1
    for o in range(2):
        assert _call(native, op, ins, [None if j == o else x for j, x in enumerate(outs)], p) == -1
    assert _call(native, op, ins, outs, None) == -1
    assert _call(native, op, ins, [ins[0], outs[1]], cf.QkNormRopeParams(**dict(OK, q_stride=512, q_out_stride=768))) == -1
    assert _call(native, op, ins, [outs[0], ins[1]], cf.QkNormRopeParams(**dict(OK, k_stride=256))) == -1
    # Nothing to do, with whatever may be absent.
    none = [None, ins[1], None, None, None, None, None]
    assert _call(native, op, none, [None, outs[1]],
                 cf.QkNormRopeParams(**dict(OK, num_tokens=0, num_heads=0, rope_base=0.0, rotary_dim=0))) == 0


@pytest.mark.parametrize("op", OPS)
def test_refuses_the_others_array(native, op):
    ins, outs, p = [DP + 64 * i for i in range(7)], [DP + 1024, DP + 2048], cf.QkNormRopeParams(**OK)
    for pair in ([outs[0], outs[0]], [ins[1], outs[1]], [outs[0], ins[0]], [ins[1], ins[0]]):
        assert _call(native, op, ins, pair, p) == -1


def test_layout(native):
    assert ctypes.sizeof(cf.QkNormRopeParams) == 112
    for op in OPS:
        e = native.operator_find(op.encode()).contents
        assert e.data_type == (b"f16" if "f16" in op else b"f32")


def test_frequencies_meet_at_their_borders():
    """What holds without arithmetic: pairs that turn often keep their frequency, slow ones are divided."""
    f = frequencies(128, 500000.0)
    for scaling in (2, 3):
        g = frequencies(128, 500000.0, scaling, 8.0, 8192.0, 1.0, 4.0)
        turns = 8192.0 * f / (2 * math.pi)
        assert np.allclose(g[turns > 8], f[turns > 8], rtol=1e-15) and (g <= f * (1 + 1e-15)).all()
        assert np.allclose(g[turns < 0.5], f[turns < 0.5] / 8, rtol=1e-15)
    assert np.allclose(frequencies(64, 10000.0, 1, 4.0), frequencies(64, 10000.0) / 4, rtol=1e-15)


# ------------------------------------------------------------------ against 64 bits (GPU) ---

@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("norm", [0, 1, 2])
@pytest.mark.parametrize("halves", [0, 1])
@pytest.mark.parametrize("H,H_kv,d,r", [(32, 8, 128, 128), (12, 12, 64, 32), (3, 1, 256, 64), (8, 2, 96, 48), (5, 5, 33, 10),
                                        (2, 2, 8, 2), (4, 1, 512, 256), (16, 16, 64, 16), (1, 1, 1024, 256), (7, 3, 80, 80)])
def test_rows(gpu, f16, norm, halves, H, H_kv, d, r):
    c = Rows(13, H, H_kv, d, f16, r, halves, norm)
    c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("scaling", [
    dict(scaling=1, factor=4.0), dict(scaling=2, factor=8.0, original_len=8192.0, low=1.0, high=4.0),
    dict(scaling=3, factor=16.0, original_len=4096.0, low=1.0, high=32.0, amplitude=1.2772589),
    dict(scaling=3, factor=2.0, original_len=64.0, low=1.0, high=32.0), dict(scaling=0, amplitude=-0.5)])
@pytest.mark.parametrize("halves", [0, 1])
def test_scalings(gpu, f16, scaling, halves):
    for base in (10000.0, 500000.0):
        c = Rows(29, 8, 2, 128, f16, 0, halves, 1, base=base, far=1 << 20, **scaling)
        c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("T", [1, 2, 63, 700])
@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("in_place", [False, True])
def test_strides_and_places(gpu, f16, T, d, in_place):
    for pads in ((0, 0, 0, 0), (64, 192, 128, 32), (3, 5, 1, 7)):
        c = Rows(T, 6, 2, d, f16, 0, 1, 2, pads=pads, seed=T)
        c.check(c.run(in_place), in_place)


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d", [64, 31])
def test_what_may_be_absent(gpu, f16, d):
    """No Q or no K, no gains, no biases, no rotation and no positions."""
    for H, H_kv in ((4, 0), (0, 4)):
        c = Rows(9, H, H_kv, d, f16, 2, 0, 1)
        c.check(c.run())
    c = Rows(9, 4, 2, d, f16, 2, 1, 2, gains=False)
    c.check(c.run())
    c = Rows(9, 4, 2, d, f16, 2, 1, 2, biases=False)
    c.check(c.run())
    for norm in (0, 2):
        c = Rows(9, 4, 2, d, f16, norm=norm, base=0.0)
        c.check(c.run(null_positions=True))


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d", [128, 36])
@pytest.mark.parametrize("norm", [1, 2])
def test_values_far_from_one(gpu, f16, d, norm):
    """Large and small heads, heads of zeros, a mean that is many times the spread."""
    for std, mean, eps in ((300.0, 0.0, 1e-6), (1e-3, 0.0, 1e-6), (1.0, 20.0, 1e-5), (0.0, 0.0, 1e-6), (0.0, 0.0, 1.0)):
        c = Rows(9, 4, 2, d, f16, 0, 1, norm, std=std, mean=mean, eps=eps)
        c.check(c.run())


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
@pytest.mark.parametrize("d", [128, 36])
def test_one_heads_infinity_stays_there(gpu, f16, d):
    c = Rows(9, 4, 2, d, f16, 0, 1, 1)
    clean = c.run()
    c.x[0][4, d + 3] = np.inf
    c.x[1][5, 2] = np.nan
    got = c.run()
    assert np.isnan(got[0][4, d:2 * d]).any() and np.isnan(got[1][5, :d]).all()
    for i, (t, h) in enumerate(((4, 1), (5, 0))):
        same = np.ones(got[i].shape, bool)
        same[t, h * d:(h + 1) * d] = False
        assert (got[i][same] == clean[i][same]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_far_positions(gpu, f16):
    """The last position of 31 bits: the angle is good to 2^31 f 2^-52 turns there, 5e-7 of one."""
    c = Rows(5, 2, 1, 64, f16, 0, 0, 0, far=2 ** 31 - 1)
    c.pos[0] = 2 ** 31 - 1
    got = c.run()
    for i in range(2):
        H = c.heads[i]
        x = c.x[i].reshape(5, H, 64)
        want, err = ref_rows(x, c.pos, None, None, 0, c.eps, 64, 0, frequencies(64, 10000.0), 1.0)
        size = np.repeat(np.abs(x.astype(np.float64)).reshape(5, H, 32, 2).sum(-1), 2, -1)
        tol = err + size * 2 * math.pi * 2.0 ** 31 * 2.0 ** -51 + (2.0 ** -11 if f16 else U) * np.abs(want) + 2.0 ** -25
        ok = np.abs(got[i].reshape(5, H, 64) - want) <= tol
        assert ok[c.pos >= 0].all()


@pytest.mark.gpu
@pytest.mark.parametrize("f16", [False, True])
def test_many_rows_and_two_streams(gpu, f16):
    a, b = cf.Stream(), cf.Stream()
    x, y = Rows(5001, 12, 12, 64, f16, 0, 1, 1, seed=3), Rows(3001, 32, 8, 128, f16, 64, 0, 2, seed=4)
    bufs = []
    for c, st in ((x, a), (y, b)):
        ins = [dev(v) for v in c.x] + [dev(c.pos)] + [dev(v) for v in c.gain + c.bias]
        outs = [dev(v) for v in c.y]
        bufs.append((c, st, ins, outs))
    for _ in range(10):
        for c, st, ins, outs in bufs:
            assert cf.call_op("qk_norm_rope_%s_cuda" % ("f16" if f16 else "f32"), ins, outs, c.params(), st) == 0
    for c, st, ins, outs in bufs:
        st.synchronize()
        c.check([o.download() for o in outs])
