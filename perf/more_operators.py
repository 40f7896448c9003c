"""The operators around the 8-bit paged KV cache: what their speed is judged on.

Between a layer's projection and its attention over a paged cache of 8-bit numbers stand
three operators (the pages of the step come from kv_page_map_i32_cuda):

  turn   qk_norm_rope_{f16,f32}_cuda: the rows of Q and K, each head normalised by itself and
         turned by its token's position, in one pass.
  store  kv_page_store_q8_{f16,f32}_cuda: new K and V rows into pages of e4m3 numbers, one
         power of two for each block of positions and head.
  attn   mha_paged_attn_q8_{f16,f32}_cuda: chunks of new tokens (one token in a decode step)
         over block tables of such pages, causal by position.

`run` computes them from elementary torch operations, or, where `own` is true, calls the
operators through operator_find(...)->func as a C program or a ctypes binding does: slot
arrays and params structs are made once, a pass is the call alone.
"""

from __future__ import annotations

import ctypes
import math
import random

import torch

own = False


# ------------------------------------------------------------------------- the cases ---

def listed():
    return [
        # The rows of a decode step, Llama-3-8B-shaped heads: positions scaled by their wavelength
        # for a long context, pairs in halves; what counts is latency.
        dict(name="turn_f16_t16", kind="turn", dtype="f16", T=16, H=32, H_kv=8, d=128, r=128, halves=True, norm=1,
             scaling=2),
        # A prefill step's rows of the same layer.
        dict(name="turn_f16_t8192", kind="turn", dtype="f16", T=8192, H=32, H_kv=8, d=128, r=128, halves=True, norm=1,
             scaling=2),
        # FP32 rows of GPT-2-small-shaped heads: half of the head turned in neighbouring pairs, norms
        # with a mean, an odd number of rows.
        dict(name="turn_f32_t1001", kind="turn", dtype="f32", T=1001, H=12, H_kv=12, d=64, r=32, halves=False, norm=2,
             scaling=0),
        # Sixteen sequences append one token each to blocks that they have begun.
        dict(name="store_f16_b16", kind="store", dtype="f16", B=16, H_kv=8, d=128, P=16, block=16, new="1",
             past="4095 1000 2900 333"),
        # Prompt chunks of a prefill step, 8192 rows in all, some of them not at a block's start.
        dict(name="store_f16_b4_t8192", kind="store", dtype="f16", B=4, H_kv=8, d=128, P=16, block=16,
             new="2048 3000 1900 1244", past="0 517 2048 5"),
        # FP32 rows, GPT-2-small-shaped, larger pages and blocks, odd lengths.
        dict(name="store_f32_b3", kind="store", dtype="f32", B=3, H_kv=12, d=64, P=64, block=32, new="300 411 129",
             past="0 517 1000"),
        # The smallest attention: one FP32 token, GPT-2-small shape, 257 positions.
        dict(name="attn_f32_b1", kind="attn", dtype="f32", B=1, H=12, H_kv=12, d=64, P=16, block=16, new="1", past="256"),
        # A decode step of 16 requests at lengths up to 4096, Llama-3-8B-shaped layer.
        dict(name="attn_f16_decode_b16", kind="attn", dtype="f16", B=16, H=32, H_kv=8, d=128, P=16, block=16,
             new="1", past="4095 4095 2900 4095 2500 4095 1777 4095"),
        # Four guessed tokens verified per request, over long contexts, larger pages and blocks.
        dict(name="attn_f16_verify_b4", kind="attn", dtype="f16", B=4, H=32, H_kv=8, d=128, P=64, block=64,
             new="4", past="28900 1501 15000 9001"),
        # A server's mixed step: prompt chunks of uneven length among decoding requests.
        dict(name="attn_f16_mixed_b35", kind="attn", dtype="f16", B=35, H=32, H_kv=8, d=128, P=16, block=16,
             new="1 1 1 1 517 1 1 1 1 1 1 230 1 1 1 1", past="3000 700 1900 4000 512 90 2200"),
        # The largest: a chunk of a long prompt (GQA, head size 128) over what is cached.
        dict(name="attn_f16_chunk_b1", kind="attn", dtype="f16", B=1, H=32, H_kv=8, d=128, P=16, block=16, new="2048",
             past="6144"),
        # FP32 chunks, GPT-2-medium-shaped layer, odd lengths.
        dict(name="attn_f32_chunk_b3", kind="attn", dtype="f32", B=3, H=16, H_kv=16, d=64, P=32, block=16,
             new="300 411 129", past="0 517 1000"),
    ]


# Head layouts the repository's configurations name (GPT-2 small / BERT-base, GPT-2 medium,
# Llama-3-8B) and a grouped one in between.
_HEADS = [(12, 12, 64), (16, 16, 64), (16, 4, 128), (32, 8, 128)]
# Most query-key pairs, times heads and head size, of one drawn attention: the largest listed case's.
_MOST_F16 = 32 * 128 * (2048 * 6144 + 2048 * 2049 // 2)
_MOST_F32 = _MOST_F16 // 24


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["turn", "turn", "store", "store", "attn", "attn", "attn", "attn"])
    H, H_kv, d = rng.choice(_HEADS)
    dtype = rng.choice(["f16", "f16", "f16", "f32"])
    if kind == "turn":
        return dict(kind=kind, dtype=dtype, T=_log_int(rng, 1, 8192 if dtype == "f16" else 4096), H=H, H_kv=H_kv, d=d,
                    r=rng.choice([d, d, d // 2, d // 4]), halves=rng.random() < 0.5, norm=rng.choice([0, 1, 1, 2]),
                    scaling=rng.randrange(4))
    P = rng.choice([16, 16, 32, 64, 128])
    block = rng.choice([x for x in (16, 16, 32, 64) if x <= P])
    base = dict(kind=kind, dtype=dtype, H_kv=H_kv, d=d, P=P, block=block)
    if kind == "attn":
        base["H"] = H
    form = rng.choice(["decode", "decode", "verify", "chunk", "chunk", "mixed"])
    most = (_MOST_F16 if dtype == "f16" else _MOST_F32) // (H * d)
    if form in ("decode", "verify"):
        B = _log_int(rng, 1, 64)
        longest = max(16, min(32768, (131072 if H_kv * d <= 1024 else 65536) // B))
        new = [1] if form == "decode" else [rng.randrange(2, 9) for _ in range(B)]
        past = [_log_int(rng, 1, longest) for _ in range(B)]
    elif form == "chunk":
        B = _log_int(rng, 1, 8)
        n = _log_int(rng, 9, 2048 if kind == "attn" else 8192 // B)
        new = [max(1, int(n * rng.uniform(0.3, 1.0))) for _ in range(B)]
        past = [rng.choice([0, _log_int(rng, 1, 8192)]) for _ in range(B)]
    else:
        B = _log_int(rng, 4, 48)
        n = _log_int(rng, 16, 768)
        new = [max(1, int(n * rng.uniform(0.3, 1.0))) if rng.random() < 0.15 else 1 for _ in range(B)]
        past = [_log_int(rng, 1, 4096) for _ in range(B)]
    # No draw does more than the largest listed case of its type.
    while kind == "attn" and sum(new[i % len(new)] * (past[i % len(past)] + new[i % len(new)]) for i in range(B)) > most:
        new = [max(1, x // 2) for x in new]
        past = [x // 2 for x in past]
    return dict(base, B=B, new=" ".join(map(str, new)), past=" ".join(map(str, past)))


# ---------------------------------------------------------------------- inputs, state ---

def _ceil(a, b):
    return -(-a // b)


def _lens(case):
    """New tokens and cached positions per sequence: the case's lists, repeated to B entries."""
    new, past = ([int(x) for x in case[k].split()] for k in ("new", "past"))
    return ([new[b % len(new)] for b in range(case["B"])], [past[b % len(past)] for b in range(case["B"])])


_BASE, _EPS = 500000.0, 1e-6
# What a scaling of the positions for a long context goes by: eight times the context that the
# model was trained on, in turns over which a pair's frequency is kept or divided.
_FACTOR, _ORIGINAL, _LOW, _HIGH = 8.0, 8192.0, 1.0, 4.0


def _amplitude(case):
    return 0.1 * math.log(_FACTOR) + 1.0 if case["scaling"] == 3 else 1.0


def _torch_dtype(case):
    return torch.float16 if case["dtype"] == "f16" else torch.float32


def _power(byte):
    """2^(byte - 127) in FP32, from its bits."""
    return (byte.to(torch.int32) << 23).view(torch.float32)


def _pages(case, n_pages, g):
    """A cache that is in use: e4m3 numbers and the powers of its blocks, heads of different size."""
    P, block, H_kv, d = case["P"], case["block"], case["H_kv"], case["d"]
    size = torch.exp(0.7 * torch.randn(H_kv, 1, device="cuda", generator=g))
    x = torch.randn(n_pages, P // block, block, H_kv, d, device="cuda", generator=g) * size
    m, k = torch.frexp(x.abs().amax((2, 4)))
    byte = (k - 9 + (m > 0.875) + 127).to(torch.uint8)
    code = (x / _power(byte)[:, :, None, :, None]).to(torch.float8_e4m3fn)
    return code.view(n_pages, P, H_kv, d), byte


def _inputs(case, seed):
    """The case's tensors by name, from the seed alone.  Pages are handed out in random order,
    as they are in a server that has run for a while."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _torch_dtype(case)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    def mk(*shape):
        return torch.randn(shape, dtype=dt, device="cuda", generator=g)

    H_kv, d = case["H_kv"], case["d"]
    if case["kind"] == "turn":
        T, H = case["T"], case["H"]
        pos = torch.randint(0, 65536, (T,), device="cuda", generator=g).to(torch.int32)
        gains = {n: (1.0 + 0.2 * torch.randn(d, device="cuda", generator=g)).to(dt) for n in ("gq", "gk")}
        shifts = {n: (0.2 * torch.randn(d, device="cuda", generator=g)).to(dt) for n in ("bq", "bk")}
        return dict(q=mk(T, H, d), k=mk(T, H_kv, d), pos=pos, **gains, **shifts)
    P, block = case["P"], case["block"]
    new, past = _lens(case)
    lens = [n + p for n, p in zip(new, past)]
    held = [_ceil(n, P) for n in lens]
    n_pages, width = sum(held) + 8, max(held)
    handed = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32)[:sum(held)]
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    t = {}
    t["kp"], t["ks"] = _pages(case, n_pages, g)
    t["vp"], t["vs"] = _pages(case, n_pages, g)
    if case["kind"] == "attn":
        t["table"] = torch.full((case["B"], width), -1, dtype=torch.int32, device="cuda")
        t["table"][torch.arange(width, device="cuda")[None, :] < ints(held)[:, None]] = handed
        return dict(t, q=mk(start[-1], case["H"], d), lens=ints(lens), start=ints(start))
    # The slots of the new rows, and (which a program knows that knows its lengths) the blocks
    # that they touch.
    first, at, slot, touched, place = 0, [], [], [], []
    for n, p, h in zip(new, past, held):
        at += [first + (p + i) // P for i in range(n)]
        slot += [(p + i) % P for i in range(n)]
        b0 = p // block
        place += [len(touched) + (p + i) // block - b0 for i in range(n)]
        touched += [(first + b * block // P, b * block % P // block) for b in range(b0, (p + n - 1) // block + 1)]
        first += h
    slots = handed[ints(at).long()] * P + ints(slot)
    pages, inner = (ints([x[i] for x in touched]) for i in (0, 1))
    blocks = handed[pages.long()] * (P // block) + inner
    T = start[-1]
    return dict(t, k=mk(T, H_kv, d) * torch.exp(0.7 * mk(1, H_kv, 1)), v=mk(T, H_kv, d), slots=slots, blocks=blocks.long(),
                place=ints(place).long())


def prepare(case, seed):
    t = _inputs(case, seed)
    state = dict(case=case, t=t)
    if case["kind"] == "turn":
        t["qo"], t["ko"] = torch.empty_like(t["q"]), torch.empty_like(t["k"])
        state["out"] = dict(q=t["qo"], k=t["ko"])
    elif case["kind"] == "store":
        state["out"] = {n: t[n] for n in ("kp", "vp", "ks", "vs")}
    else:
        t["o"] = torch.empty_like(t["q"])
        state["out"] = dict(o=t["o"])
        new, past = _lens(case)
        state["new"], state["lens"] = new, [n + p for n, p in zip(new, past)]
    if own:
        state["call"] = _own_call(case, t)
    return state


def _own_call(case, t):
    """The operator call of a case, ready to make: (function, inputs, outputs, params)."""
    import cudaforge_amd as cf

    cf.init_gpu(0)
    if case["kind"] == "turn":
        name = "qk_norm_rope_%s_cuda" % case["dtype"]
        ins = [t["q"], t["k"], t["pos"]]
        ins += [t["gq"], t["gk"]] if case["norm"] else [None, None]
        ins += [t["bq"], t["bk"]] if case["norm"] == 2 else [None, None]
        outs = [t["qo"], t["ko"]]
        params = cf.QkNormRopeParams(num_tokens=case["T"], num_heads=case["H"], num_kv_heads=case["H_kv"], head_dim=case["d"],
                                     rotary_dim=case["r"], halves=int(case["halves"]), norm=case["norm"], eps=_EPS,
                                     rope_base=_BASE, scaling=case["scaling"], factor=_FACTOR, original_len=_ORIGINAL,
                                     low=_LOW, high=_HIGH, amplitude=_amplitude(case))
    elif case["kind"] == "store":
        name = "kv_page_store_q8_%s_cuda" % case["dtype"]
        ins = [t["k"], t["v"], t["slots"]]
        outs = [t["kp"], t["vp"], t["ks"], t["vs"]]
        params = cf.KvPageStoreQ8Params(num_tokens=t["k"].shape[0], num_kv_heads=case["H_kv"], head_dim=case["d"],
                                        page_size=case["P"], num_pages=t["kp"].shape[0], block_size=case["block"])
    else:
        name = "mha_paged_attn_q8_%s_cuda" % case["dtype"]
        ins = [t["q"], t["kp"], t["vp"], t["table"], t["lens"], t["start"], t["ks"], t["vs"]]
        outs = [t["o"]]
        params = cf.MhaPagedQ8Params(batch_size=case["B"], num_tokens=t["q"].shape[0], num_heads=case["H"],
                                     num_kv_heads=case["H_kv"], head_dim=case["d"], scale=1.0 / math.sqrt(case["d"]),
                                     page_size=case["P"], num_pages=t["kp"].shape[0], max_pages=t["table"].shape[1],
                                     block_size=case["block"], max_new=max(_lens(case)[0]))

    def slots(tensors):
        arr = (ctypes.c_void_p * len(tensors))(*[None if x is None else x.data_ptr() for x in tensors])
        return ctypes.cast(arr, ctypes.POINTER(ctypes.c_void_p))

    return cf.find_op(name).func, slots(ins), slots(outs), ctypes.cast(ctypes.pointer(params), ctypes.c_void_p)


# --------------------------------------------------------------------- the plain forms ---

def _plain_frequencies(case, dev):
    """Radians per position of each pair, in 64 bits."""
    r = case["r"]
    f = _BASE ** (-torch.arange(0, r, 2, dtype=torch.float64, device=dev) / r)
    if case["scaling"] == 1:
        return f / _FACTOR
    if case["scaling"] == 2:
        keep = ((_ORIGINAL * f / (2 * math.pi) - _LOW) / (_HIGH - _LOW)).clamp(0, 1)
        return f * (keep + (1 - keep) / _FACTOR)
    if case["scaling"] == 3:
        lo, hi = (r * math.log(_ORIGINAL / (2 * math.pi * turns)) / (2 * math.log(_BASE)) for turns in (_HIGH, _LOW))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), r - 1)
        ramp = ((torch.arange(r // 2, dtype=torch.float64, device=dev) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f * (1 - ramp + ramp / _FACTOR)
    return f


def _plain_turn(case, x, pos, gain, shift):
    r, y = case["r"], x.float()
    if case["norm"] == 2:
        y = y - y.mean(-1, keepdim=True)
    if case["norm"]:
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + _EPS) * gain.float()
    if case["norm"] == 2:
        y = y + shift.float()
    angle = pos.double()[:, None] * _plain_frequencies(case, x.device)
    c, s = ((f(angle) * _amplitude(case)).float()[:, None, :] for f in (torch.cos, torch.sin))
    head, rest = y[..., :r], y[..., r:]
    if case["halves"]:
        a, b = head[..., :r // 2], head[..., r // 2:]
        head = torch.cat((a * c - b * s, a * s + b * c), -1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        head = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    return torch.cat((head, rest), -1)


def _plain_store(case, x, pages, powers, t):
    """Largest size of each touched block and head, its power of two, what the block held at that
    power, and the rows over it."""
    block, H_kv, d = case["block"], case["H_kv"], case["d"]
    cells = pages.view(torch.uint8).view(-1, block, H_kv, d)
    bytes_ = powers.view(-1, H_kv)
    x, n = x.float(), t["blocks"].numel()
    most = torch.zeros(n, H_kv, device=x.device).index_reduce_(0, t["place"], x.abs().amax(-1), "amax")
    m, k = torch.frexp(most)
    need = torch.where(most > 0, (k - 9 + (m > 0.875) + 127).clamp(0, 254), 0)
    begun = torch.zeros(n, dtype=torch.int32, device=x.device)
    begun.index_reduce_(0, t["place"], (t["slots"] % block == 0).to(torch.int32), "amax")
    old = bytes_[t["blocks"]].to(torch.int32)
    byte = torch.where(begun[:, None] > 0, need, torch.maximum(old, need))
    shift = torch.where(begun[:, None] > 0, 0, old - byte) + 127
    held = cells[t["blocks"]].view(torch.float8_e4m3fn).float() * _power(shift)[:, None, :, None]
    cells[t["blocks"]] = held.to(torch.float8_e4m3fn).view(torch.uint8)
    bytes_[t["blocks"]] = byte.to(torch.uint8)
    code = (x / _power(byte)[t["place"]][:, :, None]).to(torch.float8_e4m3fn)
    cells.view(-1, H_kv, d)[t["slots"].long()] = code.view(torch.uint8)


def _plain_cells(pages, powers, at, L):
    """Positions 0 .. L - 1 of the pages `at` in FP32: (H_kv, L, d)."""
    n, P, H_kv, d = len(at), pages.shape[1], pages.shape[2], pages.shape[3]
    x = pages.view(torch.uint8)[at].view(torch.float8_e4m3fn).float().view(n, powers.shape[1], -1, H_kv, d)
    return (x * _power(powers[at])[:, :, None, :, None]).view(n * P, H_kv, d)[:L].transpose(0, 1)


def _plain_attn(case, state):
    t, P, H, H_kv, d = state["t"], case["P"], case["H"], case["H_kv"], case["d"]
    scale, g = 1.0 / math.sqrt(d), H // H_kv
    row = 0
    for b, (n, L) in enumerate(zip(state["new"], state["lens"])):
        at = t["table"][b, :_ceil(L, P)].long()
        k = _plain_cells(t["kp"], t["ks"], at, L).transpose(1, 2).contiguous()
        v = _plain_cells(t["vp"], t["vs"], at, L).contiguous()
        q = t["q"][row:row + n].float().reshape(n, H_kv, g, d).permute(1, 2, 0, 3).reshape(H_kv, g * n, d)
        s = torch.matmul(q, k) * scale
        if n > 1:
            hidden = torch.arange(L, device=s.device) > (L - n + torch.arange(n, device=s.device))[:, None]
            s.view(H_kv, g, n, L).masked_fill_(hidden, -math.inf)
        s = torch.exp(s - s.amax(-1, keepdim=True))
        o = torch.matmul(s, v) / s.sum(-1, keepdim=True)
        t["o"][row:row + n] = o.view(H_kv, g, n, d).permute(2, 0, 1, 3).reshape(n, H, d).to(t["o"].dtype)
        row += n


def run(state):
    case, t = state["case"], state["t"]
    if own:
        func, ins, outs, params = state["call"]
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)   # a stream_t is one pointer
        rc = func(ins, outs, params, ctypes.addressof(stream))
        if rc != 0:
            raise RuntimeError("operator returned %d" % rc)
    elif case["kind"] == "turn":
        t["qo"].copy_(_plain_turn(case, t["q"], t["pos"], t["gq"], t["bq"]))
        t["ko"].copy_(_plain_turn(case, t["k"], t["pos"], t["gk"], t["bk"]))
    elif case["kind"] == "store":
        _plain_store(case, t["k"], t["kp"], t["ks"], t)
        _plain_store(case, t["v"], t["vp"], t["vs"], t)
    else:
        _plain_attn(case, state)
    return state["out"]


# --------------------------------------------------------------- what a pass has to do ---

def work(case):
    es = 2 if case["dtype"] == "f16" else 4
    H_kv, d = case["H_kv"], case["d"]
    if case["kind"] == "turn":
        T, heads = case["T"], case["H"] + H_kv
        return dict(bytes=2 * es * T * heads * d + 4 * T + (0, 2, 4)[case["norm"]] * es * d,
                    flops=T * heads * (3 * case["r"] + (0, 4, 6)[case["norm"]] * d))
    new, past = _lens(case)
    block = case["block"]
    if case["kind"] == "store":
        T = sum(new)
        touched = sum(_ceil(n + p, block) - p // block for n, p in zip(new, past))
        # Rows in; their numbers out; the powers of the blocks in and out.
        return dict(bytes=2 * T * H_kv * d * (es + 1) + 4 * T + 4 * touched * H_kv, flops=4 * T * H_kv * d)
    H, P = case["H"], case["P"]
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(new, past))
    cells = sum(n + p for n, p in zip(new, past))
    blocks = sum(_ceil(n + p, block) for n, p in zip(new, past))
    pages = sum(_ceil(n + p, P) for n, p in zip(new, past))
    return dict(bytes=2 * (cells * d + blocks) * H_kv + es * 2 * sum(new) * H * d + 4 * (pages + 2 * case["B"] + 1),
                flops=4 * pairs * H * d)


# ------------------------------------------------------------------ the same in 64 bits ---

def _exact_turn(case, x, pos, gain, shift):
    d, r, dev = case["d"], case["r"], x.device
    y = x.double()
    if case["norm"] == 1:
        y = gain.double() * y / torch.sqrt(torch.sum(y ** 2, -1, keepdim=True) / d + _EPS)
    elif case["norm"] == 2:
        var, mean = torch.var_mean(y, -1, correction=0, keepdim=True)
        y = gain.double() * (y - mean) / torch.sqrt(var + _EPS) + shift.double()
    f = []
    for i in range(r // 2):
        w = 1.0 / _BASE ** (2.0 * i / r)
        if case["scaling"] == 1:
            w /= _FACTOR
        elif case["scaling"] == 2:
            turns = _ORIGINAL / (2 * math.pi / w)
            if turns < _LOW:
                w /= _FACTOR
            elif turns <= _HIGH:
                share = (turns - _LOW) / (_HIGH - _LOW)
                w = share * w + (1 - share) * w / _FACTOR
        elif case["scaling"] == 3:
            lo = max(math.floor(r / 2 * math.log(_ORIGINAL / (_HIGH * 2 * math.pi), _BASE)), 0)
            hi = min(math.ceil(r / 2 * math.log(_ORIGINAL / (_LOW * 2 * math.pi), _BASE)), r - 1)
            share = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            w = (1 - share) * w + share * w / _FACTOR
        f.append(w)
    angle = pos.double()[:, None, None] * torch.tensor(f, dtype=torch.float64, device=dev)
    turn = torch.polar(torch.full_like(angle, _amplitude(case)), angle)
    if case["halves"]:
        z = torch.complex(y[..., :r // 2].contiguous(), y[..., r // 2:r].contiguous()) * turn
        return torch.cat((z.real, z.imag, y[..., r:]), -1)
    z = torch.view_as_complex(y[..., :r].unflatten(-1, (-1, 2)).contiguous()) * turn
    return torch.cat((torch.view_as_real(z).flatten(-2), y[..., r:]), -1)


def _exact_e4m3(x):
    """x (64 bits, at most 448 in size) rounded to 4 bits of mantissa, steps of at least 2^-9."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))).clamp(min=-6.0) - 3.0)
    return torch.round(x / step) * step


def _exact_store(case, x, pages, powers, slots):
    """Block by block on the host's list of them, the arithmetic of each on the GPU."""
    P, block = case["P"], case["block"]
    cells = pages.double().flatten(0, 1)
    bytes_ = powers.flatten(0, 1).clone()
    two = torch.tensor([2.0 ** (i - 127) for i in range(256)], dtype=torch.float64, device=x.device)
    rows = {}
    for row, s in enumerate(slots.tolist()):
        rows.setdefault(s // block, []).append((row, s))
    which, pad, marks = [], [], []
    for b, members in rows.items():
        which.append(b)
        pad.append([r for r, _ in members] + [members[0][0]] * (block - len(members)))
        marks.append(any(s % block == 0 for _, s in members))
    which = torch.tensor(which, device=x.device)
    marks = torch.tensor(marks, device=x.device)[:, None]
    size = x.double().abs().amax(-1)[torch.tensor(pad, device=x.device)].amax(1)
    e = torch.ceil(torch.log2(size / 448.0))
    e = e + (size > 448.0 * torch.exp2(e)).double() - (size <= 448.0 * torch.exp2(e - 1)).double()   # logarithms off
    need = torch.where(size > 0, (e + 127).clamp(0, 254), 0).long()
    old = bytes_[which].long()
    byte = torch.where(marks, need, torch.maximum(old, need))
    grown = torch.where(marks, 1.0, two[old] / two[byte])
    cells.view(-1, block, *cells.shape[1:])[which] = _exact_e4m3(cells.view(-1, block, *cells.shape[1:])[which] *
                                                               grown[:, None, :, None])
    bytes_[which] = byte.to(torch.uint8)
    slots = slots.long()
    cells[slots] = _exact_e4m3(x.double() / two[bytes_[slots // block].long()][:, :, None])
    return cells.view(pages.shape), bytes_.view(powers.shape)


def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "turn":
        return dict(q=_exact_turn(case, t["q"], t["pos"], t["gq"], t["bq"]),
                    k=_exact_turn(case, t["k"], t["pos"], t["gk"], t["bk"]))
    if case["kind"] == "store":
        kp, ks = _exact_store(case, t["k"], t["kp"], t["ks"], t["slots"])
        vp, vs = _exact_store(case, t["v"], t["vp"], t["vs"], t["slots"])
        return dict(kp=kp, vp=vp, ks=ks, vs=vs)
    # One head of one sequence at a time, its positions gathered by slot.
    P, block, H, H_kv, d = case["P"], case["block"], case["H"], case["H_kv"], case["d"]
    two = torch.tensor([2.0 ** (i - 127) for i in range(256)], dtype=torch.float64, device="cuda")
    kp, vp = (t[n].view(torch.uint8).flatten(0, 1) for n in ("kp", "vp"))
    ks, vs = (t[n].flatten(0, 1) for n in ("ks", "vs"))
    o = torch.empty(t["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, past) in enumerate(zip(*_lens(case))):
        j = torch.arange(n + past, device="cuda")
        at = t["table"][b].long()[j // P] * P + j % P
        seen = j[None, :] <= past + torch.arange(n, device="cuda")[:, None]
        for kvh in range(H_kv):
            k, v = (x[at, kvh].view(torch.float8_e4m3fn).double() * two[y[at // block, kvh].long()][:, None]
                    for x, y in ((kp, ks), (vp, vs)))
            for h in range(kvh * (H // H_kv), (kvh + 1) * (H // H_kv)):
                s = torch.mm(t["q"][first:first + n, h].double(), k.t()) / math.sqrt(d)
                w = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
                o[first:first + n, h] = torch.mm(w, v)
        first += n
    return dict(o=o)
