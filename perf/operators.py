"""The operators of a key/value cache held in 4 or 8 bits, measured through the framework's public entry points:
writing new rows and reading them back (ops.kvq_write, ops.kvq_read), and attention of prompts and single tokens
over such a cache (ops.kvq_attention), causal or with a sliding window and a few first tokens that stay visible.

The cache. A head row of D values is cut into groups of 32. A group has one scale s: its largest magnitude over the
largest code (7 in 4 bits, 127 in 8 bits), rounded up to four significant bits (4 bits) or to a power of two (8 bits),
in bfloat16; a value is held as c = round(x / s), half to even, and stands for c * s, which bfloat16 holds exactly. A group with a magnitude of 2^100 and more (or none: NaN) is held as NaN.
codes [B, Hk, capacity, D * bits / 8] hold c + 8 (two in a byte, the even column in the low half) or c + 128.

Attention. Query t of a sequence whose first new position is p sits at i = p + t and sees the positions j <= i with
i - j < window (where there is one) or j < sinks. Rows behind a sequence's count of new tokens are zeros.
"""
from __future__ import annotations

import math

import torch

own = False

GROUP = 32
LAYOUTS = ((9, 3, 64), (15, 5, 64), (16, 8, 128), (32, 8, 64))   # query heads, key/value heads, head size
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ---- cases --------------------------------------------------------------------------------------
def _store(B, T, Hk, D, bits, dtype, start, **k):
    return {"what": "store", "B": B, "T": T, "Hk": Hk, "D": D, "bits": bits, "dtype": dtype, "start": start, **k}


def _attend(B, T, H, Hk, D, length, bits, dtype, window=0, sinks=0, ragged=False, **k):
    return {"what": "attend", "B": B, "T": T, "H": H, "Hk": Hk, "D": D, "length": length, "bits": bits, "dtype": dtype,
            "window": window, "sinks": sinks, "ragged": ragged, **k}


def listed():
    return [
        # one new token of eight conversations, as every step of generation writes it
        _store(8, 1, 8, 128, 8, "fp32", 1000, name="store_token_8bit"),
        # a prompt of odd length behind an earlier turn, 64-wide heads
        _store(3, 1023, 5, 64, 8, "fp32", 129, name="store_prompt_8bit_odd"),
        # four long prompts at once
        _store(4, 4096, 8, 128, 4, "bf16", 0, name="store_prompt_4bit"),
        # one conversation that has just begun: latency alone
        _attend(1, 1, 9, 3, 64, 127, 4, "fp32", name="token_4bit_short"),
        # a small batch of ordinary conversations of different lengths
        _attend(8, 1, 15, 5, 64, 1023, 8, "fp32", ragged=True, name="token_8bit_batch"),
        # one conversation over a very long document
        _attend(1, 1, 32, 8, 64, 131072, 8, "fp32", name="token_8bit_long"),
        # a full server: many long conversations, the whole card's memory rate
        _attend(32, 1, 16, 8, 128, 32768, 4, "bf16", ragged=True, name="token_4bit_server"),
        # streaming chat: a window and the first tokens, whatever the conversation's length
        _attend(64, 1, 16, 8, 128, 8192, 8, "bf16", window=1024, sinks=4, ragged=True, name="token_8bit_window"),
        # five drafted tokens checked at once
        _attend(16, 5, 32, 8, 64, 2047, 4, "fp32", name="draft_4bit"),
        # prompts of different lengths padded to the longest, behind earlier turns
        _attend(4, 777, 15, 5, 64, 1500, 8, "fp32", ragged=True, name="prompt_8bit_padded"),
        # a long prompt in chunks: the last one over what is cached already
        _attend(1, 2048, 16, 8, 128, 8192, 4, "fp32", name="prompt_4bit_chunk"),
        # a whole prompt with a window
        _attend(1, 4095, 32, 8, 64, 4095, 8, "bf16", window=512, sinks=4, name="prompt_8bit_window"),
    ]


def draw(rng):
    def log(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)) - 0.5 / hi)))))

    H, Hk, D = rng.choice(LAYOUTS)
    bits, dtype = rng.choice((4, 8)), rng.choice(("fp32", "bf16"))
    kind = rng.random()
    if kind < 0.25:
        B, T = log(1, 32), log(1, 4096)
        while B * T * Hk * D > 4 * 4096 * 8 * 128:
            B, T = log(1, 32), log(1, 4096)
        return _store(B, T, Hk, D, bits, dtype, log(1, 4096) - 1)
    window = 0 if rng.random() < 0.6 else log(16, 4096)
    sinks = 0 if not window else rng.choice((0, 1, 4, 7))
    ragged = rng.random() < 0.5
    while True:
        if kind < 0.7:      # single tokens and drafts
            T = 1 if rng.random() < 0.7 else rng.randint(2, 8)
            B, length = log(1, 64), log(T, 131072)
            if B * length * Hk * D <= 20480 * 32 * 8 * 128:
                break
        else:               # prompts
            B, T = log(1, 8), log(16, 4096)
            length = T + (0 if rng.random() < 0.4 else log(1, 8192))
            if B * T * H * length <= 16 * 2048 * 8192:
                break
    return _attend(B, T, H, Hk, D, length, bits, dtype, window, sinks, ragged)


def _lengths(c):
    """Positions of each sequence once its new tokens are in, and how many of its T rows are new tokens."""
    B, T, n = c["B"], c["T"], c["length"]
    if not c["ragged"]:
        return [n] * B, [T] * B
    lengths, counts = [], []
    for b in range(B):
        part = ((b * 5 + 3) % 8 + 1) / 8             # an eighth to the whole, in no order
        counts.append(max(1, int(T * part)))
        lengths.append(max(counts[-1], int(n * part)))
    return lengths, counts


def _seen(i, window, sinks):
    """How many positions a query at position i sees."""
    n = i + 1
    if not window or n <= window:
        return n
    return window + min(sinks, n - window)


def _first(length, count, window):
    """The first position that a sequence's window reaches."""
    return max(0, length - count - window + 1) if window else 0


def work(c):
    size = 4 if c["dtype"] == "fp32" else 2
    row = c["D"] * c["bits"] / 8 + c["D"] / GROUP * 2
    if c["what"] == "store":
        rows = 2 * c["B"] * c["T"] * c["Hk"]          # keys and values; read, held, read, given back
        return {"bytes": rows * (2 * c["D"] * size + 2 * row), "flops": 0}
    keys = flops = 0
    for length, count in zip(*_lengths(c)):
        lo = _first(length, count, c["window"])
        keys += length - lo + min(c["sinks"], lo)
        flops += sum(_seen(i, c["window"], c["sinks"]) for i in range(length - count, length))
    return {"bytes": 2 * keys * c["Hk"] * row + 2 * c["B"] * c["T"] * c["H"] * c["D"] * size, "flops": 4 * flops * c["H"] * c["D"]}


# ---- the plain form -----------------------------------------------------------------------------
def _quantise(x, bits):
    """Codes (whole numbers, as bytes from 0) and scales (bfloat16) of the rows of x."""
    top, cut = (7, 20) if bits == 4 else (127, 23)
    g = x.float().unflatten(-1, (-1, GROUP))
    most = g.abs().amax(-1)
    s = (most / top).view(torch.int32)
    s = ((s + ((1 << cut) - 1)) >> cut << cut).view(torch.float32)
    s = torch.where(most < 2.0 ** 100, s, torch.full_like(s, math.nan))
    c = (g.double() / s.double().unsqueeze(-1)).round()     # 64 bits: next to a half, 32 would decide otherwise
    c = torch.where(s.unsqueeze(-1) > 0, c.clamp(-top, top), torch.zeros_like(c))
    return (c.flatten(-2) + (1 << (bits - 1))).to(torch.uint8), s.bfloat16()


def _pack(u, bits):
    return u if bits == 8 else u[..., 0::2] | (u[..., 1::2] << 4)


def _values(codes, scales, bits):
    u = codes if bits == 8 else torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    c = u.float() - (1 << (bits - 1))
    return (c.unflatten(-1, (-1, GROUP)) * scales.float().unsqueeze(-1)).flatten(-2)


def _plain_store(s):
    c = s["case"]
    at = slice(c["start"], c["start"] + c["T"])
    back = []
    for x, codes, scales in ((s["k"], s["k_codes"], s["k_scales"]), (s["v"], s["v_codes"], s["v_scales"])):
        u, sc = _quantise(x.transpose(1, 2), c["bits"])
        codes[:, :, at] = _pack(u, c["bits"])
        scales[:, :, at] = sc
        back.append(_values(codes[:, :, at], scales[:, :, at], c["bits"]).to(x.dtype))
    return back


def _plain_attend(s):
    c, q = s["case"], s["q"]
    B, T, H, D = q.shape
    Hk, n, dev = c["Hk"], c["length"], q.device
    k = _values(s["k_codes"][:, :, :n], s["k_scales"][:, :, :n], c["bits"])
    v = _values(s["v_codes"][:, :, :n], s["v_scales"][:, :, :n], c["bits"])
    rows = q.float().reshape(B, T, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, D)
    z = torch.matmul(rows, k.transpose(2, 3)).view(B, Hk, H // Hk, T, n) / math.sqrt(D)
    i = (s["pos"].long()[:, None] + torch.arange(T, device=dev))[:, :, None]
    j = torch.arange(n, device=dev)
    sees = (j <= i) & (torch.arange(T, device=dev)[:, None] < s["count"].long()[:, None, None])
    if c["window"]:
        sees &= (i - j < c["window"]) | (j < c["sinks"])
    z = z.masked_fill(~sees[:, None, None], -math.inf)
    most = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(most == -math.inf, torch.zeros_like(most), most))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(p.view(B, Hk, -1, n), v).view(B, Hk, H // Hk, T, D)
    return out.permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(q.dtype)


# ---- the framework's entry points ---------------------------------------------------------------
def _own(s):
    from emberlm_b200 import ops

    c = s["case"]
    if "cache" not in s:       # the handle that a program keeps for as long as the cache
        s["cache"] = ops.KvqCache(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"])
    if c["what"] == "store":
        ops.kvq_write(s["cache"], s["k"], s["v"], c["start"])
        return ops.kvq_read(s["cache"], c["start"], c["T"], dtype=s["k"].dtype)
    if c["ragged"]:
        return ops.kvq_attention(s["q"], s["cache"], s["pos"], count=s["count"], window=c["window"], sinks=c["sinks"])
    return ops.kvq_attention(s["q"], s["cache"], c["length"] - c["T"], window=c["window"], sinks=c["sinks"])


# ---- inputs -------------------------------------------------------------------------------------
def _rows(gen, shape, spread):
    """Projected rows: a few columns of every head are much larger than the rest."""
    x = torch.randn(shape, generator=gen, device="cuda")
    big = torch.ones(shape[-1], device="cuda")
    big[3::32] = 4.0
    return x * big * spread


def prepare(case, seed):
    c, gen = dict(case), torch.Generator(device="cuda").manual_seed(int(seed))
    B, T, Hk, D, bits, kind = c["B"], c["T"], c["Hk"], c["D"], c["bits"], DTYPES[c["dtype"]]
    end = c["start"] + T if c["what"] == "store" else c["length"]
    room = -(-end // 64) * 64
    s = {"case": c}
    for name in ("k", "v"):
        s[name + "_codes"] = torch.zeros(B, Hk, room, D * bits // 8, dtype=torch.uint8, device="cuda")
        s[name + "_scales"] = torch.zeros(B, Hk, room, D // GROUP, dtype=torch.bfloat16, device="cuda")
    if c["what"] == "store":
        packed = _rows(gen, (B, T, 2 * Hk, D), 0.5).to(kind)      # keys and values as one product leaves them
        s["k"], s["v"] = packed[:, :, :Hk], packed[:, :, Hk:]
        return s
    lengths, counts = _lengths(c)
    for b in range(B):
        for name, spread in (("k", 0.5), ("v", 1.0)):
            u, sc = _quantise(_rows(gen, (Hk, lengths[b], D), spread), bits)
            s[name + "_codes"][b, :, : lengths[b]] = _pack(u, bits)
            s[name + "_scales"][b, :, : lengths[b]] = sc
    s["q"] = torch.randn(B, T, c["H"], D, generator=gen, device="cuda").to(kind)
    s["pos"] = torch.tensor([n - m for n, m in zip(lengths, counts)], dtype=torch.int32, device="cuda")
    s["count"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
    return s


def run(s):
    if own:
        return _own(s)
    return _plain_store(s) if s["case"]["what"] == "store" else _plain_attend(s)


# ---- in 64 bits ---------------------------------------------------------------------------------
def _held64(x, bits):
    """What a group of 32 stands for once it is held in `bits` bits, from the definition."""
    x = x.double().unflatten(-1, (-1, GROUP))
    most = x.abs().amax(-1, keepdim=True)
    ratio = (most.float() / (2 ** (bits - 1) - 1)).double()       # formed in 32 bits, as the definition has it
    part, power = torch.frexp(ratio)
    keep = 16.0 if bits == 4 else 1.0
    if bits == 8:
        power = torch.where(part == 0.5, power - 1, power)        # a power of two stays
        step = torch.where(most > 0, torch.ldexp(torch.ones_like(part), power), torch.zeros_like(part))
    else:
        step = torch.ldexp(torch.ceil(part * keep) / keep, power)
    n = torch.where(step > 0, x / torch.where(step > 0, step, torch.ones_like(step)), torch.zeros_like(x))
    return (torch.round(n) * step).flatten(-2)


def exact(case, seed):
    c, s = dict(case), prepare(case, seed)
    if c["what"] == "store":
        return [_held64(x, c["bits"]).transpose(1, 2) for x in (s["k"], s["v"])]
    B, T, H, Hk, D = c["B"], c["T"], c["H"], c["Hk"], c["D"]
    if B * T * H * c["length"] > 3e9:
        return None
    out = torch.zeros(B, T, H, D, dtype=torch.float64, device="cuda")
    for b, (n, m) in enumerate(zip(*_lengths(c))):
        held = []
        for name in ("k", "v"):
            u, sc = s[name + "_codes"][b, :, :n].long(), s[name + "_scales"][b, :, :n].double()
            if c["bits"] == 4:
                u = torch.cat((u.remainder(16).unsqueeze(-1), u.div(16, rounding_mode="floor").unsqueeze(-1)), -1).reshape(Hk, n, D)
            held.append((u - 2 ** (c["bits"] - 1)).double() * sc.repeat_interleave(GROUP, -1))
        where = torch.arange(n, device="cuda")
        at = torch.arange(n - m, n, device="cuda")[:, None]
        hidden = where > at
        if c["window"]:
            hidden |= (at - where >= c["window"]) & (where >= c["sinks"])
        for h in range(H):
            key, value = held[0][h * Hk // H], held[1][h * Hk // H]
            z = (s["q"][b, :m, h].double() @ key.T) * D ** -0.5
            z[hidden] = -math.inf
            out[b, :m, h] = torch.softmax(z, -1) @ value
    return out
