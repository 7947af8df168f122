"""CPU restatement of the 8-bit KV pool and of the rotary embedding by position, in 64 bits, token by token.

Pools are lists of segments (original pool, elastic chunks); a segment is a dict of numpy arrays ``k``, ``v`` (uint8 codes
[blocks, layers, heads, block_size, head_dim]) and ``ks``, ``vs`` (float32 scales [blocks, layers, heads]).
"""
from __future__ import annotations

import numpy as np

TINY = np.float64(2.0) ** -126


def _e4m3_table():
    out = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        mag = np.nan if (e, m) == (15, 7) else m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out[c] = -mag if c & 128 else mag
    return out


E4M3 = _e4m3_table()
INT8 = np.arange(256).astype(np.uint8).view(np.int8).astype(np.float64)


def values(codes, code):
    return (INT8 if code == "int8" else E4M3)[codes]


def scale_of(amax, code):
    """The stored scale of values of up to `amax` (float64), as float32."""
    if not np.isfinite(amax):
        return np.float32(np.nan)
    if code == "int8":
        s = np.float32(amax / 127)
    else:
        if amax == 0:
            return np.float32(0)
        e = int(np.floor(np.log2(amax))) - 9
        while amax > 448 * 2.0 ** e:
            e += 1
        s = np.float32(2.0 ** e) if e > -150 else np.float32(0)
    return np.float32(0) if s < TINY else s


def inverse_of(s):
    return np.float64(np.float32(1 / np.float64(s))) if s > 0 else np.float64(0)


def encode(x, inv, code):
    """Codes (uint8) of float64 values; a factor 0 gives the code 0."""
    if inv == 0:
        return np.zeros(np.shape(x), np.uint8)
    y = np.asarray(x, np.float64) * inv
    if code == "int8":
        return np.rint(y).astype(np.int64).astype(np.int8).view(np.uint8)
    mag = E4M3[:127]                                # ascending, codes 0 ... 126
    a = np.minimum(np.abs(y), 448.0)
    hi = np.clip(np.searchsorted(mag, a), 1, 126)
    lo = hi - 1
    up, down = mag[hi] - a, a - mag[lo]
    pick = np.where(up < down, hi, np.where(down < up, lo, np.where(hi % 2 == 0, hi, lo)))
    return (pick + np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def locate(segs, blk):
    n0 = segs[0]["k"].shape[0]
    if 0 <= blk < n0:
        return segs[0], blk
    if blk < 0 or len(segs) == 1:
        return None
    n = segs[1]["k"].shape[0]
    j, r = divmod(blk - n0, n)
    return (segs[1 + j], r) if 1 + j < len(segs) else None


def page(segs, table, row, lb):
    if not (0 <= row < table.shape[0]) or lb >= table.shape[1]:
        return None
    return locate(segs, int(table[row, lb]))


def _last_entry(ids, lens, i):
    return not any(ids[j] == ids[i] and lens[j] > 0 for j in range(i + 1, len(ids)))


def store_prefill(segs, code, k, v, table, ids, starts, lens, layer, bs):
    for i, n in enumerate(lens):
        n = min(n, len(k) - starts[i])
        if n <= 0 or not _last_entry(ids, lens, i):
            continue
        for lb in range(-(-n // bs)):
            at = page(segs, table, ids[i], lb)
            if at is None:
                continue
            seg, r = at
            t0, t1 = starts[i] + lb * bs, starts[i] + min((lb + 1) * bs, n)
            for x, c, s in ((k, "k", "ks"), (v, "v", "vs")):
                for h in range(x.shape[1]):
                    y = x[t0:t1, h].astype(np.float64)
                    peak = np.inf if not np.isfinite(y).all() else np.abs(y).max()
                    seg[s][r, layer, h] = scale = scale_of(peak, code)
                    seg[c][r, layer, h, :t1 - t0] = encode(y, inverse_of(scale), code)


def store_append(segs, code, k, v, table, ids, lens, layer, bs):
    for i, n in enumerate(lens):
        if n <= 0 or not _last_entry(ids, lens, i):
            continue
        lb, slot = divmod(n - 1, bs)
        at = page(segs, table, ids[i], lb)
        if at is None:
            continue
        seg, r = at
        for x, c, s in ((k, "k", "ks"), (v, "v", "vs")):
            for h in range(x.shape[1]):
                y = x[i, h].astype(np.float64)
                held = seg[s][r, layer, h]
                fresh = scale_of(np.abs(y).max() if np.isfinite(y).all() else np.inf, code)
                scale = fresh if slot == 0 else np.float32(np.nan) if np.isnan(held) or np.isnan(fresh) else max(held, fresh)
                inv = inverse_of(scale)
                if slot > 0 and scale > held:
                    ratio = np.float64(np.float32(np.float64(held) * inv))
                    old = seg[c][r, layer, h, :slot]
                    seg[c][r, layer, h, :slot] = encode(values(old, code), ratio, code)
                seg[c][r, layer, h, slot] = encode(y, inv, code)
                seg[s][r, layer, h] = scale


def cached(segs, code, table, row, n, layer, bs):
    """(K, V) [n, heads, dim] float64 of a sequence's first n tokens; tokens whose page is not there are left out, their
    positions are in the third result."""
    ks, vs, missing = [], [], []
    for t in range(n):
        at = page(segs, table, row, t // bs)
        if at is None:
            missing.append(t)
            continue
        seg, r = at
        ks.append(values(seg["k"][r, layer, :, t % bs], code) * seg["ks"][r, layer][:, None].astype(np.float64))
        vs.append(values(seg["v"][r, layer, :, t % bs], code) * seg["vs"][r, layer][:, None].astype(np.float64))
    return (np.stack(ks), np.stack(vs), missing) if ks else (None, None, missing)


def attention(segs, code, q, table, ids, lens, layer, bs, scale, weights=16):
    """(o, slack) [batch, q_heads, dim] float64; NaN rows where nothing is attended.  `slack` bounds what a kernel may be
    off before its output is rounded: weights rounded to fp16 (2^-11 of each, 2^-25 at least), scores summed in fp32 and
    exponentials good to 2^-20.

    `weights` = 32: what a kernel may be off that holds its weights to 32 bits or as an fp16 number and what that leaves
    over (see slack_32)."""
    B, Hq, D = q.shape
    o, slack = np.full((B, Hq, D), np.nan), np.zeros((B, Hq, D))
    for i, n in enumerate(lens):
        if n <= 0:
            continue
        k, v, missing = cached(segs, code, table, ids[i], n, layer, bs)
        if k is None:
            continue
        G = Hq // k.shape[1]
        if weights == 32:
            at = [page(segs, table, ids[i], t // bs) for t in range(n) if t not in set(missing)]
            sk, sv = (np.stack([seg[c][r, layer] for seg, r in at]).astype(np.float64) for c in ("ks", "vs"))
        for h in range(Hq):
            x, kk, vv = q[i, h].astype(np.float64), k[:, h // G], v[:, h // G]
            s = kk @ x * scale
            p = np.exp(s - s.max())
            total = p.sum()
            o[i, h] = p @ vv / total
            if weights == 32:
                slack[i, h] = slack_32(code, x, kk, vv, sk[:, h // G], sv[:, h // G], p, scale)
                continue
            off = (D + 8) * 2.0 ** -24 * (np.abs(kk) @ np.abs(x)).max() * abs(scale)
            slack[i, h] = (2.0 ** -11 + 2 * off + 2.0 ** -20) * (p @ np.abs(vv)) / total + len(p) * 2.0 ** -25 * np.abs(vv).max(0) / total
    return o, slack


def slack_32(code, x, k, v, sk, sv, p, scale):
    """What one row of the attention may be off with weights to 32 bits; sk, sv: the tokens' scales, p: their weights.

    Scores: a product for each element of x that is not 0 and a few more roundings, 2^-23 each (a tensor core cuts off
    where an adder rounds), of the sum of absolute values - with int8 codes held as q + 128, whose 128 is taken off again,
    of up to 255 s |x|.  log2 of V's scale joins the exponent: good to 2^-22 of itself, and the sum rounds once more.
    A weight: exponential 2^-22, its fp16 number's remainder as fp16 2^-22, 2^-31 of the largest at least (fp16's smallest
    half step 2^-25, with the largest weight held at 2^6 or more).  The denominator's factor and the output's two take
    2^-22 each, and as much is left for the factors by which a maximum that moves scales sums down (2 * 2^-22 on what then
    has 2^-4 of the weight or less).
    Sums over tokens: up to three products for 16 tokens, a piece's merge, or one addition a token: 2^-23 each, of the sum
    of absolute values, with int8 codes again up to 255 s."""
    total, n = p.sum(), len(p)
    size = 255 * sk[:, None] if code == "int8" else np.abs(k)
    off = (np.count_nonzero(x) + 8) * 2.0 ** -23 * (size * np.abs(x)).sum(1).max() * abs(scale)
    log_sv = np.abs(np.log2(sv, out=np.zeros_like(sv), where=sv > 0)).max()
    rel = 2 * off + (1.25 * log_sv + 6) * 2.0 ** -22
    mass = p @ (255 * sv[:, None] * np.ones_like(v) if code == "int8" else np.abs(v))
    steps = 3 * -(-n // 16) + n + 16
    return (rel * (p @ np.abs(v)) + steps * 2.0 ** -23 * mass + n * 2.0 ** -31 * (p * sv).max() * 448) / total


def rotary(x, positions, inv_freq, interleaved, attention_scale):
    """x [tokens, heads, dim] -> float64."""
    y = x.astype(np.float64).copy()
    n = len(inv_freq)
    for t, pos in enumerate(positions):
        angle = np.float64(pos) * inv_freq
        c, s = np.cos(angle) * attention_scale, np.sin(angle) * attention_scale
        for h in range(y.shape[1]):
            a, b = (y[t, h, 0:2 * n:2].copy(), y[t, h, 1:2 * n:2].copy()) if interleaved else (y[t, h, :n].copy(), y[t, h, n:2 * n].copy())
            u, w = a * c - b * s, a * s + b * c
            if interleaved:
                y[t, h, 0:2 * n:2], y[t, h, 1:2 * n:2] = u, w
            else:
                y[t, h, :n], y[t, h, n:2 * n] = u, w
    return y
