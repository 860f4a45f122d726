"""Definitions of the ragged-generation operators in exact or 64-bit
arithmetic, on the host (test infrastructure: the checker, never the product).

The 4-bit history: groups of 32 channels, low = largest bf16 <= min, step =
smallest bf16 >= (max - low) / 15, code = floor((x - low) / step + 1/2)."""
import math
from fractions import Fraction

import numpy as np


def slab(D):
    return next(w for w in (256, 128, 64, 32) if D % w == 0)


def f32_bits(x):
    return int(np.float32(x).view(np.uint32))


def bits_f32(u):
    return np.uint32(u).view(np.float32)


def bf16_floor(x):
    """Largest bf16 <= x (x an fp32 number), as fp32."""
    u = f32_bits(x) & 0xFFFF0000
    if float(bits_f32(u)) > float(x):
        u += 0x10000
    return np.float32(0.0) if u == 0x80000000 else bits_f32(u)


def bf16_ceil(q):
    """Smallest bf16 >= the Fraction q >= 0, as fp32."""
    if q == 0:
        return np.float32(0.0)
    lo, hi = 0, 0x7F7F
    while lo < hi:  # bf16 bit patterns of non-negative numbers are ordered
        mid = (lo + hi) // 2
        if Fraction(float(bits_f32(mid << 16))) >= q:
            hi = mid
        else:
            lo = mid + 1
    return bits_f32(lo << 16)


def quantise_group(x):
    """(codes, step, low) of 32 fp32 values, in exact arithmetic; None for the
    codes of a group that is stored as NaN."""
    x = np.asarray(x, np.float32)
    if not np.all(np.abs(x) <= np.float32(1e37)):
        return None, np.float32(np.nan), np.float32(0)
    low = bf16_floor(x.min())
    step = bf16_ceil((Fraction(float(x.max())) - Fraction(float(low))) / 15)
    if step == 0:
        return np.zeros(32, np.int64), step, low
    fs, fl = Fraction(float(step)), Fraction(float(low))
    codes = np.array([math.floor((Fraction(float(v)) - fl) / fs + Fraction(1, 2)) for v in x])
    assert codes.min() >= 0 and codes.max() <= 15
    return codes, step, low


def pack_row(k, v):
    """The records [D/W, 5W/4] of one position's k and v [D] and the values
    (k, v) they stand for, as float64."""
    D = len(k)
    W = slab(D)
    codes, params, values = np.zeros((2, D), np.int64), np.zeros((2, D // 32, 2), np.uint16), np.zeros((2, D))
    for j, x in enumerate((k, v)):
        for g in range(D // 32):
            s = slice(32 * g, 32 * g + 32)
            c, step, low = quantise_group(x[s])
            if c is None:
                codes[j, s], params[j, g], values[j, s] = 0, (0x7FFF, 0), np.nan
                continue
            codes[j, s] = c
            params[j, g] = f32_bits(step) >> 16, f32_bits(low) >> 16
            values[j, s] = float(low) + float(step) * c
    rec = np.zeros((D // W, W * 5 // 4), np.uint8)
    for o in range(D // 8):
        at, q = divmod(8 * o, W)
        for j in (0, 1):
            for i in range(4):
                rec[at, q + 4 * j + i] = codes[j, 8 * o + 2 * i] | codes[j, 8 * o + 2 * i + 1] << 4
    for g in range(D // 32):
        at, q = divmod(32 * g, W)
        words = np.array([params[0, g, 0], params[0, g, 1], params[1, g, 0], params[1, g, 1]], np.uint16)
        rec[at, W + q // 4: W + q // 4 + 8] = words.view(np.uint8)
    return rec, values


def unpack_row(rec):
    """(k, v) [D] float64 of one position's records."""
    nslab, W = rec.shape[0], rec.shape[1] * 4 // 5
    out = np.zeros((2, nslab * W))
    for s in range(nslab):
        par = rec[s, W:].copy().view(np.uint16).astype(np.uint32) << 16
        par = par.view(np.float32).astype(np.float64).reshape(W // 32, 2, 2)
        code = rec[s, :W].reshape(W // 8, 2, 4)
        both = np.stack([code & 15, code >> 4], -1).reshape(W // 8, 2, 8).astype(np.float64)
        for j in (0, 1):
            c = both[:, j].reshape(W // 32, 32)
            out[j, s * W: (s + 1) * W] = (par[:, j, 1:] + par[:, j, :1] * c).reshape(-1)
    return out


def aft_row(q, k, v, w, hs):
    """AFT row in 64 bits: q [D], k, v [n, D], w [H, n]; zero where every
    weight is -inf."""
    x = k + np.repeat(np.asarray(w, np.float64).T, hs, 1)
    with np.errstate(invalid="ignore", over="ignore"):
        m = x.max(0)
        e = np.exp(np.where(np.isneginf(m), -np.inf, x - m))
        e = np.where(np.isneginf(m)[None], 0.0, e)
        den = e.sum(0)
        r = np.where(den == 0, 0.0, (e * v).sum(0) / np.where(den == 0, 1.0, den))
        return r / (1.0 + np.exp(-np.asarray(q, np.float64)))


def page_tables(start, count, free, head, table, page, n_slots, ld):
    """(table, slots, row_start, head, short): one request after the other."""
    table, slots, short = table.copy(), np.full(n_slots, -1, np.int64), False
    head = min(max(0, head), len(free))
    row_start = [0]
    for b in range(len(start)):
        n = max(0, int(count[b])) if start[b] >= 0 else 0
        row_start.append(row_start[-1] + n)
        s = max(0, int(start[b]))
        for c in range(-(-s // page), -(-(s + n) // page)):
            if c >= table.shape[1]:
                short = True
                break
            if head < len(free):
                table[b, c] = free[head]
            else:
                table[b, c] = -1
                short = True
            head = head + 1
        for j in range(n):
            at = b * ld + j if ld else row_start[b] + j
            if (ld and j >= ld) or at >= n_slots:
                short = True
                break
            c = (s + j) // page
            if c < table.shape[1] and table[b, c] >= 0:
                slots[at] = int(table[b, c]) * page + (s + j) % page
            else:
                short = True
    return table, slots, np.array(row_start), min(head, len(free)), short


def logits_controls(x, tokens, pos, prompt, rep, pres, freq, bias, mask):
    """Row by row in 64 bits; arrays or None."""
    x = np.array(x, np.float64)
    B, V = x.shape
    for b in range(B):
        known = [int(t) for t in tokens[b, : max(0, pos[b] + 1)]] if tokens is not None else []
        made = known[max(0, int(prompt[b])) if prompt is not None else 0:]
        for t in sorted(set(known)):
            if not 0 <= t < V:
                continue
            if rep is not None:
                x[b, t] = x[b, t] / float(rep[b]) if x[b, t] > 0 else x[b, t] * float(rep[b])
            n = made.count(t)
            if n:
                x[b, t] -= (float(freq[b]) * n if freq is not None else 0) + (float(pres[b]) if pres is not None else 0)
    if bias is not None:
        x = x + np.asarray(bias, np.float64)
    if mask is not None:
        v = np.arange(V)
        ok = (np.asarray(mask).astype(np.int64)[..., v // 32] >> (v % 32)) & 1
        x = np.where(np.broadcast_to(ok, x.shape) != 0, x, -np.inf)
    return x
