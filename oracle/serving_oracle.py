"""Definitions, in numpy and 64 bits, of the operators around attention: rotary positions, the 8-bit paged cache and its
attention, step tables.  Written from the formulas; nothing here uses the package."""
import math

import numpy as np

PAGE = 16


# ---- e4m3 --------------------------------------------------------------------------------------
def e4m3_decode(codes):
    """Values of e4m3 codes: sign, 4 exponent bits (bias 7), 3 mantissa bits; 0x7f and 0xff are NaN."""
    c = np.asarray(codes, np.uint8).astype(np.int64)
    e, m = c >> 3 & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * np.exp2(e - 10.0))
    v = np.where((c & 0x7f) == 0x7f, np.nan, v)
    return np.where(c & 0x80, -v, v)


_GRID = e4m3_decode(np.arange(127))          # 0 .. 448, ascending


def e4m3_encode(x):
    """Nearest code, ties to the even one, saturating; NaN becomes 0x7f."""
    x = np.asarray(x, np.float64)
    a = np.abs(x)
    hi = np.clip(np.searchsorted(_GRID, a, side="left"), 1, 126)
    below, above = a - _GRID[hi - 1], _GRID[hi] - a
    code = np.where((below < above) | ((below == above) & ((hi - 1) % 2 == 0)), hi - 1, hi)
    code = np.where(a >= 448.0, 126, code) | np.where(np.signbit(x), 0x80, 0)
    return np.where(np.isnan(x), 0x7f, code).astype(np.uint8)


def scale_exponent(amax):
    """Smallest e >= -100 with amax <= 448 * 2^e."""
    e = -100
    while amax > 448.0 * 2.0 ** e:
        e += 1
    return e


# ---- cache: codes [blocks, H, pages, 2, 16, D] uint8, scales [blocks, H, pages, 2] -------------------
def append(codes, scales, key, value, slots, block_size):
    """quantize_and_scatter in place, run by run."""
    x = np.stack([key, value], 2).astype(np.float64)                 # [T, H, 2, D]
    limit = codes.shape[0] * block_size
    i = 0
    while i < len(slots):
        j = i + 1
        if not 0 <= slots[i] < limit:
            i = j
            continue
        while j < len(slots) and slots[j] == slots[j - 1] + 1 and slots[j] % PAGE:
            j += 1
        b, p, at = slots[i] // block_size, slots[i] % block_size // PAGE, slots[i] % PAGE
        for h in range(x.shape[1]):
            for kv in range(2):
                rows = x[i:j, h, kv]
                finite = np.abs(rows[np.isfinite(rows)])
                e = scale_exponent(finite.max() if finite.size else 0.0)
                if at:
                    old = scales[b, h, p, kv]
                    old = int(math.log2(old)) if 2.0 ** -100 <= old <= 2.0 ** 120 else -100
                    e = max(e, old)
                    if e > old:
                        codes[b, h, p, kv, :at] = e4m3_encode(e4m3_decode(codes[b, h, p, kv, :at]) * 2.0 ** (old - e))
                scales[b, h, p, kv] = 2.0 ** e
                codes[b, h, p, kv, at:at + j - i] = e4m3_encode(rows * 2.0 ** -e)
        i = j


def gather(codes, scales, table, length, block_size, h, kv):
    """Values [length, D] of a sequence's head."""
    pos = np.arange(length)
    b, p = np.asarray(table)[pos // block_size], pos % block_size // PAGE
    return e4m3_decode(codes[b, h, p, kv, pos % PAGE]) * scales[b, h, p, kv][:, None]


def attention(q, codes, scales, tables, lens, starts, block_size, sm_scale, eps):
    """(out, tolerance) of paged_attention_8bit for q [T, Hq, D] in 64 bits.

    The tolerance of an output is half a step eps / 2 of its type, plus what the weights w_k are off.
    * Their rounding to fp16, at most 2^-11 of a weight (half a step).  Where the denominator sums rounded weights, the output is
      sum w_k (1 + d_k) v_k / sum w_k (1 + d_k), off by sum w_k d_k (v_k - out) to first order; where it sums them as they are, by
      sum w_k d_k v_k.  Both are at most 2^-11 (sum w_k |v_k| + |out|).
    * 2 ln 2 times the error of a score in units of log2 (numerator and denominator), relative to sum_k w_k |v_k|: D fp32 additions and
      products, 2^-24 each, of the sum of |q k|; a few roundings of the score itself; for queries in bf16 values below 2^-14
      of the row's largest are off by 2^-25 of it.
    * Weights below 2^-30 of the largest may vanish.
    """
    T, Hq, D = q.shape
    G = Hq // codes.shape[1]
    out, tol = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    with np.errstate(invalid="ignore", over="ignore"):
        for i in range(len(lens)):
            a, n = int(starts[i]), int(starts[i + 1] - starts[i])
            if n == 0 or lens[i] <= 0:
                continue
            for h in range(codes.shape[1]):
                k = gather(codes, scales, tables[i], int(lens[i]), block_size, h, 0)
                v = gather(codes, scales, tables[i], int(lens[i]), block_size, h, 1)
                for j in range(n):
                    L = int(lens[i]) - n + j + 1
                    if L <= 0:
                        continue
                    x = q[a + j, h * G:(h + 1) * G].astype(np.float64)
                    s = x @ k[:L].T * sm_scale
                    w = np.exp(s - s.max(1, keepdims=True))
                    w /= w.sum(1, keepdims=True)
                    out[a + j, h * G:(h + 1) * G] = w @ v[:L]
                    size = np.abs(x) @ np.abs(k[:L]).T + 2.0 ** -1 / D * np.abs(x).max(1, keepdims=True) * np.abs(k[:L]).sum(1)
                    off = (abs(sm_scale) * size * (D + 8) * 2.0 ** -24).max(1) * 2 + 2.0 ** -20 + 2.0 ** -11
                    most = np.abs(v[:L]).max(0)
                    tol[a + j, h * G:(h + 1) * G] = off[:, None] * (w @ np.abs(v[:L])) + 2.0 ** -11 * np.abs(out[a + j, h * G:(h + 1) * G]) + L * 2.0 ** -30 * most
    return out, tol + np.abs(out) * eps / 2 + 2.0 ** -24


# ---- rotary ----------------------------------------------------------------------------------------
def rotate(x, angles, factor=1.0, interleaved=False, inverse=False):
    """x [T, H, D] turned by angles [T, R / 2]."""
    y, R = x.astype(np.float64).copy(), 2 * angles.shape[1]
    c, s = np.cos(angles)[:, None] * factor, np.sin(angles)[:, None] * factor * (-1 if inverse else 1)
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    u, w = y[..., a].copy(), y[..., b].copy()
    y[..., a], y[..., b] = u * c - w * s, w * c + u * s
    return y


# ---- step tables -----------------------------------------------------------------------------------
def plan(query, context, tables, free, count, block_size, num_rows):
    """plan_step, request by request; returns (slots, positions, seq_lens, starts, count, tables, status)."""
    tables, slots, positions, status = np.array(tables), [], [], 0
    taken, wanted, lens, starts, total = 0, 0, [], [0], 0
    count = min(max(int(count), 0), len(free))
    for i, (n, ctx) in enumerate(zip(query, context)):
        n, ctx = max(int(n), 0), max(int(ctx), 0)
        held, blocks = -(-ctx // block_size), -(-(ctx + n) // block_size)
        total += n
        fits = blocks <= tables.shape[1] and total <= num_rows
        need = blocks - held if blocks <= tables.shape[1] else 0
        wanted += need
        served = fits and (need == 0 or wanted <= count)
        if served and need:
            for j in range(need):
                tables[i, held + j] = free[count - 1 - taken]
                taken += 1
        if n and not served:
            status |= 16 if fits else 32
        for p in range(ctx, ctx + min(n, num_rows - len(slots))):
            block = tables[i, p // block_size] if served else -1
            slots.append(int(block) * block_size + p % block_size if block >= 0 else -1)
            positions.append(p)
        lens.append(ctx + n if served else ctx)
        starts.append(min(total, num_rows))
    slots, positions = slots[:num_rows], positions[:num_rows]
    pad = num_rows - len(slots)
    return (np.array(slots + [-1] * pad, np.int64), np.array(positions + [0] * pad, np.int64), np.array(lens, np.int32),
            np.array(starts, np.int32), count - taken, tables, status)


def release(ended, context, tables, free, count, block_size):
    free, at = np.array(free), int(count)
    for i, e in enumerate(ended):
        if e:
            for b in tables[i, :-(-max(int(context[i]), 0) // block_size)]:
                if at < len(free):
                    free[at] = b
                at += 1
    return np.where(ended, 0, context), min(at, len(free)), free
