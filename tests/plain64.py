"""Plain 64-bit implementations of the prompt and serving operators, on the CPU, and the
error bounds their kernels are held to."""

import math

import numpy as np
import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half a step, relative


def runs_of(ids):
    """[begin, end) of each position's run of equal ids; (0, 0) where the id is negative."""
    n, out, a = len(ids), [], 0
    for i in range(n):
        if i > 0 and ids[i] != ids[i - 1]:
            a = i
        b = i + 1
        while b < n and ids[b] == ids[i]:
            b += 1
        out.append((a, b) if ids[i] >= 0 else (0, 0))
    return out


def intervals(sq, skv, causal, ids=None, prefix=None):
    """Boolean [sq, skv]: which keys each row may see."""
    pos = np.arange(sq)[:, None] + skv - sq
    key = np.arange(skv)[None]
    allowed = key <= pos if causal else np.ones((sq, skv), bool)
    if prefix is not None:
        allowed = allowed | (key < prefix)
    if ids is not None:
        r = np.array(runs_of(ids)).reshape(-1, 2)
        allowed = allowed & (key >= r[:, :1]) & (key < r[:, 1:])
    return allowed


def attend(q, k, v, allowed, pos, *, scale, cap, slope, half_p, half_out):
    """(out, bound) for one head: q [n, D], k, v [m, D] float64, allowed [n, m].

    The kernels compute scores in FP32 (products of 16-bit values are exact; D additions
    and a few factors, each off by at most 2^-23 of what is added), round probabilities to
    16 bits (half_p), add up to m products in FP32, and round the result (half_out)."""
    d, m = q.shape[1], k.shape[0]
    raw = q @ k.T * scale
    size = np.abs(q) @ np.abs(k).T * abs(scale)
    x, off = raw, (d + 8) * 2.0 ** -23 * size
    if cap:
        x = cap * np.tanh(x / cap)
        off = off + cap * 2.0 ** -20  # exponential, reciprocal and the difference from 1
    far = np.abs(pos[:, None] - np.arange(m)[None])
    if slope:
        x = x - slope * far
        off = off + slope * far * 2.0 ** -22
    off = off + np.abs(x) * 2.0 ** -22 + 2.0 ** -21  # to log2 units, minus the reference point, 2^x
    x = np.where(allowed, x, -np.inf)
    some = allowed.any(1)
    top = np.where(some, x.max(1, initial=-np.inf), 0.0)
    w = np.where(allowed, np.exp(np.where(allowed, x - top[:, None], 0.0)), 0.0)
    total = np.where(some, w.sum(1), 1.0)
    p = w / total[:, None]
    out = p @ v
    weight = p @ np.abs(v)
    worst = np.where(allowed & (p > 1e-12), off, 0.0).max(1, initial=0.0)
    # A weight is off by 2 worst (its own score and the sum's), a rounding, and the sums;
    # weights under 2^-21 of the largest round by at most 2^-32 each.
    rel = 2.2 * worst + half_p + (m + 64) * 2.0 ** -23
    bound = weight * rel[:, None] + np.abs(v).sum(0)[None] * 2.0 ** -32
    return out, bound + half_out * (np.abs(out) + bound) + 2.0 ** -25


def scale_for(amax):
    """Smallest power of two s with amax <= 448 s, at least 2^-100."""
    if amax == 0:
        return 2.0 ** -100
    e = math.frexp(amax / 448.0)
    k = e[1] - 1 if e[0] == 0.5 else e[1]
    return 2.0 ** max(k, -100)


def e4m3(x):
    """Nearest e4m3 value (ties to even) of float64 x; beyond 448 saturates, NaN stays."""
    x = np.asarray(x, np.float64)
    a = np.abs(x)
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        e = np.maximum(np.frexp(np.where(np.isfinite(a) & (a > 0), a, 1.0))[1] - 1, -6).astype(np.float64)
        step = 2.0 ** (e - 3)
        r = np.minimum(np.round(np.where(np.isfinite(a), a, 448.0) / step) * step, 448.0)
        r = np.copysign(r, x)
    return np.where(np.isnan(x), np.nan, r)


def cache_values(cache):
    """float64 numpy values of e4m3 bytes."""
    return cache.cpu().view(torch.float8_e4m3fn).float().double().numpy()


def append(x, slots, values, scales, page):
    """Appends x [T, H, D] (float64) to values [P, H, page, D], scales [P, H], in place."""
    t, n = 0, len(slots)
    n_slots = values.shape[0] * page
    while t < n:
        s = slots[t]
        if s < 0 or s >= n_slots:
            t += 1
            continue
        p, at = divmod(s, page)
        end = t + 1
        while end < n and slots[end] == s + end - t and at + end - t < page:
            end += 1
        for h in range(values.shape[1]):
            part = x[t:end, h]
            fine = np.where(np.isfinite(part), np.abs(part), 0.0)
            now = scale_for(float(fine.max()))
            if at > 0:
                now = max(now, scales[p, h])
                if now != scales[p, h]:
                    factor = np.float64(np.float32(scales[p, h]) / np.float32(now))
                    values[p, h, :at] = e4m3(values[p, h, :at] * factor)
            values[p, h, at:at + end - t] = e4m3(np.float32(part) / np.float32(now))
            scales[p, h] = now
        t = end


def plan(cached, new, page, table, free, n_free, max_tokens):
    """(lens, seq_lens, starts, slots, n_free); table is filled in place."""
    width = table.shape[1]
    n_free = max(0, min(n_free, len(free)))
    lens, seq, starts, slots = [], [], [0], [-1] * max_tokens
    wanted = used = 0
    for r, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        a = starts[-1]
        starts.append(a + n)
        have, want = -(-c // page), -(-(c + n) // page)
        fits = n > 0 and c + n <= width * page and a + n <= max_tokens
        need = want - have if fits else 0
        taken = fits and (need == 0 or wanted + need <= n_free)
        if taken:
            for i in range(need):
                table[r, have + i] = free[n_free - 1 - wanted - i]
            for i in range(n):
                owner = table[r, (c + i) // page]
                slots[a + i] = int(owner) * page + (c + i) % page if owner >= 0 else -1
            used = max(used, wanted + need) if need else used
        wanted += need
        lens.append(c + n if taken else c)
        seq.append(c + n if taken else 0)
    return lens, seq, starts, slots, n_free - used
