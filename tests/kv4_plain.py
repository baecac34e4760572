"""Plain forms of the 4-bit cache and of attention, in numpy on the CPU and in
64 bits, for the tests of the device-buffer entry points."""
from __future__ import annotations

import numpy as np

PAGE = 16
TYPE = {"f32": 0, "f16": 1, "bf16": 30}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}   # half a step, relative


def round_to(x, t):
    """x (f32) as the nearest value of type t, in f32."""
    x = np.asarray(x, np.float32)
    if t == "f32":
        return x
    if t == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float32)
    b = x.view(np.uint32)
    r = ((b.astype(np.uint64) + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.float32(np.nan), r)


def groups_padded(D):
    return (D // 32 + 1) // 2 * 2


def record_bytes(D):
    return 2 * (PAGE * D // 2 + 2 * PAGE * 2 * groups_padded(D))


def k_byte(D, d):
    g, t, n = d // 32, d % 32 // 8, d % 8
    return 4 * (D // 32) * t + 4 * g + n // 2


def v_byte(D, d, row):
    g, h, n = d // 32, d % 32 // 4, d % 4
    return 2 * (D // 32) * (h ^ (4 if row & 2 else 0)) + 2 * g + n // 2


def quantise(x):
    """(codes, d, lo) of x [..][D] f32, as the format defines them; every step rounded to f32."""
    x = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    big = np.float32(65504)
    nan = np.isnan(x)
    none = nan.all(-1)
    mn = np.where(none, 0, np.where(nan, np.float32(np.inf), x).min(-1)).astype(np.float32)
    mx = np.where(none, 0, np.where(nan, np.float32(-np.inf), x).max(-1)).astype(np.float32)
    lo = np.clip(mn, -big, big).astype(np.float16)
    with np.errstate(all="ignore"):
        d = ((np.clip(mx, -big, big) - lo.astype(np.float32)) * np.float32(1 / 15)).astype(np.float16)
        inv = np.where(d > 0, np.float32(1) / d.astype(np.float32), np.float32(0)).astype(np.float32)
        c = np.rint((x - lo.astype(np.float32)[..., None]) * inv[..., None])
    codes = np.clip(np.where(np.isnan(c), 0, c), 0, 15).astype(np.uint8)
    return codes, d, lo


def values(codes, d, lo):
    x = lo.astype(np.float32)[..., None] + d.astype(np.float32)[..., None] * codes.astype(np.float32)
    return x.reshape(*x.shape[:-2], -1)


def rope(x, cos, sin, rot, neox):
    """x [heads][D] f32 rotated by one table row, each step rounded to f32."""
    y = x.copy()
    half = rot // 2
    for i in range(half):
        a, b = (i, i + half) if neox else (2 * i, 2 * i + 1)
        y[:, a] = x[:, a] * cos[i] - x[:, b] * sin[i]
        y[:, b] = x[:, a] * sin[i] + x[:, b] * cos[i]
    return y


def store(pool, at, row, is_v, D, codes, d, lo):
    """One quantised row of one kv head into the pool (uint8) at its record's first byte."""
    gp = groups_padded(D)
    at += record_bytes(D) // 2 if is_v else 0
    flat = codes.reshape(-1)
    line = np.zeros(D // 2, np.uint8)
    for i in range(D):
        b = v_byte(D, i, row) if is_v else k_byte(D, i)
        line[b] |= flat[i] << (4 * (i & 1))
    pool[at + row * D // 2: at + (row + 1) * D // 2] = line
    sc = at + PAGE * D // 2 + row * gp * 2
    pool[sc: sc + 2 * (D // 32)] = d.view(np.uint8)
    sc += PAGE * gp * 2
    pool[sc: sc + 2 * (D // 32)] = lo.view(np.uint8)


def fetch(pool, at, D, steps=False):
    """K and V [16][D] in 64 bits of the record at byte `at`; with steps, V's d of every value too."""
    gp, out = groups_padded(D), []
    for is_v in (False, True):
        base = at + (record_bytes(D) // 2 if is_v else 0)
        x = np.zeros((PAGE, D))
        sc = pool[base + PAGE * D // 2: base + PAGE * D // 2 + 2 * PAGE * gp * 2].view(np.float16).astype(np.float64)
        d, lo = sc.reshape(2, PAGE, gp)
        for row in range(PAGE):
            at_b = np.array([v_byte(D, i, row) if is_v else k_byte(D, i) for i in range(D)])
            c = (pool[base + row * D // 2 + at_b] >> (4 * (np.arange(D) & 1)).astype(np.uint8)) & 15
            x[row] = lo[row, np.arange(D) // 32] + d[row, np.arange(D) // 32] * c
        out.append(x)
        if steps and is_v:
            out.append(d[:, np.arange(D) // 32])
    return out


def attend(q, k, v, pos, scale, softcap=0.0, window=0, steps=None):
    """Attention of queries q [rows][D] at positions pos over k, v [keys][D] in
    64 bits, and what bounds its error: sum p |v| and the largest sum |q k|;
    with steps [keys][D], sum p steps too."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    out, mean, ext, coarse = np.zeros_like(q), np.zeros_like(q), np.zeros(len(q)), np.zeros_like(q)
    for r, p in enumerate(pos):
        a = max(0, p - window + 1) if window else 0
        kk, vv = k[a:p + 1], v[a:p + 1]
        if not len(kk):
            continue
        s = kk @ q[r] * scale
        ext[r] = (np.abs(kk) @ np.abs(q[r])).max() * scale
        if softcap:
            s = softcap * np.tanh(s / softcap)
        w = np.exp(s - s.max())
        w /= w.sum()
        out[r], mean[r] = w @ vv, w @ np.abs(vv)
        if steps is not None:
            coarse[r] = w @ steps[a:p + 1]
    return (out, mean, ext) if steps is None else (out, mean, ext, coarse)


def allowed(out, mean, ext, t, weights, softcap=0.0, coarse=None):
    """How far an output of type t may be off. A score is a sum of products
    accumulated in 32 bits: off by 2^-20 of sum |q k| at most (operands of two
    f16 parts: 2^-22; sums of 128 terms in a truncating adder: under 2^-20), a
    soft cap adds 2^-21 of the cap; a weight's relative error is twice that
    (itself and its share of the sum), plus 2^-20 for the exponential and the
    sums, plus `weights`, the rounding of a weight before its product with v.
    An output is off by that share of sum p |v|, then rounded to t (with the
    smallest step of f16).

    Over the cache, v = (lo + 8 d) + d (code - 8) is summed in two parts: the
    rounded weight p d meets |code - 8| <= 8, so `weights` is a share of sum p 8
    d, and both parts together, |lo + 8 d| + 8 d <= |v| + 16 d, carry the 2^-20
    of the sums. coarse is sum p d."""
    ds = 2.0 ** -20 * ext + 2.0 ** -21 * softcap
    if coarse is None:
        off = (2 * ds + 2.0 ** -20 + weights)[:, None] * mean
    else:
        off = 2 * ds[:, None] * mean + 2.0 ** -20 * (mean + 16 * coarse) + weights * 8 * coarse
    return off * 1.01 + HALF[t] * np.abs(out) + 2.0 ** -25
