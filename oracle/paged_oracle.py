"""CPU oracle of the paged-cache operators.  TEST INFRASTRUCTURE ONLY.

Float64 / integer numpy restatements, from the definitions in
``include/mla_decode_b200.h``, of: the 4-bit latent form (quantise, pack, unpack), block
tables and slots, rotary positions, and decode over a dequantised cache.  The product
path never imports this module.
"""
from __future__ import annotations

import math

import numpy as np

GROUP = 32
NIBBLE_DIM = (0, 2, 4, 6, 1, 3, 5, 7)   # dim of eight held by each nibble of a word, lowest first


def quantise_int4(x):
    """Rows [..., 512] -> (codes 0..15 uint8 [..., 512], scales float16 [..., 16])."""
    g = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(all="ignore"):
        amax = np.nanmax(np.where(np.isnan(g), 0.0, np.abs(g)), axis=-1)
        s = np.minimum(amax / 7.0, 65504.0).astype(np.float16)
        sf = s.astype(np.float64)[..., None]
        n = np.where(sf > 0, np.clip(np.rint(g / np.where(sf > 0, sf, 1.0)), -8, 7), 0.0)
        n = np.where(np.isnan(g), 0.0, n)
    return (n + 8).astype(np.uint8).reshape(x.shape), s


def pack_int4(codes):
    """Codes [..., 512] -> bytes [..., 256]."""
    w = np.zeros((*codes.shape[:-1], codes.shape[-1] // 8), np.uint32)
    c = codes.reshape(*codes.shape[:-1], -1, 8).astype(np.uint32)
    for nib, d in enumerate(NIBBLE_DIM):
        w |= c[..., d] << np.uint32(4 * nib)
    return w.astype("<u4").view(np.uint8)


def unpack_int4(data):
    """Bytes [..., 256] -> codes [..., 512]."""
    w = np.ascontiguousarray(data).view("<u4")
    out = np.empty((*w.shape, 8), np.uint8)
    for nib, d in enumerate(NIBBLE_DIM):
        out[..., d] = (w >> np.uint32(4 * nib)) & 15
    return out.reshape(*w.shape[:-1], -1)


def dequantise_int4(codes, scales):
    """Codes [..., 512] and scales [..., 16] -> float64 rows."""
    n = codes.astype(np.float64) - 8.0
    return n * np.repeat(scales.astype(np.float64), GROUP, axis=-1)


def extend_tables(table, lens, new, free, free_pos, page, num_pages, num_tokens, q_len=0, whole=False):
    """mla_extend_block_tables (``whole``: mla_extend_block_tables_whole), request by request
    and row by row."""
    table = [list(r) for r in table]
    max_pages = len(table[0])
    cover = max_pages * page
    slots, positions = [-1] * num_tokens, [0] * num_tokens
    pos = min(max(free_pos, 0), len(free))
    out_lens, cu, at, closed = [], [0], 0, False
    for i, (length, n) in enumerate(zip(lens, new)):
        length, n = min(max(length, 0), cover), max(n, 0)
        if q_len:
            n = min(n, q_len)
            first = (i + 1) * q_len - n
            kept = n
        else:
            first, kept = at, max(0, min(n, num_tokens - at))
        held = -(-length // page)
        end = min(length + kept, cover)
        if whole:
            lacks = -(-end // page) - held
            if length + kept > cover:
                end = length
            elif lacks and (closed or lacks > len(free) - pos):
                closed, end = True, length
        got = 0
        while held + got < -(-end // page) and pos < len(free):
            table[i][held + got] = free[pos]
            pos += 1
            got += 1
        end = min(end, (held + got) * page)
        for t in range(kept):
            p = length + t
            positions[first + t] = p
            if p < end:
                pg = table[i][p // page]
                if 0 <= pg < num_pages:
                    slots[first + t] = pg * page + p % page
        out_lens.append(end)
        at += kept
        cu.append(at)
    return table, out_lens, pos, slots, positions, cu


def frequencies(rot_dim, base=10000.0, scaling=None):
    """Angle per position of every pair and the gain, as rotary_frequencies defines them."""
    d, i = rot_dim, np.arange(rot_dim // 2, dtype=np.float64)
    kind = (scaling or {}).get("type")
    f = (scaling or {}).get("factor", 1.0)
    if kind == "ntk":
        base = base * f ** (d / (d - 2))
    w = np.power(base, -2.0 * i / d)
    if kind == "linear":
        return w / f, 1.0
    if kind != "yarn":
        return w, 1.0
    n = scaling["original_max_position"]
    edge = [d * np.log(n / (2 * np.pi * scaling.get(k, v))) / (2 * np.log(base))
            for k, v in (("beta_fast", 32.0), ("beta_slow", 1.0))]
    lo, hi = max(np.floor(edge[0]), 0), min(np.ceil(edge[1]), d - 1)
    ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
    return w * (1 - ramp) + w / f * ramp, scaling.get("gain", 0.1 * np.log(f) + 1)


def rotate(x, pos, freq, gain, interleaved, offset=0):
    """float64 rotation of dims [offset, offset + 2 len(freq)) of x [tokens, heads, dim]."""
    x = np.array(x, np.float64)
    d = 2 * len(freq)
    angle = np.asarray(pos, np.float64)[:, None, None] * freq
    c, s = np.cos(angle) * gain, np.sin(angle) * gain
    part = x[..., offset:offset + d]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :d // 2], part[..., d // 2:])
    ra, rb = a * c - b * s, a * s + b * c
    if interleaved:
        part = np.stack((ra, rb), -1).reshape(part.shape)
    else:
        part = np.concatenate((ra, rb), -1)
    x[..., offset:offset + d] = part
    return x


def rotate_bound(x, freq, gain, offset=0, interleaved=True):
    """|a| + |b| of every rotated dim's pair times the gain (0 for copied dims): the scale of
    the float32 error of a rotated value."""
    x = np.abs(np.array(x, np.float64))
    d = 2 * len(freq)
    out = np.zeros_like(x)
    part = x[..., offset:offset + d]
    if interleaved:
        pair = np.repeat(part[..., 0::2] + part[..., 1::2], 2, axis=-1)
    else:
        pair = np.concatenate([part[..., :d // 2] + part[..., d // 2:]] * 2, -1)
    out[..., offset:offset + d] = pair * abs(gain)
    return out


def decode(q, q_pe, v, k_pe, scale):
    """One query sequence: q [h, 512], q_pe [h, 64], rows v [n, 512], k_pe [n, 64] (float64).

    Returns (out, lse, spread, ds): spread [h, 512] bounds the error of a kernel that rounds
    each weight and each row value once to fp16 (half a step, 2^-11 relative, each) and the
    row values in the scores too: with ds >= |error of a score|, a weight is off by at most
    exp(2 ds) - 1 relative, so the output by (2 ds + 2 * 2^-11) sum p |v| to first order
    (a twentieth is added for the rest).  A weight below fp16's normal range (2^-14 of the
    row's largest) is off by up to half the smallest step, 2^-25 of the largest weight,
    hence 2^-25 sum |v| / z.  ds counts, beside the row values, the float32 sums of 576
    products: each sum is off by at most 2^-23 (truncated) of the magnitudes' sum, together
    below 2^-13 of it.  The log-sum-exp is off by at
    most ds [h, 1], the largest error of a score.
    """
    if len(v) == 0:
        return np.zeros(q.shape), np.full(len(q), -math.inf), np.zeros(q.shape), np.zeros((len(q), 1))
    s = (q @ v.T + q_pe @ k_pe.T) * scale
    m = s.max(-1, keepdims=True)
    p = np.exp(s - m)
    z = p.sum(-1, keepdims=True)
    p /= z
    half = 2.0 ** -11
    mags = np.abs(q) @ np.abs(v).T
    sums = mags + np.abs(q_pe) @ np.abs(k_pe).T
    ds = scale * (half * mags + 2.0 ** -13 * sums).max(-1, keepdims=True) + 1e-5
    return p @ v, (np.log(z) + m)[:, 0], \
        1.05 * (2 * ds + 2 * half) * (p @ np.abs(v)) + 2.0 ** -25 * np.abs(v).sum(0) / z, ds


def rounding_gate(q, q_pe, v, k_pe, scale, dtype):
    """What relative L2 distance from the rounded result such a kernel is expected to have, as
    a square.  A rounding to fp16 is off by a uniform share of half a step, 2^-11 / m relative
    for a mantissa m in [1, 2), log-uniform: rms r = 2^-11 sqrt(0.541 / 3) = 2.07e-4.  A
    weight and a row value are rounded once each, and the row values move a score by
    r scale sqrt(sum q^2 v^2) (rms), that is the weight by as much relative: together
    d = r sqrt(2 + scale^2 sum q^2 v^2).  The result is then rounded to steps of 2^-7 / m
    (bf16; fp16 2^-10 / m) of it, 0.72 of that on average: with probability |error| / step it
    lands on the other neighbour, a whole step away, hence d^2 + step E|error| with
    E|error| = 0.8 d for a normal error.
    """
    s = (q @ v.T + q_pe @ k_pe.T) * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    r2 = 2.0 ** -22 * 0.541 / 3
    d2 = r2 * (2 + scale ** 2 * (p * ((q * q) @ (v * v).T)).sum(-1).mean())
    step = 0.72 * (2.0 ** -7 if dtype == "bf16" else 2.0 ** -10)
    return d2 + step * 0.8 * math.sqrt(d2)
