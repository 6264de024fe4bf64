"""Paged-cache operators restated in 64 bits, sequence by sequence (test infrastructure)."""
from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0


def dequantise(pages, scales):
    x = pages.double()
    return x if scales is None else x * scales.double()[:, :, None, None]


def rotate(x, cos, sin, layout):
    """x [rows, heads, dim] double, cos / sin [rows, rot] double -> rotated rows and the sum of the magnitudes of the two products."""
    rot = cos.shape[1]
    y, mag = x.clone(), x.abs()
    for d in range(rot):
        pair, sign = (d ^ 1, -1.0 if d % 2 == 0 else 1.0) if layout == "interleaved" else \
            ((d + rot // 2, -1.0) if d < rot // 2 else (d - rot // 2, 1.0))
        a, b = x[..., d] * cos[:, None, d], x[..., pair] * sin[:, None, d]
        y[..., d], mag[..., d] = a + sign * b, a.abs() + b.abs()
    return y, mag


def scale_for(amax: float) -> float:
    """Smallest power of two, exponent in [-64, 120], that brings amax to 448 or less."""
    e = -64
    while e < 120 and amax > E4M3_MAX * 2.0 ** e:
        e += 1
    return 2.0 ** e


def rows_of(cu, seqs, tokens, b):
    return (int(cu[b]), int(cu[b + 1])) if cu is not None else (b * (tokens // seqs), (b + 1) * (tokens // seqs))


def attention(q, k, v, table, lengths, cu, page, scale):
    """q [tokens, heads, dim]; k, v dequantised pages [pages, kv_heads, page, dim] in 64 bits.  Returns (out, mean of the
    weighted magnitudes of the values); rows of no sequence are NaN."""
    q = q.double()
    out = torch.full_like(q, math.nan)
    mag = torch.zeros_like(q)
    seqs, group = table.shape[0], q.shape[1] // k.shape[1]
    for b in range(seqs):
        r0, r1 = rows_of(cu, seqs, q.shape[0], b)
        length, n = max(0, min(int(lengths[b]), table.shape[1] * page)), r1 - r0
        ids = table[b, : -(-length // page)].long()
        there = ((ids >= 0) & (ids < k.shape[0])).repeat_interleave(page)[:length]
        safe = torch.where((ids >= 0) & (ids < k.shape[0]), ids, 0)
        for i in range(n):
            seen = max(0, min(length, length - n + i + 1))
            keep = there[:seen]
            for h in range(q.shape[1]):
                kk = k[safe, h // group].reshape(-1, q.shape[2])[:seen][keep]
                vv = v[safe, h // group].reshape(-1, q.shape[2])[:seen][keep]
                if kk.shape[0] == 0:
                    out[r0 + i, h] = 0.0
                    continue
                w = torch.softmax(kk @ q[r0 + i, h] * scale, dim=0)
                out[r0 + i, h], mag[r0 + i, h] = w @ vv, w @ vv.abs()
    return out, mag


def attention_tolerance(ref, mag, fp8, positions, vmax, many_rows=False):
    """Result rounded to bf16 (2^-8).  Weights: f16 (2^-11, and 2^-25 of the largest where that is less) for the 8-bit cache; two
    bf16 terms (2^-16) for a bf16 cache; one bf16 term where a sequence has more than 32 (token, head of the group) rows and the
    large-tile kernel takes it: |sum w_j (1 + e_j) v_j - sum w_j v_j| <= max |e_j| sum w_j |v_j| = 2^-8 mag.  Scores and sums in fp32
    (2^-14 is generous for up to 128 products and 2^14 positions)."""
    weight = 2.0 ** -11 if fp8 else 2.0 ** -8 if many_rows else 2.0 ** -16
    return 2.0 ** -8 * ref.abs() + (weight + 2.0 ** -14) * mag + (positions * 2.0 ** -25 * vmax if fp8 else 0.0)
