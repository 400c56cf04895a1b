"""The generation operators' definitions in numpy, in 64 bits, for the tests."""
from __future__ import annotations

import math

import numpy as np

GROUP = 32


def rotate(x, cos, sin, pos):
    """x [rows][heads][hd] fp32 at positions pos: glc_rope's arithmetic, every product and sum rounded to fp32."""
    c, s = cos[pos][:, None, :], sin[pos][:, None, :]
    a, b = x[..., 0::2], x[..., 1::2]
    out = np.empty_like(x)
    with np.errstate(all="ignore"):
        out[..., 0::2] = a * c - b * s
        out[..., 1::2] = a * s + b * c
    return out


def quantize(x):
    """(codes uint8 [..., hd], scales float16 [..., hd/32]) of fp32 x [..., hd]."""
    y = x.reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(all="ignore"):
        mag = np.abs(y)
        far = np.take_along_axis(y, np.argmax(np.where(np.isnan(mag), np.inf, mag), -1)[..., None], -1)
        d = np.clip((far.astype(np.float64) / -8), -65504, 65504).astype(np.float16)
        code = np.clip(np.rint(y.astype(np.float64) / np.where(d == 0, 1, d).astype(np.float64)), -8, 7) + 8
        bad = ~np.isfinite(y).all(-1, keepdims=True)
        code = np.where((d == 0) | bad, 8, code).astype(np.uint8)
        d = np.where(bad, np.float16(np.nan), d)
    return code.reshape(x.shape), d[..., 0]


def numbers(codes, scales):
    """fp32 numbers of codes [..., hd] and scales [..., hd/32] (exact: 15 bits)."""
    c = codes.astype(np.float32).reshape(*codes.shape[:-1], -1, GROUP) - 8
    with np.errstate(all="ignore"):
        return (c * scales.astype(np.float32)[..., None]).reshape(codes.shape)


class Pools:
    """Host image of the two pools and their layout."""

    def __init__(self, pages, page, heads, hd, rng=None):
        self.pages, self.page, self.heads, self.hd = pages, page, heads, hd
        self.chunk = page * hd * 9 // 16
        shape = (2, pages, heads, self.chunk)
        self.raw = np.zeros(shape, np.uint8)
        if rng is not None:
            self.codes[:] = rng.integers(0, 256, self.codes.shape)
            d = (2.1 + 0.4 * rng.standard_normal(self.scales.shape)) / 8 * rng.choice([-1, 1], self.scales.shape)
            self.scales[:] = d.astype(np.float16)

    @property
    def codes(self):  # [2][pages][heads][page][hd/2] bytes, a view
        return np.lib.stride_tricks.as_strided(
            self.raw, (2, self.pages, self.heads, self.page, self.hd // 2), (*self.raw.strides[:3], self.hd // 2, 1))

    @property
    def scales(self):  # [2][pages][heads][page][hd/32] halves, a view
        base = self.raw.reshape(-1)[self.page * self.hd // 2:]
        return np.lib.stride_tricks.as_strided(
            base.view(np.float16), (2, self.pages, self.heads, self.page, self.hd // GROUP),
            (*self.raw.strides[:3], self.hd // GROUP * 2, 2))

    def store(self, side, page, slot, codes, scales):
        """codes [heads][hd], scales [heads][hd/32] of one token."""
        self.codes[side, page, :, slot] = codes[:, 0::2] | (codes[:, 1::2] << 4)
        self.scales[side, page, :, slot] = scales

    def token(self, side, page, slot):
        """fp32 [heads][hd] of one token."""
        b = self.codes[side, page, :, slot]
        codes = np.stack([b & 15, b >> 4], -1).reshape(self.heads, self.hd)
        return numbers(codes, self.scales[side, page, :, slot])

    def sequence(self, side, table, length):
        """fp32 [length][heads][hd]."""
        n = -(-length // self.page)
        b = self.codes[side, table[:n]]  # [n][heads][page][hd/2]
        codes = np.stack([b & 15, b >> 4], -1).reshape(n, self.heads, self.page, self.hd)
        x = numbers(codes, self.scales[side, table[:n]])
        return x.transpose(0, 2, 1, 3).reshape(n * self.page, self.heads, self.hd)[:length]


def attend(pools, table, lens, starts, q, heads):
    """(o, lse, bound) of q [rows][heads * hd] in 64 bits; rows of no sequence are NaN.  bound [rows][heads]: the
    largest sum of |q_i k_i| / sqrt(hd) over the keys, which the kernel's error goes by."""
    rows, hd, hkv = q.shape[0], pools.hd, pools.heads
    o = np.full((rows, heads, hd), np.nan)
    lse = np.full((rows, heads), np.nan)
    bound = np.zeros((rows, heads))
    for b, length in enumerate(lens):
        first, end = (b, b + 1) if starts is None else (starts[b], starts[b + 1])
        if end <= first:
            continue
        if length > 0:
            k = pools.sequence(0, table[b], length).astype(np.float64)
            v = pools.sequence(1, table[b], length).astype(np.float64)
        for t in range(first, end):
            see = length - (end - first) + (t - first) + 1
            if see <= 0:
                o[t], lse[t] = 0, -np.inf
                continue
            for h in range(heads):
                x = q[t, h * hd:(h + 1) * hd].astype(np.float64)
                kk, vv = k[:see, h // (heads // hkv)], v[:see, h // (heads // hkv)]
                s = kk @ x / math.sqrt(hd)
                m = s.max()
                p = np.exp(s - m)
                o[t, h] = p @ vv / p.sum()
                lse[t, h] = m + np.log(p.sum())
                bound[t, h] = (np.abs(kk) @ np.abs(x)).max() / math.sqrt(hd)
    return o.reshape(rows, heads * hd), lse, bound


def kept_tokens(x, temperature, k, p, m):
    """(kept token ids in index order, their weights in 64 bits) of one row of logits, by the definition."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[x[order] > -np.inf]
    if len(order) == 0:
        return order, np.zeros(0)
    top = x[order[0]]
    if not temperature > 0:
        return order[:1], np.ones(1)
    with np.errstate(all="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / np.float64(temperature)))
    n = len(order) if k <= 0 else min(k, len(order))
    if p < 1:
        before = np.cumsum(w[:n]) - w[:n]
        n = max(1, int((before < p * w[:n].sum()).sum()))
    keep = np.ones(n, bool) if not m > 0 else (x[order[:n]] == top) if m >= 1 else w[:n] >= m
    ids = np.sort(order[:n][keep])
    inverse = np.empty(len(x), np.int64)
    inverse[order] = np.arange(len(order))
    return ids, w[inverse[ids]]
