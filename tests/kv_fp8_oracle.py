"""The 8-bit paged KV cache in plain numpy: float64 and exact e4m3 arithmetic (formats in
include/dli_hip.h). Pools are numpy uint8 arrays, positions and tables plain lists. check_attention
holds an attention's output against it."""
from __future__ import annotations

import numpy as np
import torch

LARGEST = 448.0


def _e4m3_values():
    c = np.arange(256)
    e, m = (c >> 3) & 15, (c & 7) / 8
    v = np.where(e > 0, (1 + m) * 2.0 ** (np.maximum(e, 1) - 7.0), m * 2.0 ** -6)
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >> 7 == 1, -v, v)


E4M3 = _e4m3_values()
_POSITIVE = E4M3[:127]  # ascending, 0 .. 448


def quantize(x):
    """float64 [.., D] -> codes [.., D], scale codes [..]."""
    x = np.asarray(x, np.float64)
    top = np.abs(x).max(-1)
    finite = np.isfinite(top)
    safe = np.where(finite, top, 0.0)
    code = np.zeros(top.shape, np.int64)  # least c >= 0 with top / 2^(c - 127) <= 448
    with np.errstate(divide="ignore"):
        guess = np.where(safe > 0, np.floor(np.log2(np.maximum(safe, 1e-300) / LARGEST)), -127)
    for delta in (2, 1, 0, -1):
        c = np.clip(guess + 127 + delta, 0, 254).astype(np.int64)
        code = np.where(safe <= LARGEST * 2.0 ** (c - 127.0), c, code)
    y = np.where(finite[..., None], np.abs(x), 0.0) / (2.0 ** (code - 127.0))[..., None]
    hi = np.clip(np.searchsorted(_POSITIVE, y), 0, 126)
    lo = np.maximum(hi - 1, 0)
    d_hi, d_lo = _POSITIVE[hi] - y, y - _POSITIVE[lo]
    pick_hi = (d_hi < d_lo) | ((d_hi == d_lo) & (hi % 2 == 0)) | (_POSITIVE[hi] == y)
    codes = np.where(pick_hi, hi, lo).astype(np.uint8)
    codes = np.where(finite[..., None], codes | (np.signbit(x).astype(np.uint8) << 7), 0)
    return codes.astype(np.uint8), np.where(finite, code, 255).astype(np.uint8)


def scale_values(codes):
    c = codes.astype(np.float64)
    return np.where(codes == 255, np.nan, 2.0 ** (c - 127))


class Cache:
    """key [N, H, bs, D], value [N, H, D, bs], scales [N, H, 2, bs], table [B, max_blocks]."""

    def __init__(self, key, value, scales, table):
        self.key, self.value, self.scales, self.table = (np.array(x) for x in (key, value, scales, table))
        self.block = self.key.shape[2]

    @property
    def capacity(self):
        return self.table.shape[1] * self.block

    def place(self, b, pos):
        """(page, slot), or None."""
        if pos < 0 or pos >= self.capacity:
            return None
        page = int(self.table[b, pos // self.block])
        return (page, pos % self.block) if 0 <= page < self.key.shape[0] else None

    def append(self, k, v, first):
        """k, v float64 [B, H, S, D]; first: position of each sequence's first token."""
        kc, ks = quantize(k)
        vc, vs = quantize(v)
        for b in range(k.shape[0]):
            for s in range(k.shape[2]):
                at = self.place(b, first[b] + s)
                if at is None:
                    continue
                page, slot = at
                self.key[page, :, slot] = kc[b, :, s]
                self.value[page, :, :, slot] = vc[b, :, s]
                self.scales[page, :, 0, slot] = ks[b, :, s]
                self.scales[page, :, 1, slot] = vs[b, :, s]

    def rows(self, b, pos):
        """(k, v) float64 [H, D] at a position, None where nothing is held."""
        at = self.place(b, pos)
        if at is None:
            return None
        page, slot = at
        k = E4M3[self.key[page, :, slot]] * scale_values(self.scales[page, :, 0, slot])[:, None]
        v = E4M3[self.value[page, :, :, slot]] * scale_values(self.scales[page, :, 1, slot])[:, None]
        nan = (self.scales[page, :, :, slot] == 255)
        return np.where(nan[:, :1], np.nan, k), np.where(nan[:, 1:], np.nan, v)

    def read(self, first, seq):
        B, H, D = self.table.shape[0], self.key.shape[1], self.key.shape[3]
        k, v = np.zeros((B, H, seq, D)), np.zeros((B, H, seq, D))
        for b in range(B):
            for s in range(seq):
                held = self.rows(b, first[b] + s)
                if held is not None:
                    k[b, :, s], v[b, :, s] = held
        return k, v

    def attention(self, q, past, causal, scale):
        """q float64 [B, Hq, S, D] -> (out, magnitude sum_t p_t |v_t|, largest sum_d |q_d k_d| scale
        of a row, sum_t |v_t| as if every token had the largest value scale), the last three for error
        bounds."""
        B, Hq, S, D = q.shape
        H = self.key.shape[1]
        group = Hq // H
        out, mag = np.zeros_like(q), np.zeros_like(q)
        spread, level = np.zeros((B, Hq, S, 1)), np.zeros_like(q)
        for b in range(B):
            last = min(max(past[b] + S, 0), self.capacity)
            held = [self.rows(b, p) for p in range(last)]
            at = np.array([p for p in range(last) if held[p] is not None], np.int64)
            if len(at):
                K, V = (np.stack([held[p][i] for p in at], 1) for i in (0, 1))  # [H, T, D]
                size = np.stack([scale_values(self.scales[self.place(b, p)[0], :, 1,
                                                          self.place(b, p)[1]]) for p in at], 1)
            for i in range(S):
                seen = min(max(past[b] + (i + 1 if causal else S), 0), self.capacity)
                if seen == 0:
                    continue
                use = at < seen
                for h in range(Hq):
                    if not use.any():
                        continue
                    Kh, Vh = K[h // group][use], V[h // group][use]
                    s = Kh @ q[b, h, i] * scale
                    with np.errstate(invalid="ignore"):
                        p = np.exp(s - s.max())
                        p = p / p.sum()
                        out[b, h, i], mag[b, h, i] = p @ Vh, p @ np.abs(Vh)
                    one = size[h // group][use][:, None]
                    level[b, h, i] = (np.abs(Vh) / one).sum(0) * one.max()
                    spread[b, h, i] = (np.abs(Kh) @ np.abs(q[b, h, i])).max() * abs(scale)
        return out, mag, spread, level


def check_attention(out, want, dtype, keys, dim):
    """want: (value, magnitude A = sum p |v|, spread = largest sum |q k| scale, level = sum |element|
    times the largest value scale) in float64. The output is rounded once (half a step, and another half
    of the least subnormal; half a step past the largest number to infinity). A weight is rounded to f16 once
    (bf16 outputs) or kept to 22 bits; a score's fp32 sum of `dim` products, its scaling and
    the exponential shift it by at most (dim + 8) 2^-24 of the row's spread and the largest exponent
    argument, which moves a weight by that share and its sum likewise; the outputs' fp32 sums run
    over at most 4 steps a 64-key tile and the joins. f16's least step is 2^-24, so a weight (and the
    rest of one in two terms) is off by up to 2^-25 in any case; the row's sum of weights is at least
    2^11 in those units (its reference's own weight) and an element's factor at most the largest value
    scale: 2^-36 of the level."""
    value, mag, spread, level = want
    got = out.double().cpu().numpy()
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    weight = 2.0 ** -12 if dtype == torch.bfloat16 else 2.0 ** -22
    score = 2 * (dim + 8) * 2.0 ** -24 * (spread + 30)
    sums = (4 * (keys / 64) + 96) * 2.0 ** -24
    bound = half * np.abs(value) + (1 + half) * (weight + score + sums) * mag + tiny
    bound += 2.0 ** -36 * level
    nan = np.isnan(value)
    assert np.array_equal(np.isnan(got), nan)
    over = np.abs(np.nan_to_num(value)) > (1 + half) * torch.finfo(dtype).max
    assert np.array_equal(got[over], np.copysign(np.inf, value[over]))
    with np.errstate(invalid="ignore"):
        err = np.where(nan | over, 0.0, np.abs(got - value))
    worst = np.nanmax(np.where(bound > 0, err / np.maximum(bound, 1e-300), err > 0)) if err.size else 0
    assert worst <= 1, worst
