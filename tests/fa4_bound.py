"""Attention over Q4_0 K and V: the exact result in 64 bits and how far the kernels'
arithmetic may be from it, element by element.

With s the scores, p = exp(s - max s), L = sum p, and u = 2^-24:
  scores  A_j = scale sum_b |d_b| sum_e (level_e + 8) |q_e| bounds the terms of the two
          sums that make s_j (levels 0..15 and -8 sum q), 33 terms a block: 64 u A_j;
          q held to 23 bits of the row's largest element: scale sum |k| max|q| 2^-23; the scaling by d, the sum over blocks, the row's
          scale and the mask's addition: 16 u A_j + 4 u |mask_j|
          BF16 y, many rows: k in fp16, half a step of 11 bits: 2^-11 scale sum |k| |q|
  p       2^-22 for the exponential, 2 u |s_j - max s| for its argument, and the score's
          error, doubled for the second order: rho_j
  P, V    F32 y: P as two fp16, 2^-22, and the low x low product left out, 2^-22; BF16 y: P and
          V one fp16 each, half a step of 11 significant bits, 2^-11 either; parts of P below fp16's range: 2^-33 of the largest p
  sums    up to 3 products a key in fp32: 8 sqrt(3 n) u (the probabilistic bound of Higham
          and Mary, failure below 1e-13), for the numerator and for L
  rescale one rounding each time a wave's maximum moves, at most once a tile, and once a
          merge: (tiles + 8) 2 u
  y       its own rounding, half a step: 2^-24 F32 (and the division's 2^-23), 2^-8 BF16 (8
          significant bits: a value 1 + 2^-8 lies between 1 and 1 + 2^-7)
"""
import numpy as np
import q4

U = 2.0 ** -24


def row(q, k, v, mask, scale, f32_y):
    """q (D,) float64, k and v Q4_0 bytes (n, D / 32 * 18), mask (n,) float64 or None -> (y, bound), each (D,)."""
    D, n = len(q), len(k)
    if mask is not None:
        on = mask != -np.inf
        k, v, mask = k[on], v[on], mask[on]
    if len(k) == 0:
        return np.full(D, np.nan), np.zeros(D)
    kf, vf = q4.dequantize(k), q4.dequantize(v)
    d = np.repeat(np.abs(k.reshape(len(k), -1, 18)[:, :, :2].copy().view(np.float16)[:, :, 0].astype(np.float64)), 32, axis=1)
    level = np.where(d > 0, np.abs(kf) / np.where(d > 0, d, 1) + 16, 16)  # |level - 8| + 16 >= level + 8
    s = kf @ q * scale
    A = (d * level) @ np.abs(q) * abs(scale)
    ds = 80 * U * A + 2.0 ** -23 * np.abs(kf).sum(1) * np.abs(q).max() * abs(scale)
    if not f32_y:
        ds = ds + 2.0 ** -11 * (np.abs(kf) @ np.abs(q)) * abs(scale)
    if mask is not None:
        s = s + mask
        ds = ds + 4 * U * np.abs(mask)
    top = s.max()
    p = np.exp(s - top)
    L = p.sum()
    y = p @ vf / L
    rho = 2.0 ** -22 + 2 * U * (top - s) + 2 * ds
    each = 2.0 ** -21 if f32_y else 2.0 ** -10
    rest = each + 16 * np.sqrt(3.0 * n) * U + (n / 32 + 8) * 2 * U + (p @ rho) / L
    av = np.abs(vf)
    bound = ((p * (rho + rest)) @ av + 2.0 ** -33 * av.sum(0)) / L
    bound += np.abs(y) * (2.0 ** -22 if f32_y else 2.0 ** -8 + 2.0 ** -22) + 1e-37
    return y, bound
