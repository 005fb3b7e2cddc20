"""Plain 64-bit forms of rotary positions, the paged key-value cache and the attention of one new token over it, for the
tests: loops over tokens and rows on the CPU, nothing shared with the library."""
import math

import numpy as np
import torch

E4M3_MAX = 448.0


def rotary(x, positions, inv_freq, interleaved=False, scale=1.0, inverse=False):
    """x [B,H,T,d] double, positions [B,T], inv_freq [rot/2] double."""
    y = x.double().clone()
    half = inv_freq.numel()
    a = positions.double().unsqueeze(-1) * inv_freq.double()
    c, s = scale * torch.cos(a).unsqueeze(1), scale * torch.sin(a).unsqueeze(1) * (-1.0 if inverse else 1.0)
    i0 = torch.arange(half) * 2 if interleaved else torch.arange(half)
    i1 = i0 + 1 if interleaved else i0 + half
    x0, x1 = x[..., i0].double(), x[..., i1].double()
    y[..., i0] = x0 * c - x1 * s
    y[..., i1] = x0 * s + x1 * c
    return y


def rotary_bound(x, inv_freq, interleaved=False, scale=1.0):
    """Elementwise bound of an FP32 evaluation: the fraction of a turn (at most one half) is rounded to 2^-24 of itself,
    which moves cosine and sine by at most pi * 2^-24; sincospif is within 2 ulp (2^-23); one multiplication by the
    scale, two products and a sum add a rounding each: below 12 * 2^-24 of |x0| + |x1|."""
    b = torch.zeros_like(x, dtype=torch.float64)
    half = inv_freq.numel()
    i0 = torch.arange(half) * 2 if interleaved else torch.arange(half)
    i1 = i0 + 1 if interleaved else i0 + half
    both = (x[..., i0].abs() + x[..., i1].abs()).double() * abs(scale) * 12 * 2.0 ** -24
    b[..., i0] = both
    b[..., i1] = both
    return b


def e4m3_row(row):
    """(values the 8-bit row stands for, its power of two) of a 1-D float array, NaN where the value is not finite."""
    row = np.asarray(row, dtype=np.float64)
    finite = np.isfinite(row)
    amax = float(np.abs(row[finite]).max()) if finite.any() else 0.0
    e = -126
    if amax > 0:
        m, x = math.frexp(amax / E4M3_MAX)          # exact: 448 = 7 * 2^6 only enters the comparison below
        e = x - 1
        while amax > E4M3_MAX * 2.0 ** e:
            e += 1
        while e > -126 and amax <= E4M3_MAX * 2.0 ** (e - 1):
            e -= 1
        e = max(e, -126)
    unit = 2.0 ** e
    y = np.where(finite, row, 0.0) / unit
    step = 2.0 ** (np.floor(np.log2(np.maximum(np.abs(y), 2.0 ** -6))) - 3)
    out = np.rint(y / step) * step * unit           # rint rounds half to even
    out[~finite] = np.nan
    return out, unit


def place(page_table, b, position, page_size):
    return int(page_table[b, position // page_size]), position % page_size


def attention(q, k, v, scale):
    """o, log-sum-exp and, for the bounds, sum p|v| and the largest |score| and scale * sum |q||k|; q [G,d], k, v [n,d] double."""
    s = (q @ k.T) * scale
    m = s.max(dim=1, keepdim=True).values
    p = torch.exp(s - m)
    total = p.sum(dim=1, keepdim=True)
    p = p / total
    reach = ((q.abs() @ k.abs().T) * abs(scale)).max(dim=1, keepdim=True).values
    return p @ v, (m + torch.log(total)).squeeze(1), p @ v.abs(), s.abs().max(dim=1, keepdim=True).values, reach


def attention_bound(d, n, absolute, top, reach):
    """Bounds of |o - exact| and |lse - exact| for an FP32 evaluation, roundings taken as independent (4 sigma).
    A score sums d products: 4 sqrt(d) 2^-24 of scale * sum |q||k|; scaling it to base 2 and subtracting the maximum rounds
    it by at most 3 * 2^-24 of the largest score; exp2 is within 2 ulp (2^-22).  Together delta, relative to a weight.
    Weights enter numerator and denominator: 2 delta; either sums n terms: 2 * 4 sqrt(n) 2^-24; joining parts and the
    division add a few roundings, 8 * 2^-24."""
    delta = 4 * math.sqrt(d) * 2.0 ** -24 * reach + 3 * 2.0 ** -24 * top + 2.0 ** -22
    rel = 2 * delta + 8 * math.sqrt(n) * 2.0 ** -24 + 8 * 2.0 ** -24
    return rel * absolute + 1e-30, (delta + (4 * math.sqrt(n) + 8) * 2.0 ** -24 + 2.0 ** -23 * top).squeeze(1)
