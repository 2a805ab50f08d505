"""float64 oracle of the routes attention_masked, rotary and linear_f16, each result with the bound on
its fp32 computation that the tests hold the kernels to.

Rounding: a value rounded to a type is off by at most half a step, u = 2^-24 (fp32) or 2^-11 (fp16)
relative. A sum of n terms in fp32 rounds about n times; the errors are independent, each at most u
times the sum of magnitudes so far, so four times sqrt(n) u sum|terms| holds them all (seven standard
deviations of errors uniform in half a step).
"""

from __future__ import annotations

import math

import numpy as np
from numpy.typing import NDArray

U32, U16 = 2.0**-24, 2.0**-11


def key_ranges(batch: int, seq: int, lengths: NDArray, *, mask: str, window: int = 0,
               prefix: NDArray | None = None, spans: NDArray | None = None):
    """lo and hi, [batch, seq]: token i attends the keys lo <= j < hi."""
    i = np.arange(seq, dtype=np.int64)[None, :]
    hi = np.broadcast_to(np.minimum(lengths, seq).astype(np.int64)[:, None], (batch, seq)).copy()
    lo = np.zeros((batch, seq), np.int64)
    if mask == "causal":
        hi = np.minimum(hi, i + 1)
    elif mask == "prefix":
        hi = np.minimum(hi, np.maximum(i + 1, prefix.astype(np.int64)[:, None]))
    if window:
        lo, hi = np.maximum(lo, i - window + 1), np.minimum(hi, i + window)
    if spans is not None:
        lo = np.maximum(lo, spans[..., 0].astype(np.int64))
        hi = np.minimum(hi, spans[..., 1].astype(np.int64))
    return lo, hi


def attention_masked(q: NDArray, k: NDArray, v: NDArray, lengths: NDArray, *, mask: str,
                     window: int = 0, cap: float = 0.0, scale: float | None = None,
                     prefix: NDArray | None = None, spans: NDArray | None = None,
                     slopes: NDArray | None = None, table: NDArray | None = None,
                     tokens: NDArray | None = None):
    """q [B,S,H,D], k and v [B,S,KV,D] -> (out, bound), both [B,S,H,D] (of `tokens` alone where they
    are given, zeros elsewhere). The bound, for operands of
    q's type (fp16: probabilities rounded to fp16 for the product with v, as well as the output):
      scores   4 sqrt(D) u scale sum|q k| for the sum, 8 u |s| for its scaling to log2 units, 16 u |s|
               for the tanh (s capped; fp16 up to a cap of 256: 16 u cap), 4 u |bias|; an error d of the scores changes out by at most
               2 d sum p|v|
      exp, sums over n keys   (8 + 4 sqrt(n)) u sum p|v|, numerator and denominator
      fp16     u16 (sum p|v| + |out|) for the probabilities, u16 |out| for the output
    """
    batch, seq, heads, dim = q.shape
    group = heads // k.shape[2]
    scale = dim**-0.5 if scale is None else scale
    lo, hi = key_ranges(batch, seq, lengths, mask=mask, window=window, prefix=prefix, spans=spans)
    half = q.dtype == np.float16
    out = np.zeros(q.shape)
    bound = np.zeros(q.shape)
    for b in range(batch):
        for i in range(seq) if tokens is None else tokens:
            if hi[b, i] <= lo[b, i]:
                continue
            j = np.arange(lo[b, i], hi[b, i])
            kk = np.repeat(k[b, j].astype(np.float64), group, axis=1)  # [n, H, D]
            vv = np.repeat(v[b, j].astype(np.float64), group, axis=1)
            prod = kk * q[b, i].astype(np.float64)[None]
            s = prod.sum(-1) * scale  # [n, H]
            d = 4 * math.sqrt(dim) * U32 * abs(scale) * np.abs(prod).sum(-1) + 8 * U32 * np.abs(s)
            if cap:
                s = cap * np.tanh(s / cap)
                d = d + 16 * U32 * (cap if half and cap <= 256 else np.abs(s))
            bias = np.zeros_like(s)
            if slopes is not None:
                bias = -slopes.astype(np.float64)[None] * np.abs(j - i)[:, None]
            if table is not None:
                radius = table.shape[1] // 2
                bias = table[:, np.clip(j - i, -radius, radius) + radius].T.astype(np.float64)
            with np.errstate(invalid="ignore"):
                s = s + bias
                d = d + 4 * U32 * np.where(np.isfinite(bias), np.abs(bias), 0.0)
                top = s.max(0)
                p = np.exp(s - np.where(top == -np.inf, 0.0, top))
                total = p.sum(0)
                p = p / np.where(total == 0, 1.0, total)
                out[b, i] = np.where((p == 0)[:, :, None], 0.0, p[:, :, None] * vv).sum(0)
                mass = np.where((p == 0)[:, :, None], 0.0, p[:, :, None] * np.abs(vv)).sum(0)
            # what a score's error does to out goes with its probability
            live = (p > 1e-12)
            worst = np.where(live, d, 0.0).max(0)[:, None]
            bound[b, i] = (2 * worst + (8 + 4 * math.sqrt(len(j))) * U32) * mass + U32 * np.abs(out[b, i])
            if half:
                bound[b, i] += U16 * (mass + 2 * np.abs(out[b, i])) + 2.0**-24
    return out, bound


def rotary(x: NDArray, positions: NDArray, frequencies: NDArray, *, layout: str,
           factor: float = 1.0, norm: NDArray | None = None, eps: float = 1e-6):
    """x [tokens, heads, D], positions [tokens], frequencies [rot / 2] -> (y, bound). The bound: the
    norm rounds its sum, quotient, root and two products (8 u), the table its entries (u) and the turn
    its product and fused multiply-add (2 u), so 12 u (|a| + |b|) factor; then the output's type."""
    half = x.dtype == np.float16
    r = 2 * len(frequencies)
    v = x.astype(np.float64)
    if norm is not None:
        v = v / np.sqrt((v * v).mean(-1, keepdims=True) + eps) * norm.astype(np.float64)
    angle = positions.astype(np.float64)[:, None, None] * frequencies
    cos, sin = np.cos(angle) * factor, np.sin(angle) * factor
    first, second = ((slice(0, r // 2), slice(r // 2, r)) if layout == "half"
                     else (slice(0, r, 2), slice(1, r, 2)))
    a, b = v[..., first], v[..., second]
    y, bound = v.copy(), 12 * U32 * np.abs(v)
    y[..., first], y[..., second] = a * cos - b * sin, a * sin + b * cos
    bound[..., first] = bound[..., second] = 12 * U32 * factor * (np.abs(a) + np.abs(b))
    return y, bound + (U16 * np.abs(y) + 2.0**-25 if half else U32 * np.abs(y))


_ERF = np.vectorize(math.erf, otypes=[np.float64])


def linear(x: NDArray, w: NDArray, *, bias: NDArray | None = None, residual: NDArray | None = None,
           activation: str = "none", half: bool = True):
    """x [M,K], w [N,K] -> (out, bound). The bound: 4 sqrt(K) u sum|x w| for the sum and u for the
    bias, which the activation (slope below 1.13) passes on, 16 u |y| for the activation's own
    arithmetic, u |out| for the residual, then the output's type."""
    xd, wd = x.astype(np.float64), w.astype(np.float64)
    y = xd @ wd.T
    d = 4 * math.sqrt(x.shape[1]) * U32 * (np.abs(xd) @ np.abs(wd).T)
    if bias is not None:
        y = y + bias.astype(np.float64)
        d = d + U32 * np.abs(y)
    with np.errstate(over="ignore"):
        act = {"none": lambda t: t, "relu": lambda t: np.maximum(t, 0.0),
               "gelu": lambda t: 0.5 * t * (1.0 + _ERF(t / math.sqrt(2.0))),
               "gelu_tanh": lambda t: 0.5 * t * (1.0 + np.tanh(
                   math.sqrt(2.0 / math.pi) * (t + 0.044715 * t**3))),
               "silu": lambda t: t / (1.0 + np.exp(-t))}[activation](y)
    d = 1.13 * d + (16 * U32 * np.abs(y) if activation != "none" else 0.0)
    out = act if residual is None else act + residual.astype(np.float64)
    d = d + U32 * np.abs(out)
    return out, d + (U16 * np.abs(out) + 2.0**-25 if half else 0.0)
