"""The key / value cache operators restated in float64 (numpy), from the definition in include/mm4.h. Test
infrastructure; nothing of the package is used here."""
import numpy as np

GROUP = 32


def row_bytes(D, bits):
    return D * bits // 8 + D // GROUP * 4


def half_towards_zero(x):
    """float64 >= 0 to the largest fp16 not above it."""
    h = x.astype(np.float16)
    bits = h.view(np.uint16).astype(np.int32)
    return np.where(h.astype(np.float64) > x, bits - 1, bits).astype(np.uint16).view(np.float16)


def quantise(x, bits):
    """(codes, scale, zero) of fp16 x [..., D]; codes [..., D], scale and zero [..., D / 32] fp16. The subtraction
    and the two quotients are the definition's fp32 operations."""
    top = np.float32(2 ** bits - 1)
    g = x.astype(np.float32).reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    g = np.clip(np.where(np.isnan(g), np.float32(0), g), np.float32(-65504), np.float32(65504))
    lo = g.min(-1, keepdims=True)
    scale = half_towards_zero(((g.max(-1, keepdims=True) - lo) / top).astype(np.float32).astype(np.float64))
    s = scale.astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(s > 0, np.minimum(np.rint((g - lo) / s), top), 0).astype(np.uint8)
    return c.reshape(x.shape), scale[..., 0], lo[..., 0].astype(np.float16)


def values(codes, scale, zero):
    """fp16 values that codes [..., D] stand for: code * scale + zero is exact in float64 up to 2^-42 of its
    size, then one rounding."""
    c = codes.astype(np.float64).reshape(*codes.shape[:-1], codes.shape[-1] // GROUP, GROUP)
    v = c * scale.astype(np.float64)[..., None] + zero.astype(np.float64)[..., None]
    return v.astype(np.float16).reshape(codes.shape)


def pack(x, bits):
    """Cache rows uint8 [..., row] of fp16 x [..., D]."""
    codes, scale, zero = quantise(x, bits)
    raw = codes if bits == 8 else codes[..., 0::2] | (codes[..., 1::2] << 4)
    par = np.stack([scale, zero], -1).reshape(*x.shape[:-1], 2 * (x.shape[-1] // GROUP))
    return np.concatenate([raw, np.ascontiguousarray(par).view(np.uint8)], -1)


def unpack(raw, D, bits):
    """fp16 values [..., D] of cache rows."""
    n = D * bits // 8
    codes = raw[..., :n] if bits == 8 else np.stack([raw[..., :n] & 15, raw[..., :n] >> 4], -1).reshape(
        *raw.shape[:-1], D)
    par = np.ascontiguousarray(raw[..., n:]).view(np.float16).reshape(*raw.shape[:-1], D // GROUP, 2)
    return values(codes, par[..., 0], par[..., 1])


def attention(Q, K, V, n, causal, scale):
    """(O, lse, tol_O, tol_lse) in float64 of the last n tokens Q [n][Hq][D] over K, V [len][Hk][D] (fp16 values).
    A row before position 0 attends to nothing: O = 0, lse = -inf.

    The tolerances bound what a kernel with fp16 inputs, fp32 sums and an fp16 result may be off:
      score  s = scale * max over keys of sum_d |q_d k_d|, each of the D + 8 fp32 operations off by at most one unit
             in the last place (2^-23, as accumulators may cut instead of rounding): ds = s (D + 8) 2^-23;
      P      an fp16 P is off by 2^-11 of itself, and the exponential by 2^-20 and by the score's ds in numerator
             and denominator, weighted by |v|: a (2^-11 + 2^-19 + 2 ds) with a = sum p |v| / sum p; the P V sums
             add a (len / 16 + 64) 2^-23 (accumulation in steps of 16 keys, and the joins); a P below fp16's
             normal range is off by 2^-25 of the largest: sum |v| 2^-25 / sum p;
      O      fp16 rounding 2^-11 |O|, or half of fp16's smallest step, 2^-25;
      lse    ds + 2^-20 + (len / 16 + 64) 2^-23 from the sum, and 2^-22 of its size.
    """
    Hq, Hk, ln = Q.shape[1], K.shape[1], K.shape[0]
    D = Q.shape[2]
    O, lse = np.zeros((n, Hq, D)), np.full((n, Hq), -np.inf)
    tol_O, tol_lse = np.zeros((n, Hq, D)), np.zeros((n, Hq))
    q64, k64, v64 = Q.astype(np.float64), K.astype(np.float64), V.astype(np.float64)
    for h in range(Hq):
        hk = h // (Hq // Hk)
        S = scale * (q64[:, h] @ k64[:, hk].T)
        A = abs(scale) * (np.abs(q64[:, h]) @ np.abs(k64[:, hk]).T)
        for i in range(n):
            seen = min(ln, max(0, ln - n + i + 1)) if causal else ln
            if seen == 0:
                continue
            m = S[i, :seen].max()
            p = np.exp(S[i, :seen] - m)
            total = p.sum()
            p /= total
            lse[i, h] = m + np.log(total)
            O[i, h] = p @ v64[:seen, hk]
            ds = A[i, :seen].max() * (D + 8) * 2.0 ** -23
            a = p @ np.abs(v64[:seen, hk])
            tol_O[i, h] = a * (2.0 ** -11 + 2.0 ** -19 + 2 * ds + (seen / 16 + 64) * 2.0 ** -23) \
                + np.abs(v64[:seen, hk]).sum(0) * 2.0 ** -25 / total + 2.0 ** -11 * np.abs(O[i, h]) + 2.0 ** -25
            tol_lse[i, h] = ds + 2.0 ** -20 + (seen / 16 + 64) * 2.0 ** -23 + 2.0 ** -22 * abs(lse[i, h])
    return O, lse, tol_O, tol_lse
