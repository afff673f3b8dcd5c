"""Plain implementations of the norm, the router's product and the adapters, in
64 bits where the formula has sums (CPU, numpy)."""
import numpy as np

from oracle import fp8, mx, spec


def rms_norm(x, residual, weight, eps, bf16):
    """(r, n): the new stream and the fp32 norm; x, residual, weight fp32 arrays
    whose values are those of the stored type (bf16: the stream is bf16)."""
    r = x if residual is None else (x + residual).astype(np.float32)
    if residual is not None and bf16:
        r = fp8.bf16_round(r)
    m = np.mean(np.square(r.astype(np.float64)), axis=1, keepdims=True)
    rstd = (1.0 / np.sqrt(m + eps)).astype(np.float32)
    return r, ((r * rstd).astype(np.float32) * weight).astype(np.float32)


def quantise(n, scales, scale=None):
    """(q bytes, s) of fp32 n."""
    if scales == "group":
        return spec.quant_group_1x128(n)
    if scales == "mx":
        return mx.quant_mx(n)
    if scale is None:
        q, s = spec.quant_per_tensor(n)
        return q, np.atleast_1d(np.asarray(s, np.float32))
    return fp8.f32_to_e4m3((n / np.float32(scale)).astype(np.float32)), np.array([scale], np.float32)


def lora(y, x, a, b, ids, scaling):
    """(out, bound): out in 64 bits and, per value, sum |c| |x| |A| |B| over the two
    sums' terms, which their rounding errors are measured against."""
    out, mag = y.astype(np.float64), np.zeros(y.shape)
    for l in np.unique(ids):
        if not 0 <= l < a.shape[0]:
            continue
        t = np.flatnonzero(ids == l)
        c = 1.0 if scaling is None else float(scaling[l])
        x64, a64, b64 = x[t].astype(np.float64), a[l].astype(np.float64), b[l].astype(np.float64)
        out[t] += c * (x64 @ a64.T) @ b64.T
        mag[t] = abs(c) * (np.abs(x64) @ np.abs(a64).T) @ np.abs(b64).T
    return out, mag


def lora_bound(out, mag, hidden, rank, bf16):
    """How far a value may be off: the output's rounding (half a step), and for the
    two fp32 sums at most one rounding of 2^-24 (half a step) per term of the longest
    chain, hidden + rank + 32 of them with the split parts' sums, the scaling and
    the final addition; v's terms leave 2^-17 (bf16 y) or 2^-25 of it."""
    half = 2.0 ** -8 if bf16 else 2.0 ** -24
    inner = (hidden + rank + 32) * 2.0 ** -24 + (2.0 ** -17 if bf16 else 2.0 ** -25)
    return half * np.abs(out) + (1 + half) * inner * mag + 32 * 2.0 ** -24 * np.abs(out)


def lora_exact_inputs(rng, t, h, n, r, adapters, bf16):
    """(x, a, b, c, v) of whole numbers and powers of two such that every product and every partial
    sum, in whatever order, is exact in fp32, and v = x A^T (the same for every adapter up to
    its signs) needs 24 bits: three bytes, each a value of x, at three places of K far from each other.
    fp32 output: a column is c v_r alone, with c B a power of two.  bf16 output (v of 16
    bits): a column is v_r - v_r', small, so that only v's first term would leave nothing or too much."""
    places = np.array([h // 9, h // 2, h - 1])
    x, a, b = np.zeros((t, h), np.float32), np.zeros((adapters, r, h), np.float32), np.zeros((adapters, n, r), np.float32)
    top = rng.integers(64, 128, t) if not bf16 else np.zeros(t, np.int64)
    x[:, places] = np.stack([top, rng.integers(128, 256, t), 2 * rng.integers(0, 128, t) + 1], 1)
    x *= rng.choice([-1.0, 1.0], (t, 1)).astype(np.float32)
    a[:, :, places] = [65536.0, 256.0, 1.0]
    c = (2.0 ** rng.integers(-3, 4, adapters)).astype(np.float32)
    col = np.arange(n)
    if bf16:
        # ranks differ by small multiples of x's last byte: v_r = 256 x1 + (1 + r % 2) x0
        a[:, 1::2, places[2]] = 2.0
        b[:, col, 2 * (col % (r // 2))] = -1.0
        b[:, col, 2 * (col % (r // 2)) + 1] = 1.0  # their difference: x0, at most 255
    else:
        a *= rng.choice([-1.0, 1.0], (adapters, r, 1)).astype(np.float32)
        b[:, col, col % r] = 2.0 ** rng.integers(-4, 5, (adapters, n))
    v = np.einsum("th,arh->atr", x.astype(np.float64), a.astype(np.float64))
    return x, a, b, c, v


def split_terms(v, terms):
    """v as a sum of `terms` bf16 values, each the rounding of what those before it leave."""
    left, out = np.asarray(v, np.float32).copy(), np.zeros(np.shape(v))
    for _ in range(terms):
        t = fp8.bf16_round(left)
        out, left = out + t, left - t
    return out
