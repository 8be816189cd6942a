"""The KV cache's operators in 64 bits, on the CPU, from their definitions (numpy; test infrastructure)."""
import numpy as np
import torch

BF16, FP16, E4M3, E5M2, E2M1 = range(5)
TORCH = {BF16: torch.bfloat16, FP16: torch.float16}
LARGEST = {E4M3: 448.0, E5M2: 57344.0, E2M1: 6.0}
BITS = {BF16: 16, FP16: 16, E4M3: 8, E5M2: 8, E2M1: 4}


def code_values(fmt):
    """Value of every code of an 8- or 4-bit format, in 64 bits."""
    if fmt == E2M1:
        half = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
        return np.array(half + [-x for x in half])
    mant, bias = (3, 7) if fmt == E4M3 else (2, 15)
    out = np.zeros(256)
    for c in range(256):
        e, m = (c & 127) >> mant, c & ((1 << mant) - 1)
        if fmt == E4M3 and (c & 127) == 127:
            v = np.nan
        elif fmt == E5M2 and e == 31:
            v = np.inf if m == 0 else np.nan
        else:
            v = np.ldexp(m + (1 << mant if e else 0), max(e, 1) - bias - mant)
        out[c] = -v if c & 128 else v
    return out


def nearest_code(a, fmt):
    """Code of magnitudes a (finite, at most the largest value), to nearest, ties to the even code."""
    last = int(np.flatnonzero(code_values(fmt)[:128 if fmt != E2M1 else 8] == LARGEST[fmt])[0])
    grid = code_values(fmt)[:last + 1]
    hi = np.minimum(np.searchsorted(grid, a), last)
    lo = np.maximum(hi - 1, 0)
    down, up = a - grid[lo], grid[hi] - a
    return np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)


def quantise(x, fmt, group):
    """(codes uint8 [..., dim] one per element, scale bytes [..., dim / group]) of float64 rows."""
    y = x.reshape(*x.shape[:-1], -1, group)
    fin = np.where(np.isfinite(y), np.abs(y), 0.0)
    top = fin.max(-1, keepdims=True)
    m, e = np.frexp(np.where(top == 0, 1.0, top) / LARGEST[fmt])  # m in [0.5, 1): exact powers have m = 0.5
    e = np.where(m == 0.5, e - 1, e)
    # (the quotient is rounded: settle the exponent by exact comparisons)
    e = np.where(top > np.ldexp(LARGEST[fmt], e), e + 1, e)
    e = np.where(top <= np.ldexp(LARGEST[fmt], e - 1), e - 1, e)
    e = np.where(top == 0, 0, np.maximum(e, -126))
    z = np.ldexp(y, -e)
    z = np.where(np.isinf(z), np.copysign(LARGEST[fmt], z), z)
    nan = np.isnan(z)
    mag = np.abs(np.where(nan, 0.0, z))
    sign = np.signbit(z)
    code = nearest_code(mag, fmt) | np.where(sign, 8 if fmt == E2M1 else 128, 0)
    scale = (e + 127)[..., 0]
    if fmt == E2M1:
        code = np.where(nan, 0, code)
        scale = np.where(nan.any(-1), 255, scale)
    else:
        code = np.where(nan, 127, code)  # some NaN: compared by value
    return code.reshape(x.shape).astype(np.uint8), scale.astype(np.uint8)


def dequantise(code, scale, fmt, group):
    v = code_values(fmt)[code].reshape(*code.shape[:-1], -1, group)
    s = np.where(scale == 255, np.nan, np.ldexp(1.0, scale.astype(np.int64) - 127))
    return (v * s[..., None]).reshape(code.shape)


def unpack(pool, fmt):
    """Codes, one per element, of a pool tensor (uint8 / float8)."""
    b = pool.cpu().view(torch.uint8).numpy()
    if fmt != E2M1:
        return b
    return np.stack([b & 15, b >> 4], -1).reshape(*b.shape[:-1], -1)


def pool_values(pool, scale, fmt):
    """[pages, page_size, heads, dim] in 64 bits."""
    if fmt in TORCH:
        return pool.cpu().double().numpy()
    code = unpack(pool, fmt)
    group = code.shape[-1] // scale.shape[2]
    return dequantise(code, scale.cpu().numpy().transpose(0, 3, 1, 2), fmt, group)


def attend(q, k, v, table, kv_len, cu, mask, scale):
    """q [rows, q_heads, dim] float64, k / v [pages, page_size, heads, dim] float64.  Returns
    (out, lse, weight) with weight = sum p |v| / sum p, what errors of p are measured by."""
    rows, hq, d = q.shape
    page, heads = k.shape[1], k.shape[2]
    per = hq // heads
    out, lse, wt = np.zeros((rows, hq, d)), np.full((rows, hq), -np.inf), np.zeros((rows, hq, d))
    for b in range(len(kv_len)):
        n, past = int(cu[b + 1] - cu[b]), int(kv_len[b] - (cu[b + 1] - cu[b]))
        pos = np.arange(int(kv_len[b]))
        kk, vv = k[table[b][pos // page], pos % page], v[table[b][pos // page], pos % page]
        for i in range(n):
            r = cu[b] + i
            seen = pos < past
            if mask is None:
                seen = pos <= past + i
            else:
                j = np.arange(n)
                seen[past:] = (mask[r].view(np.uint32)[j // 32] >> (j % 32).astype(np.uint32)) & 1
            if not seen.any():
                continue
            for h in range(hq):
                with np.errstate(all="ignore"):
                    s = scale * (kk[seen, h // per] @ q[r, h])
                    top = s.max()
                    p = np.exp(s - top)
                    out[r, h] = (p @ vv[seen, h // per]) / p.sum()
                    wt[r, h] = (p @ np.abs(vv[seen, h // per])) / p.sum()
                    lse[r, h] = top + np.log(p.sum())
    return out, lse, wt


def tolerance(out, weight, q, kmax, n_keys, scale, dtype):
    """Bound on |attended - out|.  u: half a step of the type.  Per weight p: its rounding u (in the
    numerator and in the divisor), its exponent's error: a product of dim terms in 32 bits, off by
    (dim + 8) 2^-24 of the sum of magnitudes, which enters p as its absolute error, and 2^-20 for
    the exponential; sums of n_keys terms in 32 bits, twice; fp16 drops weights below 2^-31 of the
    largest.  Then the output's own rounding."""
    u = torch.finfo(dtype).eps / 2
    d = q.shape[-1]
    mags = scale * np.abs(q).sum(-1, keepdims=True) * kmax
    rel = 2 * u + 2 * ((d + 8) * 2.0 ** -24 * mags * 1.5 + 2.0 ** -20) + 2 * n_keys * 2.0 ** -24 + n_keys * 2.0 ** -31
    return u * np.abs(out) + 1.01 * rel * weight + 2.0 ** -24
