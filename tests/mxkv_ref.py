"""64-bit definitions of the MX KV cache, its attention and draft verification, in numpy (CPU)."""
import numpy as np

E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def e4m3_values():
    v = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v[c] = np.ldexp(m, -9) if e == 0 else np.ldexp(8 + m, e - 10)
        if c & 127 == 127:
            v[c] = np.nan
        if c & 128:
            v[c] = -v[c]
    return v


E4M3 = e4m3_values()


def position(d, hd):
    """Code position of dimension d in a row."""
    return (d % 32 // 4 * (hd // 32) + d // 32) * 4 + d % 4


def nearest_e4m3(y):
    """Nearest E4M3 code (ties to the even code, saturating at 448), NaN -> 0x7F."""
    mags = E4M3[:127]
    a = np.minimum(np.abs(y), 448.0)
    hi = np.clip(np.searchsorted(mags, a), 1, 126)
    lo = hi - 1
    dl, dh = a - mags[lo], mags[hi] - a
    code = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    code = code | np.where(np.signbit(y), 128, 0)
    return np.where(np.isnan(y), 0x7F, code).astype(np.uint8)


def nearest_e2m1(y):
    """Nearest E2M1 code, ties to the smaller magnitude; negative values keep their sign at 0."""
    a = np.abs(y)
    d = np.abs(np.minimum(a, 100.0)[..., None] - E2M1)
    return (np.argmin(np.where(np.isnan(d), 1e300, d), -1) | np.where(y < 0, 8, 0)).astype(np.uint8)


def encode(x, fmt):
    """x [..., hd] -> (codes [..., row bytes], scales [..., hd/32]) uint8."""
    x = np.asarray(x, np.float64)
    hd = x.shape[-1]
    blocks = x.reshape(x.shape[:-1] + (hd // 32, 32))
    amax = np.max(np.where(np.isnan(blocks), 0.0, np.abs(blocks)), -1)
    amax = np.minimum(amax, np.finfo(np.float32).max)
    top = 8 if fmt == "mxfp8" else 2
    e = np.where(amax > 0, np.clip(np.frexp(amax)[1] - 1 - top + 127, 0, 254), 127).astype(np.int64)
    y = blocks * np.exp2(127.0 - e)[..., None]
    if fmt == "mxfp8":
        code = nearest_e4m3(y)
    else:
        code = nearest_e2m1(y)
        e = np.where(np.isnan(blocks).any(-1), 255, e)
    code = code.reshape(x.shape)
    row = np.zeros_like(code)
    row[..., position(np.arange(hd), hd)] = code
    if fmt == "mxfp4":
        row = row[..., 0::2] | (row[..., 1::2] << 4)
    return row.astype(np.uint8), e.astype(np.uint8)


def decode(row, scales, fmt):
    """Inverse of encode: f64 values [..., hd]."""
    hd = 32 * scales.shape[-1]
    if fmt == "mxfp4":
        code = np.stack((row & 15, row >> 4), -1).reshape(row.shape[:-1] + (hd,))
        v = np.where(code & 8, -1.0, 1.0) * E2M1[code & 7]
    else:
        v = E4M3[row]
    d = np.arange(hd)
    v = v[..., position(d, hd)]
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return v * np.repeat(s, 32, -1)


def attention(q, k, v, limits):
    """q [t][H][hd], k, v [n][KV][hd] f64, limits [t] visible positions -> (out, sum p |v|, sum |q k| / sqrt(hd) max)."""
    t, H, hd = q.shape
    group = H // k.shape[1]
    out, mass, size = np.zeros_like(q), np.zeros_like(q), np.zeros((t, H, 1))
    for i in range(t):
        n = limits[i]
        if n <= 0:
            continue
        for h in range(H):
            kk, vv = k[:n, h // group], v[:n, h // group]
            s = kk @ q[i, h] / np.sqrt(hd)
            size[i, h] = (np.abs(kk) @ np.abs(q[i, h])).max() / np.sqrt(hd)
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h], mass[i, h] = p @ vv, p @ np.abs(vv)
    return out, mass, size


def verify(logits, drafts, u, noise, probs=None, lens=None, temp=None):
    """Speculative verification in 64 bits: accepted, tokens, logprobs."""
    logits = np.asarray(logits, np.float64)
    B, K1, V = logits.shape
    acc, toks, lps = np.zeros(B, np.int32), np.full((B, K1), -1, np.int32), np.zeros((B, K1))
    for b in range(B):
        T = 1.0 if temp is None else float(temp[b])
        greedy = not T > 1e-30
        n = K1 - 1 if lens is None else min(max(int(lens[b]), 0), K1 - 1)
        for i in range(K1):
            x = np.where(np.isnan(logits[b, i]), -np.inf, np.minimum(logits[b, i], np.finfo(np.float32).max))
            best, m = int(np.argmax(x)), x.max()
            with np.errstate(invalid="ignore", over="ignore"):
                y = np.where(x == -np.inf, -np.inf, (x - m) / (1.0 if greedy else T))
            p = np.exp(y)
            total = p.sum()
            p = p / total if total > 0 else p
            with np.errstate(divide="ignore"):
                lp = y - np.log(total) if total > 0 else y
            if i < n:
                d = int(drafts[b, i])
                inside = 0 <= d < V
                q = np.zeros(V)
                if probs is not None:
                    q = np.asarray(probs[b, i], np.float64)
                elif inside:
                    q[d] = 1.0
                if inside and (d == best if greedy else float(u[b, i]) * q[d] < p[d]):
                    toks[b, i], lps[b, i] = d, lp[d]
                    continue
            if greedy:
                tok = best
            else:
                w = np.maximum(p - q, 0) if i < n else p
                w = w if w.max() > 0 else p
                tok = int(np.argmax(w / noise[b])) if w.max() > 0 else best
            toks[b, i], lps[b, i], acc[b] = tok, lp[tok], i
            break
    return acc, toks, lps
