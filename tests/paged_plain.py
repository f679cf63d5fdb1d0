"""The paged operators in 64 bits, and how far 16-bit results may be from them (numpy, from the definitions)."""
import numpy as np

# half the spacing of a 16-bit type's values, relative; and its smallest normal's half spacing
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -133}


def to_bits(x, dtype):
    """f64 / f32 -> the 16-bit patterns, to nearest even."""
    x = np.asarray(x, dtype=np.float32)
    if dtype == "f16":
        return x.astype(np.float16).view(np.uint16)
    b = x.view(np.uint32)
    r = ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bits(b, dtype):
    b = np.asarray(b, dtype=np.uint16)
    if dtype == "f16":
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def norm_rope(x, pos, w, eps, table, rot, interleaved):
    """x [tokens][heads][hd] f64; table [rows][rot/2][2] sines and cosines."""
    x = np.asarray(x, dtype=np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    y = x.copy()
    half = rot // 2
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        s, c = table[pos, i, 0].astype(np.float64)[:, None], table[pos, i, 1].astype(np.float64)[:, None]
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., a] * s + x[..., b] * c
    return y


def positions(q_len, kv_len):
    seq = np.repeat(np.arange(len(q_len)), q_len)
    pos = np.concatenate([np.arange(m - n, m) for n, m in zip(q_len, kv_len)] + [np.zeros(0, int)]).astype(int)
    return seq, pos


def attention(q, k_pages, v_pages, tables, q_len, kv_len, scale, dtype):
    """-> (out f64 [tokens][heads][hd], bound of the same shape). q [tokens][n_head][hd], pages [n][n_head_kv][page][hd], f64.

    The bound, for an output rounded to u relative from weights rounded to u relative:
      u |out|                      the output's rounding
      (u + 2 d + 2^-20) A          the weights' rounding and the scores' error d, A = sum p |v| / sum p
      tiny (1 + sum |v|)           weights and outputs below the type's normal range
    d: a score is a sum of hd <= 128 products in f32 in any order, 2^-24 hd scale sum |q k| at most (twice that is taken)."""
    n_head, n_kv = q.shape[1], k_pages.shape[1]
    page, group, u, tiny = k_pages.shape[2], n_head // n_kv, U[dtype], TINY[dtype]
    out, bound, at = np.zeros_like(q), np.zeros_like(q), 0
    for s, (n, m) in enumerate(zip(q_len, kv_len)):
        idx = np.arange(m)
        ids = np.asarray(tables[s])[idx // page] if m else np.zeros(0, int)
        k, v = k_pages[ids, :, idx % page], v_pages[ids, :, idx % page]
        seen = np.arange(m) <= np.arange(m - n, m)[:, None]
        for h in range(n_head if n else 0):
            kk, vv, row = k[:, h // group], v[:, h // group], q[at:at + n, h]
            sc = np.where(seen, scale * (row @ kk.T), -np.inf)
            d = 2.0 ** -23 * kk.shape[1] * abs(scale) * np.where(seen, np.abs(row) @ np.abs(kk).T, 0).max(1, keepdims=True)
            p = np.exp(sc - sc.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            o = p @ vv
            out[at:at + n, h] = o
            bound[at:at + n, h] = u * np.abs(o) + (u + 2 * d + 2.0 ** -20) * (p @ np.abs(vv)) + tiny * (1 + seen @ np.abs(vv))
        at += n
    return out, bound
