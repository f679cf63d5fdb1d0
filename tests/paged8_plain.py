"""Caches in 8 bits in 64 bits: codes, scales, and the append's rules (numpy, from the definitions)."""
import numpy as np

BLOCK = 16
# the largest code, the least and the largest exponent of an append's scale
FORMATS = {"i8": (127.0, -24, 9), "e4m3": (448.0, -15, 7)}


def _e4m3():
    b = np.arange(256)
    e, m = (b >> 3) & 15, b & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))  # (NaN's two codes: 480 here, and in no test)
    return np.where(b & 128, -v, v)


TABLE = {"e4m3": _e4m3(), "i8": np.arange(256, dtype=np.uint8).view(np.int8).astype(np.float64)}


def values(codes, scales, cache):
    """codes uint8 [pages][heads][page][hd], scales uint8 [pages][heads][page / 16] -> f64."""
    return TABLE[cache][codes] * np.repeat(2.0 ** (scales.astype(np.float64) - 127), BLOCK, axis=2)[..., None]


def step(x, cache):
    """The distance of neighbouring codes about x (in units of the scale), never too small: half of it is how far a rounding goes."""
    x = np.minimum(np.abs(x), FORMATS[cache][0])
    return np.ones_like(x) if cache == "i8" else 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(x, 2.0 ** -9))), -6) - 3)


def rounded(x, cache):
    """f64 -> the codes' values, to nearest even, saturating."""
    most = FORMATS[cache][0]
    x = np.clip(x, -most, most)
    s = step(x, cache)
    return np.clip(np.rint(x / s) * s, -most, most)


def exponent(top, cache):
    """The least e with top <= most 2^e, inside the format's."""
    most, low, high = FORMATS[cache]
    with np.errstate(divide="ignore"):
        m, e = np.frexp(top / most)
    return np.clip(np.where(m == 0, low, np.where(m == 0.5, e - 1, e)), low, high)


def random_pool(rng, n_pages, K, page, D, cache, low=-6, high=0):
    """Codes of a normal distribution, and scales 2^low to 2^high about where values are of size 1."""
    x = rng.standard_normal((n_pages, K, page, D)) * (36.0 if cache == "i8" else 110.0)
    at = np.argsort(TABLE[cache][:127] if cache == "e4m3" else TABLE[cache][:128])  # (from 0 up)
    v = TABLE[cache][at]
    near = np.searchsorted((v[1:] + v[:-1]) / 2, np.abs(x))
    codes = at[near].astype(np.uint8)
    neg = x < 0
    codes[neg] = (codes[neg] | 128) if cache == "e4m3" else (-codes[neg].view(np.int8)).view(np.uint8)
    scales = rng.integers(127 + low + (-5 if cache == "i8" else -7) + 3, 127 + high + (-5 if cache == "i8" else -7) + 3, (n_pages, K, page // BLOCK), endpoint=True).astype(np.uint8)
    return codes, scales
