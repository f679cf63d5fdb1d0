"""Sampling against a softmax whose weights are not rounded: how near to a border a number has to be for another token to come out, and weights over the whole range of
temperatures and logits."""
import numpy as np
import pytest

import sample_plain as plain
from test_gpu_sample import logits, run, sampling  # noqa: F401  (sampling: the fixture)

pytestmark = pytest.mark.gpu


def near(sampling, x, u, **settings):
    """The token's own stretch of [0, 1), in 80 bits, is no further from u than what the weights' errors move its ends, and its share no further from the exact one. A
    weight is off by 2^-36.6 of itself (the series up to f^9, |f| <= 1/2: (ln 2 / 2)^10 / 10! 2^(1/2)) and by a rounding to multiples of 2^-40 of the first's, 2^-41. With n weights of W in all, in
    units of the first's, a sum of some of them and of all are off by e = 2^-36.6 W + n 2^-41 at most, together, so their quotient by e / (W - e)."""
    got, share = run(sampling, x, u, **settings)
    for r, row in enumerate(x):
        T = np.longdouble(np.float32(settings.get("temperature", 1.0)))
        order = np.argsort(-row.astype(np.float64), kind="stable")
        order = np.sort(order[:settings["top_k"]]) if settings.get("top_k", 0) > 0 else np.arange(len(row))
        w = np.exp((row[order].astype(np.longdouble) - np.longdouble(row.max())) / T)
        W, n = w.sum(), len(w)
        e = 2.0 ** -36.6 * W + n * 2.0 ** -41
        e = float(e / (W - e)) + n * 2.0 ** -63
        at = int(np.flatnonzero(order == got[r])[0])
        end = w[:at + 1].sum() / W
        begin = end - w[at] / W
        assert begin - e <= u[r] < end + e, (r, float(begin), float(end), u[r], e)
        assert abs(share[r] - w[at] / W) <= 2.0 ** -23 * w[at] / W + e
    return got


@pytest.mark.parametrize("n", [40, 5000, 151936])
def test_near_a_border(sampling, n):  # noqa: F811
    rng = np.random.default_rng(n)
    for spread in (0.01, 2.0, 8.0):
        x = logits(rng, 12, n, spread)
        for rule in (dict(), dict(temperature=0.3), dict(top_k=30, temperature=1.7), dict(top_k=n // 3)):
            near(sampling, x, rng.random(12).astype(np.float32), **rule)


def test_weights_below_a_unit(sampling):  # noqa: F811
    """One token far above all others, each of which weighs less than half of 2^-40 of it, or just more: all of them together are what rounding may lose, or add."""
    for n in (151936, 393216):
        for weight in (2.0 ** -41.2, 2.0 ** -40.8, 2.0 ** -39.5):
            x = np.full((3, n), np.log(weight), np.float32)
            x[:, 0] = 0.0
            near(sampling, x, np.array([0.5, 1 - 2.0 ** -23, 1 - 2.0 ** -24], np.float32))


def test_ends_of_the_range(sampling):  # noqa: F811
    """Logits further apart than f32 reaches, with a temperature as large; and temperatures among f32's smallest, with logits nearer than a normal number to one another."""
    u = np.array([0.0, 0.3, 0.9, 0.999, 1 - 2.0 ** -24], np.float32)
    for n in (3, 700, 40000):
        x = np.tile(np.linspace(3.3e38, -3.3e38, n).astype(np.float32), (5, 1))
        for T in (1e38, 3e38, 4e37):
            for rule in (dict(), dict(top_k=2), dict(top_k=n // 2 + 1)):
                near(sampling, x, u, temperature=T, **rule)
        x = (-1e-39 * np.arange(n)).astype(np.float32)
        for T in (1e-44, 1e-41, 3e-39, 1e-38):
            for rule in (dict(), dict(top_k=2), dict(top_k=n // 2 + 1)):
                near(sampling, np.tile(x, (5, 1)), u, temperature=T, **rule)
                assert plain.sample(x, 0.0, T)[0] == 0


# The largest logit, temperature, min_p and j: logits (j - 1) 2^-53 and j 2^-53 have weights that are min_p and the number of 64 bits just below, in this order: the smaller logit's is the larger (a last
# bit of the series). Found by trying some 10^10.
TURNED = [("0x1.4e471cp-1", "0x1.085846p+1", "0x1.753a18p-1", 50), ("0x1.92d2fep-1", "0x1.3319cp+1", "0x1.70da7ap-1", -54), ("0x1.3bd1b8p-1", "0x1.2973ep+1", "0x1.88a354p-1", -45),
          ("0x1.97fa18p-1", "0x1.2a6efap+1", "0x1.6bc89cp-1", 62), ("0x1.4d82d4p-1", "0x1.0de482p+1", "0x1.77ed56p-1", -4)]


@pytest.mark.parametrize("k,n,rows", [(3, 9, 4), (3, 20000, 4), (40, 5000, 300), (400, 5000, 300), (300, 40000, 64)])
def test_a_last_bit_at_min_p(sampling, k, n, rows):  # noqa: F811
    """Two logits at min_p whose weights are in the wrong order: two tokens are kept, the largest and one of these, and every number falls on one of them."""
    u = ((np.arange(rows) + 0.5) / rows).astype(np.float32)
    for top, T, m, j in TURNED:
        top, T, m = (np.float32(float.fromhex(v)) for v in (top, T, m))
        x = np.tile(np.linspace(-3, -5, n).astype(np.float32), (rows, 1))
        x[:, :3] = [(j - 1) * 2.0 ** -53, top, j * 2.0 ** -53]
        got, share = run(sampling, x, u, temperature=T, top_k=k, min_p=m)
        assert set(got.tolist()) <= {0, 1, 2} and {0, 2} - set(got.tolist())
        assert np.allclose(share, np.where(got == 1, 1 / (1 + m), m / (1 + m)), rtol=1e-6)
        near_top = np.sum(got == 1) / rows
        assert abs(near_top - 1 / (1 + m)) <= 1.001 / rows
        assert np.array_equal(got, run(sampling, x, u, temperature=T, top_k=k, min_p=m)[0])
