"""How exact attention over caches in 8 bits is, element by element, whatever the caches' scales and whichever kernel reads them."""
import numpy as np
import pytest

import paged8_plain as plain8
import paged_plain as plain
from test_gpu_paged import close
from test_gpu_paged8 import run_attention8

pytestmark = pytest.mark.gpu
CACHES = ["i8", "e4m3"]
FEW = {"i8": 2.0 ** -33, "e4m3": 2.0 ** -37}  # `tiny` of few query rows


@pytest.fixture(scope="module")
def paged():
    from llamd_rs_b200 import backend, paged as p

    backend.stream_init()
    return p


def code_of(value, cache):
    return int(np.flatnonzero(plain8.TABLE[cache][:127] == value)[0])


def far_apart(cache, dtype, ahead):
    """An edit for run_attention8: every fourth block of V holds one element of the largest scale and zeros beside it, the others the least scale and a zero there; and
    the former's scores are `ahead` nats above the latter's (by each head's last element: 4 sqrt(hd) in q, ahead / 4 in K)."""
    _, low, high = plain8.FORMATS[cache]
    e = -5 if cache == "i8" else -7

    def edit(q, k, v, tables):
        q[..., -1] = plain.to_bits(np.float32(4 * q.shape[-1] ** 0.5), dtype)
        k[1][:] = 127 + e
        k[0][..., -1] = 0
        for table in tables:
            for i, page in enumerate(table):
                apart = i % 4 == 1
                v[1][page] = 127 + (high if apart else low)
                if apart:
                    v[0][page, :, :, 1:] = 0
                    k[0][page, :, :, -1] = code_of(ahead / 4 * 2.0 ** -e, cache)
                else:
                    v[0][page, :, :, 0] = 0
    return edit


def compare(paged, cache, H, K, D, dtype, q_len, kv_len, edit, tiny, n_shared=0, **more):
    """Outputs in f32 of pages of 16, against the definition: |got - want| <= (u + 2 d + n) A + tiny sum |v| + 2^-22 |want|,  A = sum p |v|:
      u     the weights' rounding to f16, half a step of 2^-10
      d     a score's error: hd products of 16-bit numbers summed in f32 in any order, 2^-24 hd scale sum |q k| at most (twice that is taken)
      n     both sums in f32: a 16th of a sequence's positions one behind the other, the joins of lanes, warps and pieces: (positions / 16 + 64) 2^-24 each
      tiny  half of f16's least step over the largest weight that is sure to be there: 2^-25 over 2^12 (few query rows) or 2^7 (many). Few rows of i8: weights have up
            to 2^4 of their scales in them, so the largest by itself may be 2^8
    The last term is the quotient's and the join's own arithmetic."""
    seen = {}

    def keep(q, k, v, tables):
        if edit:
            edit(q, k, v, tables)
        seen.update(q=q.copy(), k=[x.copy() for x in k], v=[x.copy() for x in v], tables=tables)

    got, want, _ = run_attention8(paged, cache, H, K, D, 16, dtype, q_len, kv_len, n_shared, out_f32=True, edit=keep, **more)
    q, scale = plain.from_bits(seen["q"], dtype), D ** -0.5
    bound, at = np.zeros_like(want), 0
    for t, n, m in zip(seen["tables"], q_len, kv_len):
        idx = np.arange(m)
        ids = np.asarray(t)[idx // 16] if m else np.zeros(0, int)
        kk, vv = (plain8.TABLE[cache][c[ids, :, idx % 16]] * 2.0 ** (e[ids, :, 0].astype(float) - 127)[..., None] for c, e in (seen["k"], seen["v"]))
        mask = idx <= np.arange(m - n, m)[:, None]
        for h in range(H if n else 0):
            g, row = h // (H // K), q[at:at + n, h]
            sc = np.where(mask, scale * (row @ kk[:, g].T), -np.inf)
            d = 2.0 ** -23 * D * scale * np.where(mask, np.abs(row) @ np.abs(kk[:, g]).T, 0).max(1, keepdims=True)
            p = np.exp(sc - sc.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            size = np.abs(vv[:, g])
            bound[at:at + n, h] = (2.0 ** -11 + 2 * d + 2 * (m / 16 + 64) * 2.0 ** -24) * (p @ size) + tiny * (mask @ size) + 2.0 ** -22 * np.abs(want[at:at + n, h]) + 2.0 ** -149
        at += n
    assert np.all(np.isfinite(got))
    worst = np.max(np.abs(got - want) / bound)
    assert worst <= 1.0, f"{worst:.3g} of the bound"


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,K,D,q_len,kv_len,n_shared", [(4, 2, 64, [1], [200], 0), (8, 1, 128, [1, 1, 2], [64, 177, 90], 0), (16, 1, 64, [1], [3000], 0), (8, 1, 128, [1], [20000], 0),
                                                         (8, 2, 128, [1, 1, 1], [70, 100, 300], 64)])
def test_scales_far_apart(paged, cache, dtype, H, K, D, q_len, kv_len, n_shared):
    """Few query rows; V's scales as far apart as an append makes them, in different elements: an element's error is in proportion to what that element is made of."""
    for ahead in (0.0, 5.0, 10.0):
        compare(paged, cache, H, K, D, dtype, q_len, kv_len, far_apart(cache, dtype, ahead), FEW[cache], n_shared)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,K,D,q_len,kv_len,n_shared", [(8, 1, 128, [70], [300], 0), (4, 2, 64, [257, 60], [257, 1000], 0), (32, 4, 128, [600], [600], 0), (8, 1, 64, [100], [9000], 0),
                                                         (32, 4, 128, [1] * 40, [1700 + i for i in range(40)], 1696)])
def test_many_rows(paged, cache, dtype, H, K, D, q_len, kv_len, n_shared):
    """The kernel of many query rows, of either type: weights and V in f16, as in that of few."""
    for edit in (None, far_apart(cache, dtype, 0.0), far_apart(cache, dtype, 5.0)):
        compare(paged, cache, H, K, D, dtype, q_len, kv_len, edit, max(2.0 ** -32, FEW[cache]), n_shared)


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("D", [64, 128])
def test_the_largest_queries(paged, cache, D):
    """bf16 rows of which each element is near the type's largest: finite scores, by a small scale, in both kernels."""
    def largest(q, k, v, tables):
        sign = np.random.default_rng(1).choice([-1.0, 1.0], q.shape)
        q[:] = plain.to_bits((sign * np.linspace(1.5e38, 3.3e38, q.size).reshape(q.shape)).astype(np.float32), "bf16")

    for q_len, kv_len in (([1, 2], [90, 40]), ([1], [2000]), ([60], [200])):
        close(*run_attention8(paged, cache, 8, 2, D, 16, "bf16", q_len, kv_len, edit=largest, scale=1.3e-38, low=-12, high=-8))
