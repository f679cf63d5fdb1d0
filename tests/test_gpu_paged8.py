"""Paged K/V caches in 8 bits on the GPU: append and attention against the definitions in 64 bits (paged_plain.py, paged8_plain.py)."""
import numpy as np
import pytest

import paged8_plain as plain8
import paged_plain as plain
from test_gpu_paged import APPEND, ATTENTION, close, dev, lib, scatter_tables

pytestmark = pytest.mark.gpu
CACHES = ["i8", "e4m3"]


@pytest.fixture(scope="module")
def paged():
    from llamd_rs_b200 import backend, paged as p

    backend.stream_init()
    return p


def run_append(paged, H, K, D, page, dtype, inputs, q_len, kv_len, rot, interleaved, norm, pad, cache, grow=1.0, edit=None, repeat=1):
    """-> everything that append8 has read and written, on the host."""
    from llamd_rs_b200 import backend

    rng = np.random.default_rng(H * 1000 + D + rot + len(q_len) + int(8 * grow))
    tables, n_pages = scatter_tables(rng, kv_len, page)
    b = paged.Batch(H, K, D, page, dtype, cache=cache)
    b.set(q_len, kv_len, tables, n_pages)
    T, eps = b.tokens, 1e-6
    rows = [rng.standard_normal((T, n * D + pad)).astype(np.float32) * (1.0 if n == H else grow) for n in (H, K, K)]
    if edit:
        edit(rows)
    if inputs == "f32":
        bufs, vals = [dev(r) for r in rows], [r.astype(np.float64) for r in rows]
    else:
        bits = [plain.to_bits(r, dtype) for r in rows]
        bufs, vals = [dev(x) for x in bits], [plain.from_bits(x, dtype) for x in bits]
    vals = [v[:, :n * D].reshape(T, n, D) for v, n in zip(vals, (H, K, K))]
    table = paged.rope_table(max(kv_len), rot, 1e6) if rot else np.zeros((1, 0, 2), np.float32)
    wq, wk = ((1 + 0.3 * rng.standard_normal(D)).astype(np.float32) for _ in range(2)) if norm else (None, None)
    before = [plain8.random_pool(rng, n_pages, K, page, D, cache) for _ in range(2)]
    pools = [[dev(x) for x in p] for p in before]
    out = dev(np.zeros((T, H, D), np.uint16))
    for _ in range(repeat):
        b.append(*bufs, out, pools[0][0], pools[1][0], rope=dev(table) if rot else None, rot=rot, interleaved=interleaved, q_norm=dev(wq) if norm else None,
                 k_norm=dev(wk) if norm else None, eps=eps, inputs=inputs, strides=[n * D + pad for n in (H, K, K)], k_scales=pools[0][1], v_scales=pools[1][1])
    backend.sync()
    seq, pos = plain.positions(q_len, kv_len)
    want = [plain.norm_rope(vals[0], pos, wq, eps, table, rot, interleaved), plain.norm_rope(vals[1], pos, wk, eps, table, rot, interleaved), vals[2]]
    got_q = plain.from_bits(out.download(np.uint16, T * H * D), dtype).reshape(T, H, D)
    after = [[buf.download(np.uint8, a.size).reshape(a.shape) for buf, a in zip(p, x)] for p, x in zip(pools, before)]
    ids = np.array([tables[s][p // page] for s, p in zip(seq, pos)], int)
    return want, got_q, before, after, seq, pos, ids


def check_pool(want, before, after, seq, pos, ids, q_len, kv_len, page, tables_of, cache, D, f32=None):
    """want [T][K][D] f64: the scales that the rules give, the older codes exactly, the new ones within a rounding, all else as it was."""
    codes, scales = before[0].copy(), before[1].astype(int) - 127
    got, got_e = after[0], after[1].astype(int) - 127
    most, low, high = plain8.FORMATS[cache]
    slot = pos % page
    block = ids * (page // 16) + slot // 16
    noise = 2.0 ** -24 * (D / 2 + 8) * 2 * np.abs(want).max(-1) if f32 is None else np.zeros(want.shape[:2])  # of f32 arithmetic: test_append's
    for x in np.unique(block):
        rows = np.nonzero(block == x)[0]
        page_id, at = x // (page // 16), x % (page // 16)
        held = int(pos[rows[0]] % 16)
        for h in range(want.shape[1]):
            top, off = np.abs(want[rows, h]).max(), noise[rows, h].max()
            own = scales[page_id, h, at] if held else -1000
            e = got_e[page_id, h, at]
            # (where the largest value is that near to a power's border, either)
            assert e in {max(int(plain8.exponent(top + d, cache)), own) for d in (-off, 0.0, off)}
            part = codes[page_id, h, at * 16:at * 16 + held]
            if held:
                now = got[page_id, h, at * 16:at * 16 + held]
                if e == own:
                    assert np.array_equal(now, part)
                else:
                    assert np.array_equal(plain8.TABLE[cache][now], plain8.rounded(plain8.TABLE[cache][part] * 2.0 ** (own - e), cache))
            y = want[rows, h] * 2.0 ** -float(e)
            new = plain8.TABLE[cache][got[page_id, h, slot[rows]]]
            near = np.clip(y, -most, most)
            assert np.all(np.abs(new - near) <= plain8.step(np.abs(near) + noise[rows, h][:, None] * 2.0 ** -float(e), cache) / 2 + noise[rows, h][:, None] * 2.0 ** -float(e))
            codes[page_id, h, at * 16:at * 16 + held] = got[page_id, h, at * 16:at * 16 + held]
            codes[page_id, h, slot[rows]] = got[page_id, h, slot[rows]]
            scales[page_id, h, at] = e
    assert np.array_equal(codes, got) and np.array_equal(scales, got_e)


MORE = [
    # blocks that begin and end anywhere, and pages of one
    (8, 2, 128, 16, "f16", "f32", [5, 16, 17, 31, 33, 2], [5, 32, 17, 40, 70, 16], 128, False, True, 0),
    (14, 2, 64, 32, "bf16", "bf16", [1, 15, 1, 14], [17, 32, 16, 31], 64, True, True, 0),
    (5, 5, 64, 128, "f16", "f16", [300, 1], [301, 129], 32, False, True, 6),
    (32, 4, 128, 64, "bf16", "f32", [1] * 40, [24 + 6 * i for i in range(40)], 128, False, True, 0),
]


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("grow", [0.01, 1.0, 40.0])
@pytest.mark.parametrize("H,K,D,page,dtype,inputs,q_len,kv_len,rot,interleaved,norm,pad", APPEND + MORE)
def test_append(paged, H, K, D, page, dtype, inputs, q_len, kv_len, rot, interleaved, norm, pad, grow, cache):
    """New rows a hundredth to forty times as large as the older ones: scales that stay and that grow."""
    args = (paged, H, K, D, page, dtype, inputs, q_len, kv_len, rot, interleaved, norm, pad, cache, grow)
    want, got_q, before, after, seq, pos, ids = run_append(*args)
    size = np.abs(want[0]).max(-1, keepdims=True)
    assert np.all(np.abs(got_q - want[0]) <= plain.U[dtype] * np.abs(want[0]) + 2.0 ** -24 * (D / 2 + 8) * 2 * size + plain.TINY[dtype])
    check_pool(want[1], before[0], after[0], seq, pos, ids, q_len, kv_len, page, None, cache, D)
    check_pool(want[2], before[1], after[1], seq, pos, ids, q_len, kv_len, page, None, cache, D, f32=0)
    again = run_append(*args, repeat=2)[3]  # the same rows once more: nothing changes
    assert all(np.array_equal(x, y) for p, o in zip(after, again) for x, y in zip(p, o))


@pytest.mark.parametrize("cache", CACHES)
def test_append_of_extremes(paged, cache):
    """Nothing but zeros, values below the least and above the largest scale, infinities and NaN."""
    def edit(rows):
        v = rows[2].reshape(-1, 2, 64)
        v[0:16] = 0.0
        v[16:32, 0] *= 1e-12
        v[16:32, 1] *= 1e12
        v[32, 0, 5], v[33, 1, 7], v[34, 0, 9] = np.inf, -np.inf, np.nan

    most, low, high = plain8.FORMATS[cache]
    want, _, before, after, seq, pos, ids = run_append(paged, 4, 2, 64, 16, "f16", "f32", [48], [48], 0, False, False, 0, cache, edit=edit)
    e = after[1][1].astype(int)[ids[::16], :, 0] - 127  # [3 blocks][2 heads]
    assert np.all(e[0] == low) and e[1, 0] == low and e[1, 1] == high and np.all(e[2] == high)
    got = plain8.values(*after[1], cache)[ids, :, pos % 16]
    assert np.all(got[:16] == 0) and np.all(np.abs(got[16:32, 1]) == most * 2.0 ** high)
    assert got[32, 0, 5] == most * 2.0 ** high and got[33, 1, 7] == -most * 2.0 ** high
    assert after[1][0][ids[34], 0, 34 % 16, 9] in ([0] if cache == "i8" else [0x7F, 0xFF])


def run_attention8(paged, cache, H, K, D, page, dtype, q_len, kv_len, n_shared=0, scale=None, out_f32=False, q_scale=1.0, seed=0, edit=None, repeat=1, low=-6, high=0,
                   pad=0, shift=0):
    from llamd_rs_b200 import backend

    rng = np.random.default_rng(seed + H * 100 + D + sum(kv_len))
    tables, n_pages = scatter_tables(rng, kv_len, page, n_shared)
    b = paged.Batch(H, K, D, page, dtype, cache=cache)
    b.set(q_len, kv_len, tables, n_pages, n_shared)
    T = b.tokens
    q = plain.to_bits(q_scale * rng.standard_normal((T, H, D)), dtype)
    k, v = (plain8.random_pool(rng, n_pages, K, page, D, cache, low, high) for _ in range(2))
    if edit:
        edit(q, k, v, tables)
    # whatever no sequence holds: the largest codes and NaN's, scales of every kind
    live = np.zeros((n_pages, page), bool)
    for t, m in zip(tables, kv_len):
        idx = np.arange(m)
        live[t[idx // page], idx % page] = True
    dead = np.broadcast_to(~live[:, None, :, None], k[0].shape)
    empty = np.broadcast_to(~live.reshape(n_pages, 1, page // 16, 16).any(-1), k[1].shape)
    for codes, scales in (k, v):
        codes[dead] = rng.choice([0x7F, 0x80, 0xFF, 0x7E], int(dead.sum()))
        scales[empty] = rng.choice([0, 254, 255], int(empty.sum()))
    wide, n = np.uint32 if out_f32 else np.uint16, H * D + pad
    rows = np.full((T, n), 0x7FFF, np.uint16)
    rows[:, :H * D] = q.reshape(T, H * D)
    rows = dev(np.concatenate([np.full(shift, 0x7FFF, np.uint16), rows.ravel()]))
    out = dev(np.full(shift + T * n, np.iinfo(wide).max, wide))
    pools = [dev(x) for x in (*k, *v)]
    for _ in range(repeat):
        if pad or shift:
            assert lib().llamd_fwd_paged_attention8(b.ptr, rows.ptr + 2 * shift, n, pools[0].ptr, pools[2].ptr, pools[1].ptr, pools[3].ptr,
                                                    out.ptr + wide().itemsize * shift, n, int(out_f32), D ** -0.5 if scale is None else scale) == 0
        else:
            b.attention(rows, pools[0], pools[2], out, scale=scale, out_f32=out_f32, k_scales=pools[1], v_scales=pools[3])
    backend.sync()
    assert paged.status() == 0
    got = out.download(wide, shift + T * n)
    assert np.all(got[:shift] == np.iinfo(wide).max)
    got = got[shift:].reshape(T, n)
    assert np.all(got[:, H * D:] == np.iinfo(wide).max)
    got = np.ascontiguousarray(got[:, :H * D])
    got = (got.view(np.float32).astype(np.float64) if out_f32 else plain.from_bits(got, dtype)).reshape(T, H, D)
    kv = []
    for codes, scales in (k, v):
        codes, scales = codes.copy(), scales.copy()
        codes[dead], scales[empty] = 0, 127
        kv.append(plain8.values(codes, scales, cache))
    # The bound of 16 bits, whose values these are exactly; and one term more, of either type. The kernel of few rows keeps weights w = 2^12 2^(x + l - m) in f16, x a score
    # times log2 e, 2^l its V scale and m no more than the largest x + l, M. One that ends in f16's subnormals is off by half their step, 2^-25: the numerator by
    # 2^-37 2^M sum |c|, c the codes. The denominator sum 2^x is 2^(M - l') at least, l' the largest's own l: an output by no more than 2^-37 2^l' sum |c|.
    want, bound = plain.attention(plain.from_bits(q, dtype), *kv, tables, q_len, kv_len, D ** -0.5 if scale is None else scale, dtype)
    at = 0
    for t, n, m in zip(tables, q_len, kv_len):
        idx = np.arange(m)
        codes = np.abs(plain8.TABLE[cache][v[0][t[idx // page], :, idx % page]]).sum(0)                      # [K][D]
        most = 2.0 ** (v[1][t[idx // page], :, idx % page // 16].astype(float) - 127).max(0, initial=0.0)    # [K]
        bound[at:at + n] += np.repeat(2.0 ** -37 * most[:, None] * codes, H // K, axis=0)
        at += n
    return got, want, bound


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("H,K,D,page,dtype,q_len,kv_len,n_shared", ATTENTION)
def test_attention(paged, cache, H, K, D, page, dtype, q_len, kv_len, n_shared):
    close(*run_attention8(paged, cache, H, K, D, page, dtype, q_len, kv_len, n_shared))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("q_len,kv_len", [([1], [300]), ([70], [300])])
def test_attention_sharp_and_flat(paged, cache, dtype, q_len, kv_len):
    """Keys that grow along the sequence, block by block; scores far apart and all alike; another scale; f32 out; scales 2^14 apart."""
    def ramp(q, k, v, tables):
        for i in range(-(-kv_len[0] // 16)):
            k[1][tables[0][i], :, 0] = 127 - 12 + i // 2

    args = (paged, cache, 8, 1, 128, 16, dtype, q_len, kv_len)
    close(*run_attention8(*args, q_scale=2.0, edit=ramp))
    close(*run_attention8(*args, q_scale=6.0))
    close(*run_attention8(*args, q_scale=0.0))
    close(*run_attention8(*args, scale=0.5))
    close(*run_attention8(*args, out_f32=True))
    close(*run_attention8(*args, q_scale=0.1, low=-7, high=7))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("size", [1e-30, 1e-6, 3e4, 1e30])
def test_queries_of_any_size(paged, cache, size):
    """bf16 rows far beyond f16's range, with a scale that brings the scores back."""
    for q_len, kv_len in (([1, 2], [90, 40]), ([60], [200])):
        close(*run_attention8(paged, cache, 8, 2, 64, 16, "bf16", q_len, kv_len, q_scale=size, scale=0.125 / size))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("n", [9, 41, 90])
@pytest.mark.parametrize("D,dtype", [(128, "bf16"), (64, "f16")])
def test_attention_joins(paged, cache, n, D, dtype):
    close(*run_attention8(paged, cache, 32, 4, D, 16, dtype, [1] * n, [401 + 5 * i for i in range(n)], 400))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("H,K,D,page,dtype,q_len,kv_len,n_shared", [c for c in ATTENTION if max(c[5]) > 3 and not c[7]])
def test_attention_beside_a_long_prompt(paged, cache, H, K, D, page, dtype, q_len, kv_len, n_shared):
    """Prompts that would be too little work for the tensor cores by themselves, in one batch with another that is not."""
    long = 300 + 2400 // (H // K)
    close(*run_attention8(paged, cache, H, K, D, page, dtype, q_len + [long], kv_len + [long], n_shared))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("H,D,dtype", [(8, 128, "f16"), (5, 64, "bf16"), (1, 128, "bf16"), (2, 64, "f16")])
def test_attention_many_pieces(paged, cache, H, D, dtype):
    """Several pieces to every CTA, of one tile and of two, of one block and of several, tails of every length, and short sequences between them."""
    rng = np.random.default_rng(H)
    q_len, kv_len = [], []
    for _ in range(260):
        n = int(rng.choice([0, 1, 3, rng.integers(13, 17), rng.integers(17, 60), rng.integers(100, 140)], p=[.05, .1, .1, .3, .35, .1])) * (8 if H == 1 else 1)
        q_len.append(n)
        kv_len.append(n + int(rng.choice([0, 0, rng.integers(0, 40), rng.integers(0, 400)])))
    close(*run_attention8(paged, cache, H, 1, D, 16, dtype, q_len, kv_len, repeat=2))
    close(*run_attention8(paged, cache, H, 1, D, 32, dtype, q_len, [m + 256 for m in kv_len], 256, repeat=2))


@pytest.mark.parametrize("cache", CACHES)
def test_attention_beside(paged, cache):
    """A batch large enough that the prefix and the sequences' own positions are read at the same time; three times."""
    rng = np.random.default_rng(3)
    own = [int(x) for x in rng.integers(900, 1100, 64)]
    close(*run_attention8(paged, cache, 32, 4, 128, 64, "bf16", [1] * 64, [7552 + m for m in own], 7552, repeat=3))


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("prompt", [True, False])
def test_every_code_and_scale(paged, cache, dtype, D, prompt):
    """V holds all codes but e4m3's NaN (-128 is none of i8's: with the largest scale it is beyond f16) with all of an append's scales, and each query's weight is 1 at one
    position and below 2^-700 at all others: out is that value. One prompt for the tensor cores' kernel, as many sequences of one token for the other.

    The weight itself is 2^d, |d| <= 2^-12 (a score of 2560 log2 e has a rounding of half a step of 2^-12), and is rounded by u for the product, not for the
    sum that the product is divided by: u and 2^-22 of the quotient's own arithmetic. Neighbouring codes are 2^-7 apart at least."""
    from llamd_rs_b200 import backend

    _, low, high = plain8.FORMATS[cache]
    n_blocks = high - low + 1
    n = 16 * n_blocks
    codes = np.tile(np.arange(256, dtype=np.uint8), n * D // 256 + 1)[:n * D].reshape(n_blocks, 1, 16, D)
    codes[codes == 0x80] = 0x81
    if cache == "e4m3":
        codes[codes & 0x7F == 0x7F] = 0x7E
    scales = np.arange(127 + low, 128 + high, dtype=np.uint8).reshape(n_blocks, 1, 1)
    # position i's key is its number in base 2, 16 and -16 by bit: a token scores 2560 at its own, 2048 at most at those before it
    kv = np.zeros((n, D))
    kv[:, :10] = np.where((np.arange(n)[:, None] >> np.arange(10)) & 1, 16.0, -16.0)
    k_codes = np.searchsorted(plain8.TABLE[cache][:127], np.abs(kv)).astype(np.uint8)
    k_codes = np.where(kv < 0, (k_codes | 128) if cache == "e4m3" else (-k_codes.view(np.int8)).view(np.uint8), k_codes).astype(np.uint8)
    assert np.array_equal(plain8.TABLE[cache][k_codes], kv)
    b = paged.Batch(1, 1, D, 16, dtype, cache=cache)
    table = list(range(n_blocks))
    if prompt:
        b.set([n], [n], [table], n_blocks)
    else:
        b.set([1] * n, np.arange(1, n + 1), [table] * n, n_blocks)
    q, out = dev(plain.to_bits(kv.reshape(n, 1, D), dtype)), dev(np.zeros((n, 1, D), np.uint32))
    b.attention(q, dev(k_codes.reshape(n_blocks, 1, 16, D)), dev(codes), out, scale=1.0, out_f32=True, k_scales=dev(np.full((n_blocks, 1, 1), 127, np.uint8)), v_scales=dev(scales))
    backend.sync()
    got = out.download(np.uint32, n * D).view(np.float32).astype(np.float64).reshape(n, D)
    want = plain8.values(codes, scales, cache).reshape(n, D)
    assert np.all(np.abs(got - want) <= (plain.U[dtype if prompt else "f16"] + 2.0 ** -22) * np.abs(want))


@pytest.mark.parametrize("cache", CACHES)
def test_attention_long(paged, cache):
    """More than 32 slices to a warp, pages that end inside a piece, a group of its own size."""
    close(*run_attention8(paged, cache, 6, 2, 64, 32, "f16", [1, 1], [9001, 4000]))
    close(*run_attention8(paged, cache, 32, 4, 128, 128, "bf16", [1], [20011]))


@pytest.mark.parametrize("q_len,kv_len,n_shared", [([1, 2], [300, 90], 0), ([1] * 6, [100 + i for i in range(6)], 96), ([90, 60], [200, 60], 0)])
def test_attention_rows_apart(paged, q_len, kv_len, n_shared):
    for pad, shift in ((8, 0), (24, 8), (0, 8)):
        close(*run_attention8(paged, "e4m3", 8, 2, 64, 16, "f16", q_len, kv_len, n_shared, pad=pad, shift=shift))
    close(*run_attention8(paged, "i8", 8, 2, 64, 16, "f16", q_len, kv_len, n_shared, pad=8, shift=8, out_f32=True))


def test_refusals(paged):
    from llamd_rs_b200.backend import Malformed, ShapeError, Unsupported

    with pytest.raises(Unsupported):
        paged.Batch(8, 2, 64, 16, "f16", cache="e5m2")
    with pytest.raises(Malformed):
        paged.Batch(8, 3, 64, 16, "f16", cache="i8")
    assert lib().llamd_cuda_paged_new8(8, 2, 64, 16, 0, 0) is None
    lib().llamd_fwd_last_error()
    pool, scales, rows = dev(np.zeros(6 * 2 * 16 * 64, np.uint8)), dev(np.zeros(12, np.uint8)), dev(np.zeros(64 * 8 * 64, np.uint16))
    b = paged.Batch(8, 2, 64, 16, "f16", cache="i8")
    s = dict(k_scales=scales, v_scales=scales)
    with pytest.raises(Malformed):  # not set
        b.attention(rows, pool, pool, rows, **s)
    b.set([2], [20], [[3, 1]], 6)
    b.append(rows, rows, rows, rows, pool, pool, inputs="f16", **s)
    b.attention(rows, pool, pool, rows, **s)
    for call in (lambda **x: b.attention(rows, pool, pool, rows, **x), lambda **x: b.append(rows, rows, rows, rows, pool, pool, inputs="f16", **x)):
        with pytest.raises(Malformed):
            call()
        with pytest.raises(Malformed):
            call(k_scales=scales)
        with pytest.raises(ShapeError):
            call(k_scales=scales, v_scales=dev(np.zeros(11, np.uint8)))
    with pytest.raises(ShapeError):
        b.attention(rows, dev(np.zeros(6 * 2 * 16 * 64 - 1, np.uint8)), pool, rows, **s)
    # the other kind's calls
    wide = paged.Batch(8, 2, 64, 16, "f16")
    wide.set([2], [20], [[3, 1]], 6)
    with pytest.raises(Malformed):
        wide.attention(rows, rows, rows, rows, **s)
    L, a = lib(), (rows.ptr, 512)
    assert L.llamd_fwd_paged_attention(b.ptr, *a, rows.ptr, rows.ptr, *a, 0, 0.1) == -1
    assert L.llamd_fwd_paged_attention8(wide.ptr, *a, pool.ptr, pool.ptr, scales.ptr, scales.ptr, *a, 0, 0.1) == -1
    assert L.llamd_fwd_paged_attention8(b.ptr, *a, pool.ptr, pool.ptr, None, scales.ptr, *a, 0, 0.1) == -1
    L.llamd_fwd_last_error()
    # two sequences whose new tokens go to one page, and one that lists a page twice
    for q_len, kv_len, tables in (([1, 1], [1, 2], [[4], [4]]), ([20], [20], [[5, 5]])):
        b.set(q_len, kv_len, tables, 6)
        with pytest.raises(Malformed):
            b.append(rows, rows, rows, rows, pool, pool, inputs="f16", **s)
        b.attention(rows, pool, pool, rows, **s)  # (reading is no harm)


def test_tensors(paged):
    """torch tensors of the 8-bit types on torch's current stream; another type's are refused."""
    torch = pytest.importorskip("torch")
    from llamd_rs_b200.backend import ShapeError

    H, K, D, page, n = 8, 2, 64, 16, 50
    b = paged.Batch(H, K, D, page, "bf16", cache="e4m3")
    b.set([n], [n], [[2, 0, 3, 1]], 4)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # (without the order the calls would read what is not there yet)
        qkv = torch.randn(n, H + 2 * K, D, device="cuda").bfloat16()
        kp, vp = (torch.zeros(4, K, page, D, device="cuda").to(torch.float8_e4m3fn) for _ in range(2))
        ks = torch.zeros(4, K, 1, device="cuda", dtype=torch.uint8)
        vs = ks.clone().view(torch.float8_e8m0fnu)
        q, out = (torch.zeros(n, H, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        b.append(qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:], q, kp, vp, k_scales=ks, v_scales=vs)
        b.attention(q, kp, vp, out, k_scales=ks, v_scales=vs)
        got = out.clone()
    side.synchronize()
    pages = [(p.float() * torch.exp2(s.view(torch.uint8).float() - 127)[..., None]).double().cpu().numpy() for p, s in ((kp, ks), (vp, vs))]
    want, bound = plain.attention(qkv[:, :H].double().cpu().numpy(), *pages, [[2, 0, 3, 1]], [n], [n], D ** -0.5, "bf16")
    close(got.double().cpu().numpy(), want, bound)
    with pytest.raises(ShapeError):
        b.attention(q, kp.view(torch.int8), vp, out, k_scales=ks, v_scales=vs)
    with pytest.raises(ShapeError):
        b.attention(q, kp, vp, out, k_scales=ks.float(), v_scales=vs)
    with pytest.raises(ShapeError):
        b.attention(q, kp, vp, out, k_scales=ks[:3], v_scales=vs)


def test_graph(paged):
    """append and attention captured once and replayed over new values; the blocks' scales go on from replay to replay."""
    from llamd_rs_b200 import backend

    H, K, D, page, dtype, cache = 8, 1, 128, 16, "f16", "i8"
    q_len, kv_len = [1, 1, 40], [130, 17, 40]
    rng = np.random.default_rng(5)
    tables, n_pages = scatter_tables(rng, kv_len, page)
    b = paged.Batch(H, K, D, page, dtype, cache=cache)
    b.set(q_len, kv_len, tables, n_pages)
    T = b.tokens
    x = [rng.standard_normal((2, T, n, D)).astype(np.float32) for n in (H, K, K)]
    bufs = [dev(v[0]) for v in x]
    pools = [[dev(y) for y in plain8.random_pool(rng, n_pages, K, page, D, cache)] for _ in range(2)]
    q, out = dev(np.zeros((T, H, D), np.uint16)), dev(np.zeros((T, H, D), np.uint16))
    s = dict(k_scales=pools[0][1], v_scales=pools[1][1])
    backend.sync()
    assert lib().llamd_fwd_begin_capture() == 0
    b.append(*bufs, q, pools[0][0], pools[1][0], **s)
    b.attention(q, pools[0][0], pools[1][0], out, **s)
    assert lib().llamd_fwd_end_capture() == 0
    try:
        for i in range(2):
            for buf, v in zip(bufs, x):
                buf.upload(v[i])
            assert lib().llamd_fwd_graph_launch() == 0
            backend.sync()
            kv = [plain8.values(p[0].download(np.uint8, n_pages * K * page * D).reshape(n_pages, K, page, D), p[1].download(np.uint8, n_pages * K).reshape(n_pages, K, 1), cache)
                  for p in pools]
            want, bound = plain.attention(plain.from_bits(plain.to_bits(x[0][i], dtype), dtype), *kv, tables, q_len, kv_len, D ** -0.5, dtype)
            close(plain.from_bits(out.download(np.uint16, T * H * D), dtype).reshape(T, H, D), want, bound)
            seq, pos = plain.positions(q_len, kv_len)
            ids = np.array([tables[s_][p // page] for s_, p in zip(seq, pos)])
            new = kv[1][ids, :, pos % page]
            assert np.all(np.abs(new - x[2][i]) <= np.abs(x[2][i]).max() * 2 / 127 + 1e-6)  # (a step at most: scales only grow over the replays)
    finally:
        lib().llamd_fwd_graph_destroy()
    assert paged.status() == 0
