"""Paged K/V caches on the GPU: append and attention against the definitions in 64 bits (paged_plain.py)."""
import numpy as np
import pytest

import paged_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    from llamd_rs_b200 import backend, paged as p

    backend.stream_init()
    return p


def scatter_tables(rng, kv_len, page, n_shared=0, spare=2):
    """Tables of shuffled pages; the first n_shared positions' pages are common. -> (tables, n_pages)"""
    first = n_shared // page
    own = [-(-m // page) - first for m in kv_len]
    n_pages = first + sum(own) + spare
    ids = rng.permutation(n_pages).astype(np.int32)
    tables, at = [], first
    for n in own:
        tables.append(np.concatenate([ids[:first], ids[at:at + n]]).astype(np.int32))
        at += n
    return tables, n_pages


def dev(a):
    from llamd_rs_b200.backend import DevBuf

    return DevBuf.from_array(a)


def make_append(paged, rng, H, K, D, page, dtype, q_len, kv_len, inputs, stride_pad=0):
    tables, n_pages = scatter_tables(rng, kv_len, page)
    b = paged.Batch(H, K, D, page, dtype)
    b.set(q_len, kv_len, tables, n_pages)
    T = b.tokens
    rows = [rng.standard_normal((T, n * D + stride_pad)).astype(np.float32) for n in (H, K, K)]
    if inputs == "f32":
        bufs, vals = [dev(r) for r in rows], [r.astype(np.float64) for r in rows]
    else:
        bits = [plain.to_bits(r, dtype) for r in rows]
        bufs, vals = [dev(x) for x in bits], [plain.from_bits(x, dtype) for x in bits]
    vals = [v[:, :n * D].reshape(T, n, D) for v, n in zip(vals, (H, K, K))]
    return b, tables, n_pages, bufs, vals


APPEND = [
    # H, K, D, page, dtype, inputs, q_len, kv_len, rot, interleaved, norm, stride_pad
    (32, 4, 128, 16, "f16", "f32", [1], [1], 128, False, True, 0),
    (32, 4, 128, 16, "f16", "f32", [1], [17], 128, False, True, 0),
    (32, 4, 128, 32, "bf16", "bf16", [3, 0, 1, 18], [3, 5, 40, 50], 64, False, True, 8),
    (14, 2, 64, 16, "f16", "f16", [33, 1], [35, 16], 32, True, False, 0),
    (14, 2, 64, 64, "bf16", "f32", [7], [70], 16, True, True, 4),
    (5, 1, 128, 16, "f16", "f16", [21], [21], 128, True, True, 0),
    (5, 1, 128, 16, "bf16", "f32", [2, 2], [2, 33], 0, False, True, 0),
    (8, 8, 64, 4096, "f16", "f32", [9], [4100], 64, False, False, 0),
    (3, 3, 64, 16, "f16", "f32", [5], [6], 48, False, True, 1),     # rows off the 16-byte boundary
    (3, 3, 64, 16, "bf16", "bf16", [5], [6], 64, True, True, 3),
]


@pytest.mark.parametrize("H,K,D,page,dtype,inputs,q_len,kv_len,rot,interleaved,norm,pad", APPEND)
def test_append(paged, H, K, D, page, dtype, inputs, q_len, kv_len, rot, interleaved, norm, pad):
    rng = np.random.default_rng(H * 1000 + D + rot + len(q_len))
    b, tables, n_pages, bufs, vals = make_append(paged, rng, H, K, D, page, dtype, q_len, kv_len, inputs, pad)
    T, eps = b.tokens, 1e-6
    table = paged.rope_table(max(kv_len), rot, 1e6) if rot else None
    wq, wk = ((1 + 0.3 * rng.standard_normal(D)).astype(np.float32) for _ in range(2)) if norm else (None, None)
    before = [plain.to_bits(rng.standard_normal((n_pages, K, page, D)), dtype) for _ in range(2)]
    kp, vp = dev(before[0]), dev(before[1])
    out = dev(np.zeros((T, H, D), np.uint16))
    b.append(*bufs, out, kp, vp, rope=dev(table) if rot else None, rot=rot, interleaved=interleaved, q_norm=dev(wq) if norm else None,
             k_norm=dev(wk) if norm else None, eps=eps, inputs=inputs, strides=[n * D + pad for n in (H, K, K)])
    from llamd_rs_b200 import backend

    backend.sync()
    seq, pos = plain.positions(q_len, kv_len)
    got_q = plain.from_bits(out.download(np.uint16, T * H * D), dtype).reshape(T, H, D)
    got = [p.download(np.uint16, before[0].size).reshape(before[0].shape) for p in (kp, vp)]
    ids, slot = np.array([tables[s][p // page] for s, p in zip(seq, pos)]), pos % page
    tab = table if rot else np.zeros((1, 0, 2), np.float32)
    want = [plain.norm_rope(vals[0], pos, wq, eps, tab, rot, interleaved), plain.norm_rope(vals[1], pos, wk, eps, tab, rot, interleaved), vals[2]]
    have = [got_q] + [plain.from_bits(g[ids, :, slot], dtype) for g in got]
    for g, w in zip(have, want):
        # f32 arithmetic: a norm of D terms and a rotation, 2^-24 (D / 2 + 8) of the pair's magnitude; then one rounding
        size = np.abs(w).max(-1, keepdims=True)
        assert np.all(np.abs(g - w) <= plain.U[dtype] * np.abs(w) + 2.0 ** -24 * (D / 2 + 8) * 2 * size + plain.TINY[dtype])
    if inputs != "f32" and not norm and not rot:
        assert np.array_equal(have[0], want[0])
    # nothing but the new tokens' slots has changed
    for g, w in zip(got, before):
        g, w = g.copy(), w.copy()
        g[ids, :, slot] = 0
        w[ids, :, slot] = 0
        assert np.array_equal(g, w)


def lib():
    from llamd_rs_b200._lib import lib as load

    return load()


def run_attention(paged, H, K, D, page, dtype, q_len, kv_len, n_shared=0, scale=None, out_f32=False, q_scale=1.0, poison=True, seed=0, edit=None,
                  repeat=1, pad=0, shift=0):
    rng = np.random.default_rng(seed + H * 100 + D + sum(kv_len))
    tables, n_pages = scatter_tables(rng, kv_len, page, n_shared)
    b = paged.Batch(H, K, D, page, dtype)
    b.set(q_len, kv_len, tables, n_pages, n_shared)
    T = b.tokens
    q = plain.to_bits(q_scale * rng.standard_normal((T, H, D)), dtype)
    kp, vp = (plain.to_bits(rng.standard_normal((n_pages, K, page, D)), dtype) for _ in range(2))
    if edit:
        edit(q, kp, vp, tables)
    if poison:  # whatever no sequence holds: NaN and infinities
        live = np.zeros((n_pages, page), bool)
        for t, m in zip(tables, kv_len):
            idx = np.arange(m)
            live[t[idx // page], idx % page] = True
        nan, inf = (0x7E00, 0x7C00) if dtype == "f16" else (0x7FC0, 0x7F80)
        dead = np.broadcast_to(~live[:, None, :, None], kp.shape)
        kp[dead], vp[dead] = nan, nan
        vp[..., ::2][dead[..., ::2]] = inf
    from llamd_rs_b200 import backend

    wide, n = np.uint32 if out_f32 else np.uint16, H * D + pad
    rows = np.full((T, n), 0x7FFF, np.uint16)
    rows[:, :H * D] = q.reshape(T, H * D)
    rows = dev(np.concatenate([np.full(shift, 0x7FFF, np.uint16), rows.ravel()]))
    out = dev(np.full(shift + T * n, np.iinfo(wide).max, wide))
    dk, dv = dev(kp), dev(vp)
    for _ in range(repeat):
        if pad or shift:
            assert lib().llamd_fwd_paged_attention(b.ptr, rows.ptr + 2 * shift, n, dk.ptr, dv.ptr, out.ptr + wide().itemsize * shift, n, int(out_f32),
                                                   D ** -0.5 if scale is None else scale) == 0
        else:
            b.attention(rows, dk, dv, out, scale=scale, out_f32=out_f32)
    backend.sync()
    assert paged.status() == 0
    got = out.download(wide, shift + T * n)
    assert np.all(got[:shift] == np.iinfo(wide).max)
    got = got[shift:].reshape(T, n)
    assert np.all(got[:, H * D:] == np.iinfo(wide).max)  # nothing between the rows is written
    got = np.ascontiguousarray(got[:, :H * D])
    got = (got.view(np.float32).astype(np.float64) if out_f32 else plain.from_bits(got, dtype)).reshape(T, H, D)
    want, bound = plain.attention(plain.from_bits(q, dtype), plain.from_bits(kp, dtype), plain.from_bits(vp, dtype), tables, q_len, kv_len,
                                  D ** -0.5 if scale is None else scale, dtype)
    return got, want, bound


def close(got, want, bound):
    assert np.all(np.isfinite(got))
    worst = np.max(np.abs(got - want) / bound) if got.size else 0.0
    assert worst <= 1.0, f"{worst:.3g} of the bound"


ATTENTION = [
    # H, K, D, page, dtype, q_len, kv_len, n_shared
    (32, 4, 128, 16, "f16", [1], [1], 0),
    (32, 4, 128, 16, "f16", [1], [2], 0),
    (32, 4, 128, 16, "bf16", [1], [16], 0),
    (32, 4, 128, 16, "f16", [1], [17], 0),
    (32, 4, 128, 32, "bf16", [1], [700], 0),
    (32, 4, 128, 16, "f16", [1, 1, 1, 1], [1, 129, 64, 500], 0),
    (8, 8, 64, 16, "f16", [1, 1], [33, 257], 0),
    (14, 2, 64, 64, "bf16", [1, 3, 1], [63, 65, 128], 0),
    (5, 1, 128, 16, "f16", [2, 0, 1], [130, 7, 31], 0),
    (16, 1, 128, 16, "bf16", [1, 1], [200, 90], 0),
    (40, 1, 64, 16, "f16", [1, 2], [40, 300], 0),              # a group of 40
    (64, 1, 128, 16, "f16", [3], [130], 0),
    (4, 2, 128, 4096, "f16", [1], [4097], 0),
    # prompts
    (8, 1, 128, 16, "f16", [5], [5], 0),
    (8, 1, 128, 16, "f16", [16], [16], 0),
    (8, 1, 128, 32, "bf16", [129], [129], 0),
    (4, 2, 64, 16, "f16", [128], [128], 0),
    (4, 2, 64, 16, "bf16", [257, 1, 40], [257, 1, 40], 0),
    (2, 2, 128, 64, "f16", [300], [300], 0),                    # no grouping: a tile is many tokens
    (5, 1, 128, 16, "f16", [100], [230], 0),
    (14, 2, 64, 128, "f16", [60, 77], [360, 77], 0),
    (7, 1, 128, 16, "bf16", [190, 0, 33], [1000, 3, 200], 0),
    (40, 1, 64, 16, "f16", [40], [170], 0),
    # a shared prefix
    (32, 4, 128, 16, "f16", [1, 1], [17, 17], 16),
    (32, 4, 128, 16, "bf16", [1, 1, 1], [65, 100, 200], 64),
    (8, 2, 64, 16, "f16", [1] * 9, [257 + 3 * i for i in range(9)], 256),
    (8, 1, 128, 32, "f16", [1] * 40, [161 + i for i in range(40)], 160),
    (5, 1, 128, 16, "bf16", [1, 2, 0, 3] * 6, [150 + i for i in range(24)], 144),
    (8, 1, 128, 16, "f16", [60, 1, 90], [400, 290, 290 + 90], 272),
    (4, 2, 64, 16, "f16", [0, 1], [32, 33], 32),
]


@pytest.mark.parametrize("H,K,D,page,dtype,q_len,kv_len,n_shared", ATTENTION)
def test_attention(paged, H, K, D, page, dtype, q_len, kv_len, n_shared):
    close(*run_attention(paged, H, K, D, page, dtype, q_len, kv_len, n_shared))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("q_len,kv_len", [([1], [300]), ([70], [300])])
def test_attention_sharp_and_flat(paged, dtype, q_len, kv_len):
    """Scores far apart (one key takes nearly everything, the maximum moves late) and all alike; another scale; f32 out."""
    def ramp(q, kp, vp, tables):
        # keys grow along the sequence: the running maximum moves in every tile
        t = np.asarray(tables[0])
        for i in range(kv_len[0]):
            kp[t[i // 16], :, i % 16] = plain.to_bits(plain.from_bits(kp[t[i // 16], :, i % 16], dtype) * (0.02 * i), dtype)

    close(*run_attention(paged, 8, 1, 128, 16, dtype, q_len, kv_len, q_scale=2.0, edit=ramp))
    close(*run_attention(paged, 8, 1, 128, 16, dtype, q_len, kv_len, q_scale=6.0))
    close(*run_attention(paged, 8, 1, 128, 16, dtype, q_len, kv_len, q_scale=0.0))
    close(*run_attention(paged, 8, 1, 128, 16, dtype, q_len, kv_len, scale=0.5))
    close(*run_attention(paged, 8, 1, 128, 16, dtype, q_len, kv_len, out_f32=True))


@pytest.mark.parametrize("H,K,D,page,dtype,q_len,kv_len,n_shared", [c for c in ATTENTION if max(c[5]) > 3 and not c[7]])
def test_attention_beside_a_long_prompt(paged, H, K, D, page, dtype, q_len, kv_len, n_shared):
    """Prompts that would be too little work for the tensor cores by themselves, in one batch with another that is not."""
    long = 300 + 2400 // (H // K)
    close(*run_attention(paged, H, K, D, page, dtype, q_len + [long], kv_len + [long], n_shared))


@pytest.mark.parametrize("n", [9, 24, 41, 90])
@pytest.mark.parametrize("D,dtype", [(128, "bf16"), (64, "f16")])
def test_attention_joins(paged, n, D, dtype):
    """A shared prefix of several parts behind 288 to 2880 rows: they are joined by 8, 4, 2 and 1 warps each."""
    close(*run_attention(paged, 32, 4, D, 16, dtype, [1] * n, [401 + 5 * i for i in range(n)], 400))


@pytest.mark.parametrize("q_len,kv_len", [([9], [300]), ([32], [70]), ([33], [70]), ([20, 1, 31], [20, 400, 131]), ([8] * 5, [600 + i for i in range(5)]),
                                          ([8] * 24, [500 + i for i in range(24)])])
def test_attention_few_rows(paged, q_len, kv_len):
    """Stretches of 64 to 264 query rows, on both sides of the lines between the two kernels."""
    close(*run_attention(paged, 32, 4, 128, 16, "f16", q_len, kv_len))
    close(*run_attention(paged, 16, 2, 64, 32, "bf16", q_len, [m + 64 for m in kv_len], 64))


def test_attention_beside(paged):
    """A batch large enough that the prefix and the sequences' own positions are read at the same time; twice, the second over the first's results."""
    rng = np.random.default_rng(3)
    own = [int(x) for x in rng.integers(380, 520, 64)]
    args = (paged, 32, 4, 128, 64, "bf16", [1] * 64, [7552 + m for m in own], 7552)
    close(*run_attention(*args, repeat=3))


@pytest.mark.parametrize("H,D,dtype", [(8, 128, "f16"), (5, 64, "bf16"), (1, 128, "bf16")])
def test_attention_many_pieces(paged, H, D, dtype):
    """Several pieces to every CTA, of one tile and of two, of one block and of several, tails of every length, and short sequences between them."""
    rng = np.random.default_rng(H)
    q_len, kv_len = [], []
    for _ in range(260):
        n = int(rng.choice([0, 1, 3, rng.integers(13, 17), rng.integers(17, 60), rng.integers(100, 140)], p=[.05, .1, .1, .3, .35, .1])) * (8 if H == 1 else 1)
        q_len.append(n)
        kv_len.append(n + int(rng.choice([0, 0, rng.integers(0, 40), rng.integers(0, 400)])))
    close(*run_attention(paged, H, 1, D, 16, dtype, q_len, kv_len, repeat=2))
    close(*run_attention(paged, H, 1, D, 32, dtype, q_len, [m + 256 for m in kv_len], 256, repeat=2))


@pytest.mark.parametrize("q_len,kv_len,n_shared", [([1, 2], [300, 90], 0), ([1] * 6, [100 + i for i in range(6)], 96), ([90, 60], [200, 60], 0)])
def test_attention_rows_apart(paged, q_len, kv_len, n_shared):
    """Rows of q and out further apart than their values, and starting at 16 bytes but not at 32."""
    for pad, shift in ((8, 0), (24, 8), (0, 8)):
        close(*run_attention(paged, 8, 2, 64, 16, "f16", q_len, kv_len, n_shared, pad=pad, shift=shift))
    close(*run_attention(paged, 8, 2, 64, 16, "f16", q_len, kv_len, n_shared, pad=8, shift=8, out_f32=True))


def test_graph(paged):
    """append and attention of a set batch captured once and replayed over new values."""
    from llamd_rs_b200 import backend

    H, K, D, page, dtype = 8, 1, 128, 16, "f16"
    q_len, kv_len = [1, 1, 40], [130, 17, 40]
    rng = np.random.default_rng(5)
    tables, n_pages = scatter_tables(rng, kv_len, page)
    b = paged.Batch(H, K, D, page, dtype)
    b.set(q_len, kv_len, tables, n_pages)
    T = b.tokens
    x = [rng.standard_normal((2, T, n, D)).astype(np.float32) for n in (H, K, K)]
    bufs = [dev(v[0]) for v in x]
    cache = [plain.to_bits(rng.standard_normal((n_pages, K, page, D)), dtype) for _ in range(2)]
    kp, vp, q, out = dev(cache[0]), dev(cache[1]), dev(np.zeros((T, H, D), np.uint16)), dev(np.zeros((T, H, D), np.uint16))
    backend.sync()
    assert lib().llamd_fwd_begin_capture() == 0
    b.append(*bufs, q, kp, vp)
    b.attention(q, kp, vp, out)
    assert lib().llamd_fwd_end_capture() == 0
    try:
        for i in range(2):
            for buf, v in zip(bufs, x):
                buf.upload(v[i])
            assert lib().llamd_fwd_graph_launch() == 0
            backend.sync()
            seq, pos = plain.positions(q_len, kv_len)
            ids = np.array([tables[s][p // page] for s, p in zip(seq, pos)])
            for c, v in zip(cache, x[1:]):
                c[ids, :, pos % page] = plain.to_bits(v[i], dtype)
            want, bound = plain.attention(plain.from_bits(plain.to_bits(x[0][i], dtype), dtype), plain.from_bits(cache[0], dtype),
                                          plain.from_bits(cache[1], dtype), tables, q_len, kv_len, D ** -0.5, dtype)
            close(plain.from_bits(out.download(np.uint16, T * H * D), dtype).reshape(T, H, D), want, bound)
    finally:
        lib().llamd_fwd_graph_destroy()
    assert paged.status() == 0


def test_no_tokens(paged):
    """A batch without sequences, and one whose sequences have nothing new: calls that do nothing."""
    b = paged.Batch(8, 2, 64, 16, "f16")
    buf = dev(np.full(4 * 8 * 16 * 64, 7, np.uint16))
    for q_len, kv_len, tables in (([], [], np.zeros((0, 1), np.int32)), ([0, 0], [5, 0], [[1], []])):
        b.set(q_len, kv_len, tables, 4)
        b.attention(buf, buf, buf, buf)
        b.append(buf, buf, buf, buf, buf, buf, inputs="f16")
    from llamd_rs_b200 import backend

    backend.sync()
    assert np.all(buf.download(np.uint16, 4 * 8 * 16 * 64) == 7)


def test_refusals(paged):
    from llamd_rs_b200 import backend
    from llamd_rs_b200.backend import Malformed, ShapeError, Unsupported

    for bad in ((8, 3, 64, 16), (8, 2, 96, 16), (8, 2, 64, 24), (8, 2, 64, 8), (130, 1, 64, 16), (0, 1, 64, 16)):
        with pytest.raises(Malformed):
            paged.Batch(*bad)
    with pytest.raises(Unsupported):
        paged.Batch(8, 2, 64, 16, "f32")
    b = paged.Batch(8, 2, 64, 16, "f16")
    pool, rows = dev(np.zeros(6 * 2 * 16 * 64, np.uint16)), dev(np.zeros(64 * 8 * 64, np.uint16))
    with pytest.raises(Malformed):  # not set
        b.attention(rows, pool, pool, rows)
    b.set([2], [20], [[3, 1]], 6)
    for q_len, kv_len, tables, n_pages, shared in (
            ([3], [2], [[0]], 6, 0),                    # more new tokens than positions
            ([-1], [2], [[0]], 6, 0),
            ([1], [17], [[0]], 6, 0),                   # a table too short
            ([1], [17], [[0, 6]], 6, 0),                # a page that is not there
            ([1], [17], [[0, -1]], 6, 0),
            ([1, 1], [17, 17], [[0, 1], [0, 2]], 6, 8),     # part of a page is shared
            ([1, 1], [17, 17], [[0, 1], [3, 2]], 6, 16),    # not the same pages
            ([1, 2], [17, 17], [[0, 1], [0, 2]], 6, 16),    # a new token inside the shared prefix
            ([1], [17], [[0, 1]], 0, 0)):
        with pytest.raises(Malformed):
            b.set(q_len, kv_len, tables, n_pages, shared)
    with pytest.raises(ShapeError):
        b.set([1, 1], [17], [[0, 1]], 6)
    b.attention(rows, pool, pool, rows)  # the batch as it was set before the refusals
    small = dev(np.zeros(64, np.uint16))
    for args in ((small, pool, pool, rows), (rows, small, pool, rows), (rows, pool, small, rows), (rows, pool, pool, small)):
        with pytest.raises(ShapeError):
            b.attention(*args)
    with pytest.raises(Malformed):
        b.attention(rows.ptr + 2, pool, pool, rows)  # off the 16-byte boundary
    table = dev(paged.rope_table(20, 64, 1e4))
    with pytest.raises(Malformed):  # 19 rows for positions up to 19
        b.append(rows, rows, rows, rows, pool, pool, rope=table, inputs="f16", rope_rows=19)
    with pytest.raises(Malformed):
        b.append(rows, rows, rows, rows, pool, pool, rope=table, rot=24, inputs="f16")
    with pytest.raises(Malformed):
        b.append(rows, rows, rows, rows, pool, pool, rot=16, inputs="f16")
    with pytest.raises(Unsupported):
        b.append(rows, rows, rows, rows, pool, pool, inputs="bf16")
    with pytest.raises(ShapeError):
        b.append(small, rows, rows, rows, pool, pool, inputs="f16")
    with pytest.raises(Unsupported):
        paged.rope_table(4, 64, 1e4, "spiral")
    with pytest.raises(Malformed):
        paged.rope_table(4, 64, 1e4, "linear", 0.5)
    backend.sync()


def test_refuses_odd_addresses_and_other_tables(paged):
    torch = pytest.importorskip("torch")
    from llamd_rs_b200.backend import Malformed, ShapeError

    with pytest.raises(Malformed):
        paged.Batch(8192, 4096, 64, 16)
    b = paged.Batch(8, 2, 64, 16, "f16")
    b.set([2], [20], [[3, 1]], 6)
    pool, rows = dev(np.zeros(6 * 2 * 16 * 64, np.uint16)), dev(np.zeros(64 * 8 * 64, np.uint16))
    for i in range(3):  # q, k or v inside an element
        with pytest.raises(Malformed):
            b.append(*[rows.ptr + (i == j) for j in range(3)], rows, pool, pool, inputs="f16")
    x = torch.zeros(2, 12, 64, dtype=torch.float16, device="cuda")
    with pytest.raises(ShapeError):  # a table of 64 rotated elements read as one of 32
        b.append(x[:, :8], x[:, 8:10], x[:, 10:], rows, pool, pool, rope=torch.zeros(20, 32, 2, device="cuda"), rot=32)


def test_tensors(paged):
    """torch tensors on a stream of their own: strided rows of one projection, types checked, order kept by wait_for / ready_for."""
    torch = pytest.importorskip("torch")
    from llamd_rs_b200.backend import ShapeError

    side = torch.cuda.Stream()
    H, K, D, page, n = 8, 2, 64, 16, 50
    b = paged.Batch(H, K, D, page, "bf16")
    b.set([n], [n], [list(range(4))], 4)
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # the side stream is behind: without the order the calls would read what is not there yet
        qkv = torch.randn(n, H + 2 * K, D, device="cuda").bfloat16()
        kp, vp = (torch.zeros(4, K, page, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        q, out = (torch.zeros(n, H, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    paged.wait_for(side.cuda_stream)
    b.append(qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:], q, kp, vp)
    b.attention(q, kp, vp, out)
    paged.ready_for(side.cuda_stream)
    with torch.cuda.stream(side):
        got = out.clone()
    side.synchronize()
    assert torch.equal(q, qkv[:, :H]) and torch.equal(kp.transpose(1, 2).reshape(64, K, D)[:n], qkv[:, H:H + K])
    x = qkv.double().cpu().numpy()
    pages = [y.double().cpu().numpy() for y in (kp, vp)]
    want, bound = plain.attention(x[:, :H], *pages, [list(range(4))], [n], [n], D ** -0.5, "bf16")
    close(got.double().cpu().numpy(), want, bound)
    with pytest.raises(ShapeError):
        b.attention(q.float(), kp, vp, out)
    with pytest.raises(ShapeError):
        b.attention(q.transpose(0, 1), kp, vp, out)
    with pytest.raises(ShapeError):
        b.attention(q, kp[:3], vp, out)
    with pytest.raises(ShapeError):
        b.attention(q, kp, vp, out[:-1])


def test_pages(paged):
    p = paged.Pages(6, 16)
    a = []
    p.grow(a, 33)
    assert len(a) == 3 and p.free() == 3
    c = p.fork(a, 32)
    p.grow(c, 40)
    assert c[:2] == a[:2] and c[2] != a[2] and p.free() == 2
    p.release(a)
    assert a == [] and p.free() == 3          # the shared two are still held
    with pytest.raises(paged.OutOfPages):
        p.grow(c, 16 * 7)
    assert len(c) == 3
    with pytest.raises(paged.Malformed):
        p.fork(c, 17)
    d = list(c)
    p.release(c)
    assert p.free() == 6
    with pytest.raises(paged.Malformed):
        p.release(d)


@pytest.mark.parametrize("scaling,factor,original", [("none", 1.0, 0), ("linear", 4.0, 0), ("base", 4.0, 0), ("by_frequency", 8.0, 512)])
def test_rope_table(paged, scaling, factor, original):
    rot, base, rows = 64, 1e4, 40
    got = paged.rope_table(rows, rot, base, scaling, factor, original).astype(np.float64)
    i, mag = np.arange(rot // 2), 1.0
    b = base * factor ** (rot / (rot - 2)) if scaling == "base" else base
    f = b ** (-2.0 * i / rot)
    if scaling == "linear":
        f = f / factor
    if scaling == "by_frequency":
        keep = np.clip((original * f / (2 * np.pi) - 1) / 31, 0, 1)
        f, mag = keep * f + (1 - keep) * f / factor, 0.1 * np.log(factor) + 1
    a = np.arange(rows)[:, None] * f
    want = mag * np.stack([np.sin(a), np.cos(a)], -1)
    assert np.max(np.abs(got - want)) <= mag * 2.0 ** -24 + 1e-12
