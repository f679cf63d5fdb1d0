"""Paged attention and append at the edges of their use."""
import numpy as np
import pytest

import paged_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    from llamd_rs_b200 import backend, paged as p

    backend.stream_init()
    return p


def dev(a):
    from llamd_rs_b200.backend import DevBuf

    return DevBuf.from_array(a)


@pytest.mark.parametrize("n_seq,q_len,more", [(1, 1, 15), (230, 1, 15), (1, 40, 7), (150, 40, 7)])
@pytest.mark.parametrize("nats", [11, 15, 17])
@pytest.mark.parametrize("out_f32", [False, True])
def test_many_small_weights(paged, n_seq, q_len, more, nats, out_f32):
    """One key far above 131072 alike: each of their weights is small, their sum is not. The sequences hold the same pages; where there are many,
    each is one piece, with one maximum.

    The scores are exact, so an output is off by its own rounding, by the weights' (u of each, and half a step of f16's subnormals
    where they end there: 2^-25, of weights scaled by 2^more) and by 2^-20 of f32 arithmetic."""
    from llamd_rs_b200 import backend

    n, H, D, page = 131072 + q_len, 8, 128, 64
    n_pages = -(-n // page)
    k, v = np.zeros((n_pages * page, D)), np.zeros((n_pages * page, D))
    k[0, 0], v[0, 1::2], v[1:, ::2] = nats, 1, 1
    q = np.zeros((n_seq, q_len, H, D))
    q[..., 0] = 1
    kp, vp = (dev(plain.to_bits(x.reshape(n_pages, 1, page, D), "f16")) for x in (k, v))
    b = paged.Batch(H, 1, D, page, "f16")
    b.set([q_len] * n_seq, [n] * n_seq, np.tile(np.arange(n_pages, dtype=np.int32), (n_seq, 1)), n_pages)
    wide = np.uint32 if out_f32 else np.uint16
    out = dev(np.zeros(q.shape, wide))
    b.attention(dev(plain.to_bits(q, "f16")), kp, vp, out, scale=1.0, out_f32=out_f32)
    backend.sync()
    got = out.download(wide, q.size)
    got = (got.view(np.float32).astype(np.float64) if out_f32 else plain.from_bits(got, "f16")).reshape(q.shape)
    far = np.arange(n - q_len, n)[:, None, None] * np.exp(-float(nats))  # the small weights' sum, token by token
    want = np.where(np.arange(D) % 2, 1, far) / (1 + far)
    u, tiny = plain.U["f16"], plain.TINY["f16"]
    rounded = 0.0 if out_f32 else u * want + tiny
    bound = rounded + (u + 2.0 ** -20) * want + (n - 1) * tiny * 2.0 ** -more / (1 + far)
    assert np.all(np.abs(got - want) <= bound), np.max(np.abs(got - want) / bound)


def test_streams_are_not_ordered_inside_a_capture(paged):
    """Events of or for another stream would end the capture, or draw that stream into it."""
    torch = pytest.importorskip("torch")
    from llamd_rs_b200 import backend
    from llamd_rs_b200._lib import lib

    side, L = torch.cuda.Stream(), lib()
    a, c = dev(np.arange(256, dtype=np.float32)), dev(np.zeros(256, np.float32))
    backend.sync()
    assert L.llamd_fwd_begin_capture() == 0
    paged.wait_for(side.cuda_stream)
    L.llamd_fwd_add(a.ptr, a.ptr, c.ptr, 256)
    paged.ready_for(side.cuda_stream)
    assert L.llamd_fwd_end_capture() == 0
    try:
        assert not any(c.download_f32(256))
        assert side.query() and L.llamd_fwd_graph_launch() == 0
        backend.sync()
        assert np.array_equal(c.download_f32(256), 2 * np.arange(256, dtype=np.float32))
        paged.wait_for(side.cuda_stream)  # and they do again afterwards
        paged.ready_for(side.cuda_stream)
        side.synchronize()
    finally:
        L.llamd_fwd_graph_destroy()


def test_tensors_of_another_stream(paged):
    """Tensors that torch's current stream is still making, outputs that it reads right after the calls: nobody has to say so."""
    torch = pytest.importorskip("torch")

    H, K, D, page, n = 8, 2, 64, 16, 50
    b = paged.Batch(H, K, D, page, "bf16")
    b.set([n], [n], [list(range(4))], 4)
    side = torch.cuda.Stream()
    for stream in (side, torch.cuda.default_stream()):
        with torch.cuda.stream(stream):
            qkv = torch.randn(n, H + 2 * K, D, device="cuda").bfloat16()
            source = qkv.clone()
            kp, vp = (torch.zeros(4, K, page, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
            q, out = (torch.zeros(n, H, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
            torch.cuda.synchronize()
            qkv.zero_()
            torch.cuda._sleep(20_000_000)
            qkv.copy_(source)  # (in front of this, and of the sleep before it, the calls would read zeros)
            b.append(qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:], q, kp, vp)
            qkv.zero_()        # (this must not come before they have read it)
            b.attention(q, kp, vp, out)
            got = [x.clone() for x in (q, kp, vp, out)]
            torch.cuda.synchronize()
        assert torch.equal(got[0], source[:, :H]) and torch.equal(got[1].transpose(1, 2).reshape(64, K, D)[:n], source[:, H:H + K])
        x = source.double().cpu().numpy()
        want, bound = plain.attention(x[:, :H], *(y.double().cpu().numpy() for y in got[1:3]), [list(range(4))], [n], [n], D ** -0.5, "bf16")
        assert np.all(np.abs(got[3].double().cpu().numpy() - want) <= bound)


def test_refused_attention_launches_nothing(paged):
    """Rows of q further apart than a tensor map can say, behind a shared prefix, whose parts another launch joins: refused before any of them."""
    from llamd_rs_b200 import backend
    from llamd_rs_b200._lib import lib

    L, H, D, n = lib(), 64, 128, 40
    b = paged.Batch(H, 1, D, 16, "f16")
    b.set([1], [n], [[0, 1, 2]], 3, 16)
    rng = np.random.default_rng(0)
    q, kp, vp = (plain.to_bits(rng.standard_normal(s), "f16") for s in ((1, H, D), (3, 1, 16, D), (3, 1, 16, D)))
    dq, dk, dv, out = dev(q), dev(kp), dev(vp), dev(np.full((1, H, D), 7, np.uint16))
    backend.sync()
    before = L.llamd_fwd_launch_count()
    assert L.llamd_fwd_paged_attention(b.ptr, dq.ptr, 1 << 40, dk.ptr, dv.ptr, out.ptr, H * D, 0, D ** -0.5) == -1  # (one row: nothing lies that far)
    assert L.llamd_fwd_launch_count() == before and L.llamd_fwd_last_error() == -1
    assert np.all(out.download(np.uint16, H * D) == 7)
    b.attention(dq, dk, dv, out)
    backend.sync()
    want, bound = plain.attention(*(plain.from_bits(x, "f16") for x in (q, kp, vp)), [[0, 1, 2]], [1], [n], D ** -0.5, "f16")
    assert np.all(np.abs(plain.from_bits(out.download(np.uint16, H * D), "f16").reshape(1, H, D) - want) <= bound)


@pytest.mark.parametrize("dtype,out_f32", [("f16", False), ("bf16", True)])
@pytest.mark.parametrize("q_len,kv_len,n_shared", [([90, 300], [90, 900], 0), ([20, 1, 20], [6048, 6016, 6040], 6000), ([1] * 40, [6001] * 40, 6000)])
def test_given_up(paged, dtype, out_f32, q_len, kv_len, n_shared):
    """Waits that may take no time: every row of the tensor-core kernel, or that joins one of its parts, is NaN, the status says so once, calls refuse
    until it has been read, and then all is as before."""
    from llamd_rs_b200 import backend

    H, D, page = 8, 128, 16
    rng = np.random.default_rng(1)
    first, n_pages, tables = list(range(n_shared // page)), n_shared // page, []
    for m in kv_len:
        own = -(-m // page) - n_shared // page
        tables.append(first + list(range(n_pages, n_pages + own)))
        n_pages += own
    b = paged.Batch(H, 1, D, page, dtype)
    b.set(q_len, kv_len, tables, n_pages, n_shared)
    T, wide = b.tokens, np.uint32 if out_f32 else np.uint16
    q, kp, vp = (plain.to_bits(rng.standard_normal(s), dtype) for s in ((T, H, D), (n_pages, 1, page, D), (n_pages, 1, page, D)))
    dq, dk, dv, out = dev(q), dev(kp), dev(vp), dev(np.zeros((T, H, D), wide))

    def result():
        got = out.download(wide, T * H * D)
        return (got.view(np.float32).astype(np.float64) if out_f32 else plain.from_bits(got, dtype)).reshape(T, H, D)

    want, bound = plain.attention(*(plain.from_bits(x, dtype) for x in (q, kp, vp)), tables, q_len, kv_len, D ** -0.5, dtype)
    b.attention(dq, dk, dv, out, out_f32=out_f32)
    backend.sync()
    assert np.all(np.abs(result() - want) <= bound) and paged.status() == 0
    paged.wait_limit(0)
    try:
        b.attention(dq, dk, dv, out, out_f32=out_f32)
    finally:
        paged.wait_limit(2)
    backend.sync()
    assert np.all(np.isnan(result()))
    for _ in range(2):
        with pytest.raises(paged.Other, match="ran out"):
            b.attention(dq, dk, dv, out, out_f32=out_f32)
    with pytest.raises(paged.Other, match="ran out"):
        b.append(dq, dq, dq, dq, dk, dv, inputs=dtype)
    assert paged.status() > 0 and paged.status() == 0
    b.attention(dq, dk, dv, out, out_f32=out_f32)
    backend.sync()
    assert np.all(np.abs(result() - want) <= bound) and paged.status() == 0


def test_given_up_beside_the_decode_kernel(paged):
    """A batch of which the decode kernel takes some sequences by itself: those are right, the others NaN."""
    from llamd_rs_b200 import backend

    H, D, page, q_len, kv_len = 8, 128, 16, [1, 400, 2], [20, 400, 33]
    rng = np.random.default_rng(2)
    tables = [[0, 1], list(range(2, 27)), [27, 28, 29]]
    b = paged.Batch(H, 1, D, page, "f16")
    b.set(q_len, kv_len, tables, 30)
    q, kp, vp = (plain.to_bits(rng.standard_normal(s), "f16") for s in ((403, H, D), (30, 1, page, D), (30, 1, page, D)))
    out = dev(np.zeros(q.shape, np.uint16))
    paged.wait_limit(0)
    try:
        b.attention(dev(q), dev(kp), dev(vp), out)
    finally:
        paged.wait_limit(2)
    backend.sync()
    assert paged.status() > 0 and paged.status() == 0
    got = plain.from_bits(out.download(np.uint16, q.size), "f16").reshape(q.shape)
    want, bound = plain.attention(*(plain.from_bits(x, "f16") for x in (q, kp, vp)), tables, q_len, kv_len, D ** -0.5, "f16")
    assert np.all(np.isnan(got[1:401]))
    assert np.all(np.abs(got - want)[[0, 401, 402]] <= bound[[0, 401, 402]])


def test_set_inside_a_capture_is_refused(paged):
    """The batch stays as it was, and the capture goes on."""
    from llamd_rs_b200 import backend
    from llamd_rs_b200._lib import lib

    L, H, D = lib(), 8, 64
    rng = np.random.default_rng(4)
    q, kp, vp = (plain.to_bits(rng.standard_normal(s), "f16") for s in ((2, H, D), (2, 1, 16, D), (2, 1, 16, D)))
    dq, dk, dv, out = dev(q), dev(kp), dev(vp), dev(np.zeros((2, H, D), np.uint16))
    b = paged.Batch(H, 1, D, 16, "f16")
    b.set([2], [20], [[1, 0]], 2)
    backend.sync()
    assert L.llamd_fwd_begin_capture() == 0
    for tables in ([[0, 1]], [[1, 0]]):
        with pytest.raises(paged.Malformed, match="captured"):
            b.set([1], [18], tables, 2)
    b.attention(dq, dk, dv, out)
    assert L.llamd_fwd_end_capture() == 0
    try:
        assert L.llamd_fwd_graph_launch() == 0
        backend.sync()
    finally:
        L.llamd_fwd_graph_destroy()
    want, bound = plain.attention(*(plain.from_bits(x, "f16") for x in (q, kp, vp)), [[1, 0]], [2], [20], D ** -0.5, "f16")
    assert np.all(np.abs(plain.from_bits(out.download(np.uint16, q.size), "f16").reshape(q.shape) - want) <= bound)


def large_batch(paged):
    """A batch whose partial results are some 40 MB: 1280 sequences behind a shared prefix."""
    b = paged.Batch(32, 4, 128, 16, "f16")
    b.set([1] * 1280, [2049] * 1280, np.tile(np.arange(129, dtype=np.int32), (1280, 1)), 129, 2048)
    return b


def test_memory_of_large_batches_is_kept(paged):
    """A batch made and given back every step: from the second on nothing is allocated or returned."""
    from llamd_rs_b200 import backend

    large_batch(paged).free()
    at = []
    for _ in range(3):
        b = large_batch(paged)
        at.append(backend.free_memory())
        b.free()
        at.append(backend.free_memory())
    assert len(set(at)) == 1


def test_free_waits_for_nothing_and_may_be_inside_a_capture(paged):
    torch = pytest.importorskip("torch")
    import time

    from llamd_rs_b200 import backend
    from llamd_rs_b200._lib import lib

    L = lib()
    batches = [large_batch(paged)] + [paged.Batch(8, 2, 64, 16) for _ in range(12)]
    for b in batches[1:]:
        b.set([1], [1], [[0]], 1)
    backend.sync()
    a, c = dev(np.arange(256, dtype=np.float32)), dev(np.zeros(256, np.float32))
    with torch.cuda.stream(torch.cuda.ExternalStream(L.llamd_fwd_stream())):
        torch.cuda._sleep(1_000_000_000)  # half a second
    t = time.perf_counter()
    for b in batches[:6]:
        b.free()
    assert time.perf_counter() - t < 0.1
    backend.sync()
    assert L.llamd_fwd_begin_capture() == 0
    for b in batches[6:]:
        b.free()
    L.llamd_fwd_add(a.ptr, a.ptr, c.ptr, 256)
    assert L.llamd_fwd_end_capture() == 0
    try:
        assert L.llamd_fwd_graph_launch() == 0
        backend.sync()
        assert np.array_equal(c.download_f32(256), 2 * np.arange(256, dtype=np.float32))
    finally:
        L.llamd_fwd_graph_destroy()


@pytest.mark.parametrize("how", ["set", "free"])
def test_graph_whose_batch_is_gone(paged, how):
    """A graph reads its batch's tables: once they are another's it is not launched any more. A refused set leaves it valid."""
    from llamd_rs_b200 import backend
    from llamd_rs_b200._lib import lib

    L, H, D = lib(), 8, 64
    q, pool, out = (dev(np.zeros(n * 16 * D, np.uint16)) for n in (2 * H, 2, 2 * H))
    b = paged.Batch(H, 1, D, 16, "f16")
    b.set([2], [20], [[1, 0]], 2)
    backend.sync()
    assert L.llamd_fwd_begin_capture() == 0
    b.append(q, q, q, q, pool, pool, inputs="f16")
    b.attention(q, pool, pool, out)
    assert L.llamd_fwd_end_capture() == 0
    try:
        assert L.llamd_fwd_graph_launch() == 0
        with pytest.raises(paged.Malformed):
            b.set([2], [20], [[1, 7]], 2)
        assert L.llamd_fwd_graph_launch() == 0
        if how == "set":
            b.set([2], [20], [[1, 0]], 2)
        else:
            b.free()
        assert L.llamd_fwd_graph_launch() == -1 and "freed" in backend._last_error()
        assert L.llamd_fwd_last_error() == -1
        backend.sync()
        assert L.llamd_fwd_begin_capture() == 0  # another graph has nothing to do with it
        L.llamd_fwd_add(out.ptr, out.ptr, out.ptr, 16)
        assert L.llamd_fwd_end_capture() == 0 and L.llamd_fwd_graph_launch() == 0
        backend.sync()
    finally:
        L.llamd_fwd_graph_destroy()


@pytest.mark.parametrize("q_len,kv_len,n_shared", [([0, 1, 0, 1], [0, 40, 0, 70], 32), ([0, 0, 2, 1], [50, 16, 34, 33], 32), ([1, 0, 90], [65, 3, 400], 64)])
def test_idle_slots_behind_a_shared_prefix(paged, q_len, kv_len, n_shared):
    """Sequences without new tokens need not have the prefix, nor any position, wherever they stand."""
    from llamd_rs_b200 import backend

    H, K, D, page = 8, 2, 64, 16
    rng = np.random.default_rng(6)
    shared = [5, 2, 9, 1][:n_shared // page]
    tables, at = [], 10
    for n, m in zip(q_len, kv_len):
        own = -(-m // page) - (len(shared) if n else 0)
        tables.append((shared if n else []) + list(range(at, at + own)))
        at += own
    b = paged.Batch(H, K, D, page, "f16")
    b.set(q_len, kv_len, tables, at, n_shared)
    T = b.tokens
    q, kp, vp = (plain.to_bits(rng.standard_normal(s), "f16") for s in ((T, H, D), (at, K, page, D), (at, K, page, D)))
    out = dev(np.zeros(q.shape, np.uint16))
    b.attention(dev(q), dev(kp), dev(vp), out)
    backend.sync()
    want, bound = plain.attention(*(plain.from_bits(x, "f16") for x in (q, kp, vp)), tables, q_len, kv_len, D ** -0.5, "f16")
    assert np.all(np.abs(plain.from_bits(out.download(np.uint16, q.size), "f16").reshape(q.shape) - want) <= bound)


def test_angles_need_not_reach_idle_sequences(paged):
    """A table of angles as long as the sequences with new tokens; one without is longer."""
    from llamd_rs_b200 import backend

    H, D, page = 2, 64, 16
    b = paged.Batch(H, 1, D, page, "f16")
    b.set([1, 0], [20, 90], [[0, 1], list(range(2, 8))], 8)
    rng = np.random.default_rng(7)
    x = rng.standard_normal((1, H, D)).astype(np.float32)
    table, pool, out = paged.rope_table(20, D, 1e4), dev(np.zeros(8 * page * D, np.uint16)), dev(np.zeros(H * D, np.uint16))
    b.append(dev(x), dev(x[:, :1]), dev(x[:, :1]), out, pool, pool, rope=dev(table))
    backend.sync()
    want = plain.norm_rope(x, np.array([19]), None, 0, table, D, False)
    got = plain.from_bits(out.download(np.uint16, H * D), "f16").reshape(want.shape)
    assert np.all(np.abs(got - want) <= plain.U["f16"] * np.abs(want) + 2.0 ** -22 * np.abs(want).max() + plain.TINY["f16"])
    with pytest.raises(paged.Malformed, match="angles"):
        b.append(dev(x), dev(x[:, :1]), dev(x[:, :1]), out, pool, pool, rope=dev(table), rope_rows=19)


def test_strides_that_point_elsewhere_are_refused(paged):
    """Negative strides between tokens: before anything is read."""
    from llamd_rs_b200._lib import lib

    b = paged.Batch(8, 2, 64, 16, "f16")
    b.set([3], [20], [[3, 1]], 6)
    pool, rows = dev(np.zeros(6 * 2 * 16 * 64, np.uint16)), dev(np.zeros(64 * 8 * 64, np.uint16))
    before = lib().llamd_fwd_launch_count()
    for i in range(3):
        strides = [None] * 3
        strides[i] = -1024
        for q in (rows, rows.ptr):
            with pytest.raises(paged.Malformed, match="between tokens"):
                b.append(q, q, q, rows, pool, pool, inputs="f16", strides=strides)
    assert lib().llamd_fwd_launch_count() == before


@pytest.mark.parametrize("q_len,n_shared", [([31] * 6, 272), ([33] * 6, 272), ([90] + [1] * 12, 272), ([300] + [1] * 12, 1008), ([40], 512), ([0, 1, 0], 512)])
@pytest.mark.parametrize("K,D,dtype", [(1, 128, "bf16"), (2, 64, "f16")])
def test_prefix_apart_and_whole(paged, q_len, n_shared, K, D, dtype):
    """Prompts and tokens behind a prefix on both sides of the line from which it is read once for all."""
    from llamd_rs_b200 import backend

    H, page = 8 * K, 16
    kv_len = [n_shared + n + 5 * i if n else 0 for i, n in enumerate(q_len)]
    rng, first, tables = np.random.default_rng(len(q_len)), n_shared // page, []
    ids, at = rng.permutation(sum(-(-m // page) for m in kv_len) + first), first
    for m in kv_len:
        own = max(0, -(-m // page) - first)
        tables.append(np.concatenate([ids[:first] if m else ids[:0], ids[at:at + own]]).astype(np.int32))
        at += own
    b = paged.Batch(H, K, D, page, dtype)
    b.set(q_len, kv_len, tables, len(ids), n_shared)
    T = b.tokens
    q, kp, vp = (plain.to_bits(rng.standard_normal(s), dtype) for s in ((T, H, D), (len(ids), K, page, D), (len(ids), K, page, D)))
    out = dev(np.zeros(q.shape, np.uint16))
    b.attention(dev(q), dev(kp), dev(vp), out)
    backend.sync()
    want, bound = plain.attention(*(plain.from_bits(x, dtype) for x in (q, kp, vp)), tables, q_len, kv_len, D ** -0.5, dtype)
    assert np.all(np.abs(plain.from_bits(out.download(np.uint16, q.size), dtype).reshape(q.shape) - want) <= bound)


def test_graph_with_the_side_stream(paged):
    """A batch whose prefix and own positions are read at the same time, captured and replayed over new queries; a launch before and behind it on the
    library's stream, so that fork and join are inside."""
    from llamd_rs_b200 import backend
    from llamd_rs_b200._lib import lib

    L, H, K, D, page, n_shared = lib(), 32, 4, 128, 64, 7552
    rng = np.random.default_rng(8)
    q_len = [1] * 64
    kv_len = [n_shared + int(x) for x in rng.integers(380, 520, 64)]
    first, tables, at = n_shared // page, [], n_shared // page
    for m in kv_len:
        own = -(-m // page) - first
        tables.append(list(range(first)) + list(range(at, at + own)))
        at += own
    b = paged.Batch(H, K, D, page, "bf16")
    b.set(q_len, kv_len, tables, at, n_shared)
    kp, vp = (plain.to_bits(rng.standard_normal((at, K, page, D)), "bf16") for _ in range(2))
    q = [plain.to_bits(rng.standard_normal((64, H, D)), "bf16") for _ in range(3)]
    dq, dk, dv, out, x = dev(q[0]), dev(kp), dev(vp), dev(np.zeros((64, H, D), np.float32)), dev(np.ones(64 * H * D, np.float32))
    total = dev(np.zeros(64 * H * D, np.float32))
    backend.sync()
    assert L.llamd_fwd_begin_capture() == 0
    L.llamd_fwd_add(x.ptr, x.ptr, out.ptr, 64 * H * D)
    b.attention(dq, dk, dv, out, out_f32=True)
    L.llamd_fwd_add(out.ptr, x.ptr, total.ptr, 64 * H * D)
    assert L.llamd_fwd_end_capture() == 0
    pages = [plain.from_bits(y, "bf16") for y in (kp, vp)]
    try:
        for i in range(3):
            dq.upload(q[i])
            for _ in range(1 + i):
                assert L.llamd_fwd_graph_launch() == 0
            backend.sync()
            got = total.download_f32(64 * H * D).astype(np.float64).reshape(64, H, D) - 1
            want, bound = plain.attention(plain.from_bits(q[i], "bf16"), *pages, tables, q_len, kv_len, D ** -0.5, "bf16")
            assert np.all(np.abs(got - want) <= bound + 2.0 ** -22)  # (the sum with 1 is rounded once)
    finally:
        L.llamd_fwd_graph_destroy()
    assert paged.status() == 0


def test_tensors_in_torchs_own_graph(paged):
    """torch captures its stream: the calls' launches and orders become part of its graph."""
    torch = pytest.importorskip("torch")

    H, K, D, page, n = 8, 2, 64, 16, 50
    b = paged.Batch(H, K, D, page, "bf16")
    b.set([n], [n], [list(range(4))], 4)
    qkv = torch.randn(n, H + 2 * K, D, device="cuda").bfloat16()
    kp, vp = (torch.zeros(4, K, page, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    q, out = (torch.zeros(n, H, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    b.append(qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:], q, kp, vp)
    b.attention(q, kp, vp, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        qkv.mul_(0.5)
        b.append(qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:], q, kp, vp)
        b.attention(q, kp, vp, out)
        doubled = out * 2
    for _ in range(2):
        before = qkv.clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(qkv, before * 0.5) and torch.equal(q, qkv[:, :H]) and torch.equal(doubled, out * 2)
        x = qkv.double().cpu().numpy()
        want, bound = plain.attention(x[:, :H], *(y.double().cpu().numpy() for y in (kp, vp)), [list(range(4))], [n], [n], D ** -0.5, "bf16")
        assert np.all(np.abs(out.double().cpu().numpy() - want) <= bound)
