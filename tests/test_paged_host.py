"""The host side of paged caches, without a device: pages and who holds them, the angles' tables, what is refused before any launch."""
import numpy as np
import pytest


@pytest.fixture(scope="module")
def paged():
    import __graft_entry__ as g

    g.build()
    from llamd_rs_b200 import paged as p

    return p


def test_pages_are_neither_lost_nor_held_twice(paged):
    """Conversations that begin, fork, grow and end in random order: every page is free or held by exactly the tables that list it."""
    rng = np.random.default_rng(1)
    pool, live = paged.Pages(40, 16), []
    for _ in range(600):
        what = rng.integers(4)
        if what == 0 or not live:
            live.append([[], 0])
        elif what == 1 and len(live) < 12:
            table, n = live[rng.integers(len(live))]
            share = int(rng.integers(0, n // 16 + 1)) * 16
            live.append([pool.fork(table, share), share])
        elif what == 2:
            c = live[rng.integers(len(live))]
            more = c[1] + int(rng.integers(1, 60))
            before = list(c[0])
            try:
                pool.grow(c[0], more)
                c[1] = more
            except paged.OutOfPages:
                assert c[0] == before
        else:
            table, _ = live.pop(rng.integers(len(live)))
            pool.release(table)
        held = np.zeros(40, int)
        for table, n in live:
            assert len(table) * 16 >= n and len(set(table)) == len(table)
            for p in table:
                held[p] += 1
        assert pool.free() == np.sum(held == 0)
        assert pool._held == held.tolist()


def test_pages_refuse(paged):
    for n, size in ((0, 16), (4, 8), (4, 24), (4, 8192)):
        with pytest.raises(paged.ShapeError):
            paged.Pages(n, size)
    p = paged.Pages(2, 16)
    t = []
    p.grow(t, 20)
    with pytest.raises(paged.Malformed):
        p.fork(t, 33)
    with pytest.raises(paged.Malformed):
        p.fork(t, 8)


@pytest.mark.parametrize("rot,base", [(128, 1e6), (64, 1e4), (2, 1e4)])
def test_table_of_angles(paged, rot, base):
    """Rounded once from double: within half a step of f32 of the definition, at far positions too."""
    rows = 5000
    got = paged.rope_table(rows, rot, base).astype(np.float64)
    a = np.arange(rows)[:, None] * float(np.float32(base)) ** (-2.0 * np.arange(rot // 2) / rot)
    assert np.max(np.abs(got - np.stack([np.sin(a), np.cos(a)], -1))) <= 2.0 ** -25 + 1e-11


def test_linear_scaling_stretches_positions(paged):
    assert np.array_equal(paged.rope_table(64, 32, 1e4, "linear", 4.0)[::4], paged.rope_table(16, 32, 1e4))


def test_refused_without_a_device(paged):
    from llamd_rs_b200 import backend

    if backend.available():
        pytest.skip("a device is present")
    with pytest.raises(paged.Unsupported):
        paged.Batch(8, 2, 64, 16)


def test_pages_refuse_what_is_not_held(paged):
    """A negative length, pages that are free or not there: refused, and nothing has changed."""
    p = paged.Pages(6, 16)
    a = []
    p.grow(a, 60)
    before = list(p._held)
    for table, n in ((a, -16), ([5], 16), ([9], 16), ([-1], 16)):
        with pytest.raises(paged.Malformed):
            p.fork(table, n)
        assert p._held == before
    for table in ([a[0], 5], a[:2] + a[:1], [a[1], 6], [a[1], -1]):
        kept = list(table)
        with pytest.raises(paged.Malformed):
            p.release(table)
        assert p._held == before and p.free() == 2 and table == kept
    twice = a + p.fork(a, 32)  # a table may list a page twice, as often as it is held
    p.release(twice)
    assert p.free() == 6 and sorted(p._free) == list(range(6)) and not any(p._held)


def test_numbers_that_would_lose_bits_are_refused(paged):
    """What int32 cannot hold, and fractions: refused by name, not cut to the low bits (a batch that is never made serves: nothing reaches the library)."""
    b = paged.Batch.__new__(paged.Batch)
    b.ptr = None
    big = np.array([2 ** 32 + 1], np.int64)
    for q, kv, pages, n_pages, shared, what in (
            (big, [1], [[0]], 4, 0, "new-token counts"), ([1], big, [[0]], 4, 0, "lengths"), ([1], [1], big[None], 4, 0, "page ids"), ([1], [1], [big], 4, 0, "page ids"),
            ([1.5], [2], [[0]], 4, 0, "new-token counts"), ([1], [2], [[0.5]], 4, 0, "page ids"), ([1], [1], np.array([[2 ** 31]], np.uint32), 4, 0, "page ids"),
            ([1], [1], [[0]], 2 ** 32 + 4, 0, "pages"), ([1], [1], [[0]], 4, 2 ** 32, "shared positions"), ([1], [1], [[0]], 4.0, 0, "pages"),
            ([1], [1], [[0]], 4, -16, "shared positions")):
        with pytest.raises(paged.Malformed, match=what):
            b.set(q, kv, pages, n_pages, shared)
    for rows, rot, original in ((2 ** 32, 2, 0), (4, 2 ** 33, 0), (4, 8, 2 ** 32 + 1), (4, 8, -1)):
        with pytest.raises(paged.Malformed):
            paged.rope_table(rows, rot, 1e4, "by_frequency", 2.0, original)
    b.tokens, b.head_dim = 3, 64
    for stride in (-64, 2 ** 40, 64.0):
        with pytest.raises(paged.Malformed, match="elements between tokens"):
            b._rows(1 << 20, 64, 0, "q", stride)
    assert b._rows(1 << 20, 64, 0, "q", 72) == (1 << 20, 72) and b._rows(1 << 20, 64, 0, "q") == (1 << 20, 64)
