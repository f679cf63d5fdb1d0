"""What is kept of the memory of paged batches that are gone (csrc/paged_keep.h); no GPU is needed."""
import ctypes as C
import os
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llamd_rs_b200", "csrc")
SOURCE = r"""
#include <atomic>
#include <map>
#include <thread>
#include "paged_keep.h"
using namespace llamd;
static Kept *k = nullptr;
static uintptr_t made = 0;
extern "C" {
void start(size_t most, size_t bytes) { delete k; k = new Kept(most, bytes); made = 0; }
// n bytes: kept ones, or new ones (a number in place of an address). -> the block's number; its size in *have
size_t want(size_t n, size_t *have) {
    KeptBlock b = k->take(n);
    if (!b.p) b.p = (uint8_t *)++made, b.n = Kept::rounded(n);
    *have = b.n;
    return (size_t)b.p;
}
void let_go() { k->let_go(); }
void give(size_t p, size_t n) { KeptBlock b; b.p = (uint8_t *)p, b.n = n; k->keep(b); }
size_t n_made() { return made; }
size_t gone(size_t *out, size_t room) {
    size_t n = 0;
    for (const KeptBlock &b : k->gone()) if (n < room) out[n++] = (size_t)b.p;
    return n;
}
// Threads that take, hold and give back: 0, or how often a block was handed to two of them at once.
int threads(int n, int rounds) {
    start(6, 6 << 20);
    static std::atomic<int> held[1 << 20];
    for (auto &h : held) h = 0;
    std::atomic<int> twice{0};
    std::atomic<size_t> number{0};
    std::vector<std::thread> all;
    for (int t = 0; t < n; t++)
        all.emplace_back([&, t] {
            for (int i = 0; i < rounds; i++) {
                const size_t bytes = (size_t)(1 + (i * 7 + t * 13) % 23) << 14;
                KeptBlock b = k->take(bytes);
                if (!b.p) b.p = (uint8_t *)++number, b.n = Kept::rounded(bytes);
                if (held[(size_t)b.p].fetch_add(1)) twice++;
                std::this_thread::yield();
                held[(size_t)b.p].fetch_sub(1);
                k->keep(b);
                if (i % 50 == 0) for (const KeptBlock &g : k->gone()) if (held[(size_t)g.p].fetch_add(1)) twice++;
            }
        });
    for (auto &t : all) t.join();
    return twice;
}
}
"""


@pytest.fixture(scope="module")
def keep(tmp_path_factory):
    d = tmp_path_factory.mktemp("keep")
    (d / "k.cpp").write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-pthread", "-shared", "-fPIC", "-I", CSRC, str(d / "k.cpp"), "-o", str(d / "k.so")])
    L = C.CDLL(str(d / "k.so"))
    for f in (L.want, L.n_made, L.gone):
        f.restype = C.c_size_t
    L.want.argtypes, L.give.argtypes, L.start.argtypes = [C.c_size_t, C.c_void_p], [C.c_size_t, C.c_size_t], [C.c_size_t, C.c_size_t]
    L.gone.argtypes = [C.c_void_p, C.c_size_t]
    return L


def want(keep, n):
    have = C.c_size_t()
    return keep.want(n, C.byref(have)), have.value


def gone(keep):
    out = (C.c_size_t * 64)()
    return list(out[:keep.gone(out, 64)])


def test_larger_batches_after_many_small_ones(keep):
    """Blocks of small batches fill the list; one of a large batch still takes a place, and is found again."""
    keep.start(6, 1 << 30)
    small = [want(keep, 1000) for _ in range(9)]
    for b in small:
        keep.give(*b)
    assert len(gone(keep)) == 3
    p, n = want(keep, 200 << 20)
    made = keep.n_made()
    for _ in range(5):
        keep.give(p, n)
        assert want(keep, 200 << 20) == (p, n)
    assert keep.n_made() == made and len(gone(keep)) == 1


def test_sizes_that_creep_up(keep):
    """A batch a little larger each step: blocks double, so few are made."""
    keep.start(6, 1 << 30)
    held = want(keep, 1 << 20)
    for n in range(1 << 20, 5 << 20, 1 << 14):
        if held[1] < n:
            keep.give(*held)
            held = want(keep, n)
    assert keep.n_made() <= 4


def test_bytes_are_bounded(keep):
    keep.start(100, 10 << 20)
    blocks = [want(keep, 4 << 20) for _ in range(3)]
    for b in blocks:
        keep.give(*b)
    assert gone(keep) == [blocks[0][0]]         # the one kept longest
    big = want(keep, 100 << 20)
    keep.give(*big)
    assert gone(keep) == [big[0]]               # more than all may be: the others stay
    assert want(keep, 4 << 20) in blocks[1:] and want(keep, 4 << 20) in blocks[1:] and keep.n_made() == 4


def test_a_small_batch_does_not_take_a_large_block(keep):
    keep.start(6, 1 << 30)
    big = want(keep, 64 << 20)
    keep.give(*big)
    assert want(keep, 1000)[0] != big[0] and want(keep, 20 << 20)[0] == big[0]


def test_all_of_it_can_go(keep):
    keep.start(6, 1 << 30)
    blocks = [want(keep, n << 20) for n in (1, 5, 40)]
    for b in blocks:
        keep.give(*b)
    keep.let_go()
    assert sorted(gone(keep)) == sorted(b[0] for b in blocks) and not gone(keep)
    made = keep.n_made()
    assert want(keep, 1 << 20)[0] == made + 1


def test_threads(keep):
    assert keep.threads(8, 4000) == 0
