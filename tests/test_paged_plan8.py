"""The plan of a batch over caches in 8 bits, on random batches (no GPU): test_paged_plan.py's checks of every piece and join, the decode CTAs' lists, the pages that are
widened for the tensor-core kernel, the blocks that new tokens go to."""
import ctypes as C
import random
import subprocess

import numpy as np
import pytest

from test_paged_plan import CSRC, SOURCE

MORE = r"""
extern "C" {
// Null, or what is wrong with the CTAs' lists, the widened pages and the blocks of a batch. numbers: CTAs, positions of the longest list, widened pages, blocks.
const char *check8(int n_seq, const int32_t *q_len, const int32_t *kv_len, const int32_t *pages, int n_head, int n_head_kv, int hd, int page, int n_shared, int sms, long long *numbers) {
    PagedView v = {};
    v.n_head = n_head, v.n_head_kv = n_head_kv, v.group = n_head / n_head_kv, v.hd = hd, v.page = page, v.n_seq = n_seq, v.n_shared = n_shared, v.table_stride = 1;
    for (int s = 0; s < n_seq; s++) v.table_stride = std::max(v.table_stride, (kv_len[s] + page - 1) / page), v.tokens += q_len[s];
    Plan plan;
    make_plan(plan, v, q_len, kv_len, sms, true);
    const auto &begin = plan.small_begin;
    if (plan.small.empty() != begin.empty()) return wrong("small pieces without lists");
    numbers[0] = begin.empty() ? 0 : begin.size() - 1, numbers[1] = 0;
    if (!begin.empty() && (begin[0] != 0 || begin.back() != (int)plan.small.size())) return wrong("the lists' ends");
    for (size_t c = 1; c < begin.size(); c++) {
        long long n = 0;
        if (begin[c] <= begin[c - 1]) return wrong("an empty list");
        for (int i = begin[c - 1]; i < begin[c]; i++) {
            n += plan.small[i].kv_end - plan.small[i].kv_begin;
            if (plan.small[i].kv_begin % kScaleBlock) return wrong("a piece that begins inside a scale block");
        }
        numbers[1] = std::max(numbers[1], n);
    }
    std::vector<PagedItem> before = plan.large;
    std::vector<PagedWide> wide;
    std::vector<int32_t> table;
    wide_pages(wide, table, plan, v, pages, v.table_stride);
    numbers[2] = wide.size();
    std::map<int, int> times;
    for (size_t i = 0; i < plan.large.size(); i++) {
        const PagedItem &it = plan.large[i], &was = before[i];
        if (it.table - n_seq * v.table_stride != was.table || it.kv_begin != was.kv_begin || it.kv_end != was.kv_end) return wrong("a piece that is another");
        for (int pos = it.kv_begin; pos < it.kv_end; pos++) {
            const int w = table[was.table + pos / page];
            if (w < 0 || w >= (int)wide.size()) return wrong("a widened page that is not there");
            if (wide[w].page != pages[was.table + pos / page]) return wrong("another page's values");
            if (pos % page >= wide[w].valid) return wrong("a position that is not widened");
        }
    }
    for (const PagedWide &w : wide)
        if (w.valid < 1 || w.valid > page) return wrong("a page without positions");
    std::vector<PagedBlock> block;
    blocks_of(block, n_seq, q_len, kv_len);
    numbers[3] = block.size();
    size_t b = 0;
    for (int s = 0, t = 0; s < n_seq; t += q_len[s], s++)
        for (int pos = kv_len[s] - q_len[s]; pos < kv_len[s]; b++) {
            if (b >= block.size() || block[b].token != t + pos - (kv_len[s] - q_len[s])) return wrong("a token without a block");
            if (block[b].n < 1 || pos % kScaleBlock + block[b].n > kScaleBlock || pos + block[b].n > kv_len[s]) return wrong("a block that reaches into the next");
            pos += block[b].n;
            if (pos < kv_len[s] && pos % kScaleBlock) return wrong("a block that ends early");
        }
    return b == block.size() ? nullptr : wrong("blocks of no token");
}
int shared_write(int page, int n_seq, const int32_t *q_len, const int32_t *kv_len, const int32_t *pages, int stride) { return writes_shared(page, n_seq, q_len, kv_len, pages, stride); }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan8")
    assert SOURCE.count("make_plan(plan, v, q_len, kv_len, sms);") == 1
    (d / "p.cpp").write_text(SOURCE.replace("make_plan(plan, v, q_len, kv_len, sms);", "make_plan(plan, v, q_len, kv_len, sms, true);") + MORE)
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I", CSRC, str(d / "p.cpp"), "-o", str(d / "p.so")])
    lib = C.CDLL(str(d / "p.so"))
    lib.check.restype, lib.check.argtypes = C.c_char_p, [C.c_int, C.c_void_p, C.c_void_p] + [C.c_int] * 7 + [C.c_void_p]
    lib.check8.restype, lib.check8.argtypes = C.c_char_p, [C.c_int, C.c_void_p, C.c_void_p, C.c_void_p] + [C.c_int] * 6 + [C.c_void_p]
    lib.shared_write.argtypes = [C.c_int, C.c_int, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int]
    return lib


def check(lib, q, kv, n_head=32, n_head_kv=4, hd=128, page=32, n_shared=0, sms=148):
    """-> (rows of partial results, joins, small pieces, large pieces, CTAs, positions of the longest list, widened pages, blocks)"""
    q, kv, numbers, more = np.asarray(q, np.int32), np.asarray(kv, np.int32), (C.c_longlong * 4)(), (C.c_longlong * 4)()
    why = lib.check(len(q), q.ctypes.data, kv.ctypes.data, n_head, n_head_kv, hd, page, n_shared, sms, 0, numbers)
    assert why is None, (why.decode(), q.tolist(), kv.tolist(), n_head, n_head_kv, page, n_shared)
    stride = max([1] + [-(-int(m) // page) for m in kv])
    pages = np.random.default_rng(len(q)).permutation(len(q) * stride).astype(np.int32).reshape(len(q), stride)
    pages[:, :n_shared // page] = pages[:1, :n_shared // page]
    why = lib.check8(len(q), q.ctypes.data, kv.ctypes.data, pages.ctypes.data, n_head, n_head_kv, hd, page, n_shared, sms, more)
    assert why is None, (why.decode(), q.tolist(), kv.tolist(), n_head, n_head_kv, page, n_shared)
    return list(numbers) + list(more)


@pytest.mark.parametrize("seed", range(8))
def test_random_batches(lib, seed):
    r = random.Random(seed)
    for _ in range(200):
        group, heads = r.choice([1, 2, 3, 4, 5, 7, 8, 16, 33, 40, 64]), r.choice([1, 2, 3, 8, 200])
        page, n = r.choice([16, 32, 64, 256, 4096]), r.choice([1, 1, 2, 3, 9, 40])
        shared = page * r.choice([0, 0, 0, 1, 2, 300 // page])
        q, kv = [], []
        for _ in range(n):
            q.append(r.choice([0, 1, 1, 1, 2, 3, r.randint(1, 30), r.randint(1, 400)]))
            kv.append(r.choice([0, r.randint(0, 2000)]) if q[-1] == 0 else shared + q[-1] + r.choice([0, r.randint(0, 40), r.randint(0, 3000)]))
        if any(n_ and m - n_ < shared for n_, m in zip(q, kv)):
            continue
        # (tables of idle sequences may be shorter than the prefix)
        kv = [m if n_ or m <= shared else shared for n_, m in zip(q, kv)]
        check(lib, q, kv, group * heads, heads, r.choice([64, 128]), page, shared, r.choice([148, 148, 132, 16]))


def test_lists_are_even(lib):
    """Sequences of very different lengths: no CTA has much more than its share, and no more CTAs than run at once."""
    r = random.Random(3)
    for _ in range(20):
        kv = [r.randint(150, 8000) for _ in range(32)]
        numbers = check(lib, [1] * 32, kv)
        if numbers[4] <= 74:  # cut
            assert numbers[5] <= 1.15 * sum(kv) / 74 + 200


def test_short_sequences_are_not_cut(lib):
    assert check(lib, [1] * 64, [512] * 64)[:3] == [0, 0, 64]


def test_a_shared_prefix_is_widened_once(lib):
    rows = check(lib, [40] * 6 + [1], [4096 + 40] * 6 + [4097], n_shared=4096)
    assert 4096 // 32 <= rows[6] <= 4096 // 32 + 7 * 2


def test_long_sequences(lib):
    q, kv = np.array([1] * 500, np.int32), np.array([1 << 30] * 500, np.int32)
    numbers = (C.c_longlong * 4)()
    assert lib.check(500, q.ctypes.data, kv.ctypes.data, 8, 8, 128, 4096, 0, 148, 0, numbers) is None


def test_pages_that_two_write(lib):
    a = lambda x: np.asarray(x, np.int32)  # noqa: E731

    def two(q, kv, pages, page=16):
        q, kv, pages = a(q), a(kv), a(pages)
        return bool(lib.shared_write(page, len(q), q.ctypes.data, kv.ctypes.data, pages.ctypes.data, pages.shape[1]))

    assert two([1, 1], [5, 6], [[3], [3]]) and two([20], [20], [[1, 1]]) and two([1, 3], [17, 18], [[0, 4], [4, 0]])
    assert not two([1, 1], [17, 17], [[0, 1], [0, 2]])      # a prefix in common
    assert not two([1, 0], [5, 6], [[3], [3]]) and not two([0, 0], [0, 5], [[3], [3]])
