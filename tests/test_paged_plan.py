"""How attention over paged caches is cut into pieces (csrc/paged_plan.h), as the kernels read it: on random batches, no GPU is needed."""
import ctypes as C
import os
import random
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llamd_rs_b200", "csrc")
SOURCE = r"""
#include <map>
#include <string>
#include <tuple>
#include "paged_plan.h"
using namespace llamd;
static std::string why;
static const char *wrong(const std::string &s) { why = s; return why.c_str(); }
struct Seen { int begin, end, row; };  // positions, and the row its result goes to (-1: out)
extern "C" {
// The plan of a batch: null, or what is wrong with it. numbers: rows of partial results, joined (token, head)s, pieces of either kernel.
const char *check(int n_seq, const int32_t *q_len, const int32_t *kv_len, int n_head, int n_head_kv, int hd, int page, int n_shared, int sms, int plant,
                  long long *numbers) {
    PagedView v = {};
    v.n_head = n_head, v.n_head_kv = n_head_kv, v.group = n_head / n_head_kv, v.hd = hd, v.page = page, v.n_seq = n_seq, v.n_shared = n_shared, v.table_stride = 1;
    std::vector<int> seq, pos;
    int lead = -1;
    for (int s = 0; s < n_seq; s++) {
        v.table_stride = std::max(v.table_stride, (kv_len[s] + page - 1) / page);
        if (q_len[s] && lead < 0) lead = s;
        for (int i = 0; i < q_len[s]; i++) seq.push_back(s), pos.push_back(kv_len[s] - q_len[s] + i);
    }
    v.tokens = (int)seq.size();
    Plan plan;
    make_plan(plan, v, q_len, kv_len, sms);
    if (plant == 1) (plan.small.empty() ? plan.large : plan.small)[0].kv_begin += 128;
    if (plant == 2) plan.part.back().row += v.group;
    if (plant == 3) plan.merge.pop_back();
    if (plant == 4) plan.large.back().part -= 1;
    numbers[0] = plan.rows, numbers[1] = plan.merge.size(), numbers[2] = plan.small.size(), numbers[3] = plan.large.size();
    const int G = v.group, K = n_head_kv;
    std::vector<std::vector<Seen>> seen((size_t)v.tokens * K);
    std::vector<char> used(plan.rows, 0);
    auto piece = [&](const PagedItem &it, int head, int row0) -> const char * {
        if (it.kv_begin >= it.kv_end || it.n_tok < 1) return wrong("an empty piece");
        for (int i = 0; i < it.n_tok; i++) {
            const int t = it.token + i, s = it.table / v.table_stride;
            if (t >= v.tokens || it.table % v.table_stride) return wrong("a token or table that is not there");
            if (s != seq[t] && !(s == lead && it.kv_end <= n_shared)) return wrong("another sequence's positions");
            if ((it.kv_end + page - 1) / page > v.table_stride || it.kv_end > kv_len[s]) return wrong("positions behind the end");
            const int end = std::min(it.kv_end, it.limit + i * it.step);
            for (int g = 0; g < G && row0 >= 0; g++) {
                const size_t r = (size_t)row0 + i * G + g;
                if (r >= used.size()) return wrong("a row outside the partial results");
                if (used[r]++) return wrong("a row that two pieces write");
            }
            seen[(size_t)t * K + head].push_back({it.kv_begin, std::max(end, it.kv_begin), row0 < 0 ? -1 : row0 + i * G});
        }
        return nullptr;
    };
    int longest = 0;
    for (const PagedItem &it : plan.small) {
        if (it.n_tok * G > kPagedSmallRows || it.n_tok * G > plan.small_rows) return wrong("too many rows for the decode kernel");
        if (it.kv_begin % 16) return wrong("a slice across pages");
        if (it.part >= 0 && it.part_rows != it.n_tok * G) return wrong("rows between heads");
        for (int h = 0; h < K; h++)
            if (const char *e = piece(it, h, it.part < 0 ? -1 : it.part + h * it.part_rows)) return e;
        longest = std::max(longest, it.kv_end - it.kv_begin);
    }
    if (plan.begin.empty() || plan.begin[0] != 0 || plan.begin.back() != (int)plan.large.size() || (int)plan.begin.size() - 1 > sms) return wrong("the CTAs' lists");
    for (size_t c = 1; c < plan.begin.size(); c++)
        if (plan.begin[c] < plan.begin[c - 1]) return wrong("the CTAs' lists");
    for (const PagedItem &it : plan.large) {
        if (it.n_tok > 2 * (kPagedTileRows / G)) return wrong("too many tokens for two tiles");
        if (it.kv_begin % std::min(page, kPagedBlock)) return wrong("a box across pages");
        if (it.head < 0 || it.head >= K) return wrong("a head that is not there");
        if (const char *e = piece(it, it.head, it.part < 0 ? -1 : it.part)) return e;
    }
    std::map<std::pair<int, int>, const PagedMerge *> joins;
    for (const PagedMerge &m : plan.merge) {
        if (m.count < 1 || m.begin < 0 || m.begin + m.count > (int)plan.part.size() || m.count > plan.most) return wrong("a join's list");
        if (!joins.insert({{m.token, m.head}, &m}).second) return wrong("a token and head joined twice");
    }
    for (int t = 0; t < v.tokens; t++)
        for (int h = 0; h < K; h++) {
            auto &s = seen[(size_t)t * K + h];
            const auto j = joins.find({t, h});
            if (s.size() == 1 && s[0].row < 0) {
                if (j != joins.end()) return wrong("a row that is out is joined");
            } else {
                if (j == joins.end()) return wrong("parts that nobody joins");
                std::map<int, int> rows;
                for (const Seen &x : s) {
                    if (x.row < 0) return wrong("a piece writes out beside others");
                    rows[x.row]++;
                }
                for (int i = 0; i < j->second->count; i++) {
                    const PagedPart &p = plan.part[j->second->begin + i];
                    if (--rows[p.row + (t - p.token) * G]) return wrong("a part joined twice, or not the row's own");
                }
                for (const auto &r : rows)
                    if (r.second) return wrong("a part left out");
            }
            std::sort(s.begin(), s.end(), [](const Seen &a, const Seen &b) { return std::make_pair(a.begin, a.end) < std::make_pair(b.begin, b.end); });
            int at = 0;
            for (const Seen &x : s) {
                if (x.end == x.begin) continue;  // (cut by the causal limit: nothing)
                if (x.begin != at) return wrong("positions left out or seen twice");
                at = x.end;
            }
            if (at != pos[t] + 1) return wrong("not up to the token's own position");
        }
    return nullptr;
}
}
"""


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "p.cpp").write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I", CSRC, str(d / "p.cpp"), "-o", str(d / "p.so")])
    f = C.CDLL(str(d / "p.so")).check
    f.restype, f.argtypes = C.c_char_p, [C.c_int, C.c_void_p, C.c_void_p] + [C.c_int] * 7 + [C.c_void_p]

    def run(q, kv, n_head=32, n_head_kv=4, hd=128, page=32, n_shared=0, sms=148, plant=0):
        q, kv, numbers = np.asarray(q, np.int32), np.asarray(kv, np.int32), (C.c_longlong * 4)()
        why = f(len(q), q.ctypes.data, kv.ctypes.data, n_head, n_head_kv, hd, page, n_shared, sms, plant, numbers)
        assert why is None, (why.decode(), q.tolist(), kv.tolist(), n_head, n_head_kv, page, n_shared)
        return list(numbers)  # rows of partial results, joins, pieces for the decode kernel, for the prompt kernel

    return run


@pytest.mark.parametrize("seed", range(8))
def test_every_position_once_and_every_part_joined(check, seed):
    r = random.Random(seed)
    for _ in range(250):
        group, heads = r.choice([1, 2, 3, 4, 5, 7, 8, 16, 33, 40, 64]), r.choice([1, 2, 3, 8])
        page, n = r.choice([16, 32, 64, 256, 4096]), r.choice([1, 1, 2, 3, 9, 40])
        shared = page * r.choice([0, 0, 0, 1, 2, 300 // page])
        q, kv = [], []
        for _ in range(n):
            q.append(r.choice([0, 1, 1, 1, 2, 3, r.randint(1, 30), r.randint(1, 400)]))
            idle = q[-1] == 0
            kv.append(r.choice([0, r.randint(0, 2000)]) if idle else shared + q[-1] + r.choice([0, r.randint(0, 40), r.randint(0, 3000)]))
        check(q, kv, group * heads, heads, r.choice([64, 128]), page, shared, r.choice([148, 148, 132, 16]))


@pytest.mark.parametrize("n,tokens,shared", [(16, 2048, 4096), (32, 200, 1024), (4, 1000, 2048), (1, 2000, 2048), (1, 8192, 16), (8, 1000, 1024), (1, 1, 1024)])
def test_prompts_behind_a_prefix_need_no_more_room_than_without(check, n, tokens, shared):
    """Long prompts save nothing by reading the prefix once for all, and one sequence has nobody to share with: planned as if there were no prefix."""
    q, kv = [tokens] * n, [shared + tokens] * n
    assert check(q, kv, n_shared=shared) == check(q, kv)


def test_few_tokens_read_the_prefix_once(check):
    for q in ([1] * 64, [31] * 16, [512] + [1] * 100):
        kv = [4096 + n for n in q]
        assert check(q, kv, n_shared=4096)[0] >= 2 * 32 * sum(q) and check(q, kv, n_shared=4096) != check(q, kv)


def test_as_long_as_sequences_may_be(check):
    """An even share of the positions that is more than 32 bits hold."""
    check([1] * 500, [1 << 30] * 500, 8, 8, page=4096)
    check([1, 40], [1 << 30] * 2, 8, 8, page=4096, n_shared=1 << 29)


@pytest.mark.parametrize("plant", [1, 2, 3, 4])
def test_the_checks_find_a_wrong_plan(check, plant):
    check([1] * 30, [3000 + i for i in range(30)], n_shared=2048)
    with pytest.raises(AssertionError):
        check([1] * 30, [3000 + i for i in range(30)], n_shared=2048, plant=plant)
