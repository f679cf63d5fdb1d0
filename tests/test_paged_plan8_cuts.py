"""How runs of positions over a cache in 8 bits are dealt to the decode kernel's CTAs (csrc/paged_plan.h): every position once, no list longer than its share by more than a step, and no
piece shorter than the header says (no GPU)."""
import ctypes as C
import random
import subprocess

import numpy as np
import pytest

from test_paged_plan import CSRC

SOURCE = r"""
#include "paged_plan.h"
using namespace llamd;
extern "C" int deal(int n, const int32_t *positions, int ctas, long long share, int32_t *out, int room, long long *used) {
    std::vector<Run> runs;
    for (int i = 0; i < n; i++) runs.push_back({positions[i]});
    std::vector<RunCut> cuts;
    const int c = share ? deal_runs(runs, share, cuts) : deal_runs_evenly(runs, ctas, cuts, share);
    *used = share;
    if ((int)cuts.size() > room) return -1;
    for (size_t i = 0; i < cuts.size(); i++) out[4 * i] = cuts[i].run, out[4 * i + 1] = cuts[i].first, out[4 * i + 2] = cuts[i].n, out[4 * i + 3] = cuts[i].cta;
    out[4 * cuts.size()] = -1;
    return c;
}
extern "C" int numbers(int i) { const int n[] = {kDecode8Piece, kDecode8Least}; return n[i]; }
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("cuts")
    (d / "p.cpp").write_text(SOURCE)
    subprocess.check_call(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I", CSRC, str(d / "p.cpp"), "-o", str(d / "p.so")])
    lib = C.CDLL(str(d / "p.so"))
    lib.deal.argtypes = [C.c_int, C.c_void_p, C.c_int, C.c_longlong, C.c_void_p, C.c_int, C.c_void_p]
    return lib


def check(lib, runs, ctas=0, share=0):
    runs, room, used = np.asarray(runs, np.int32), 200000, C.c_longlong()
    out = np.zeros(4 * room + 4, np.int32)
    n = lib.deal(len(runs), runs.ctypes.data, ctas, share, out.ctypes.data, room, C.byref(used))
    cuts = out[:4 * room].reshape(-1, 4)
    cuts = cuts[:int(np.flatnonzero(out[::4] == -1)[0])]
    piece, share = lib.numbers(0), used.value
    assert n == cuts[-1, 3] + 1 and np.all(np.isin(np.diff(cuts[:, 3]), (0, 1))) and cuts[0, 3] == 0
    at = {}
    for run, first, m, _ in cuts:
        assert first == at.get(run, 0) and m > 0
        at[run] = first + m
        whole, last = m == runs[run], first + m == runs[run]
        assert whole or m >= (32 if last else 64) and (last or m % 32 == 0)
    assert at == dict(enumerate(runs))
    for c in range(n):
        assert sum(m + piece for m in cuts[cuts[:, 3] == c, 2]) <= share + 32 + piece
    return n, share


@pytest.mark.parametrize("seed", range(6))
def test_random_runs(lib, seed):
    r = random.Random(seed)
    for _ in range(120):
        runs = [r.choice([1, r.randint(1, 40), r.randint(1, 300), r.randint(1, 9000)]) for _ in range(r.choice([1, 2, 9, 200]))]
        check(lib, runs, share=r.randint(lib.numbers(0) + lib.numbers(1), 2000))
        ctas = r.choice([1, 2, 18, 74, 296])
        n, share = check(lib, runs, ctas)
        assert n <= ctas and share >= lib.numbers(0) + lib.numbers(1)
