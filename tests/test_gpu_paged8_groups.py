"""Attention over caches in 8 bits with 17 to 32 query heads to a kv head: pieces of three and four groups of 8 query rows, whole and cut, with and without a shared prefix."""
import pytest

from test_gpu_paged import close
from test_gpu_paged8 import run_attention8
from test_gpu_paged8_accuracy import FEW, compare, far_apart

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def paged():
    from llamd_rs_b200 import backend, paged as p

    backend.stream_init()
    return p


BATCHES = [
    # q_len, kv_len, n_shared
    ([1], [1], 0),
    ([1, 1, 1], [31, 32, 33], 0),
    ([1], [3003], 0),                                             # cut
    ([1] * 3, [1500 + 37 * i for i in range(3)], 0),              # cut, lists of several pieces
    ([1] * 40, [20 + 3 * i for i in range(40)], 0),               # whole
    ([1, 2, 0, 3], [150, 90, 7, 230], 0),
    ([1, 1, 2], [65, 100, 200], 64),
    ([1] * 36, [801 + i for i in range(36)], 800),                # the prefix by the kernel of many rows
]


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("group", [17, 24, 32])
def test_wide_groups(paged, group, D, dtype, cache):
    for i, (q_len, kv_len, n_shared) in enumerate(BATCHES):
        close(*run_attention8(paged, cache, 2 * group, 2, D, 16 << i % 2 if not n_shared else 16, dtype, q_len, kv_len, n_shared, out_f32=i % 3 == 1))
    close(*run_attention8(paged, cache, group, 1, D, 16, dtype, [1, 1], [700, 20], 0, pad=8, shift=8))
    compare(paged, cache, group, 1, D, dtype, [1, 1], [400, 70], far_apart(cache, dtype, 5.0), FEW[cache])
