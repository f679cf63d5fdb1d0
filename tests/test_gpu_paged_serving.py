"""examples/paged_serving.py on small sizes: attention layers over paged caches against the same layers on the exact ops."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("paged_serving", os.path.join(ROOT, "examples", "paged_serving.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.backend.stream_init()
    return m


# One layer: the paged path differs by the rounding of q, k, v and the softmax's weights to 11 bits, each at most 2^-11 relative, and the Q8_K form of
# its output then steps by up to 1/127 of a block's largest value where a value lies at a rounding's edge: a few such of 256 are well within 1e-2.
@pytest.mark.parametrize("conversations,system,steps,page", [(3, 64, 3, 16), (1, 0, 2, 32), (9, 192, 2, 64)])
def test_one_layer_against_the_exact_ops(example, conversations, system, steps, page):
    hp = dict(n_embd=512, n_head=8, n_head_kv=2, head_dim=128)
    far = example.serve(hp, 1, conversations, system, steps, page, check=True, say=lambda *a: None)
    assert far < 1e-2


def test_layers(example):
    """Several layers deep nothing but the sizes is new: finite, and pages all given back."""
    hp = dict(n_embd=256, n_head=4, n_head_kv=4, head_dim=64)
    lines = []
    assert example.serve(hp, 3, 5, 48, 4, 16, check=False, say=lines.append) is None
    assert len(lines) == 6
