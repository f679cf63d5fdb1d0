"""The host side of sampling and of caches in 8 bits, without a device: what is refused before any launch."""

import numpy as np
import pytest


@pytest.fixture(scope="module")
def built():
    import __graft_entry__ as g

    g.build()
    from llamd_rs_b200 import backend, paged, sampling

    return backend, paged, sampling


def test_tensors_that_are_not_on_a_device(built):
    backend, _, sampling = built
    torch = pytest.importorskip("torch")
    x, u, t = torch.zeros(2, 10), torch.zeros(2), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(backend.ShapeError):
        sampling.sample(x, u, t)
    with pytest.raises(backend.Unsupported):
        sampling.sample(x.double(), u, t)


def test_numbers(built):
    backend, _, sampling = built
    for kw in (dict(rows=-1, n_vocab=5), dict(rows=2 ** 31, n_vocab=5), dict(rows=1.5, n_vocab=5), dict(rows=1), dict(n_vocab=5), dict(rows=1, n_vocab=5, stride=2 ** 40)):
        with pytest.raises(backend.Malformed):
            sampling.sample(1 << 20, 1 << 20, 1 << 20, **kw)
    with pytest.raises(backend.Malformed):
        sampling.sample(1 << 20, None, 1 << 20, rows=1, n_vocab=5)
    with pytest.raises(backend.ShapeError):
        sampling.sample(1 << 20, 1 << 20, 1 << 20, rows=2, n_vocab=5, stride=4)
    with pytest.raises(backend.Unsupported):
        sampling.sample(1 << 20, 1 << 20, 1 << 20, rows=2, n_vocab=5, dtype="e4m3")


def test_scales_of_a_batch(built):
    backend, paged, _ = built
    b = paged.Batch.__new__(paged.Batch)
    b.ptr, b.type, b.cache, b._pool, b.head_dim = None, 0, 3, 4 * 2 * 16 * 64, 64
    with pytest.raises(backend.Malformed):
        b._scales_of(None, 1 << 20)
    assert b._scales_of(1 << 20, 1 << 21) == (1 << 20, 1 << 21)
    b.cache = 0
    assert b._scales_of(None, None) == ()
    with pytest.raises(backend.Malformed):
        b._scales_of(1 << 20, 1 << 20)


class OnDevice:
    """As much of a tensor as is looked at before an address is taken."""

    is_cuda = True

    def __init__(self, x, device):
        self.x, self.device = x, device

    def get_device(self):
        return self.device

    def __getattr__(self, name):
        return getattr(self.x, name)


def test_one_device(built):
    """Tensors of two devices, or of one that is not the current one, are refused before anything is enqueued."""
    backend, paged, sampling = built
    torch = pytest.importorskip("torch")
    f, i = (lambda n, d: OnDevice(torch.zeros(n), d)), (lambda n, d: OnDevice(torch.zeros(n, dtype=torch.int32), d))
    rows = OnDevice(torch.zeros(2, 10), 0)
    for kw in (dict(uniform=f(2, 1), token=i(2, 0)), dict(uniform=f(2, 0), token=i(2, 1)), dict(uniform=f(2, 0), token=i(2, 0), top_k=i(2, 1)),
               dict(uniform=f(2, 0), token=i(2, 0), prob=f(2, 1))):
        with pytest.raises(backend.ShapeError, match="devices 0 and 1"):
            sampling.sample(rows, **kw)
    b = paged.Batch.__new__(paged.Batch)
    b.ptr, b.type, b.cache, b._pool, b.head_dim = None, 0, 3, 4 * 2 * 16 * 64, 64
    scales = lambda d: OnDevice(torch.zeros(4, 2, 1, dtype=torch.uint8), d)  # noqa: E731
    b.tokens, b.n_head, b.n_head_kv, b.scale = 1, 8, 2, 0.125
    b._wait = b._ready = b._attention = b._append = None  # (nothing is called)
    codes = lambda d: OnDevice(torch.zeros(b._pool, dtype=torch.int8), d)  # noqa: E731
    paged._type_of(codes(0)), paged._type_of(scales(0))
    wanted = lambda d: ((codes(0), 3, b._pool, None), (codes(d), 3, b._pool, None))  # noqa: E731
    assert len(paged.Batch._tensors(*wanted(0))) == 2 and paged.Batch._tensors(*wanted(1)) is None
    for d in range(1, 64):
        q, kp, vp, out, ks, vs = (make(d >> i & 1) for i, make in enumerate((lambda d: OnDevice(torch.zeros(1, 512, dtype=torch.float16), d), codes, codes,
                                                                             lambda d: OnDevice(torch.zeros(1, 512), d), scales, scales)))
        if d < 63:
            with pytest.raises(backend.ShapeError, match="devices [01] and [01]"):
                b.attention(q, kp, vp, out, k_scales=ks, v_scales=vs)
        if d & 55 not in (0, 55):  # (all but `out`)
            with pytest.raises(backend.ShapeError, match="devices [01] and [01]"):
                b.append(q, q, q, q, kp, vp, k_scales=ks, v_scales=vs, inputs="f16")
    paged._one_device(None, 1 << 20)  # (addresses are the caller's word)


def test_current_device(built, monkeypatch):
    backend, paged, _ = built
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    paged._one_device(OnDevice(torch.zeros(2), 0))
    with pytest.raises(backend.ShapeError, match="device 1 where 0"):
        paged._one_device(OnDevice(torch.zeros(2), 1), OnDevice(torch.zeros(2), 1))


def test_refused_without_a_device(built):
    backend, paged, _ = built
    if backend.available():
        pytest.skip("a device is present")
    with pytest.raises(backend.Unsupported):
        paged.Batch(8, 2, 64, 16, cache="e4m3")
    from llamd_rs_b200._lib import lib

    assert lib().llamd_fwd_sample(None, 2, 10, 1, 10, None, None, None, None, None, None, None) == -1
    assert lib().llamd_cuda_paged_new8(8, 2, 64, 16, 0, 7) is None
    lib().llamd_fwd_last_error()


def test_plain_forms_agree():
    """The definition that the GPU tests compare with, against frequencies counted another way."""
    import sample_plain

    rng = np.random.default_rng(0)
    x = rng.standard_normal(12) * 2
    kept = [i for i in np.argsort(-x)[:7]]
    w = np.exp((x - x.max()) / 0.9)
    order, total = sorted(kept, key=lambda i: -w[i]), sum(w[i] for i in kept)
    nucleus, before = [], 0.0
    for i in order:
        if before < 0.8 * total:
            nucleus.append(i)
        before += w[i]
    nucleus = [i for i in nucleus if w[i] >= 0.1]
    share = {int(i): w[i] / sum(w[j] for j in nucleus) for i in nucleus}
    drawn = [sample_plain.sample(x.astype(np.float64), u, 0.9, 7, 0.8, 0.1)[0] for u in (np.arange(2000) + 0.5) / 2000]
    assert set(drawn) == set(share) and all(abs(drawn.count(i) / 2000 - share[i]) < 1e-3 for i in share)
