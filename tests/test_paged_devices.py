"""Tensors that are not all on the current device, given to the calls over 16-bit caches: refused before anything is enqueued, as over those in 8 bits (no GPU)."""
import pytest

from test_sampling_host import OnDevice, built  # noqa: F401  (built: the fixture)


def batch(paged):
    b = paged.Batch.__new__(paged.Batch)
    b.ptr, b.type, b.cache, b.head_dim, b.tokens, b.n_head, b.n_head_kv, b.scale = None, 0, 0, 64, 1, 8, 2, 0.125
    b._pool = 4 * 2 * 16 * 64

    def never(*args):
        raise AssertionError("enqueued")

    b._wait = b._ready = b._attention = b._append = never
    return b


def halves(n, device, rows=1):
    import torch

    return OnDevice(torch.zeros(rows, n // rows, dtype=torch.float16), device)


@pytest.mark.parametrize("whole", [True, False])
def test_two_devices(built, whole):  # noqa: F811
    """Of one call's tensors each may be the one that is elsewhere; rows that follow one another, and rows that do not (looked at one by one)."""
    backend, paged, _ = built
    pytest.importorskip("torch")
    b = batch(paged)
    rows = (lambda n, d: halves(n, d)) if whole else (lambda n, d: OnDevice(halves(2 * n, d).x[:, :n], d))
    for d in range(1, 15):
        q, kp, vp, out = (x(n, d >> i & 1) for i, (x, n) in enumerate(((rows, 512), (halves, b._pool), (halves, b._pool), (rows, 512))))
        with pytest.raises(backend.ShapeError, match="devices [01] and [01]"):
            b.attention(q, kp, vp, out)
    for d in range(1, 63):
        q, k, v, out, kp, vp = (x(n, d >> i & 1) for i, (x, n) in enumerate(((rows, 512), (rows, 128), (rows, 128), (rows, 512), (halves, b._pool), (halves, b._pool))))
        with pytest.raises(backend.ShapeError, match="devices [01] and [01]"):
            b.append(q, k, v, out, kp, vp)


def test_another_device(built, monkeypatch):  # noqa: F811
    """All on one device, which is not the current one: with norms and angles (looked at all at once) and without."""
    backend, paged, _ = built
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    b, f = batch(paged), lambda *shape: OnDevice(torch.zeros(*shape), 1)
    q, k, out, pool = halves(512, 1), halves(128, 1), halves(512, 1), halves(b._pool, 1)
    for x in (q, f(64)):
        paged._type_of(x)
    for call in (lambda: b.attention(q, pool, pool, out), lambda: b.append(q, k, k, out, pool, pool),
                 lambda: b.append(q, k, k, out, pool, pool, rope=f(9, 64), rot=64, q_norm=f(64), k_norm=f(64))):
        with pytest.raises(backend.ShapeError, match="device 1 where 0"):
            call()
