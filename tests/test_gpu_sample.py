"""Sampling on the GPU against its definition (sample_plain.py): the same token, and its share to f32's rounding."""
import numpy as np
import pytest

import paged_plain as bits
import sample_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def sampling():
    from llamd_rs_b200 import backend, sampling as s

    backend.stream_init()
    return s


def dev(a):
    from llamd_rs_b200.backend import DevBuf

    return DevBuf.from_array(a)


def run(sampling, x, u, dtype="f32", pad=0, shift=0, **settings):
    """x f32 [rows][n] whose values `dtype` holds exactly -> (tokens, shares)."""
    from llamd_rs_b200 import backend

    rows, n = x.shape
    wide = np.full((rows, n + pad), 7.0, np.float32)  # (what lies between the rows is above them)
    wide[:, :n] = x
    raw = wide.ravel() if dtype == "f32" else bits.to_bits(wide.ravel(), dtype)
    raw = np.concatenate([np.zeros(shift, raw.dtype), raw])
    logits = dev(raw)
    token, prob = dev(np.full(rows + 2, -7, np.int32)), dev(np.full(rows + 2, -7, np.float32))
    keep = {k: dev(np.ascontiguousarray(np.broadcast_to(np.asarray(v, np.int32 if k == "top_k" else np.float32), (rows,)))) for k, v in settings.items()}
    du = dev(np.asarray(u, np.float32))
    at = {k: v.ptr for k, v in keep.items()}
    sampling.sample(logits.ptr + shift * raw.itemsize, du, token, prob=prob, rows=rows, n_vocab=n, dtype=dtype, stride=n + pad, **at)
    backend.sync()
    t, s = token.download(np.int32, rows + 2), prob.download(np.float32, rows + 2)
    assert np.all(t[rows:] == -7) and np.all(s[rows:] == -7)
    return t[:rows], s[:rows]


def check(sampling, x, u, dtype="f32", **more):
    if dtype != "f32":
        x = bits.from_bits(bits.to_bits(x, dtype), dtype).astype(np.float32)
    got, share = run(sampling, x, u, dtype, **more)
    settings = {k: np.broadcast_to(np.asarray(v), (len(x),)) for k, v in more.items() if k in ("temperature", "top_k", "top_p", "min_p")}
    for r in range(len(x)):
        want, s = plain.sample(x[r], u[r], **{k: v[r] for k, v in settings.items()})
        assert got[r] == want, (r, got[r], want, {k: v[r] for k, v in settings.items()}, u[r])
        assert abs(share[r] - s) <= 2.0 ** -23 * s + 2.0 ** -39  # (a rounding to f32; a weight's last unit)
    return got


def logits(rng, rows, n, spread=2.0, boosted=40):
    x = (spread * rng.standard_normal((rows, n))).astype(np.float32)
    for r in range(rows):
        x[r, rng.integers(0, n, boosted)] += (2 * spread * rng.exponential(size=boosted)).astype(np.float32)
    return x


RULES = [dict(), dict(temperature=0.7, top_k=20, top_p=0.8), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=1), dict(top_k=3000, top_p=0.99, min_p=0.001, temperature=1.3),
         dict(top_p=0.5, min_p=0.02, temperature=2.5), dict(top_k=5000), dict(temperature=0.0), dict(top_p=0.0), dict(top_p=0.9999, temperature=3.0)]


@pytest.mark.parametrize("rule", range(len(RULES)))
@pytest.mark.parametrize("n", [1, 2, 5, 31, 300, 1024, 1025, 8192, 8193, 20001, 65537, 151936])
def test_rules(sampling, n, rule):
    rng = np.random.default_rng(n + rule)
    rows = 9
    check(sampling, logits(rng, rows, n), rng.random(rows), **RULES[rule])


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 0), (64, 1), (8, 3), (0, 5)])
@pytest.mark.parametrize("n", [7, 1000, 50257])
def test_types_and_strides(sampling, dtype, pad, shift, n):
    """16-bit logits, of which many are alike; rows that start anywhere."""
    rng = np.random.default_rng(n + pad)
    x = logits(rng, 6, n, spread=1.0)
    for rule in RULES[:6]:
        check(sampling, x, rng.random(6), dtype, pad=pad, shift=shift, **rule)
    check(sampling, x, rng.random(6), "f32", pad=pad, shift=shift, **RULES[5])


def test_each_row_its_own(sampling):
    rng = np.random.default_rng(5)
    rows, n = 64, 32003
    x = logits(rng, rows, n)
    x[rng.random(x.shape) < 0.3] = -np.inf
    x[11] = -np.inf
    x[12], x[12, 0] = -np.inf, 1.0
    got = check(sampling, x, rng.random(rows), temperature=rng.choice([0.0, 0.3, 1.0, 2.0], rows), top_k=rng.choice([-3, 0, 1, 2, 40, 1024, 1025, 6000, 10 ** 9], rows),
                top_p=rng.choice([-1.0, 0.0, 0.1, 0.6, 0.95, 1.0, 2.0], rows), min_p=rng.choice([-1.0, 0.0, 0.01, 0.5, 1.0], rows))
    assert got[11] == -1 and got[12] == 0


@pytest.mark.parametrize("n", [6, 1024, 4000, 100003])
def test_alike(sampling, n):
    """Logits that are all alike, or of two, three and nine kinds: ties go by index, and shares end inside them."""
    rng = np.random.default_rng(n)
    for kinds in (1, 2, 3, 9):
        x = rng.integers(0, kinds, (8, n)).astype(np.float32)
        for rule in (dict(), dict(top_k=2), dict(top_k=n // 2 + 1), dict(top_p=0.5), dict(top_p=0.25, top_k=n // 2 + 2), dict(top_p=0.125, min_p=0.5), dict(min_p=1.0)):
            check(sampling, x, rng.random(8), **rule)


def test_masked_rows(sampling):
    """One token left, few, none; the type's lowest value as a mask; infinities and NaN."""
    rng = np.random.default_rng(2)
    n = 20000
    for fill in (-np.inf, np.finfo(np.float32).min, np.nan):
        x = logits(rng, 12, n)
        for r, left in enumerate((0, 1, 2, 3, 50, 1500, 1, 2, 30, 1024, 1025, 2000)):
            x[r, rng.permutation(n)[left:]] = fill
        for rule in (dict(), dict(top_k=40, top_p=0.9), dict(top_p=0.95), dict(min_p=0.1), dict(temperature=0.0), dict(top_k=1500)):
            got = check(sampling, x, rng.random(12), **rule)
            assert fill == np.finfo(np.float32).min or got[0] == -1
    x = logits(rng, 4, n)
    x[0, 777] = np.inf
    x[1, [5, 99, 19999]] = np.inf
    x[2], x[2, 3] = -np.inf, 3e38
    x[3, 0], x[3, 1] = 3e38, -3e38
    for rule in RULES:
        got = check(sampling, x, [0.5, 0.5, 0.5, 0.5], **rule)
        assert got[0] == 777 and got[1] in (5, 99) and got[2] == 3 and got[3] == 0


@pytest.mark.parametrize("u", [0.0, 1e-30, 2.0 ** -24, 0.25, 1 - 2.0 ** -24, 1.0, 5.0, -1.0, np.nan])
def test_numbers_at_the_ends(sampling, u):
    rng = np.random.default_rng(3)
    x = logits(rng, 3, 9000)
    for rule in (dict(), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.1)):
        check(sampling, x, [0.0 if np.isnan(u) else u] * 3, **rule)
    assert np.array_equal(run(sampling, x, [u] * 3)[0], run(sampling, x, [0.0 if not u > 0 else min(u, 1 - 2.0 ** -24)] * 3)[0])


def test_finite_masks(sampling):
    """Masks that are numbers: most of a row far below the rest, all of it, and rows whose own logits are that low."""
    rng = np.random.default_rng(13)
    n = 40000
    for mask in (-1e4, -65504.0, -1e9, -3e38):
        x = logits(rng, 5, n)
        x[:, rng.random(n) < 0.9] = mask
        x[3] = mask
        x[4] = x[4] + np.float32(-2e4)
        for rule in (dict(), dict(top_k=20, top_p=0.9), dict(top_k=3000), dict(top_p=0.95), dict(min_p=0.1)):
            check(sampling, x, rng.random(5), **rule)
            if mask == -65504.0:
                check(sampling, np.maximum(x, mask), rng.random(5), "f16", **rule)


def test_answers_over_settings(sampling):
    """Tokens written where k was, shares where the temperature was: each row's settings have been read by then."""
    from llamd_rs_b200 import backend

    rng = np.random.default_rng(14)
    rows, n = 24, 50000
    x, u, t = logits(rng, rows, n), rng.random(rows).astype(np.float32), rng.choice([0.0, 0.7, 1.5], rows).astype(np.float32)
    k = rng.choice([0, 1, 30, 2000], rows).astype(np.int32)
    dx, du, dt, dk = dev(x), dev(u), dev(t), dev(k)
    sampling.sample(dx, du, dk, temperature=dt, top_k=dk, prob=dt, rows=rows, n_vocab=n)
    backend.sync()
    want = [plain.sample(x[r], u[r], t[r], k[r])[0] for r in range(rows)]
    assert dk.download(np.int32, rows).tolist() == want


def test_settings_beyond_their_ranges(sampling):
    rng = np.random.default_rng(12)
    x, u = logits(rng, 6, 5000), rng.random(6)
    for got, as_if in ((dict(min_p=7.0), dict(min_p=1.0)), (dict(min_p=np.nan), dict()), (dict(top_p=np.nan), dict()), (dict(top_p=9.0), dict()), (dict(top_p=-2.0), dict(top_p=0.0)),
                       (dict(temperature=np.nan), dict(temperature=0.0)), (dict(temperature=-3.0), dict(temperature=0.0)), (dict(top_k=-5), dict()), (dict(min_p=-1.0), dict())):
        assert np.array_equal(run(sampling, x, u, **got)[0], run(sampling, x, u, **as_if)[0])


@pytest.mark.parametrize("rows", [1, 2, 18, 19, 37, 75, 149, 300])
@pytest.mark.parametrize("n", [3000, 40001])
def test_rows(sampling, rows, n):
    """Clusters of every size, rows kept in shared memory and read again."""
    rng = np.random.default_rng(rows + n)
    x = logits(rng, rows, n, spread=1.0)
    for rule in (RULES[1], RULES[2], RULES[3], RULES[5], RULES[10]):
        check(sampling, x, rng.random(rows), **rule)


@pytest.mark.parametrize("temperature", [1e-45, 1e-30, 1e-4, 50.0, 1e30, np.inf])
def test_temperatures(sampling, temperature):
    rng = np.random.default_rng(4)
    x = logits(rng, 5, 12345)
    for rule in (dict(), dict(top_k=50), dict(top_p=0.9), dict(min_p=0.1)):
        check(sampling, x, rng.random(5), temperature=temperature, **rule)


def test_logits_of_any_size(sampling):
    rng = np.random.default_rng(6)
    for spread in (1e-20, 1e-3, 300.0, 1e20, 1e37):
        x = np.clip(logits(rng, 5, 30000, spread=1.0).astype(np.float64) * spread, -3.4e38, 3.4e38).astype(np.float32)
        for rule in (dict(), dict(top_k=50), dict(top_k=2000), dict(top_p=0.9), dict(top_p=0.9, top_k=4000)):
            check(sampling, x, rng.random(5), temperature=spread, **rule)
            check(sampling, x, rng.random(5), **rule)


def test_no_settings_and_no_share(sampling):
    """NULL settings, NULL shares; the largest vocabulary, and one token."""
    from llamd_rs_b200 import backend

    rng = np.random.default_rng(7)
    for n in (1, 262147, 393216):
        x = logits(rng, 2, n)
        u = rng.random(2).astype(np.float32)
        token, dx, du = dev(np.zeros(2, np.int32)), dev(x), dev(u)
        sampling.sample(dx, du, token, rows=2, n_vocab=n)
        backend.sync()
        assert token.download(np.int32, 2).tolist() == [plain.sample(x[r], u[r])[0] for r in range(2)]
        check(sampling, x, u, top_p=0.9)
        check(sampling, x, u, top_k=60)
    sampling.sample(dx, du, token, rows=0, n_vocab=5)


def test_frequencies(sampling):
    """Many numbers, spread evenly: each token as often as its share says, to within one."""
    rng = np.random.default_rng(8)
    x = np.repeat(logits(rng, 1, 500), 4096, 0)
    u = (np.arange(4096) + 0.5) / 4096
    for rule in (dict(), dict(top_k=30, top_p=0.9, temperature=0.8)):
        got, share = run(sampling, x, u, **rule)
        assert np.all(np.diff(got) >= 0)
        for t in np.unique(got):
            assert abs(np.sum(got == t) - 4096 * share[got == t][0]) <= 1.001


def test_graph_and_repeats(sampling):
    """Captured once, replayed over new logits and numbers; and the same answer every time."""
    from llamd_rs_b200 import backend
    from llamd_rs_b200._lib import lib

    rng = np.random.default_rng(9)
    rows, n = 6, 40000
    x, u = [logits(rng, rows, n) for _ in range(3)], rng.random((3, rows)).astype(np.float32)
    dx, du, k, p = dev(x[0]), dev(u[0]), dev(np.full(rows, 50, np.int32)), dev(np.linspace(0.5, 1.0, rows).astype(np.float32))
    token, prob = dev(np.zeros(rows, np.int32)), dev(np.zeros(rows, np.float32))
    sampling.sample(dx, du, token, top_p=p, prob=prob, rows=rows, n_vocab=n)
    backend.sync()
    assert lib().llamd_fwd_begin_capture() == 0
    sampling.sample(dx, du, token, top_p=p, prob=prob, rows=rows, n_vocab=n)
    assert lib().llamd_fwd_end_capture() == 0
    try:
        for i in (1, 2, 0, 0, 0):
            dx.upload(x[i])
            du.upload(u[i])
            assert lib().llamd_fwd_graph_launch() == 0
            backend.sync()
            want = [plain.sample(x[i][r], u[i][r], top_p=np.linspace(0.5, 1.0, rows).astype(np.float32)[r])[0] for r in range(rows)]
            assert token.download(np.int32, rows).tolist() == want
    finally:
        lib().llamd_fwd_graph_destroy()


def test_tensors(sampling):
    """torch tensors on a stream of their own: rows of a padded vocabulary, order with that stream, types and shapes checked."""
    torch = pytest.importorskip("torch")
    from llamd_rs_b200.backend import ShapeError, Unsupported

    rows, n = 5, 3001
    f = lambda v: torch.full((rows,), v, device="cuda")  # noqa: E731
    token, prob, u = torch.zeros(rows, dtype=torch.int32, device="cuda"), f(0.0), torch.rand(rows, device="cuda")
    k = torch.full((rows,), 40, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(20_000_000)  # (without the order the call would read what is not there yet)
        x = torch.randn(rows, n + 63, device="cuda").bfloat16()[:, :n]
        sampling.sample(x, u, token, temperature=f(0.9), top_k=k, top_p=f(0.95), prob=prob)
        got = token.clone()
    side.synchronize()
    want = [plain.sample(x[r].float().cpu().numpy(), u[r].item(), 0.9, 40, 0.95)[0] for r in range(rows)]
    assert got.tolist() == want
    for bad in (dict(logits=x.double()), dict(logits=x.to(torch.int32))):
        with pytest.raises(Unsupported):
            sampling.sample(bad["logits"], u, token)
    for args in ((x[0], u, token), (x.t(), u, token), (x, u[:4], token), (x, u, token.float()), (x, u, token.long()), (x.cpu(), u, token), (x, u.cpu(), token)):
        with pytest.raises(ShapeError):
            sampling.sample(*args)
    with pytest.raises(ShapeError):
        sampling.sample(x, u, token, top_k=k.float())
    with pytest.raises(ShapeError):
        sampling.sample(x.expand(rows, n)[:1].expand(rows, n), u, token)  # rows that are one
    sampling.sample(x[:1], u[:1], token[:1])


def test_refusals(sampling):
    from llamd_rs_b200._lib import lib
    from llamd_rs_b200.backend import Malformed, ShapeError, Unsupported

    L, x, w = lib(), dev(np.zeros((2, 100), np.float32)), dev(np.zeros(8, np.int32))
    good = [x.ptr, 2, 100, 2, 100, None, None, None, None, w.ptr, w.ptr + 16, None]
    assert L.llamd_fwd_sample(*good) == 0
    for at, bad in ((0, None), (0, x.ptr + 2), (1, 3), (1, -1), (2, 99), (3, -1), (4, 0), (4, 393217), (4, -5), (9, None), (10, None), (10, w.ptr + 17), (6, w.ptr + 1)):
        args = list(good)
        args[at] = bad
        assert L.llamd_fwd_sample(*args) == -1, (at, bad)
        assert L.llamd_fwd_last_error() != 0
    with pytest.raises(Unsupported):
        sampling.sample(x, w, w, rows=2, n_vocab=100, dtype="i8")
    with pytest.raises(Malformed):
        sampling.sample(x, w, w)
    with pytest.raises(Malformed):
        sampling.sample(x, None, w, rows=2, n_vocab=100)
    for kw in (dict(rows=3, n_vocab=100), dict(rows=2, n_vocab=101), dict(rows=2, n_vocab=100, stride=50)):
        with pytest.raises(ShapeError):
            sampling.sample(x, w, w, **kw)
    with pytest.raises(ShapeError):
        sampling.sample(x, w, dev(np.zeros(1, np.int32)), rows=2, n_vocab=100)
    with pytest.raises(Malformed):
        sampling.sample(x, w, w, rows=-1, n_vocab=100)


def test_ops(sampling):
    from llamd_rs_b200 import ops

    rng = np.random.default_rng(10)
    x, u = logits(rng, 4, 700), rng.random(4).astype(np.float32)
    token, share = ops.sample(x, u, temperature=0.8, top_k=30, top_p=0.9)
    want = [plain.sample(x[r], u[r], 0.8, 30, 0.9) for r in range(4)]
    assert token.tolist() == [t for t, _ in want] and np.allclose(share, [s for _, s in want], rtol=1e-6)
    assert np.array_equal(ops.sample(x, 0.5, temperature=0.0)[0], ops.argmax(x))


def test_model(sampling):
    """A model's logits sampled where they are: decoding that draws every token, greedy where the temperature is 0, settings checked."""
    from llamd_rs_b200 import backend, synth
    from llamd_rs_b200.model import CudaModel

    hp = synth.TINY
    m = CudaModel.load_batched(hp, synth.make_model(hp, seed=7), max_kv=64, max_seq=4)
    try:
        rng = np.random.default_rng(11)
        u = rng.random(8).astype(np.float32)
        tokens, shares = m.sample_decode(3, 0, u, temperature=1.2, top_k=50, top_p=0.95)
        at = 3
        for i in range(8):
            m.forward(at, i)
            want, share = plain.sample(m.logits(1)[0], u[i], 1.2, 50, 0.95)
            assert tokens[i] == want and abs(shares[i] - share) <= 1e-6
            at = want
        greedy = [m.forward(t, 8 + i) for i, t in enumerate([at, 5])]
        assert m.sample([0.3], temperature=0.0)[0][0] == greedy[1]
        m.forward_batch([1, 2, 3], [0, 0, 0])
        x, u = m.logits(3), rng.random(3).astype(np.float32)
        got, _ = m.sample(u, temperature=[0.5, 1.0, 2.0], min_p=0.01)
        assert got.tolist() == [plain.sample(x[r], u[r], t, min_p=0.01)[0] for r, t in enumerate((0.5, 1.0, 2.0))]
        for bad in (dict(temperature=-1.0), dict(top_p=1.5), dict(min_p=-0.1), dict(top_p=np.nan), dict(temperature=np.nan)):
            with pytest.raises(backend.Malformed):
                m.sample([0.5], **bad)
        for u in ([1.0], [-0.5], [np.nan]):
            with pytest.raises(backend.Malformed):
                m.sample(u)
        with pytest.raises(backend.ShapeError):
            m.sample([0.5] * 5)
        with pytest.raises(backend.Malformed):
            m.sample([0.5, 0.5], top_k=[1, 2, 3])
        with pytest.raises(backend.Malformed):
            m.sample([0.5], top_k=1.5)
    finally:
        m.free()
