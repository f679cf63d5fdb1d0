"""Decode steps as a server makes them: append to caches in 8 bits, attention over them, logits, a token drawn from each row, the next step. Every call's results against the
definitions, on what the calls before it have left."""
import numpy as np
import pytest

import paged8_plain as plain8
import paged_plain as plain
import sample_plain
from test_gpu_paged import close, dev
from test_gpu_paged_serving import example  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype,D,page", [("f16", 64, 16), ("bf16", 128, 32)])
def test_conversations(cache, dtype, D, page):
    """Three conversations behind a common beginning: their prompts in one step, then tokens one by one, drawn from what attention gave."""
    from llamd_rs_b200 import backend, paged, sampling

    backend.stream_init()
    rng = np.random.default_rng(D)
    H, K, V, n_pages, shared, steps = 8, 2, 600, 40, 2 * page, 20
    embed = [rng.standard_normal((V, n, D)).astype(np.float32) for n in (H, K, K)]
    out_head = rng.standard_normal((H * D, V)).astype(np.float32) / np.sqrt(H * D)
    table = paged.rope_table(512, D, 1e4)
    rope, pages = dev(table), paged.Pages(n_pages, page)
    pools = [[dev(rng.integers(0, 256, (n_pages, K, page, D)).astype(np.uint8)), dev(rng.integers(0, 256, (n_pages, K, page // 16)).astype(np.uint8))] for _ in range(2)]
    s = dict(k_scales=pools[0][1], v_scales=pools[1][1])
    b = paged.Batch(H, K, D, page, dtype, cache=cache)

    def step(tokens, q_len, tables, lengths, n_shared):
        """All new tokens (a list of each conversation's) -> attention's rows, checked."""
        for i, n in enumerate(q_len):
            lengths[i] += n
            pages.grow(tables[i], lengths[i])
        b.set(q_len, lengths, tables, n_pages, n_shared)
        t = np.concatenate(tokens)
        x = [e[t] for e in embed]
        q, out = dev(np.zeros((len(t), H, D), np.uint16)), dev(np.zeros((len(t), H, D), np.uint32))
        b.append(*[dev(v) for v in x], q, pools[0][0], pools[1][0], rope=rope, **s)
        b.attention(q, pools[0][0], pools[1][0], out, out_f32=True, **s)
        backend.sync()
        assert paged.status() == 0
        got_q = plain.from_bits(q.download(np.uint16, len(t) * H * D), dtype).reshape(-1, H, D)
        seq, pos = plain.positions(q_len, lengths)
        raw = [[p[0].download(np.uint8, n_pages * K * page * D).reshape(n_pages, K, page, D), p[1].download(np.uint8, n_pages * K * page // 16).reshape(n_pages, K, page // 16)]
               for p in pools]
        # the new rows, to within a step of their block's scale (half of it, and half again where later rows made it larger)
        ids = np.array([tables[i][p // page] for i, p in zip(seq, pos)])
        for (codes, scales), v, turned in zip(raw, x[1:], (True, False)):
            want = plain.norm_rope(v.astype(np.float64), pos, None, 0, table, D if turned else 0, False)
            have = plain8.values(codes, scales, cache)[ids, :, pos % page]
            e = scales[ids, :, pos % page // 16].astype(int) - 127
            assert np.all(np.abs(have - want) <= plain8.step(want * 2.0 ** -e[..., None].astype(float), cache) * 2.0 ** e[..., None] + 1e-5)
        live = np.zeros((n_pages, page), bool)
        for tb, m in zip(tables, lengths):
            live[np.asarray(tb)[np.arange(m) // page], np.arange(m) % page] = True
        kv = []
        for codes, scales in raw:  # (whatever no conversation holds is as it was made: anything)
            v = plain8.values(codes, np.where(live.reshape(n_pages, 1, page // 16, 16).any(-1), scales, 127), cache)
            kv.append(np.where(live[:, None, :, None], v, 0.0))
        got = out.download(np.uint32, len(t) * H * D).view(np.float32).astype(np.float64).reshape(-1, H, D)
        want, bound = plain.attention(got_q, *kv, tables, q_len, lengths, D ** -0.5, dtype)
        close(got, want, bound + 2.0 ** -37 * 448 * 8)
        return got

    first, n0 = [], [0]
    step([rng.integers(0, V, shared)], [shared], [first], n0, 0)
    tables, lengths = [pages.fork(first, shared) for _ in range(3)], [shared] * 3
    q_len = [int(x) for x in rng.integers(1, 60, 3)]
    got = step([rng.integers(0, V, n) for n in q_len], q_len, tables, lengths, shared)
    last = got[np.cumsum(q_len) - 1]
    settings = dict(temperature=0.7, top_k=40, top_p=0.9, min_p=0.02)
    on_device = {k: dev(np.full(3, v, np.int32 if k == "top_k" else np.float32)) for k, v in settings.items()}
    for _ in range(steps):
        logits, u = (4 * last.reshape(3, -1) @ out_head).astype(np.float32), rng.random(3).astype(np.float32)
        token = dev(np.zeros(3, np.int32))
        sampling.sample(dev(logits), dev(u), token, rows=3, n_vocab=V, **on_device)
        backend.sync()
        tokens = token.download(np.int32, 3)
        assert tokens.tolist() == [sample_plain.sample(logits[r], u[r], **settings)[0] for r in range(3)]
        last = step([tokens[r:r + 1] for r in range(3)], [1] * 3, tables, lengths, shared)
    for t in [first] + tables:
        pages.release(t)
    assert pages.free() == n_pages


@pytest.mark.parametrize("cache", ["i8", "e4m3"])
def test_example(example, cache):  # noqa: F811
    """The example with caches in 8 bits and a head that tokens are drawn from: it runs, and gives its pages back."""
    hp = dict(n_embd=256, n_head=4, n_head_kv=2, head_dim=64)
    lines = []
    assert example.serve(hp, 2, 5, 48, 6, 16, say=lines.append, cache=cache, vocab=1024) is None
    assert len(lines) == 8


# One layer: keys and values differ from the exact ones by half a step of their block's scale: i8 1/127 of the block's largest value at most, e4m3 2^-4 of the value. Scores are off by
# that of |q| |k| / sqrt(hd) at random, weights and values by as much: some hundredths of the attention's rows, and less of rows that the residual is most of.
@pytest.mark.parametrize("cache,most", [("i8", 0.03), ("e4m3", 0.1)])
def test_one_layer_against_the_exact_ops(example, cache, most):  # noqa: F811
    hp = dict(n_embd=512, n_head=8, n_head_kv=2, head_dim=128)
    assert example.serve(hp, 1, 3, 64, 3, 16, check=True, say=lambda *a: None, cache=cache) < most
