"""Attention layers of a Qwen3MoE-shaped model serving several conversations over paged caches, one system prompt for all.

Every layer is norm -> Q/K/V projections (Q6_K) -> append -> attention -> output projection -> residual, all on the library's stream,
the conversations' rows packed. The experts between the layers are left out: they do not see the caches. Weights and inputs are
random; a decode step's row is the last layer's normed output, or with --vocab the embedding of the token that is drawn from its logits. Steps:

  1. the system prompt goes in once;
  2. the conversations fork its pages, and their own prompts, of different lengths, go in packed in one step;
  3. decode steps of one token per conversation, the system prompt's pages read once for all of them.

    python examples/paged_serving.py [--layers 4] [--conversations 32] [--system 1024] [--steps 16] [--cache e4m3] [--vocab 32768] [--check]

--cache i8 or e4m3 keeps keys and values in 8 bits. --vocab n: an output head of n tokens, each conversation's next token drawn by
temperature, top-k, top-p and min-p. --check sends one conversation through the exact ops as well (f32 slab caches, attention in the reference's order) and
prints how far the paged layers' outputs are from theirs.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from llamd_rs_b200 import backend, paged, sampling, synth  # noqa: E402
from llamd_rs_b200._lib import lib  # noqa: E402
from llamd_rs_b200.backend import DevBuf  # noqa: E402

EPS, FREQ_BASE = 1e-6, 1e6


class Layers:
    """The weights, and the device buffers for up to max_tokens rows."""

    def __init__(self, hp, n_layer, max_tokens, max_positions, seed=0, vocab=0):
        self.hp, self.n_layer = hp, n_layer
        E, D = hp["n_embd"], hp["head_dim"]
        self.E, self.qd, self.kvd = E, hp["n_head"] * D, hp["n_head_kv"] * D
        w = lambda rows, k, *key: backend.DeviceWeights.upload(synth.q6k_blocks(rows * k // 256, seed, *key), rows, k // 256)  # noqa: E731
        ones = lambda n, *key: DevBuf.from_array((1 + 0.1 * synth.normal_f32(n, seed, *key)).astype(np.float32))  # noqa: E731
        self.layers = [dict(norm=ones(E, il, "norm"), qn=ones(D, il, "qn"), kn=ones(D, il, "kn"), q=w(self.qd, E, il, "q"), k=w(self.kvd, E, il, "k"),
                            v=w(self.kvd, E, il, "v"), o=w(E, self.qd, il, "o")) for il in range(n_layer)]
        self.vocab = vocab
        if vocab:
            self.head, self.embedding = w(vocab, E, "head"), synth.normal_f32(vocab * E, seed, "embedding").reshape(vocab, E)
            self.head_norm = ones(E, "head norm")
        self.rope = DevBuf.from_array(paged.rope_table(max_positions, D, FREQ_BASE))
        f32 = lambda n: DevBuf(4 * max_tokens * n)  # noqa: E731
        self.x, self.q, self.k, self.v, self.att, self.o = f32(E), f32(self.qd), f32(self.kvd), f32(self.kvd), f32(self.qd), f32(E)
        wide = max(E, self.qd)
        self.qs, self.d = DevBuf(max_tokens * wide), DevBuf(4 * max_tokens * wide // 256)
        self.q16 = DevBuf(2 * max_tokens * self.qd)

    def project(self, il, n):
        """Q, K and V of the n rows of x."""
        L, w = lib(), self.layers[il]
        L.llamd_fwd_rms_norm_quant(self.x.ptr, w["norm"].ptr, None, self.qs.ptr, self.d.ptr, self.E, EPS, n)
        L.llamd_fwd_matvec_tokens(w["q"].ptr, w["k"].ptr, w["v"].ptr, self.qs.ptr, self.d.ptr, self.q.ptr, self.k.ptr, self.v.ptr, self.E // 256, self.qd,
                                  self.kvd, self.kvd, n)

    def finish(self, il, n):
        """x += the output projection of the n attended rows."""
        L = lib()
        L.llamd_fwd_quantize(self.att.ptr, self.qs.ptr, self.d.ptr, n * self.qd // 256)
        L.llamd_fwd_matvec_tokens(self.layers[il]["o"].ptr, None, None, self.qs.ptr, self.d.ptr, self.o.ptr, None, None, self.qd // 256, self.E, 0, 0, n)
        L.llamd_fwd_add(self.x.ptr, self.o.ptr, self.x.ptr, n * self.E)

    def out(self, n):
        backend.sync()
        return self.x.download_f32(n * self.E).reshape(n, self.E)


class Head:
    """The output head over up to `rows` rows, and the draw of a token from each."""

    def __init__(self, layers, rows, temperature=0.8, top_k=50, top_p=0.95, min_p=0.01):
        self.m, self.rng = layers, np.random.default_rng(1)
        each = lambda v, t: DevBuf.from_array(np.full(rows, v, t))  # noqa: E731
        self.logits, self.uniform, self.token = DevBuf(4 * rows * layers.vocab), DevBuf(4 * rows), DevBuf(4 * rows)
        self.settings = dict(temperature=each(temperature, np.float32), top_k=each(top_k, np.int32), top_p=each(top_p, np.float32), min_p=each(min_p, np.float32))

    def draw(self, rows):
        """The next tokens behind the rows."""
        m, L, n = self.m, lib(), len(rows)
        m.x.upload(rows.astype(np.float32))
        L.llamd_fwd_rms_norm_quant(m.x.ptr, m.head_norm.ptr, None, m.qs.ptr, m.d.ptr, m.E, EPS, n)
        L.llamd_fwd_matvec_tokens(m.head.ptr, None, None, m.qs.ptr, m.d.ptr, self.logits.ptr, None, None, m.E // 256, m.vocab, 0, 0, n)
        self.uniform.upload(self.rng.random(n, dtype=np.float32))
        sampling.sample(self.logits, self.uniform, self.token, rows=n, n_vocab=m.vocab, **self.settings)
        backend.sync()
        return self.token.download_i32(n)


class Server:
    """Conversations over paged caches: a pool of K and of V pages per layer, one table per conversation for all layers."""

    def __init__(self, layers, n_pages, page_size=32, dtype="f16", cache=None):
        hp = layers.hp
        self.layers, self.pages = layers, paged.Pages(n_pages, page_size)
        pool = (1 if cache else 2) * n_pages * page_size * layers.kvd
        self.scales = [{}] * layers.n_layer
        if cache:
            n = n_pages * hp["n_head_kv"] * page_size // paged.SCALE_BLOCK
            self.scales = [dict(k_scales=DevBuf(n), v_scales=DevBuf(n)) for _ in range(layers.n_layer)]
        self.k = [DevBuf(pool) for _ in range(layers.n_layer)]
        self.v = [DevBuf(pool) for _ in range(layers.n_layer)]
        self.batch = paged.Batch(hp["n_head"], hp["n_head_kv"], hp["head_dim"], page_size, dtype, cache=cache)

    def step(self, rows, q_lens, tables, lengths, n_shared=0):
        """The new rows of every conversation through all layers; grows the tables and the lengths. -> the last layer's rows."""
        m, n = self.layers, len(rows)
        for i, more in enumerate(q_lens):
            lengths[i] += more
            self.pages.grow(tables[i], lengths[i])
        self.batch.set(q_lens, lengths, tables, self.pages.n_pages, n_shared)
        m.x.upload(rows.astype(np.float32))
        for il, w in enumerate(m.layers):
            m.project(il, n)
            self.batch.append(m.q, m.k, m.v, m.q16, self.k[il], self.v[il], rope=m.rope, q_norm=w["qn"], k_norm=w["kn"], eps=EPS, **self.scales[il])
            self.batch.attention(m.q16, self.k[il], self.v[il], m.att, out_f32=True, **self.scales[il])
            m.finish(il, n)
        return m.out(n)


def exact(layers, steps, max_positions):
    """One conversation's steps ([tokens][E] each) through the exact ops over f32 slab caches. -> the rows of the last step."""
    m, hp, L = layers, layers.hp, lib()
    H, K, D = hp["n_head"], hp["n_head_kv"], hp["head_dim"]
    caches = [(DevBuf.zeroed(4 * max_positions * m.kvd), DevBuf.zeroed(4 * max_positions * m.kvd)) for _ in m.layers]
    table = np.empty((max_positions, D // 2, 2), np.float32)
    L.llamd_cuda_rope_table(backend._ptr(table), max_positions, D, FREQ_BASE)
    rope, at, out = DevBuf.from_array(table), 0, None
    for rows in steps:
        n = len(rows)
        meta = DevBuf.from_array(np.stack([np.zeros(n, np.int32), np.arange(at, at + n, dtype=np.int32)], 1))
        scores = DevBuf(4 * n * H * max_positions)
        m.x.upload(rows.astype(np.float32))
        for il, w in enumerate(m.layers):
            kc, vc = caches[il]
            m.project(il, n)
            L.llamd_fwd_qk_norm_rope_store_tile(m.q.ptr, w["qn"].ptr, m.k.ptr, w["kn"].ptr, m.v.ptr, kc.ptr, vc.ptr, H, K, D, meta.ptr, rope.ptr, EPS, n)
            L.llamd_fwd_attention_prefill(m.q.ptr, kc.ptr, vc.ptr, m.att.ptr, scores.ptr, H, K, D, meta.ptr, max_positions, n, at + n)
            m.finish(il, n)
        out = m.out(n)
        at += n
    return out


def normed(rows):
    return rows / np.sqrt((rows * rows).mean(-1, keepdims=True) + EPS)


def serve(hp, n_layer, conversations, system, steps, page_size=32, check=False, say=print, cache=None, vocab=0):
    """-> with check: the relative distance of conversation 0's last row from the exact ops', else None."""
    rng = np.random.default_rng(0)
    E, system = hp["n_embd"], system // page_size * page_size  # (whole pages can be shared)
    own = rng.integers(1, 200, conversations)
    longest = system + int(own.max()) + steps
    layers = Layers(hp, n_layer, max(system, int(own.sum()), conversations, 1), longest, vocab=vocab)
    server = Server(layers, -(-system // page_size) + int(sum(-(-(n + steps) // page_size) for n in own)) + 8, page_size, cache=cache)
    head = Head(layers, conversations) if vocab else None
    rows = lambda n: rng.standard_normal((n, E)).astype(np.float32)  # noqa: E731

    def timed(what, *a):
        t = time.perf_counter()
        got = server.step(*a)
        say(f"{what:28s} {1e3 * (time.perf_counter() - t):8.3f} ms, {server.pages.free()} of {server.pages.n_pages} pages free")
        return got

    first, lengths0 = [], [0]
    prompt = rows(system)
    if system:
        timed(f"system prompt, {system} rows", prompt, [system], [first], lengths0)
    tables, lengths = [server.pages.fork(first, system) for _ in own], [system] * conversations
    prompts = [rows(n) for n in own]
    out = timed(f"{conversations} prompts, {int(own.sum())} rows", np.concatenate(prompts), own, tables, lengths, system)
    last = out[np.cumsum(own) - 1]
    history = [prompt, prompts[0]] if system else [prompts[0]]
    for s in range(steps):
        x = layers.embedding[head.draw(last)] if head else normed(last)
        history.append(x[:1])
        last = timed(f"decode step {s}", x, [1] * conversations, tables, lengths, system)
    for t in [first] + tables:
        server.pages.release(t)
    if paged.status() != 0:
        raise RuntimeError("a wait inside the attention ran out")
    if not check:
        return None
    # (the last rows of one conversation; its inputs are those that the paged layers produced)
    want = exact(layers, history, longest)[-1]
    far = float(np.linalg.norm(last[0] - want) / np.linalg.norm(want))
    say(f"conversation 0, last row: {far:.2e} from the exact ops (relative)")
    return far


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--conversations", type=int, default=32)
    ap.add_argument("--system", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--page", type=int, default=32)
    ap.add_argument("--cache", choices=sorted(paged.CACHES))
    ap.add_argument("--vocab", type=int, default=0)
    ap.add_argument("--check", action="store_true")
    a = ap.parse_args()
    backend.stream_init()
    serve(synth.QWEN3MOE_30B, a.layers, a.conversations, a.system, a.steps, a.page, a.check, cache=a.cache, vocab=a.vocab)


if __name__ == "__main__":
    main()
