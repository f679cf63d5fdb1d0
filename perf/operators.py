"""Operators over a paged K/V cache: what a server of many sequences calls once per layer and step.

append      the new tokens' queries and keys normed per head and rotated, keys and values written to their pages
prompt      causal attention of whole prompts (or chunks of them) of different lengths, packed one behind the other
decode      attention of a batch with one or a few new tokens per sequence; sequences may share a prefix, whose pages are
            then the same and which is read once for all

Layouts: q, k, v [tokens][heads][hd], the tokens of all sequences packed; pages [n_pages][n_head_kv][page][hd] in 16 bits;
a table of page ids per sequence. Position i of a sequence sits in slot i % page of its page i // page. A sequence's new
tokens are the last q_len of its kv_len positions, and each attends to every position up to its own.
"""
import json
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _case(name, kind, n_seq, q, ctx, heads=(32, 4, 128), page=16, type="f16", shared=0, **more):
    """q, ctx: (least, most) new tokens and positions in front of them (behind a shared prefix), per sequence."""
    return dict(name=name, kind=kind, n_seq=n_seq, q_lo=q[0], q_hi=q[1], ctx_lo=ctx[0], ctx_hi=ctx[1], n_head=heads[0], n_head_kv=heads[1], hd=heads[2],
                page=page, type=type, shared=shared, **more)


def _append(name, *a, inputs="f32", rot=128, interleaved=False, norm=True, stretch=1.0, **k):
    return _case(name, "append", *a, inputs=inputs, rot=rot, interleaved=interleaved, norm=norm, stretch=stretch, **k)


def listed():
    return [
        # one token of one long conversation: the call's latency is what counts
        _append("append_one", 1, (1, 1), (4001, 4001)),
        # a decode step of a serving batch, projections in f32 as the quantized matrices leave them
        _append("append_batch_128", 128, (1, 1), (24, 264), type="bf16"),
        # a step that takes several prompts in, one projection for q, k and v in 16 bits (so rows with a stride)
        _append("append_prompts", 7, (1, 1999), (0, 300), inputs="f16", page=64),
        # a long prompt of a model that rotates half of each head, neighbouring elements paired, positions stretched fourfold
        _append("append_part_rotated", 1, (8192, 8192), (0, 0), heads=(14, 2, 64), inputs="f32", type="bf16", rot=32, interleaved=True, norm=False,
                stretch=4.0, page=32),
        # the benchmark's prompt
        _case("prompt_512", "prompt", 1, (512, 512), (0, 0)),
        # prompts of a serving step, packed
        _case("prompt_packed", "prompt", 9, (1, 1999), (0, 0), type="bf16", page=32),
        # one long prompt
        _case("prompt_8192", "prompt", 1, (8192, 8192), (0, 0), type="bf16", page=64),
        # chunks of prompts whose beginnings are cached already; small heads, a group of seven
        _case("prompt_chunks", "prompt", 4, (37, 301), (900, 8000), heads=(14, 2, 64)),
        # one long conversation
        _case("decode_one", "decode", 1, (1, 1), (4001, 4001)),
        # a serving batch of conversations of very different lengths
        _case("decode_batch_32", "decode", 32, (1, 1), (150, 8000), type="bf16", page=32),
        # a few short conversations behind one system prompt
        _case("decode_shared_8", "decode", 8, (1, 1), (0, 264), shared=512),
        # many behind a long one
        _case("decode_shared_256", "decode", 256, (1, 1), (3, 600), type="bf16", shared=4096),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 4, 128), (32, 4, 128), (16, 1, 128), (8, 8, 64), (14, 2, 64), (5, 1, 128), (40, 8, 64)]


def draw(rng):
    kind = rng.choice(["append", "prompt", "decode"])
    heads, page, type_ = rng.choice(HEADS), rng.choice([16, 32, 64, 128]), rng.choice(["f16", "bf16"])
    common = dict(heads=heads, page=page, type=type_)
    if kind == "append":
        n_seq = _log_int(rng, 1, 200)
        most = _log_int(rng, 1, max(1, 8192 // n_seq))
        rot = rng.choice([heads[2], heads[2], heads[2] // 2, heads[2] // 4])
        c = _append("", n_seq, (rng.randint(1, most), most), (0, _log_int(rng, 1, 4000)), inputs=rng.choice(["f32", type_]), rot=rot,
                    interleaved=rng.random() < 0.5, norm=rng.random() < 0.6, stretch=rng.choice([1.0, 4.0]), **common)
    elif kind == "prompt":
        n_seq = _log_int(rng, 1, 12)
        most = _log_int(rng, 20, 8000 // n_seq)
        ctx = rng.choice([0, _log_int(rng, 1, 8000 // n_seq)])
        c = _case("", "prompt", n_seq, (rng.randint(1, most), most), (0, ctx), **common)
    else:
        n_seq = _log_int(rng, 1, 256)
        shared = rng.choice([0, 0, page * _log_int(rng, 1, 2560 // page)])
        most = _log_int(rng, 1, min(30000, 100000 // n_seq))
        c = _case("", "decode", n_seq, (1, rng.choice([1, 1, 1, 3])), (rng.randint(0, most), most), shared=shared, **common)
    del c["name"]
    return draw(rng) if 3072 in c.values() else c


# ---- the shapes of a case ------------------------------------------------------------------------------------------------

def _lengths(case):
    """(new tokens, positions in all) of every sequence: the case's own, whatever the seed."""
    r = random.Random(json.dumps([case[k] for k in ("kind", "n_seq", "q_lo", "q_hi", "ctx_lo", "ctx_hi", "shared")]))
    q, kv = [], []
    for _ in range(case["n_seq"]):
        q.append(r.randint(case["q_lo"], case["q_hi"]))
        kv.append(q[-1] + r.randint(case["ctx_lo"], case["ctx_hi"]) + case["shared"])
    return q, kv


def _pairs(case):
    q, kv = _lengths(case)
    return sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(q, kv))


def work(case):
    (q, kv), H, K, D = _lengths(case), case["n_head"], case["n_head_kv"], case["hd"]
    tokens = sum(q)
    if case["kind"] == "append":
        wide = 4 if case["inputs"] == "f32" else 2
        positions = len({m - 1 - i for n, m in zip(q, kv) for i in range(n)})
        values = tokens * (H + 2 * K) * D
        return dict(bytes=values * (wide + 2) + positions * case["rot"] * 4 + 4 * tokens,
                    flops=tokens * (H + K) * (case["rot"] * 3 + (4 * D if case["norm"] else 0)))
    cached = case["shared"] + sum(m - case["shared"] for m in kv)
    return dict(bytes=4 * tokens * H * D + 4 * cached * K * D + 4 * -(-cached // case["page"]), flops=4 * D * H * _pairs(case))


# ---- what a program has in hand ------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rope_table(case, rows):
    """[rows][rot / 2][2]: sine and cosine of position / stretch * base^(-2 i / rot), as a model loader tabulates them once."""
    pos = torch.arange(rows, dtype=torch.float64, device="cuda") / case["stretch"]
    freq = 1e6 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"])
    a = pos[:, None] * freq
    return torch.stack([a.sin(), a.cos()], dim=-1).float().contiguous()


def _inputs(case, seed):
    """Everything that is data, on the GPU; the same for either side."""
    gen, (q, kv) = _gen(seed), _lengths(case)
    H, K, D, page, t = case["n_head"], case["n_head_kv"], case["hd"], case["page"], TYPES[case["type"]]
    tokens, own_pages = sum(q), [-(-m // page) - case["shared"] // page for m in kv]
    n_pages = sum(own_pages) + case["shared"] // page + 3  # (a pool has free pages too)
    ids = torch.randperm(n_pages, device="cuda", generator=gen).to(torch.int32).cpu().numpy()
    table = np.zeros((len(q), max(-(-m // page) for m in kv)), np.int32)
    first, at = case["shared"] // page, case["shared"] // page
    for s, n in enumerate(own_pages):  # the shared prefix's pages, then the sequence's own
        table[s, :first] = ids[:first]
        table[s, first:first + n] = ids[at:at + n]
        at += n
    rand = lambda *shape: torch.randn(shape, device="cuda", generator=gen)  # noqa: E731
    d = dict(case, q_len=np.array(q, np.int32), kv_len=np.array(kv, np.int32), table=table, n_pages=n_pages, tokens=tokens,
             k_pages=rand(n_pages, K, page, D).to(t), v_pages=rand(n_pages, K, page, D).to(t))
    if case["kind"] == "append":
        t_in = TYPES[case["inputs"]]
        if case["inputs"] == "f32":
            d.update(q=rand(tokens, H, D), k=rand(tokens, K, D), v=rand(tokens, K, D))
        else:  # one projection made all three: rows of q, k and v side by side
            qkv = rand(tokens, H + 2 * K, D).to(t_in)
            d.update(qkv=qkv, q=qkv[:, :H], k=qkv[:, H:H + K], v=qkv[:, H + K:])
        d.update(rope=_rope_table(case, max(kv)), wq=1 + 0.3 * rand(D), wk=1 + 0.3 * rand(D), q_out=torch.empty(tokens, H, D, dtype=t, device="cuda"))
    else:
        d.update(q=(1.5 * rand(tokens, H, D)).to(t), out=torch.empty(tokens, H, D, dtype=t, device="cuda"))
    return d


def prepare(case, seed):
    s = _inputs(case, seed)
    # what both sides keep of the batch's shape: the sequence, position, page and slot of every new token
    seq = np.repeat(np.arange(len(s["q_len"])), s["q_len"])
    pos = np.concatenate([np.arange(m - n, m) for n, m in zip(s["q_len"], s["kv_len"])])
    s.update(seq=torch.from_numpy(seq).cuda(), pos=torch.from_numpy(pos).cuda(), pages=torch.from_numpy(s["table"]).cuda().long(),
             kv=torch.from_numpy(s["kv_len"]).cuda().long(), first=torch.from_numpy(np.cumsum(s["q_len"]) - s["q_len"]).cuda())
    if own:
        from llamd_rs_b200 import paged
        # the batch's plan: made once per step, used by every layer of a model
        s["batch"] = paged.Batch(s["n_head"], s["n_head_kv"], s["hd"], s["page"], s["type"])
        s["batch"].set(s["q_len"], s["kv_len"], s["table"], s["n_pages"], n_shared=s["shared"])
    return s


# ---- the plain forms -----------------------------------------------------------------------------------------------------

def _rotated(x, s):
    """x [tokens][heads][hd] in 32 bits, its first `rot` elements rotated by the position's angles."""
    sc, rot = s["rope"][s["pos"]][:, None], s["rot"]
    sin, cos = sc[..., 0], sc[..., 1]
    x, rest = x[..., :rot], x[..., rot:]
    a, b = (x[..., 0::2], x[..., 1::2]) if s["interleaved"] else (x[..., :rot // 2], x[..., rot // 2:])
    a, b = a * cos - b * sin, a * sin + b * cos
    x = torch.stack([a, b], dim=-1).flatten(-2) if s["interleaved"] else torch.cat([a, b], dim=-1)
    return torch.cat([x, rest], dim=-1)


def _normed(x, w, s):
    x = x.float()
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w if s["norm"] else x


def _plain_append(s):
    page, slot = s["pages"][s["seq"], s["pos"] // s["page"]], s["pos"] % s["page"]
    t = s["k_pages"].dtype
    s["q_out"] = _rotated(_normed(s["q"], s["wq"], s), s).to(t)
    s["k_pages"][page, :, slot] = _rotated(_normed(s["k"], s["wk"], s), s).to(t)
    s["v_pages"][page, :, slot] = s["v"].float().to(t)
    return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _rows(pages, table):
    """The cached rows of a table of pages [..., n]: [..., n * page][heads][hd], in 32 bits."""
    x = pages[table].float().transpose(-3, -2)
    return x.flatten(-4, -3)


def _attended(q, k, v, seen):
    """q [..., tokens, heads, hd], k and v [..., positions, heads_kv, hd], seen [..., tokens, positions]."""
    group = q.shape[-2] // k.shape[-2]
    q = q.unflatten(-2, (k.shape[-2], group)).movedim(-4, -2)              # [..., heads_kv, group, tokens, hd]
    k, v = (x.movedim(-3, -2).unsqueeze(-3) for x in (k, v))               # [..., heads_kv, 1, positions, hd]
    x = q @ k.transpose(-1, -2) * q.shape[-1] ** -0.5
    x = x.masked_fill(~seen[..., None, None, :, :], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x @ v / x.sum(-1, keepdim=True)
    return x.movedim(-2, -4).flatten(-3, -2)


def _plain_prompt(s):
    out, at = [], 0
    for i, (n, m) in enumerate(zip(s["q_len"].tolist(), s["kv_len"].tolist())):
        table = s["pages"][i, :-(-m // s["page"])]
        k, v = _rows(s["k_pages"], table)[:m], _rows(s["v_pages"], table)[:m]
        seen = torch.arange(m, device="cuda") <= torch.arange(m - n, m, device="cuda")[:, None]
        out.append(_attended(s["q"][at:at + n].float(), k, v, seen))
        at += n
    return torch.cat(out).to(s["q"].dtype)


def _plain_decode(s):
    """Every sequence padded to the longest, its tokens to the most."""
    most, wide = int(s["q_len"].max()), int(s["kv_len"].max())
    k, v = _rows(s["k_pages"], s["pages"])[:, :wide], _rows(s["v_pages"], s["pages"])[:, :wide]
    at = s["pos"] - s["pos"][s["first"]][s["seq"]]
    q = torch.zeros((len(s["q_len"]), most) + s["q"].shape[1:], device="cuda")
    q[s["seq"], at] = s["q"].float()
    last = s["pos"][s["first"]][:, None] + torch.arange(most, device="cuda")
    out = _attended(q, k, v, torch.arange(wide, device="cuda") <= last[:, :, None])
    return out[s["seq"], at].to(s["q"].dtype)


def run(s):
    if own:
        if s["kind"] == "append":
            s["batch"].append(s["q"], s["k"], s["v"], s["q_out"], s["k_pages"], s["v_pages"], rope=s["rope"], rot=s["rot"], interleaved=s["interleaved"],
                              q_norm=s["wq"] if s["norm"] else None, k_norm=s["wk"] if s["norm"] else None, eps=EPS)
            return {"q": s["q_out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        s["batch"].attention(s["q"], s["k_pages"], s["v_pages"], s["out"])
        return s["out"]
    return {"append": _plain_append, "prompt": _plain_prompt, "decode": _plain_decode}[s["kind"]](s)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------

def _exact_append(s):
    k_pages, v_pages, outs = s["k_pages"].double(), s["v_pages"].double(), []
    seq = np.repeat(np.arange(len(s["q_len"])), s["q_len"])
    pos = np.concatenate([np.arange(m - n, m) for n, m in zip(s["q_len"], s["kv_len"])])
    page = torch.from_numpy(s["table"][seq, pos // s["page"]]).cuda().long()
    slot, pos = torch.from_numpy(pos % s["page"]).cuda(), torch.from_numpy(pos).cuda()
    angle = torch.complex(s["rope"][pos, :, 1].double(), s["rope"][pos, :, 0].double())[:, None]  # cos + i sin
    half = s["rot"] // 2
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        x = x.double()
        if s["norm"]:
            x = x * (x.square().sum(-1, keepdim=True) / s["hd"] + EPS).rsqrt() * w.double()
        at = torch.arange(half, device="cuda")
        i, j = (2 * at, 2 * at + 1) if s["interleaved"] else (at, at + half)
        z, y = torch.complex(x[..., i], x[..., j]) * angle, x.clone()
        y[..., i], y[..., j] = z.real, z.imag
        outs.append(y)
    k_pages[page, :, slot] = outs[1]
    v_pages[page, :, slot] = s["v"].double()
    return {"q": outs[0], "k_pages": k_pages, "v_pages": v_pages}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "append":
        return _exact_append(s)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    group, at, page = s["n_head"] // s["n_head_kv"], 0, s["page"]
    for i, (n, m) in enumerate(zip(s["q_len"].tolist(), s["kv_len"].tolist())):
        pos = np.arange(m)
        where = torch.from_numpy(s["table"][i, pos // page]).cuda().long(), torch.from_numpy(pos % page).cuda()
        k, v = s["k_pages"][where[0], :, where[1]].double(), s["v_pages"][where[0], :, where[1]].double()
        for h in range(s["n_head_kv"]):
            for g in range(group):
                for t in range(0, n, 1024):  # (a slice of the tokens at a time: the scores of all would not fit)
                    e = min(n, t + 1024)
                    x = torch.einsum("td,pd->tp", s["q"][at + t:at + e, h * group + g].double(), k[:, h]) / math.sqrt(s["hd"])
                    ahead = torch.arange(m, device="cuda")[None] > torch.arange(m - n + t, m - n + e, device="cuda")[:, None]
                    out[at + t:at + e, h * group + g] = torch.softmax(x.masked_fill(ahead, -math.inf), -1) @ v[:, h]
        at += n
    return out
