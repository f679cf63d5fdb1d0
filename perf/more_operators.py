"""What a server's decode step calls beyond the operators over 16-bit caches: the same ones over caches in 8 bits, and the choice of the next tokens.

append8     the new tokens' queries and keys normed per head and rotated, keys and values written to their pages in 8 bits
attention8  "prompt8": causal attention of packed prompts, or chunks of them, over such pages; "decode8": of one or a few new tokens per
            sequence, whose beginnings may be shared
sample      a token for each row of logits, by temperature, top-k, top-p and min-p, from given uniform numbers

Pages [n_pages][heads][page][hd] hold codes c in 8 bits (e4m3, or whole numbers from -127 to 127), and each 16 neighbouring positions of a page and
head one scale 2^e (e8m0: e + 127 in a byte); a value is c 2^e. An append gives a block of 16 positions the least e with which its values
fit, those that it holds from earlier among them: the earlier codes are rounded again where e has grown. Infinities and values too large
for the largest e saturate. The rest as in operators.py beside this file.

A token is drawn from softmax(x / temperature) over the first top_k tokens by falling logit (equal ones by rising index), of those the
first whose weights before them are less than top_p of the k's together, of those the ones that weigh min_p of the first's or more: by rising index, the
first at which the sum of weights is above u times all of them. Temperature 0 is the first token itself. A row with no token above -inf gives -1.
"""
import json
import math
import random

import numpy as np
import torch

own = False

EPS = 1e-6
BLOCK = 16
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# largest code, least and largest exponent of a block's scale: what stays exact in f16
FORMATS = {"e4m3": (448.0, -15, 7), "i8": (127.0, -24, 9)}


def _case(name, kind, n_seq, q, ctx, heads=(32, 4, 128), page=16, type="f16", cache="e4m3", shared=0, **more):
    """q, ctx: (least, most) new tokens and positions in front of them (behind a shared prefix), per sequence."""
    return dict(name=name, kind=kind, n_seq=n_seq, q_lo=q[0], q_hi=q[1], ctx_lo=ctx[0], ctx_hi=ctx[1], n_head=heads[0], n_head_kv=heads[1], hd=heads[2],
                page=page, type=type, cache=cache, shared=shared, **more)


def _append(name, *a, inputs="f32", rot=128, interleaved=False, norm=True, **k):
    # (codes that are whole numbers compare by equality, and where a value falls between two of them the last bit of a norm decides: e4m3 only)
    return _case(name, "append8", *a, inputs=inputs, rot=rot, interleaved=interleaved, norm=norm, **k)


def _sample(name, rows, vocab, mix, type="f32", spread=2.0, masked=0.0, pad=0):
    return dict(name=name, kind="sample", rows=rows, vocab=vocab, mix=mix, type=type, spread=spread, masked=masked, pad=pad)


def listed():
    return [
        # one token of one long conversation: the call's latency is what counts
        _append("append8_one", 1, (1, 1), (4001, 4001)),
        # a decode step of a serving batch, projections in f32 as the quantized matrices leave them
        _append("append8_batch_128", 128, (1, 1), (24, 264), type="bf16"),
        # a step that takes several prompts in, one projection for q, k and v in 16 bits (so rows with a stride)
        _append("append8_prompts", 7, (1, 1999), (0, 300), inputs="f16", page=64),
        # the benchmark's prompt
        _case("prompt8_512", "prompt8", 1, (512, 512), (0, 0)),
        # one long prompt
        _case("prompt8_8192", "prompt8", 1, (8192, 8192), (0, 0), type="bf16", page=64),
        # chunks of prompts whose beginnings are cached already; small heads, a group of seven
        _case("prompt8_chunks", "prompt8", 4, (37, 301), (900, 8000), heads=(14, 2, 64), cache="i8"),
        # one long conversation
        _case("decode8_one", "decode8", 1, (1, 1), (4001, 4001)),
        # a serving batch of conversations of very different lengths
        _case("decode8_batch_32", "decode8", 32, (1, 1), (150, 8000), type="bf16", cache="i8", page=32),
        # many conversations behind a long system prompt
        _case("decode8_shared_256", "decode8", 256, (1, 1), (3, 600), type="bf16", shared=4096),
        # the next token of one conversation, by the settings that its model's makers recommend
        _sample("sample_one", 1, 151936, "top_k"),
        # a decode step of a serving batch, each request with settings of its own, one of them with nothing left by its grammar
        _sample("sample_batch_128", 128, 151936, "mixed", masked=0.2),
        # undecided rows of a 16-bit head, many tokens in each nucleus; rows of a padded vocabulary
        _sample("sample_flat_64", 64, 151936, "top_p", type="bf16", spread=1.0, pad=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 4, 128), (32, 4, 128), (16, 1, 128), (8, 8, 64), (14, 2, 64), (5, 1, 128), (40, 8, 64)]


def draw(rng):
    kind = rng.choice(["append8", "prompt8", "decode8", "sample"])
    heads, page, type_, cache = rng.choice(HEADS), rng.choice([16, 32, 64, 128]), rng.choice(["f16", "bf16"]), rng.choice(["e4m3", "i8"])
    common = dict(heads=heads, page=page, type=type_)
    if kind == "append8":
        n_seq = _log_int(rng, 1, 200)
        most = _log_int(rng, 1, max(1, 8192 // n_seq))
        rot = rng.choice([heads[2], heads[2], heads[2] // 2, heads[2] // 4])
        c = _append("", n_seq, (rng.randint(1, most), most), (0, _log_int(rng, 1, 4000)), inputs=rng.choice(["f32", type_]), rot=rot,
                    interleaved=rng.random() < 0.5, norm=rng.random() < 0.6, **common)
    elif kind == "prompt8":
        n_seq = _log_int(rng, 1, 12)
        most = _log_int(rng, 20, 8000 // n_seq)
        ctx = rng.choice([0, _log_int(rng, 1, 8000 // n_seq)])
        c = _case("", "prompt8", n_seq, (rng.randint(1, most), most), (0, ctx), cache=cache, **common)
    elif kind == "decode8":
        n_seq = _log_int(rng, 1, 256)
        shared = rng.choice([0, 0, page * _log_int(rng, 1, 2560 // page)])
        most = _log_int(rng, 1, min(30000, 100000 // n_seq))
        c = _case("", "decode8", n_seq, (1, rng.choice([1, 1, 1, 3])), (rng.randint(0, most), most), cache=cache, shared=shared, **common)
    else:
        c = _sample("", _log_int(rng, 1, 128), _log_int(rng, 300, 151936), rng.choice(["mixed", "mixed", "top_k", "top_p", "min_p", "none"]),
                    type=rng.choice(["f32", "f32", "f16", "bf16"]), spread=round(rng.uniform(0.5, 5.0), 2), masked=rng.choice([0.0, 0.0, 0.3, 0.999]),
                    pad=rng.choice([0, 0, 1, 64]))
    del c["name"]
    return c


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
    if case["kind"] == "sample":
        values = case["rows"] * case["vocab"]
        return dict(bytes=values * (4 if case["type"] == "f32" else 2) + 28 * case["rows"], flops=4 * values)
    (q, kv), H, K, D = _lengths(case), case["n_head"], case["n_head_kv"], case["hd"]
    tokens = sum(q)
    if case["kind"] == "append8":
        wide = 4 if case["inputs"] == "f32" else 2
        positions = len({m - 1 - i for n, m in zip(q, kv) for i in range(n)})
        blocks = sum(-(-m // BLOCK) - (m - n) // BLOCK for n, m in zip(q, kv))
        return dict(bytes=tokens * (H * D * (wide + 2) + 2 * K * D * (wide + 1)) + positions * case["rot"] * 4 + 4 * tokens + 2 * blocks * K,
                    flops=tokens * (H + K) * (case["rot"] * 3 + (4 * D if case["norm"] else 0)) + tokens * 4 * K * D)
    cached = case["shared"] + sum(m - case["shared"] for m in kv)
    return dict(bytes=4 * tokens * H * D + 2 * cached * K * D + 2 * -(-cached // BLOCK) * K + 4 * -(-cached // case["page"]), flops=4 * D * H * _pairs(case))


# ---- what a program has in hand ------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _rope_table(case, rows):
    """[rows][rot / 2][2]: sine and cosine of position * base^(-2 i / rot), as a model loader tabulates them once."""
    pos = torch.arange(rows, dtype=torch.float64, device="cuda")
    freq = 1e6 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"])
    a = pos[:, None] * freq
    return torch.stack([a.sin(), a.cos()], dim=-1).float().contiguous()


def _cached(case, n_pages, gen):
    """A pool's codes and scales: values of about 1, of some blocks a few times as large as of others."""
    K, D, page = case["n_head_kv"], case["hd"], case["page"]
    e4m3 = case["cache"] == "e4m3"
    codes = torch.randn(n_pages, K, page, D, device="cuda", generator=gen) * (110.0 if e4m3 else 36.0)
    codes = codes.clamp(-448, 448).to(torch.float8_e4m3fn) if e4m3 else codes.round().clamp(-127, 127).to(torch.int8)
    scales = torch.randint(117 if e4m3 else 120, 121 if e4m3 else 124, (n_pages, K, page // BLOCK), dtype=torch.uint8, device="cuda", generator=gen)
    return codes, scales.view(torch.float8_e8m0fnu)


def _inputs(case, seed):
    """Everything that is data, on the GPU; the same for either side."""
    gen = _gen(seed)
    rand = lambda *shape: torch.randn(shape, device="cuda", generator=gen)  # noqa: E731
    if case["kind"] == "sample":
        return _rows_of_logits(case, gen, rand)
    q, kv = _lengths(case)
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
    d = dict(case, q_len=np.array(q, np.int32), kv_len=np.array(kv, np.int32), table=table, n_pages=n_pages, tokens=tokens)
    d["k_pages"], d["k_scales"] = _cached(case, n_pages, gen)
    d["v_pages"], d["v_scales"] = _cached(case, n_pages, gen)
    if case["kind"] == "append8":
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


def _rows_of_logits(case, gen, rand):
    """Logits of `spread`, some dozens in each row well above the others, as a language model's are; the rows' settings and uniform numbers."""
    n, V, t = case["rows"], case["vocab"], TYPES[case["type"]]
    uniform = lambda *shape: torch.rand(shape, device="cuda", generator=gen)  # noqa: E731
    x = rand(n, V + case["pad"]) * case["spread"]
    at = torch.randint(0, V, (n, 40), device="cuda", generator=gen)
    x.scatter_add_(1, at, -2.0 * case["spread"] * torch.log(uniform(n, 40).clamp_min(1e-6)))
    if case["masked"]:
        x.masked_fill_(uniform(n, V + case["pad"]) < case["masked"], -math.inf)
        x[n // 2] = -math.inf if n > 3 else x[n // 2]
    whole = x.to(t)
    mix, row = case["mix"], torch.arange(n, device="cuda")
    on = lambda what, by, off: torch.where(row % 5 != by, what, off) if mix == "mixed" else what  # noqa: E731
    none_k, none_p, none_m = (torch.zeros(n, dtype=torch.int32, device="cuda"), torch.ones(n, device="cuda"), torch.zeros(n, device="cuda"))
    ks = torch.tensor([20, 50, 1, 300, 5000], dtype=torch.int32, device="cuda")[row % 5]
    ps = torch.tensor([0.8, 0.95, 0.9, 0.5, 0.99], device="cuda")[row % 5]
    ms = torch.tensor([0.05, 0.01, 0.1, 0.02, 0.3], device="cuda")[row % 5]
    temperature = 0.6 + 0.8 * uniform(n)
    return dict(case, whole=whole, logits=whole[:, :V], u=uniform(n), token=torch.empty(n, dtype=torch.int32, device="cuda"), prob=torch.empty(n, device="cuda"),
                temperature=torch.where(row % 8 == 7, torch.zeros_like(temperature), temperature) if mix == "mixed" else temperature,
                top_k=on(torch.full_like(ks, 20) if mix == "top_k" else ks, 1, none_k) if mix in ("mixed", "top_k") else none_k,
                top_p=on(ps, 2, none_p) if mix in ("mixed", "top_k", "top_p") else none_p,
                min_p=on(ms, 3, none_m) if mix in ("mixed", "min_p") else none_m)


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "sample":
        return s
    # what both sides keep of the batch's shape: the sequence, position, page and slot of every new token
    seq = np.repeat(np.arange(len(s["q_len"])), s["q_len"])
    pos = np.concatenate([np.arange(m - n, m) for n, m in zip(s["q_len"], s["kv_len"])])
    s.update(seq=torch.from_numpy(seq).cuda(), pos=torch.from_numpy(pos).cuda(), pages=torch.from_numpy(s["table"]).cuda().long(),
             kv=torch.from_numpy(s["kv_len"]).cuda().long(), first=torch.from_numpy(np.cumsum(s["q_len"]) - s["q_len"]).cuda())
    if own:
        from llamd_rs_b200 import paged
        # the batch's plan: made once per step, used by every layer of a model
        s["batch"] = paged.Batch(s["n_head"], s["n_head_kv"], s["hd"], s["page"], s["type"], cache=s["cache"])
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


def _store(y, s, pages, scales):
    """The rows y [tokens][heads][hd] into their slots; blocks whose largest value has grown take a larger scale, and their older rows with it."""
    high, low_e, high_e = FORMATS[s["cache"]]
    t, sc = pages.dtype, scales.view(torch.uint8)
    page, slot = s["pages"][s["seq"], s["pos"] // s["page"]], s["pos"] % s["page"]
    P, K, B = sc.shape
    of = page * B + slot // BLOCK                                                       # a token's block, of all pages'
    last = s["pos"][s["first"]][s["seq"]]                                               # positions that the sequence had before
    held = (last - s["pos"] // BLOCK * BLOCK).clamp(0, BLOCK)                           # rows that the block had
    most = torch.zeros(P * B, K, device="cuda").index_reduce_(0, of, y.abs().amax(-1), "amax")
    fraction, e = torch.frexp(most / high)
    e = torch.where(fraction == 0.5, e - 1, e).masked_fill(most == 0, low_e).clamp(low_e, high_e)
    rows = torch.zeros(P * B, dtype=torch.long, device="cuda").index_put_((of,), held)
    was = sc.permute(0, 2, 1).reshape(P * B, K).int() - 127
    touched = torch.zeros(P * B, dtype=torch.bool, device="cuda").index_fill_(0, of, True)
    e = torch.where(rows[:, None] > 0, torch.maximum(e, was), e)
    e = torch.where(touched[:, None], e, was)
    # the older rows of blocks with new ones
    old = pages.unflatten(2, (B, BLOCK)).permute(0, 2, 1, 3, 4).reshape(P * B, K, BLOCK, -1).float()
    again = _coded(old * torch.exp2((was - e).float())[..., None, None], s["cache"]).float()
    mine = (torch.arange(BLOCK, device="cuda") < rows[:, None])[:, None, :, None]
    old = torch.where(mine, again, old).to(t)
    pages.copy_(old.unflatten(0, (P, B)).permute(0, 2, 1, 3, 4).flatten(2, 3))
    sc.copy_((e + 127).to(torch.uint8).unflatten(0, (P, B)).permute(0, 2, 1))
    codes = _coded(y * torch.exp2(-e[of].float())[..., None], s["cache"])
    pages.view(torch.uint8)[page, :, slot] = codes.view(torch.uint8)


def _coded(x, cache):
    high = FORMATS[cache][0]
    x = x.clamp(-high, high)
    return x.to(torch.float8_e4m3fn) if cache == "e4m3" else x.round().to(torch.int8)


def _plain_append(s):
    s["q_out"] = _rotated(_normed(s["q"], s["wq"], s), s).to(TYPES[s["type"]])
    _store(_rotated(_normed(s["k"], s["wk"], s), s), s, s["k_pages"], s["k_scales"])
    _store(s["v"].float(), s, s["v_pages"], s["v_scales"])
    return _appended(s)


def _appended(s):
    return {"q": s["q_out"], **{x: s[x] for x in ("k_pages", "k_scales", "v_pages", "v_scales")}}


def _rows(pages, scales, table):
    """The cached rows of a table of pages [..., n]: [..., n * page][heads][hd], in 32 bits."""
    x = pages[table].float()
    e = scales.view(torch.uint8)[table].float() - 127
    x = x * torch.exp2(e).repeat_interleave(BLOCK, -1)[..., None]
    return x.transpose(-3, -2).flatten(-4, -3)


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
        k, v = _rows(s["k_pages"], s["k_scales"], table)[:m], _rows(s["v_pages"], s["v_scales"], table)[:m]
        seen = torch.arange(m, device="cuda") <= torch.arange(m - n, m, device="cuda")[:, None]
        out.append(_attended(s["q"][at:at + n].float(), k, v, seen))
        at += n
    return torch.cat(out).to(s["q"].dtype)


def _plain_decode(s):
    """Every sequence padded to the longest, its tokens to the most."""
    most, wide = int(s["q_len"].max()), int(s["kv_len"].max())
    k, v = _rows(s["k_pages"], s["k_scales"], s["pages"])[:, :wide], _rows(s["v_pages"], s["v_scales"], s["pages"])[:, :wide]
    at = s["pos"] - s["pos"][s["first"]][s["seq"]]
    q = torch.zeros((len(s["q_len"]), most) + s["q"].shape[1:], device="cuda")
    q[s["seq"], at] = s["q"].float()
    last = s["pos"][s["first"]][:, None] + torch.arange(most, device="cuda")
    out = _attended(q, k, v, torch.arange(wide, device="cuda") <= last[:, :, None])
    return out[s["seq"], at].to(s["q"].dtype)


def _plain_sample(s):
    """In 64 bits: which token a number falls on, and where a nucleus ends, is decided by values next to a border."""
    x = s["logits"].double()
    n, V = x.shape
    sorted_x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    top = sorted_x[:, :1]
    greedy, empty = (s["temperature"] <= 0)[:, None], top == -math.inf
    z = (sorted_x - top.masked_fill(empty, 0.0)) / s["temperature"].double()[:, None].masked_fill(greedy, 1.0)
    w = torch.exp(z)
    rank = torch.arange(V, device="cuda")
    k = torch.where((s["top_k"] > 0) & ~greedy[:, 0], s["top_k"].long(), torch.where(greedy[:, 0], 1, V))[:, None]
    w = w.masked_fill(rank >= k, 0.0)
    before = w.cumsum(-1) - w
    p = s["top_p"].double()[:, None]
    out = (p < 1) & (before >= p * w.sum(-1, keepdim=True)) & (rank > 0)
    w = w.masked_fill(out | (w < s["min_p"].double()[:, None] * w[:, :1]), 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    total = w.cumsum(-1)
    over = total > s["u"].double()[:, None] * total[:, -1:]
    token = over.int().argmax(-1, keepdim=True)
    s["token"].copy_(token.masked_fill(empty, -1)[:, 0])
    s["prob"].copy_((w.gather(1, token) / total[:, -1:]).masked_fill(empty, 0.0)[:, 0])
    return {"token": s["token"], "prob": s["prob"]}


def run(s):
    if own:
        if s["kind"] == "append8":
            s["batch"].append(s["q"], s["k"], s["v"], s["q_out"], s["k_pages"], s["v_pages"], rope=s["rope"], rot=s["rot"], interleaved=s["interleaved"],
                              q_norm=s["wq"] if s["norm"] else None, k_norm=s["wk"] if s["norm"] else None, eps=EPS, k_scales=s["k_scales"], v_scales=s["v_scales"])
            return _appended(s)
        if s["kind"] == "sample":
            from llamd_rs_b200 import sampling
            sampling.sample(s["logits"], s["u"], s["token"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"], prob=s["prob"])
            return {"token": s["token"], "prob": s["prob"]}
        s["batch"].attention(s["q"], s["k_pages"], s["v_pages"], s["out"], k_scales=s["k_scales"], v_scales=s["v_scales"])
        return s["out"]
    return {"append8": _plain_append, "prompt8": _plain_prompt, "decode8": _plain_decode, "sample": _plain_sample}[s["kind"]](s)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------

def _values(pages, scales, page, slot):
    """Cached rows [n][heads][hd] in 64 bits."""
    e = scales.view(torch.uint8)[page, :, slot // BLOCK].double() - 127
    return pages[page].double()[torch.arange(len(page), device="cuda"), :, slot] * torch.pow(2.0, e)[..., None]


def _exact_append(s):
    """q as it is defined; the caches' codes and scales are roundings, with no value in 64 bits."""
    pos = np.concatenate([np.arange(m - n, m) for n, m in zip(s["q_len"], s["kv_len"])])
    pos = torch.from_numpy(pos).cuda()
    angle = torch.complex(s["rope"][pos, :, 1].double(), s["rope"][pos, :, 0].double())[:, None]  # cos + i sin
    half, x = s["rot"] // 2, s["q"].double()
    if s["norm"]:
        x = x * (x.square().sum(-1, keepdim=True) / s["hd"] + EPS).rsqrt() * s["wq"].double()
    at = torch.arange(half, device="cuda")
    i, j = (2 * at, 2 * at + 1) if s["interleaved"] else (at, at + half)
    z, y = torch.complex(x[..., i], x[..., j]) * angle, x.clone()
    y[..., i], y[..., j] = z.real, z.imag
    return {"q": y, "k_pages": None, "k_scales": None, "v_pages": None, "v_scales": None}


def _exact_sample(s):
    """Row by row on the host: the kept tokens one after the other."""
    logits, u = s["logits"].float().cpu().numpy().astype(np.float64), s["u"].cpu().numpy().astype(np.float64)
    get = lambda x: s[x].cpu().numpy()  # noqa: E731
    T, k, p, m = get("temperature").astype(np.float64), get("top_k"), get("top_p").astype(np.float64), get("min_p").astype(np.float64)
    token, prob = np.full(len(u), -1, np.int64), np.zeros(len(u))
    for r, x in enumerate(logits):
        if x.max() == -np.inf:
            continue
        order = np.argsort(-x, kind="stable")
        order = order[x[order] > -np.inf]
        if T[r] <= 0:
            token[r], prob[r] = order[0], 1.0
            continue
        if k[r] > 0:
            order = order[:k[r]]
        w = np.exp((x[order] - x[order[0]]) / T[r])
        if p[r] < 1:
            reached = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            order = order[:max(1, int(np.searchsorted(reached, p[r] * w.sum(), side="left")))]
            w = w[:len(order)]
        order, w = order[w >= m[r] * w[0]], w[w >= m[r] * w[0]]
        by = np.argsort(order)
        order, w = order[by], w[by]
        c = np.cumsum(w)
        j = min(len(c) - 1, int(np.searchsorted(c, u[r] * c[-1], side="right")))
        token[r], prob[r] = order[j], w[j] / c[-1]
    return {"token": torch.from_numpy(token), "prob": torch.from_numpy(prob)}


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "append8":
        return _exact_append(s)
    if case["kind"] == "sample":
        return _exact_sample(s)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    group, at, page = s["n_head"] // s["n_head_kv"], 0, s["page"]
    for i, (n, m) in enumerate(zip(s["q_len"].tolist(), s["kv_len"].tolist())):
        pos = np.arange(m)
        where = torch.from_numpy(s["table"][i, pos // page]).cuda().long(), torch.from_numpy(pos % page).cuda()
        k, v = _values(s["k_pages"], s["k_scales"], *where), _values(s["v_pages"], s["v_scales"], *where)
        for h in range(s["n_head_kv"]):
            for g in range(group):
                for t in range(0, n, 1024):  # (a slice of the tokens at a time: the scores of all would not fit)
                    e = min(n, t + 1024)
                    x = torch.einsum("td,pd->tp", s["q"][at + t:at + e, h * group + g].double(), k[:, h]) / math.sqrt(s["hd"])
                    ahead = torch.arange(m, device="cuda")[None] > torch.arange(m - n + t, m - n + e, device="cuda")[:, None]
                    out[at + t:at + e, h * group + g] = torch.softmax(x.masked_fill(ahead, -math.inf), -1) @ v[:, h]
        at += n
    return out
