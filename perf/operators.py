"""Workloads of the paged-cache serving operators: writing tokens into pages,
attention of one new token over them, copying pages, and the likelihoods of
the emitted tokens.

``listed()`` names the cases, ``draw(rng)`` gives one more of the same
ranges, ``prepare`` makes a case's inputs on the GPU and ``run`` is one pass:
with ``own`` false in elementary torch operations, with ``own`` true through
the package's entry points.  ``exact`` is the same result in 64 bits."""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

D = 128                      # head dimension of the cache
F8 = torch.float8_e4m3fn     # equals the cache codec on every byte its encoder emits
HEADS = {"40/8": (40, 8), "32/4": (32, 4), "16/2": (16, 2), "8/8": (8, 8), "16/1": (16, 1)}
_mod = None


def _ops():
    global _mod
    if _mod is None:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        pkg = os.path.join(root, "rdna4-quant_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from r4q import ops
        _mod = ops
    return _mod


# ------------------------------------------------------------------- cases ---
def listed():
    return [
        # one decode step of a served batch of 16, the dense model's heads: the new tokens' q, k, v into the cache
        dict(name="write-decode-16", op="write", heads="40/8", tokens=16, seqs=16, page=64, norm=True, scaled=False),
        # several prompts admitted together, ragged, written as they are prefilled
        dict(name="write-prompts-2051", op="write", heads="40/8", tokens=2051, seqs=5, page=32, norm=True, scaled=True),
        # a long prompt in chunks of the mixture model: keys already rotated, a plain write
        dict(name="write-plain-8192", op="write", heads="32/4", tokens=8192, seqs=3, page=16, norm=False, scaled=False),
        # a single short chat: latency
        dict(name="attn-1x128", op="attn", heads="40/8", batch=1, ctx=128, spread="even", page=16, scaled=False, fwht=True),
        # one long document
        dict(name="attn-1x32768", op="attn", heads="40/8", batch=1, ctx=32768, spread="even", page=64, scaled=True, fwht=True),
        # an ordinary served batch, every request at its own length
        dict(name="attn-16x2048-ragged", op="attn", heads="40/8", batch=16, ctx=2048, spread="ragged", page=64, scaled=False, fwht=True),
        # the mixture model's heads at its largest batch, odd lengths, small pages
        dict(name="attn-64x2047-moe", op="attn", heads="32/4", batch=64, ctx=2047, spread="ragged", page=16, scaled=False, fwht=True),
        # the largest: a batch of long documents
        dict(name="attn-16x32768", op="attn", heads="40/8", batch=16, ctx=32768, spread="ragged", page=128, scaled=True, fwht=False),
        # a forked request: its shared tail pages become its own, in every layer
        dict(name="pages-fork-2", op="pages", layers=40, kv=8, page=64, pages=64, moves=2, seqs=4),
        # compaction of a fragmented pool
        dict(name="pages-compact-300", op="pages", layers=24, kv=4, page=32, pages=900, moves=300, seqs=16),
        # the sampled tokens of one decode step, with alternatives
        dict(name="logprobs-16-top20", op="logprobs", rows=16, vocab=151936, k=20, dtype="float16"),
        # the likelihood of a whole prompt
        dict(name="logprobs-2048-top5", op="logprobs", rows=2048, vocab=151936, k=5, dtype="float16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    op = rng.choice(["write", "attn", "pages", "logprobs"])
    if op == "write":
        tokens = _log(rng, 1, 8192)
        return dict(op=op, heads=rng.choice(sorted(HEADS)), tokens=tokens, seqs=min(tokens, _log(rng, 1, 64)),
                    page=rng.choice([16, 32, 48, 64, 128]), norm=rng.random() < 0.7, scaled=rng.random() < 0.5)
    if op == "attn":
        heads = rng.choice(sorted(HEADS))
        ctx = _log(rng, 1, 32768)
        most = max(1, min(64, 16 * 32768 * 8 // (ctx * HEADS[heads][1])))
        return dict(op=op, heads=heads, batch=_log(rng, 1, most), ctx=ctx,
                    spread=rng.choice(["even", "ragged", "one_long"]), page=rng.choice([16, 32, 48, 64, 128]),
                    scaled=rng.random() < 0.5, fwht=rng.random() < 0.5)
    if op == "pages":
        layers, kv, page = rng.choice([2, 24, 40, 48]), rng.choice([1, 2, 4, 8]), rng.choice([16, 32, 48, 64, 128])
        pages = max(4, min(_log(rng, 4, 4096), 450_000_000 // (layers * 2 * kv * page * D)))
        return dict(op=op, layers=layers, kv=kv, page=page, pages=pages, moves=_log(rng, 1, max(1, pages // 3)),
                    seqs=_log(rng, 1, 64))
    vocab = rng.choice([151936, 32003, 50257, 128256, _log(rng, 40, 200000)])
    dtype = rng.choice(["float16", "float16", "bfloat16", "float32"])
    return dict(op=op, rows=_log(rng, 1, 2048 if dtype != "float32" else 1024), vocab=vocab,
                k=rng.choice([0, 1, 5, 20, 32]), dtype=dtype)


def _lengths(case):
    """Lengths of a batch: all alike, spread from a quarter of the longest on, or one long among short ones."""
    b, ctx = case["batch"], case["ctx"]
    if case["spread"] == "even":
        return [ctx] * b
    if case["spread"] == "one_long":
        return [ctx] + [max(1, ctx // 16 - 3 * i) for i in range(1, b)]
    return [max(1, ctx - (i * 2654435761 % (1 << 32)) * (3 * ctx // 4) // (1 << 32)) for i in range(b)]


def _pieces(case):
    """Tokens of each sequence of a ragged write: near equal shares, the last takes the rest."""
    t, s = case["tokens"], case["seqs"]
    at = [0] + sorted(min(t, (i * t + (i * 7919) % max(1, t // (2 * s) + 1)) // s) for i in range(1, s)) + [t]
    return [b - a for a, b in zip(at, at[1:])]


# ------------------------------------------------------------------ inputs ---
def _codes(x):
    """Cache bytes of x as the encoder leaves them: no code below 2^-6, none above 448."""
    x = x.clamp(-448.0, 448.0)
    return torch.where(x.abs() < 2.0 ** -6, torch.zeros_like(x), x).to(F8).view(torch.uint8)


def _pool(pages, kv, page, g, scale):
    out = torch.empty(pages, kv, page, D, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (kv * page * D))
    for i in range(0, pages, step):
        x = torch.randn(out[i:i + step].shape, generator=g, device="cuda")
        out[i:i + step] = _codes(x if scale is None else x / scale[:, None, None])
    return out


def _scales(kv, g):
    """Per-head scales that bring values of a few units near the top of the 8-bit range."""
    return (0.008 + 0.004 * torch.rand(kv, generator=g, device="cuda")).float()


def _table(counts, page, extra, seed):
    """A block table over pages in the scattered order that a pool gets after some use: [seqs, most blocks] and the pool's size."""
    blocks = [-(-n // page) for n in counts]
    total = sum(blocks) + extra
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).int()
    table = torch.zeros(len(counts), max(1, max(blocks)), dtype=torch.int32)
    at = 0
    for i, n in enumerate(blocks):
        table[i, :n] = order[at:at + n]
        at += n
    return table.cuda(), total


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op == "write":
        h, kv = HEADS[case["heads"]]
        m, page = case["tokens"], case["page"]
        pieces = _pieces(case)
        start = [(173 * i + 5) % 900 for i in range(len(pieces))]
        table, total = _table([a + n for a, n in zip(start, pieces)], page, 3, seed)
        scale = _scales(kv, g) if case["scaled"] else None
        qkv = torch.randn(m, (h + 2 * kv) * D, generator=g, device="cuda").half()
        freq = 1e6 ** (-torch.arange(0, D, 2, device="cuda").float() / D)
        rows_of_table = table.shape[1] * page
        angle = torch.outer(torch.arange(rows_of_table, device="cuda").float(), freq)
        return dict(case=case, q=qkv[:, :h * D].view(m, h, D), k=qkv[:, h * D:(h + kv) * D].view(m, kv, D),
                    v=qkv[:, (h + kv) * D:].view(m, kv, D), table=table,
                    kp=_pool(total, kv, page, g, scale), vp=_pool(total, kv, page, g, scale),
                    pos=torch.cat([torch.arange(a, a + n) for a, n in zip(start, pieces)]).cuda(),
                    rows=torch.cat([torch.full((n,), i) for i, n in enumerate(pieces)]).int().cuda(),
                    scale=scale, cos=angle.cos().half(), sin=angle.sin().half(),
                    qw=(1 + 0.1 * torch.randn(D, generator=g, device="cuda")).half(),
                    kw=(1 + 0.1 * torch.randn(D, generator=g, device="cuda")).half())
    if op == "attn":
        h, kv = HEADS[case["heads"]]
        lens = _lengths(case)
        table, total = _table(lens, case["page"], 3, seed)
        scale = _scales(kv, g) if case["scaled"] else None
        return dict(case=case, q=torch.randn(case["batch"], h, D, generator=g, device="cuda").half(), table=table,
                    seq=torch.tensor(lens, dtype=torch.int64).cuda(), scale=scale,
                    kp=_pool(total, kv, case["page"], g, scale), vp=_pool(total, kv, case["page"], g, scale))
    if op == "pages":
        n, moves = case["pages"], min(case["moves"], case["pages"] // 2)
        r = random.Random(seed)
        ids = list(range(n))
        r.shuffle(ids)
        src, dst = ids[:moves], ids[moves:2 * moves]
        cols = max(1, -(-n // case["seqs"]))
        cells = r.sample(range(case["seqs"] * cols), moves)
        pool = torch.randn(case["layers"], 2, n, case["kv"], case["page"], D, generator=g, device="cuda",
                           dtype=torch.float16)
        return dict(case=case, pool=_codes(pool), src=src, dst=dst, rows=[c // cols for c in cells],
                    cols=[c % cols for c in cells],
                    table=torch.randint(0, n, (case["seqs"], cols), generator=g, device="cuda", dtype=torch.int32))
    m, v = case["rows"], case["vocab"]
    x = torch.randn(m, v, generator=g, device="cuda").mul_(2.5)
    # a few likely tokens stand out, as they do in a model's logits
    hot = torch.randint(0, v, (m, min(8, v)), generator=g, device="cuda")
    x.scatter_(1, hot, 8 + 6 * torch.rand(hot.shape, generator=g, device="cuda"))
    tok = torch.where(torch.rand(m, generator=g, device="cuda") < 0.7, hot[:, 0],
                      torch.randint(0, v, (m,), generator=g, device="cuda"))
    return dict(case=case, logits=x.to(getattr(torch, case["dtype"])), tokens=tok)


# ------------------------------------------------------------- plain forms ---
def _rotate(x, cos, sin):
    a, b = x[..., :D // 2], x[..., D // 2:]
    c, s = cos.float()[:, None], sin.float()[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _normed(x, w, eps=1e-6):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.float()


def _encoded(x):
    """The cache codec: three mantissa bits, ties away from zero, below 2^-6 nothing, above 448 that."""
    a = x.abs().clamp(max=448.0)
    step = torch.ldexp(torch.ones_like(a), torch.frexp(a).exponent - 4)
    r = torch.floor(a / step + 0.5) * step
    r = torch.where(r < 2.0 ** -6, torch.zeros_like(r), r).clamp(max=448.0)
    return torch.copysign(r, x).to(F8).view(torch.uint8)


def _plain_write(s):
    c = s["case"]
    page = c["page"]
    k, v = s["k"].float(), s["v"].float()
    if c["norm"]:
        cos, sin = s["cos"][s["pos"]], s["sin"][s["pos"]]
        q, k = (_rotate(_normed(x, w), cos, sin) for x, w in ((s["q"], s["qw"]), (k, s["kw"])))
    where = s["table"][s["rows"].long(), s["pos"] // page].long()
    sc = 1.0 if s["scale"] is None else s["scale"][None, :, None]
    s["kp"][where, :, s["pos"] % page] = _encoded(k / sc)
    s["vp"][where, :, s["pos"] % page] = _encoded(v / sc)
    out = {"k": s["kp"].view(F8), "v": s["vp"].view(F8)}
    return dict(out, q=q.half()) if c["norm"] else out


def _hadamard32(dtype):
    h = torch.ones(1, 1, dtype=dtype, device="cuda")
    for _ in range(5):
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h / math.sqrt(32)


def _plain_attn(s):
    b, h, _ = s["q"].shape
    kv = s["kp"].shape[1]
    table = s["table"].long()
    k, v = (p.view(torch.uint8)[table].permute(0, 2, 1, 3, 4).reshape(b, kv, -1, D).view(F8).float()
            for p in (s["kp"], s["vp"]))
    scores = s["q"].float().view(b, kv, h // kv, D) @ k.transpose(-1, -2) / math.sqrt(D)
    if s["scale"] is not None:
        scores = scores * s["scale"][None, :, None, None]
    out_of = torch.arange(k.shape[2], device="cuda")[None, :] >= s["seq"][:, None]
    scores = scores.masked_fill(out_of[:, None, None], float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    o = p @ v / p.sum(-1, keepdim=True)
    if s["scale"] is not None:
        o = o * s["scale"][None, :, None, None]
    o = o.view(b, h, D)
    if s["case"]["fwht"]:
        o = (o.view(b, h, D // 32, 32) @ _hadamard32(torch.float32)).view(b, h, D)
    return o.half()


def _plain_pages(s):
    src, dst, rows, cols = (torch.tensor(s[n], device="cuda") for n in ("src", "dst", "rows", "cols"))
    s["pool"][:, :, dst] = s["pool"][:, :, src]
    s["table"][rows, cols] = dst.int()
    return {"pool": s["pool"].view(F8), "table": s["table"]}


def _plain_logprobs(s):
    x, k = s["logits"].float(), s["case"]["k"]
    m, v = x.shape
    t = s["tokens"][:, None]
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    entropy = torch.log(total) - (e * (x - top)).sum(-1, keepdim=True) / total
    xt = x.gather(1, t)
    index = torch.arange(v, device="cuda")
    rank = (x > xt).sum(-1) + ((x == xt) & (index < t)).sum(-1) + 1
    if k:
        bits = (x + 0.0).view(torch.int32)
        key = (bits ^ ((bits >> 31) & 0x7fffffff)).long() * (1 << 32) + (v - 1 - index)
        ids = v - 1 - (torch.topk(key, k, -1, sorted=True).values & 0xffffffff)
    else:
        ids = torch.empty(m, 0, dtype=torch.int64, device="cuda")
    return {"logprob": (xt - lse)[:, 0], "rank": rank, "entropy": entropy[:, 0], "ids": ids,
            "top": x.gather(1, ids) - lse}


# ---------------------------------------------------------------- one pass ---
def run(state):
    op = state["case"]["op"]
    if not own:
        return {"write": _plain_write, "attn": _plain_attn, "pages": _plain_pages, "logprobs": _plain_logprobs}[op](state)
    ops, s = _ops(), state
    if op == "write":
        norm = dict(q=s["q"], q_w=s["qw"], k_w=s["kw"], cos=s["cos"], sin=s["sin"]) if s["case"]["norm"] else {}
        q = ops.paged_kv_write(s["k"], s["v"], s["kp"], s["vp"], s["table"], s["pos"], rows=s["rows"],
                               k_scale=s["scale"], v_scale=s["scale"], **norm)
        out = {"k": s["kp"].view(F8), "v": s["vp"].view(F8)}
        return dict(out, q=q) if s["case"]["norm"] else out
    if op == "attn":
        return ops.paged_flash_decode(s["q"], s["kp"], s["vp"], s["table"], s["seq"], k_scale=s["scale"],
                                      v_scale=s["scale"], fwht=s["case"]["fwht"])
    if op == "pages":
        ops.kv_copy_pages(s["pool"], s["src"], s["dst"])
        ops.kv_table_set(s["table"], s["rows"], s["cols"], s["dst"])
        return {"pool": s["pool"].view(F8), "table": s["table"]}
    r = ops.token_logprobs(s["logits"], s["tokens"], s["case"]["k"])
    return {"logprob": r.logprob, "rank": r.rank, "entropy": r.entropy, "ids": r.top_ids, "top": r.top_logprobs}


def work(case):
    op = case["op"]
    if op == "write":
        h, kv = HEADS[case["heads"]]
        m = case["tokens"]
        norm = (h * D * 4 + D * 2) * case["norm"]     # q in and out, a row of the angle tables
        return {"bytes": m * (2 * kv * D * 3 + 12 + norm), "flops": m * (h + kv) * D * 7 * case["norm"]}
    if op == "attn":
        h, kv = HEADS[case["heads"]]
        lens = _lengths(case)
        n = sum(lens)
        return {"bytes": n * kv * D * 2 + len(lens) * h * D * 4 + 4 * sum(-(-x // case["page"]) for x in lens),
                "flops": 4 * n * h * D}
    if op == "pages":
        moves = min(case["moves"], case["pages"] // 2)
        return {"bytes": 2 * moves * case["layers"] * 2 * case["kv"] * case["page"] * D + 4 * moves, "flops": 0}
    size = 4 if case["dtype"] == "float32" else 2
    return {"bytes": case["rows"] * (case["vocab"] * size + 24 + 12 * case["k"]), "flops": 6 * case["rows"] * case["vocab"]}


# ---------------------------------------------------------------- in 64 bits ---
def exact(case, seed):
    op = case["op"]
    if op == "pages":
        return None                                   # bytes and whole numbers alone
    s = prepare(case, seed)
    if op == "write":
        if not case["norm"]:
            return None                               # the codes alone
        h = s["q"].double()
        h = h / (h.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * s["qw"].double()
        z = torch.complex(h[..., :64], h[..., 64:]) * torch.complex(s["cos"].double(), s["sin"].double())[s["pos"]][:, None]
        return {"q": torch.cat([z.real, z.imag], -1), "k": None, "v": None}
    if op == "attn":
        h, kv = HEADS[case["heads"]]
        value = torch.arange(256, dtype=torch.uint8, device="cuda").view(F8).double()
        page, out = case["page"], torch.zeros(case["batch"], h, D, dtype=torch.float64, device="cuda")
        for b, n in enumerate(_lengths(case)):
            ids = s["table"][b, :-(-n // page)].long()
            for j in range(kv):
                key, val = (value[p[ids, j].reshape(-1, D)[:n].long()] for p in (s["kp"], s["vp"]))
                sc = 1.0 if s["scale"] is None else s["scale"][j].double()
                heads = slice(j * (h // kv), (j + 1) * (h // kv))
                w = torch.softmax(s["q"][b, heads].double() @ key.t() * (sc / math.sqrt(D)), -1)
                out[b, heads] = w @ val * sc
        if case["fwht"]:
            x = out.view(-1, 2, 2, 2, 2, 2)
            for axis in range(1, 6):
                x = torch.stack([x.sum(axis), x.select(axis, 0) - x.select(axis, 1)], axis)
            out = (x / math.sqrt(32)).reshape(out.shape)
        return out
    t, k = s["tokens"], case["k"]
    parts = []
    for i in range(0, case["rows"], 256):
        x = s["logits"][i:i + 256].double()
        lp = torch.log_softmax(x, -1)
        parts.append((lp.gather(1, t[i:i + 256, None])[:, 0], -(lp.exp() * lp).sum(-1), lp.topk(k, -1).values))
    lp, ent, top = (torch.cat(p) for p in zip(*parts))
    return {"logprob": lp, "rank": None, "entropy": ent, "ids": None, "top": top}
