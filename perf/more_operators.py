"""Cases of rotary positions with several axes, the 4-bit paged cache and page tables planned on the GPU.

Each case is one call (or one training step) of an operator as a program makes it:

* ``rotate``: qknorm_rope_scale_gqa forward and backward, each rotation pair turned by the position of its axis;
* ``append``: append_paged_kv_int4 of new tokens to a paged cache held in 4 bits;
* ``attend``: paged_attention_int4 of new tokens over such a cache;
* ``plan``: plan_paged_step, a step's pages, lengths, positions and slots from the requests' lengths.

The 4-bit format: a row's channels are in D / 32 groups of 32, group g the channels c with
(c // 8) % (D / 32) == g. A group has a scale s: -1/8 of its value of largest magnitude, cut to five
significant bits; a channel has a code clamp(rint(x / s), -8, 7) and stands for s * code.

``own`` selects the framework's kernels; otherwise the same results come from elementary torch
operations in 32 bits (the statistic of a row that is rounded to codes in 64), rounded once at the end.
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = float(np.float32(1e-5))


def listed():
    return [
        # one image with its question: latency of one fine-tuning step (time, height, width in blocks of pairs)
        dict(name="rotate image", op="rotate", dense=False, rows=300, batch=1, heads=16, kv_heads=4, dim=64, axes=3,
             interleaved=False, dtype="bf16"),
        # packed video documents, the axes' pairs interleaved
        dict(name="rotate video", op="rotate", dense=False, rows=65536, batch=1, heads=32, kv_heads=8, dim=128, axes=3,
             interleaved=True, dtype="bf16"),
        # a dense batch of images in full precision: two axes, odd length
        dict(name="rotate dense fp32", op="rotate", dense=True, rows=1023, batch=4, heads=24, kv_heads=8, dim=128, axes=2,
             interleaved=False, dtype="fp32"),
        # one decoding step of 32 running requests
        dict(name="append decode", op="append", batch=32, chunk=1, length=200, heads=32, kv_heads=8, dim=128, page=16,
             dtype="bf16", norm=True, axes=0, mix=1),
        # prompts with images: ragged chunks, positions of three axes
        dict(name="append chunks", op="append", batch=8, chunk=4096, length=4500, heads=32, kv_heads=8, dim=128, page=64,
             dtype="bf16", norm=True, axes=3, mix=2),
        # a lone conversation: latency
        dict(name="attend one", op="attend", batch=1, chunk=1, length=1000, heads=32, kv_heads=8, dim=128, page=16,
             dtype="bf16", window=0, lse=False, mix=3),
        # a decoding step of a busy server: 64 requests of uneven lengths
        dict(name="attend batch", op="attend", batch=64, chunk=1, length=8192, heads=32, kv_heads=8, dim=128, page=16,
             dtype="bf16", window=0, lse=False, mix=4),
        # two long documents, few key heads: the work has to be split along the cache
        dict(name="attend long", op="attend", batch=2, chunk=1, length=131071, heads=16, kv_heads=2, dim=128, page=64,
             dtype="fp16", window=0, lse=True, mix=5),
        # uneven chunks of prompts with a sliding window
        dict(name="attend chunks", op="attend", batch=6, chunk=2000, length=6000, heads=16, kv_heads=4, dim=64, page=16,
             dtype="fp16", window=1024, lse=False, mix=6),
        # a long prompt's last chunk over what is cached already
        dict(name="attend prompt", op="attend", batch=1, chunk=4096, length=16384, heads=32, kv_heads=8, dim=128, page=64,
             dtype="bf16", window=0, lse=False, mix=7),
        # the tables of a decoding step of 256 requests, some of which have ended
        dict(name="plan decode", op="plan", batch=256, chunk=1, length=8192, page=16, ended=0.05, mix=8),
        # the tables of a step of prompts
        dict(name="plan prompts", op="plan", batch=33, chunk=4096, length=30000, page=16, ended=0.1, mix=9),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _most():
    """The costliest listed case's bytes and operations."""
    got = [work(c) for c in listed()]
    return max(w["bytes"] for w in got), max(w["flops"] for w in got)


def draw(rng):
    most_bytes, most_flops = _most()
    while True:
        op = rng.choice(["rotate", "append", "attend", "attend", "attend", "plan"])
        case = dict(op=op)
        if op != "plan":
            group, kv = rng.choice([(1, 16), (2, 8), (4, 8), (8, 4), (4, 4), (8, 2), (5, 8), (16, 1), (3, 5), (7, 4)])
            case.update(heads=group * kv, kv_heads=kv)
        if op == "rotate":
            dense = rng.random() < 0.4
            case.update(dense=dense, rows=_log_int(rng, 1, 4096 if dense else 65536),
                        batch=rng.randint(1, 6) if dense else 1, dim=rng.choice([32, 64, 128, 256]),
                        axes=rng.randint(2, 4), interleaved=rng.random() < 0.5,
                        dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
        elif op == "plan":
            case.update(batch=_log_int(rng, 1, 1024), chunk=1 if rng.random() < 0.5 else _log_int(rng, 2, 4096),
                        length=_log_int(rng, 1, 32768), page=rng.choice([8, 16, 32, 64, 128, 256]),
                        ended=rng.choice([0.0, 0.1, 0.5]), mix=rng.randint(10, 1 << 20))
            case["chunk"] = min(case["chunk"], case["length"])
            if case["batch"] * case["chunk"] > 1 << 18:
                continue
        else:
            case.update(batch=_log_int(rng, 1, 96), page=rng.choice([8, 16, 32, 64, 128, 256]),
                        dim=rng.choice([64, 128]), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                        mix=rng.randint(10, 1 << 20))
            length = _log_int(rng, 1, 131072 if op == "attend" else 8192)
            chunk = 1 if rng.random() < 0.4 else min(length, _log_int(rng, 2, 4096))
            case.update(length=length, chunk=chunk)
            if op == "append":
                case.update(norm=rng.random() < 0.7, axes=rng.choice([0, 0, 1, 2, 3, 4]))
            else:
                case.update(window=rng.choice([0, 0, 0, 128, 1000, 4096]), lse=rng.random() < 0.3)
            padded = case["batch"] * length
            most = 8 * 4500 * 8 * 128 if op == "append" else 64 * 8192 * 8 * 128
            if padded * case["kv_heads"] * case["dim"] > most or (
                    op == "attend" and padded * chunk * case["heads"] > 32 * 4096 * 16384):
                continue
        w = work(case)
        if w["bytes"] <= most_bytes and w["flops"] <= most_flops:
            return case


def _ragged(case):
    """New tokens and total lengths of each request: the first one's are the case's largest, the others' uneven."""
    rng = random.Random(case["mix"])
    news, totals = [], []
    for b in range(case["batch"]):
        new = case["chunk"] if b == 0 or case["chunk"] == 1 else rng.randint(0, case["chunk"])
        total = case["length"] if b == 0 else rng.randint(max(new, case["length"] // 8), case["length"])
        news.append(new)
        totals.append(total)
    return news, totals


def _requests(case):
    """A plan's requests: tokens held before the step, and new ones (-1: the request has ended)."""
    news, totals = _ragged(case)
    rng = random.Random(case["mix"] + 1)
    ended = [b > 0 and rng.random() < case["ended"] for b in range(case["batch"])]
    return [t - n for n, t in zip(news, totals)], [-1 if e else n for e, n in zip(ended, news)]


def _pairs(new, total, window):
    """Key/query pairs that causal attention of the last `new` of `total` tokens has, and the keys it reaches."""
    first = total - new + 1
    if not window or total <= window:
        return new * (first + total) // 2, total if new else 0
    full = max(0, total - max(first, window) + 1)
    rest = new - full
    return full * window + rest * (2 * first + rest - 1) // 2, min(total, new + window - 1) if new else 0


def work(case):
    if case["op"] == "plan":
        held, news = _requests(case)
        page, tokens = case["page"], sum(max(n, 0) for n in news)
        pages = [-(-h // page) for h in held]
        moved = sum(p if n < 0 else -(-(h + n) // page) - p for h, n, p in zip(held, news, pages))
        # lengths in and out, starts; a page in and out; position, slot and request of each token
        return {"bytes": 16 * case["batch"] + 8 * moved + 16 * tokens, "flops": 0}
    es, D, H, K = BYTES[case["dtype"]], case["dim"], case["heads"], case["kv_heads"]
    if case["op"] == "rotate":
        rows = case["rows"] * case["batch"]
        act = rows * (H + K) * D
        # forward: q, k in and out; backward: q, k and both upstream gradients in, dq, dk out; the tables, the positions twice
        return {"bytes": act * es * 5 + 2 * 4 * case["rows"] * D // 2 + 2 * 4 * rows * case["axes"], "flops": 30 * act}
    news, totals = _ragged(case)
    tokens, row = sum(news), D // 2 + D // 16
    pages = sum(-(-t // case["page"]) for t in totals)
    if case["op"] == "append":
        # q, k, v in, q out, the rows of K and V; and all values that the cache stands for, out
        values = pages * case["page"] * K
        return {"bytes": tokens * ((2 * H + 2 * K) * D * es + 2 * K * row + 4 * D + 4 * case["axes"]) + 4 * pages
                + 2 * values * (row + D * es), "flops": 12 * tokens * (H + 2 * K) * D + 4 * values * D}
    pairs, keys = (sum(x) for x in zip(*(_pairs(n, t, case["window"]) for n, t in zip(news, totals))))
    return {"bytes": 2 * tokens * H * D * es + 2 * keys * K * row + (4 * tokens * H if case["lse"] else 0) + 4 * pages,
            "flops": 4 * pairs * H * D}


def _tables(positions, dim, device):
    inv = 10000.0 ** (-torch.arange(0, dim, 2, device=device, dtype=torch.float64) / dim)
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * inv
    return angle.sin().float(), angle.cos().float()


def _axes(case):
    """The axis of each rotation pair: uneven blocks of pairs, or the axes in turn."""
    half, n = case["dim"] // 2, case["axes"]
    if case.get("interleaved", True):
        return tuple(j % n for j in range(half))
    first = half // (n + 1)
    return tuple(0 if j < first else 1 + (j - first) * (n - 1) // (half - first) for j in range(half))


def _grid_positions(case, shape, g, device):
    """Positions [axes, *shape] of documents of text and pictures: the axes agree in text and part in a picture's grid."""
    n = shape[-1]
    index = torch.arange(n, device=device).expand(shape)
    starts = torch.rand(shape, generator=g, device=device) < 1 / 700
    starts[..., 0] = True
    first = torch.where(starts, index, torch.zeros_like(index)).cummax(-1).values
    at = index - first
    picture = torch.rand(shape, generator=g, device=device).gather(-1, first) < 0.6
    wide = 16
    parts = [at // (wide * wide), at // wide % wide, at % wide, at % 7]
    return torch.stack([torch.where(picture, p, at) for p in parts[:case["axes"]]]).to(torch.int32)


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "plan":
        return _prepare_plan(case, g, device)
    dtype, D, H, K = DTYPES[case["dtype"]], case["dim"], case["heads"], case["kv_heads"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device)

    if case["op"] != "attend":
        s["weight"] = 1 + 0.1 * normal(2, 1, D)
        s["scales"] = math.log(D ** -0.5) + 0.1 * normal(H, 1, 1)
    if case["op"] == "rotate":
        B, N = case["batch"], case["rows"]
        shape = (lambda h: (B, h, N, D)) if case["dense"] else (lambda h: (N, h, D))
        s["q"], s["k"] = (normal(*shape(h)).to(dtype) for h in (H, K))
        s["gq"], s["gk"] = (normal(*shape(h)).to(dtype) for h in (H, K))
        for name in ("q", "k", "weight", "scales"):
            s[name].requires_grad_()
        s["sin"], s["cos"] = _tables(N, D, device)
        s["positions"] = _grid_positions(case, (B, N) if case["dense"] else (N,), g, device)
        s["axes"] = _axes(case)
        s["axis"] = torch.tensor(s["axes"], device=device)
        return s
    news, totals = _ragged(case)
    page, B, tokens = case["page"], case["batch"], sum(news)
    counts = [-(-t // page) for t in totals]
    width, pool = max(counts), sum(counts)
    order = torch.randperm(pool, generator=g, device=device).to(torch.int32)
    rows, columns = torch.arange(B, device=device)[:, None], torch.arange(width, device=device)[None, :]
    used = torch.tensor(counts, device=device)[:, None] > columns
    table = torch.zeros(B, width, dtype=torch.int32, device=device)
    table[used] = order
    s["table"] = table
    s["seq_lens"] = torch.tensor(totals, dtype=torch.int32, device=device)
    ends = torch.tensor([0] + news).cumsum(0)
    s["cu_seqlens"] = None if case["chunk"] == 1 else ends.to(torch.int32).to(device)
    # where the plain form finds each token: its request, and its position in it
    s["request"] = torch.repeat_interleave(torch.arange(B), torch.tensor(news)).to(device)
    s["position"] = (torch.arange(tokens) - ends[:-1].repeat_interleave(torch.tensor(news))
                     + torch.tensor([t - n for n, t in zip(news, totals)]).repeat_interleave(torch.tensor(news))).to(device)
    for name in ("k", "v"):
        s[name + "_cache"] = torch.empty(pool, page, K, D // 2, dtype=torch.uint8, device=device)
        s[name + "_scale"] = torch.empty(pool, page, K, D // 32, dtype=torch.bfloat16, device=device)
        step = max(1, (1 << 25) // (page * K * D))
        for p in range(0, pool, step):
            q = min(pool, p + step)
            s[name + "_cache"][p:q], s[name + "_scale"][p:q] = _pack(normal(q - p, page, K, D).to(dtype).float(), dtype)
    if case["op"] == "append":
        qkv = normal(tokens, H + 2 * K, D).to(dtype)  # the projection's output: strided views of it
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:]
        s["sin"], s["cos"] = _tables(max(totals), D, device)
        if not case["norm"]:
            s["weight"] = None
        s["positions"] = s["axes"] = None
        if case["axes"]:  # text and pictures of each prompt, not beyond its length
            near = _grid_positions(case, (tokens,), g, device)
            s["positions"] = torch.minimum(near, s["position"].to(torch.int32))
            s["axes"] = _axes(case)
            s["axis"] = torch.tensor(s["axes"], device=device)
        return s
    q = normal(tokens, H, D)
    s["q"] = (2 * D ** -0.5 * q * torch.rsqrt(q.square().mean(-1, keepdim=True))).to(dtype)
    # slots that no token was written to yet hold anything
    keys = torch.arange(width * page, device=device)
    slots = table.long()[rows, keys // page] * page + keys % page
    stale = torch.ones(pool * page, dtype=torch.bool, device=device)
    stale[slots[keys < s["seq_lens"][:, None]]] = False
    s["k_scale"][stale.view(pool, page)] = float("nan")
    s["v_scale"][stale.view(pool, page)] = float("nan")
    return s


def _prepare_plan(case, g, device):
    held, news = _requests(case)
    page, B = case["page"], case["batch"]
    counts = [-(-h // page) for h in held]
    width = max(-(-(h + max(n, 0)) // page) for h, n in zip(held, news))
    need = sum(-(-(h + n) // page) - c for h, n, c in zip(held, news, counts) if n >= 0)
    pool = sum(counts) + need + 7
    order = torch.randperm(pool, generator=g, device=device).to(torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32, device=device)
    used = torch.tensor(counts, device=device)[:, None] > torch.arange(width, device=device)
    table[used] = order[:sum(counts)]
    free = torch.full((pool,), -1, dtype=torch.int32, device=device)
    free[:pool - sum(counts)] = order[sum(counts):]
    return {"case": case, "table": table, "free": free, "tokens": sum(max(n, 0) for n in news),
            "free_count": torch.tensor([pool - sum(counts)], dtype=torch.int32, device=device),
            "seq_lens": torch.tensor(held, dtype=torch.int32, device=device),
            "new_lens": torch.tensor(news, dtype=torch.int32, device=device)}


def _pack(x, dtype):
    """FP32 rows [..., D] as codes [..., D/2] (uint8) and scales [..., D/32] (BF16) for a model of type `dtype`."""
    lead, D = x.shape[:-1], x.shape[-1]
    G = D // 32
    x = x.reshape(*lead, 4, G, 8)
    high, low = x.amax((-3, -1), keepdim=True), x.amin((-3, -1), keepdim=True)
    s = -0.125 * torch.where(high >= -low, high, low)
    s = (s.contiguous().view(torch.int32) & -524288).view(torch.float32)  # sign, exponent and four bits of the fraction
    least, most = (2.0 ** -20, 7936.0) if dtype is torch.float16 else (2.0 ** -100, math.inf)
    s = torch.where(s == 0, s, s.sign() * s.abs().clamp(least, most))
    s = torch.where(s.isfinite(), s, math.nan)
    code = torch.where((s == 0) | s.isnan(), 0, (x / s).round().clamp(-8, 7)).to(torch.int32) + 8
    # a byte holds channels 4i and 4i + 2 of its half of eight: bytes 0, 1 the even ones, bytes 2, 3 the odd ones
    c = code.reshape(*lead, D // 8, 2, 2, 2)  # channel 4 h + 2 n + o: [h, n, o]
    b = (c[..., 0, :] | c[..., 1, :] << 4).transpose(-1, -2)  # [o, h]
    return b.reshape(*lead, D // 2).to(torch.uint8), s.reshape(*lead, G).to(torch.bfloat16)


def _values(codes, scales):
    """The FP32 values [..., D] that codes and scales stand for."""
    lead, D = codes.shape[:-1], 2 * codes.shape[-1]
    b = codes.reshape(*lead, D // 8, 2, 2)  # [o, h]
    c = torch.stack((b & 15, b >> 4), -1)  # [o, h, n]
    c = c.permute(*range(len(lead) + 1), -2, -1, -3).reshape(*lead, 4, D // 32, 8)
    return ((c.float() - 8) * scales.float()[..., None, :, None]).reshape(*lead, D)


def _turn(s, positions):
    """sin, cos [..., D/2] of each token by the axes of its pairs, positions [axes, ...] or [...]."""
    if s["axes"] is None:
        return s["sin"][positions], s["cos"][positions]
    at = positions.long()[s["axis"]].movedim(0, -1)
    pair = torch.arange(at.shape[-1], device=at.device)
    return s["sin"][at, pair], s["cos"][at, pair]


def _rotate(x, weight, sin, cos, scale, careful=False):
    """The prologue of rows x [..., D] in 32 bits; sin/cos broadcast to [..., D/2]. careful: the statistic in 64."""
    x = x.float()
    if weight is not None:
        y = x.double() if careful else x
        x = x * (1 / (y.square().mean(-1, keepdim=True) + EPS).sqrt()).float() * weight
    a, b = x.chunk(2, dim=-1)
    x = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return x if scale is None else x * scale.exp()


def _plain_rotate(s):
    sin, cos = _turn(s, s["positions"])
    if s["case"]["dense"]:
        sin, cos, scale = sin[:, None], cos[:, None], s["scales"]
    else:
        sin, cos, scale = sin[:, None], cos[:, None], s["scales"].reshape(-1, 1)
    q, k = s["q"], s["k"]
    return (_rotate(q, s["weight"][0], sin, cos, scale).to(q.dtype),
            _rotate(k, s["weight"][1], sin, cos, None).to(k.dtype))


def _plain_append(s):
    sin, cos = (t[:, None] for t in _turn(s, s["position"] if s["positions"] is None else s["positions"]))
    wq, wk = (None, None) if s["weight"] is None else (s["weight"][0], s["weight"][1])
    page, dtype = s["case"]["page"], s["q"].dtype
    where = (s["table"][s["request"], s["position"] // page].long(), s["position"] % page)
    for name, rows in (("k", _rotate(s["k"], wk, sin, cos, None, careful=True)), ("v", s["v"].float())):
        s[name + "_cache"][where], s[name + "_scale"][where] = _pack(rows, dtype)
    return _rotate(s["q"], wq, sin, cos, s["scales"].reshape(-1, 1)).to(dtype)


def _plain_attention(s):
    case = s["case"]
    B, K, D, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    G = case["heads"] // K
    L = s["table"].shape[1] * page
    keys = torch.arange(L, device=s["q"].device)
    held = keys < s["seq_lens"][:, None]  # [B, L]
    pages = s["table"].long()

    def gathered(name):
        x = _values(s[name + "_cache"][pages], s[name + "_scale"][pages]).reshape(B, L, K, D)
        return torch.where(held[:, :, None, None], x, 0).permute(0, 2, 1, 3)  # [B, K, L, D]

    n = case["chunk"]
    news = torch.bincount(s["request"], minlength=B)
    slot = s["position"] - (s["seq_lens"].long() - news)[s["request"]]
    q = torch.zeros(B, n, K, G, D, device=s["q"].device)
    q[s["request"], slot] = s["q"].float().reshape(-1, K, G, D)
    at = torch.full((B, n), -1, device=s["q"].device)
    at[s["request"], slot] = s["position"]
    seen = held[:, None] & (keys <= at[:, :, None])
    if case["window"]:
        seen &= keys > at[:, :, None] - case["window"]
    hidden = ~seen[:, None, :, None]  # [B, 1, n, 1, L]
    scores = q.permute(0, 2, 1, 3, 4).reshape(B, K, n * G, D) @ gathered("k").transpose(-1, -2)
    scores = scores.view(B, K, n, G, L).masked_fill_(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top.isinf(), 0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(B, K, n * G, L) @ gathered("v")).view(B, K, n, G, D) / torch.where(total > 0, total, 1)
    out = out.permute(0, 2, 1, 3, 4)[s["request"], slot].reshape(-1, K * G, D).to(s["q"].dtype)
    if not case["lse"]:
        return out
    lse = (top + total.log())[..., 0].permute(0, 2, 1, 3)[s["request"], slot]
    return out, lse.reshape(-1, K * G)


def _plain_plan(s):
    page, table, free, old, new = s["case"]["page"], s["table"], s["free"], s["seq_lens"], s["new_lens"]
    (B, width), size = table.shape, free.shape[0]
    column = torch.arange(width, device=table.device)
    ended = new < 0
    fresh = new.clamp(min=0)
    lens = torch.where(ended, 0, old + fresh)
    held, wanted = (old + page - 1) // page, (lens + page - 1) // page
    # the pages of ended requests, in order, on top of the stack
    back = (ended[:, None] & (column < held[:, None])).flatten()
    rank = back.cumsum(0) - 1
    stack = torch.cat((free, free[:1]))
    stack[torch.where(back, s["free_count"] + rank, size)] = table.flatten()
    available = s["free_count"] + back.sum()
    # new pages from its top, in order
    take = (~ended[:, None] & (column >= held[:, None]) & (column < wanted[:, None])).flatten()
    rank = take.cumsum(0) - 1
    table[:] = torch.where(take, stack[(available - 1 - rank).clamp(0, size)], table.flatten()).view(B, width)
    free[:] = stack[:size]
    cu = torch.cat((fresh.new_zeros(1), fresh.cumsum(0, dtype=torch.int32)))
    token = torch.arange(s["tokens"], device=table.device, dtype=torch.int32)
    request = torch.searchsorted(cu[1:], token, right=True, out_int32=True)
    position = (lens - fresh)[request] + token - cu[request]
    slots = table[request, position // page].long() * page + position % page
    return {"table": table, "free": free, "free_count": (available - take.sum()).to(torch.int32), "seq_lens": lens,
            "cu_seqlens": cu, "positions": position, "slots": slots, "requests": request}


def run(s):
    case = s["case"]
    if own:
        import flash_attn_prologue_b200 as fap
    if case["op"] == "rotate":
        if own:
            out = fap.qknorm_rope_scale_gqa(s["q"], s["k"], s["weight"], s["scales"], s["sin"], s["cos"], s["positions"],
                                            EPS, axes=s["axes"])
        else:
            out = _plain_rotate(s)
        grads = torch.autograd.grad(out, (s["q"], s["k"], s["weight"], s["scales"]), (s["gq"], s["gk"]))
        return {"out": tuple(out), "grads": grads}
    if case["op"] == "append":
        if own:
            q = fap.append_paged_kv_int4(s["q"], s["k"], s["v"], s["weight"], s["scales"], s["sin"], s["cos"],
                                         s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"],
                                         s["seq_lens"], s["cu_seqlens"], EPS, positions=s["positions"], axes=s["axes"])
            k, v = (fap.unpack_int4(s[name + "_cache"], s[name + "_scale"], q.dtype) for name in ("k", "v"))
        else:
            q = _plain_append(s)
            k, v = (_values(s[name + "_cache"], s[name + "_scale"]).to(q.dtype) for name in ("k", "v"))
        return {"q": q, "k": k, "v": v}
    if case["op"] == "plan":
        if own:
            p = fap.plan_paged_step(s["table"], s["seq_lens"], s["new_lens"], s["free"], s["free_count"], case["page"],
                                    s["tokens"])
            return {"table": s["table"], "free": s["free"], "free_count": p.free_count, "seq_lens": p.seq_lens,
                    "cu_seqlens": p.cu_seqlens, "positions": p.positions, "slots": p.slots, "requests": p.requests}
        return _plain_plan(s)
    if own:
        return fap.paged_attention_int4(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["table"],
                                        s["seq_lens"], s["cu_seqlens"], softmax_scale=1.0, window=case["window"],
                                        return_lse=case["lse"])
    return _plain_attention(s)


def _exact_angles(s, positions):
    """cos + i sin of every token's pairs in 64 bits."""
    angle = torch.complex(s["cos"].double(), s["sin"].double())
    if s["axes"] is None:
        return angle[positions]
    return torch.stack([angle[positions[a].long(), j] for j, a in enumerate(s["axes"])], -1)


def _exact_rows(x, weight, angle, gain):
    """Normed, rotated and scaled rows x [rows, H, D] in 64 bits, as complex pairs of the two halves."""
    if weight is not None:
        x = weight * x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half], x[..., half:]) * angle[:, None]
    return gain * torch.cat((z.real, z.imag), -1)


def _exact_rotate(s):
    case, outs, grads = s["case"], [], []
    D, N = case["dim"], case["rows"]
    angle = _exact_angles(s, s["positions"].flatten(1))
    dw, ds = torch.zeros(2, 1, D, dtype=torch.float64, device="cuda"), None
    for i, name in enumerate(("q", "k")):
        x, up = (t.detach().double() for t in (s[name], s["g" + name]))
        if case["dense"]:
            x, up = (t.permute(0, 2, 1, 3).flatten(0, 1) for t in (x, up))
        w = s["weight"].detach()[i].double()
        gain = s["scales"].detach().double().exp().reshape(1, -1, 1) if name == "q" else 1.0
        out = _exact_rows(x, w, angle, gain)
        # the rotation's transpose turns the upstream gradient back; then the norm's derivative
        back = torch.complex(up[..., :D // 2], up[..., D // 2:]) * angle.conj()[:, None]
        dy = gain * torch.cat((back.real, back.imag), -1)
        r = (x.pow(2).sum(-1, keepdim=True) / D + EPS).rsqrt()
        dw[i, 0] = (dy * x * r).sum((0, 1))
        if name == "q":
            ds = (up * out).sum((0, 2)).reshape(-1, 1, 1)
        dn = dy * w
        dx = r * dn - x * r.pow(3) * (dn * x).sum(-1, keepdim=True) / D
        if case["dense"]:
            out, dx = (t.unflatten(0, (case["batch"], N)).permute(0, 2, 1, 3) for t in (out, dx))
        outs.append(out)
        grads.append(dx)
    return {"out": tuple(outs), "grads": (*grads, dw, ds)}


def _exact_values(codes, scales):
    """What the cache's rows stand for, channel by channel, in 64 bits."""
    D = 2 * codes.shape[-1]
    out = torch.empty(*codes.shape[:-1], D, dtype=torch.float64, device=codes.device)
    for c in range(D):
        byte, high = c // 8 * 4 + c % 2 * 2 + c % 8 // 4, c % 4 // 2
        out[..., c] = scales[..., c // 8 % (D // 32)].double() * ((codes[..., byte] >> 4 * high & 15).double() - 8)
    return out


def _exact_rounded(x, half_floats):
    """Rows [..., D] rounded to four bits as the format says, in 64 bits."""
    D = x.shape[-1]
    out = torch.empty_like(x)
    channel = torch.arange(D, device=x.device)
    for g in range(D // 32):
        mine = channel // 8 % (D // 32) == g
        part = x[..., mine]
        size, where = part.abs().max(-1, keepdim=True)
        # of two that are as large the positive one
        e = torch.where((part == size).any(-1, keepdim=True), size, -size) / 8
        power = torch.exp2(torch.floor(torch.log2(e.abs().clamp(min=2.0 ** -120))) - 4)
        s = -e.sign() * torch.floor(e.abs() / power) * power
        if half_floats:
            s = torch.where(s == 0, s, s.sign() * s.abs().clamp(2.0 ** -20, 7936))
        out[..., mine] = torch.where(s == 0, 0, s * torch.clamp(torch.round(part / torch.where(s == 0, 1, s)), -8, 7))
    return out


def _exact_append(s):
    case = s["case"]
    angle = _exact_angles(s, s["position"] if s["positions"] is None else s["positions"])
    w = (None, None) if s["weight"] is None else s["weight"].double().unbind(0)
    q = _exact_rows(s["q"].double(), w[0], angle, s["scales"].double().exp().reshape(1, -1, 1))
    k = _exact_rounded(_exact_rows(s["k"].double(), w[1], angle, 1.0), case["dtype"] == "fp16")
    v = _exact_rounded(s["v"].double(), case["dtype"] == "fp16")
    caches = [_exact_values(s[name + "_cache"], s[name + "_scale"]) for name in ("k", "v")]
    pages = s["table"].long()
    begin = 0
    for b, new in enumerate(torch.bincount(s["request"], minlength=case["batch"]).tolist()):
        end = int(s["seq_lens"][b])
        slots = torch.arange(end - new, end, device="cuda")
        for cache, rows in zip(caches, (k, v)):
            cache[pages[b, slots // case["page"]], slots % case["page"]] = rows[begin:begin + new]
        begin += new
    return {"q": q, "k": caches[0], "v": caches[1]}


def _exact_attention(s):
    case = s["case"]
    G, page = case["heads"] // case["kv_heads"], case["page"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    begin = 0
    for b, new in enumerate(torch.bincount(s["request"], minlength=case["batch"]).tolist()):
        total = int(s["seq_lens"][b])
        at = torch.arange(total - new, total, device="cuda")
        low = max(0, total - new - case["window"] + 1) if case["window"] else 0
        keys = torch.arange(low, total, device="cuda")
        where = (s["table"][b].long()[keys // page], keys % page)
        bias = torch.zeros(new, len(keys), dtype=torch.float64, device="cuda")
        bias[keys[None] > at[:, None]] = -math.inf
        if case["window"]:
            bias[keys[None] <= at[:, None] - case["window"]] = -math.inf
        for h in range(case["kv_heads"] if new else 0):
            k, v = (_exact_values(s[n + "_cache"][..., h, :][where], s[n + "_scale"][..., h, :][where]) for n in ("k", "v"))
            for i in range(h * G, h * G + G):
                logits = s["q"][begin:begin + new, i].double() @ k.T + bias
                lse[begin:begin + new, i] = torch.logsumexp(logits, -1)
                out[begin:begin + new, i] = torch.exp(logits - lse[begin:begin + new, i, None]) @ v
        begin += new
    return (out, lse) if case["lse"] else out


def exact(case, seed):
    if case["op"] == "plan":  # whole numbers
        return None
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return _exact_rotate(s)
    return _exact_append(s) if case["op"] == "append" else _exact_attention(s)
