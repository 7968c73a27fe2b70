"""Cases of the grouped-query prologue, the paged cache append and paged attention.

Each case is one call (or one training step) of an operator as a program makes it:

* ``prologue``: qknorm_rope_scale_gqa forward and backward, packed [T, H, D] or dense [B, H, N, D],
  rows of the sin/cos table picked by row number or by position ids;
* ``append``: append_paged_kv of new tokens to a paged cache (single tokens, or ragged chunks);
* ``attend``: paged_attention of new tokens over the cache (single tokens, drafted tokens, prefill chunks).

``own`` selects the framework's kernels; otherwise the same results come from elementary torch
operations in 32 bits, rounded once at the end.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5


def listed():
    return [
        # a short fine-tuning document: 16 query heads on 4 key heads, latency of one step
        dict(name="train short doc", op="prologue", dense=False, rows=257, batch=1, heads=16, kv_heads=4, dim=64,
             dtype="bf16", ids=True),
        # packed pre-training documents: positions restart at each document
        dict(name="train packed docs", op="prologue", dense=False, rows=65536, batch=1, heads=32, kv_heads=8,
             dim=128, dtype="bf16", ids=True),
        # dense batch in full precision with an odd length and two key heads
        dict(name="train dense fp32", op="prologue", dense=True, rows=2047, batch=4, heads=32, kv_heads=2, dim=128,
             dtype="fp32", ids=False),
        # one decoding step of 32 running requests
        dict(name="append decode", op="append", batch=32, chunk=1, length=1500, heads=32, kv_heads=8, dim=128,
             page=16, dtype="bf16", hnd=False, norm=True, mix=1),
        # prefill of several prompts at once, some of them continuing an earlier chunk
        dict(name="append chunks", op="append", batch=8, chunk=4096, length=8192, heads=32, kv_heads=8, dim=128,
             page=64, dtype="bf16", hnd=False, norm=True, mix=2),
        # rotation only (a model without query/key norms), heads-outer pages, odd chunk lengths
        dict(name="append rope fp16", op="append", batch=5, chunk=999, length=1777, heads=16, kv_heads=16, dim=64,
             page=32, dtype="fp16", hnd=True, norm=False, mix=3),
        # the first tokens of a lone conversation: latency
        dict(name="decode one", op="attend", batch=1, chunk=1, length=1000, heads=32, kv_heads=8, dim=128, page=16,
             dtype="bf16", hnd=False, window=0, lse=False, mix=4),
        # a decoding step of a busy server: 64 requests of uneven lengths
        dict(name="decode batch", op="attend", batch=64, chunk=1, length=8192, heads=32, kv_heads=8, dim=128, page=16,
             dtype="bf16", hnd=False, window=0, lse=False, mix=5),
        # two long documents, few key heads: the work has to be split along the cache
        dict(name="decode long", op="attend", batch=2, chunk=1, length=131071, heads=16, kv_heads=2, dim=128, page=64,
             dtype="fp16", hnd=True, window=0, lse=True, mix=6),
        # drafted tokens of 16 requests, checked in one call
        dict(name="drafted tokens", op="attend", batch=16, chunk=6, length=4096, heads=16, kv_heads=4, dim=64, page=32,
             dtype="bf16", hnd=False, window=0, lse=False, mix=7),
        # uneven prefill chunks with a sliding window
        dict(name="prefill window", op="attend", batch=6, chunk=2000, length=6000, heads=16, kv_heads=4, dim=64,
             page=16, dtype="fp16", hnd=False, window=1024, lse=False, mix=8),
        # a long prompt's last chunk over what is cached already
        dict(name="prefill long", op="attend", batch=1, chunk=4096, length=16384, heads=32, kv_heads=8, dim=128,
             page=64, dtype="bf16", hnd=False, window=0, lse=False, mix=9),
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
        group, kv = rng.choice([(1, 16), (2, 8), (4, 8), (8, 4), (4, 4), (8, 2), (5, 8), (16, 1), (3, 5), (7, 4)])
        op = rng.choice(["prologue", "append", "attend", "attend"])
        case = dict(op=op, heads=group * kv, kv_heads=kv)
        if op == "prologue":
            dense = rng.random() < 0.4
            case.update(dense=dense, rows=_log_int(rng, 1, 4096 if dense else 100000),
                        batch=rng.randint(1, 6) if dense else 1, dim=rng.choice([32, 64, 128, 256]),
                        dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), ids=rng.random() < 0.5)
        else:
            case.update(batch=_log_int(rng, 1, 96), page=rng.choice([8, 16, 32, 64, 128, 256]),
                        dim=rng.choice([64, 128]), dtype=rng.choice(["bf16", "bf16", "fp16"]),
                        hnd=rng.random() < 0.4, mix=rng.randint(10, 1 << 20))
            length = _log_int(rng, 1, 131072)
            chunk = 1 if rng.random() < 0.4 else min(length, _log_int(rng, 2, 4096))
            case.update(length=length, chunk=chunk)
            if op == "append":
                case.update(norm=rng.random() < 0.7)
            else:
                case.update(window=rng.choice([0, 0, 0, 128, 1000, 4096]), lse=rng.random() < 0.3)
            padded = case["batch"] * length
            scores = padded * chunk * case["heads"]
            if padded * kv * case["dim"] > 64 * 8192 * 8 * 128 or (op == "attend" and scores > 32 * 4096 * 16384):
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


def _pairs(new, total, window):
    """Key/query pairs that causal attention of the last `new` of `total` tokens has, and the keys it reaches."""
    first = total - new + 1
    if not window or total <= window:
        return new * (first + total) // 2, total if new else 0
    full = max(0, total - max(first, window) + 1)
    rest = new - full
    return full * window + rest * (2 * first + rest - 1) // 2, min(total, new + window - 1) if new else 0


def work(case):
    es, D, H, K = BYTES[case["dtype"]], case["dim"], case["heads"], case["kv_heads"]
    if case["op"] == "prologue":
        rows = case["rows"] * case["batch"]
        act = rows * (H + K) * D
        # forward: q, k in and out; backward: q, k and both upstream gradients in, dq, dk out; one table
        return {"bytes": act * es * 5 + 2 * 4 * case["rows"] * D // 2 + (8 * rows if case["ids"] else 0),
                "flops": 30 * act}
    news, totals = _ragged(case)
    tokens = sum(news)
    pages = sum(-(-t // case["page"]) for t in totals)
    if case["op"] == "append":
        return {"bytes": tokens * (H + 2 * K) * D * es * 2 + tokens * 4 * D + 4 * pages, "flops": 10 * tokens * (H + K) * D}
    pairs, keys = (sum(x) for x in zip(*(_pairs(n, t, case["window"]) for n, t in zip(news, totals))))
    return {"bytes": 2 * tokens * H * D * es + 2 * keys * K * D * es + (4 * tokens * H if case["lse"] else 0) + 4 * pages,
            "flops": 4 * pairs * H * D}


def _tables(positions, dim, device):
    inv = 10000.0 ** (-torch.arange(0, dim, 2, device=device, dtype=torch.float64) / dim)
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * inv
    return angle.sin().float(), angle.cos().float()


def prepare(case, seed):
    device = torch.device("cuda")
    g = torch.Generator(device=device).manual_seed(seed)
    dtype, D, H, K = DTYPES[case["dtype"]], case["dim"], case["heads"], case["kv_heads"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device)

    s = {"case": case}
    if case["op"] != "attend":
        s["weight"] = 1 + 0.1 * normal(2, 1, D)
        s["scales"] = math.log(D ** -0.5) + 0.1 * normal(H, 1, 1)
    if case["op"] == "prologue":
        B, N = case["batch"], case["rows"]
        shape = (lambda h: (B, h, N, D)) if case["dense"] else (lambda h: (N, h, D))
        s["q"], s["k"] = (normal(*shape(h)).to(dtype) for h in (H, K))
        s["gq"], s["gk"] = (normal(*shape(h)).to(dtype) for h in (H, K))
        for name in ("q", "k", "weight", "scales"):
            s[name].requires_grad_()
        s["sin"], s["cos"] = _tables(N, D, device)
        s["positions"] = None
        if case["ids"]:  # documents one after the other, each counted from 0
            starts = torch.rand(N, generator=g, device=device) < 1 / 700
            starts[0] = True
            index = torch.arange(N, device=device)
            first = torch.where(starts, index, torch.zeros_like(index)).cummax(0).values
            s["positions"] = (index - first).expand(B, N).contiguous() if case["dense"] else index - first
        return s
    news, totals = _ragged(case)
    page, B, tokens = case["page"], case["batch"], sum(news)
    counts = [-(-t // page) for t in totals]
    width, pool = max(counts), sum(counts) + 3
    order = torch.randperm(pool, generator=g, device=device)[:sum(counts)].to(torch.int32)
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
    dims = (pool, K, page, D) if case["hnd"] else (pool, page, K, D)
    for name in ("k_cache", "v_cache"):
        cache = torch.empty(dims, dtype=dtype, device=device).normal_(generator=g)
        s[name] = cache.transpose(1, 2) if case["hnd"] else cache
    if case["op"] == "append":
        qkv = normal(tokens, H + 2 * K, D).to(dtype)  # the projection's output: strided views of it
        s["q"], s["k"], s["v"] = qkv[:, :H], qkv[:, H:H + K], qkv[:, H + K:]
        s["sin"], s["cos"] = _tables(max(totals), D, device)
        if not case["norm"]:
            s["weight"] = None
        return s
    q = normal(tokens, H, D)
    s["q"] = (2 * D ** -0.5 * q * torch.rsqrt(q.square().mean(-1, keepdim=True))).to(dtype)
    # slots that no token was written to yet hold anything
    keys = torch.arange(width * page, device=device)
    slots = table.long()[rows, keys // page] * page + keys % page
    stale = torch.ones(pool * page, dtype=torch.bool, device=device)
    stale[slots[keys < s["seq_lens"][:, None]]] = False
    s["k_cache"][stale.view(pool, page)] = float("nan")
    s["v_cache"][stale.view(pool, page)] = float("nan")
    return s


def _rotate(x, weight, sin, cos, scale):
    """The prologue of rows x [..., D] in 32 bits; sin/cos broadcast to [..., D/2]."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    a, b = x.chunk(2, dim=-1)
    x = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return x if scale is None else x * scale.exp()


def _plain_prologue(s):
    sin, cos = s["sin"], s["cos"]
    if s["positions"] is not None:
        sin, cos = sin[s["positions"]], cos[s["positions"]]
    if s["case"]["dense"]:
        sin, cos = (t[:, None] if t.ndim == 3 else t for t in (sin, cos))
        scale = s["scales"]
    else:
        sin, cos, scale = sin[:, None], cos[:, None], s["scales"].reshape(-1, 1)
    q, k = s["q"], s["k"]
    return (_rotate(q, s["weight"][0], sin, cos, scale).to(q.dtype),
            _rotate(k, s["weight"][1], sin, cos, None).to(k.dtype))


def _plain_append(s):
    sin, cos = s["sin"][s["position"]][:, None], s["cos"][s["position"]][:, None]
    wq, wk = (None, None) if s["weight"] is None else (s["weight"][0], s["weight"][1])
    page = s["case"]["page"]
    where = (s["table"][s["request"], s["position"] // page].long(), s["position"] % page)
    s["k_cache"][where] = _rotate(s["k"], wk, sin, cos, None).to(s["k"].dtype)
    s["v_cache"][where] = s["v"]
    return _rotate(s["q"], wq, sin, cos, s["scales"].reshape(-1, 1)).to(s["q"].dtype)


def _plain_attention(s):
    case = s["case"]
    B, K, D, page = case["batch"], case["kv_heads"], case["dim"], case["page"]
    G = case["heads"] // K
    L = s["table"].shape[1] * page
    keys = torch.arange(L, device=s["q"].device)
    held = keys < s["seq_lens"][:, None]  # [B, L]

    def gathered(cache):
        x = cache[s["table"].long()].float().reshape(B, L, K, D)
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
    scores = q.permute(0, 2, 1, 3, 4).reshape(B, K, n * G, D) @ gathered(s["k_cache"]).transpose(-1, -2)
    scores = scores.view(B, K, n, G, L).masked_fill_(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(top.isinf(), 0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(B, K, n * G, L) @ gathered(s["v_cache"])).view(B, K, n, G, D) / torch.where(total > 0, total, 1)
    out = out.permute(0, 2, 1, 3, 4)[s["request"], slot].reshape(-1, K * G, D).to(s["q"].dtype)
    if not case["lse"]:
        return out
    lse = (top + total.log())[..., 0].permute(0, 2, 1, 3)[s["request"], slot]
    return out, lse.reshape(-1, K * G)


def run(s):
    case = s["case"]
    if case["op"] == "prologue":
        if own:
            import flash_attn_prologue_b200 as fap
            out = fap.qknorm_rope_scale_gqa(s["q"], s["k"], s["weight"], s["scales"], s["sin"], s["cos"],
                                            s["positions"], EPS)
        else:
            out = _plain_prologue(s)
        grads = torch.autograd.grad(out, (s["q"], s["k"], s["weight"], s["scales"]), (s["gq"], s["gk"]))
        return {"out": tuple(out), "grads": grads}
    if case["op"] == "append":
        if own:
            import flash_attn_prologue_b200 as fap
            q = fap.append_paged_kv(s["q"], s["k"], s["v"], s["weight"], s["scales"], s["sin"], s["cos"],
                                    s["k_cache"], s["v_cache"], s["table"], s["seq_lens"], s["cu_seqlens"], EPS)
        else:
            q = _plain_append(s)
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if own:
        import flash_attn_prologue_b200 as fap
        return fap.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["seq_lens"], s["cu_seqlens"],
                                   softmax_scale=1.0, window=case["window"], return_lse=case["lse"])
    return _plain_attention(s)


def _exact_rows(x, weight, angle, gain):
    """Normed, rotated and scaled rows x [rows, H, D] in 64 bits, as complex pairs of the two halves."""
    if weight is not None:
        x = weight * x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
    half = x.shape[-1] // 2
    z = torch.complex(x[..., :half], x[..., half:]) * angle[:, None]
    return gain * torch.cat((z.real, z.imag), -1)


def _exact_prologue(s):
    case, outs, grads = s["case"], [], []
    D, N = case["dim"], case["rows"]
    ids = s["positions"]
    dw, ds = torch.zeros(2, 1, D, dtype=torch.float64, device="cuda"), None
    for i, name in enumerate(("q", "k")):
        x, up = (t.detach().double() for t in (s[name], s["g" + name]))
        if case["dense"]:
            x, up = (t.permute(0, 2, 1, 3).flatten(0, 1) for t in (x, up))
            at = torch.arange(N, device=x.device).repeat(case["batch"]) if ids is None else ids.flatten()
        else:
            at = torch.arange(N, device=x.device) if ids is None else ids
        angle = torch.complex(s["cos"].double(), s["sin"].double())[at]
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


def _exact_append(s):
    case = s["case"]
    angle = torch.complex(s["cos"].double(), s["sin"].double())[s["position"]]
    w = (None, None) if s["weight"] is None else s["weight"].double().unbind(0)
    q = _exact_rows(s["q"].double(), w[0], angle, s["scales"].double().exp().reshape(1, -1, 1))
    k = _exact_rows(s["k"].double(), w[1], angle, 1.0)
    caches = [s[name].double() for name in ("k_cache", "v_cache")]
    pages = s["table"].long()
    begin = 0
    for b, new in enumerate(torch.bincount(s["request"], minlength=case["batch"]).tolist()):
        end = int(s["seq_lens"][b])
        slots = torch.arange(end - new, end, device="cuda")
        for cache, rows in zip(caches, (k, s["v"].double())):
            cache[pages[b, slots // case["page"]], slots % case["page"]] = rows[begin:begin + new]
        begin += new
    return {"q": q, "k_cache": caches[0], "v_cache": caches[1]}


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
        for h in range(case["heads"] if new else 0):
            k, v = (s[name][..., h // G, :][where].double() for name in ("k_cache", "v_cache"))
            logits = s["q"][begin:begin + new, h].double() @ k.T + bias
            lse[begin:begin + new, h] = torch.logsumexp(logits, -1)
            out[begin:begin + new, h] = torch.exp(logits - lse[begin:begin + new, h, None]) @ v
        begin += new
    return (out, lse) if case["lse"] else out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prologue":
        return _exact_prologue(s)
    return _exact_append(s) if case["op"] == "append" else _exact_attention(s)
