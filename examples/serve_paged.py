"""Trains a small grouped-query attention model for a few steps, then serves it from a paged cache.

Training runs the prologue over packed documents (positions restart in each) with
``qknorm_rope_scale_gqa`` and its backward; serving feeds prompts in chunks and then single
tokens through ``append_paged_kv`` and ``paged_attention``, with several requests in one step,
and checks each request against the model run over its whole text at once.

    python examples/serve_paged.py [--steps 30] [--requests 6] [--new 24]
"""
import argparse
import math
import sys
import time
from pathlib import Path

import torch
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import flash_attn_prologue_b200 as fap  # noqa: E402

VOCAB, HIDDEN, HEADS, KV_HEADS, DIM, MAX_LEN = 64, 256, 8, 2, 64, 1024


class Layer(nn.Module):
    """Attention with query/key norms; the Q scale is learned, so attention's own scale is 1."""

    def __init__(self):
        super().__init__()
        self.norm = nn.RMSNorm(HIDDEN)
        self.qkv = nn.Linear(HIDDEN, (HEADS + 2 * KV_HEADS) * DIM, bias=False)
        self.out = nn.Linear(HEADS * DIM, HIDDEN, bias=False)
        self.qk_weight = nn.Parameter(torch.ones(2, 1, DIM))
        self.scales = nn.Parameter(torch.full((HEADS, 1, 1), math.log(DIM ** -0.5)))

    def rows(self, x):
        qkv = self.qkv(self.norm(x)).to(torch.bfloat16).view(-1, HEADS + 2 * KV_HEADS, DIM)
        return qkv.split((HEADS, KV_HEADS, KV_HEADS), dim=1)


class Model(nn.Module):
    def __init__(self, layers=2):
        super().__init__()
        self.embed = nn.Embedding(VOCAB, HIDDEN)
        self.layers = nn.ModuleList(Layer() for _ in range(layers))
        self.head = nn.Linear(HIDDEN, VOCAB)
        inv = 10000.0 ** (-torch.arange(0, DIM, 2, dtype=torch.float64) / DIM)
        angle = torch.arange(MAX_LEN, dtype=torch.float64)[:, None] * inv
        self.register_buffer("sin", angle.sin().float())
        self.register_buffer("cos", angle.cos().float())

    def forward(self, tokens, positions, document):
        """Logits of packed documents; a token sees its document's tokens up to itself."""
        x = self.embed(tokens)
        sees = (document[:, None] == document) & (positions[:, None] >= positions)
        for layer in self.layers:
            q, k, v = layer.rows(x)
            q, k = fap.qknorm_rope_scale_gqa(q, k, layer.qk_weight, layer.scales, self.sin, self.cos, positions)
            k, v = (t.float().repeat_interleave(HEADS // KV_HEADS, 1) for t in (k, v))
            scores = torch.einsum("ihd,jhd->hij", q.float(), k).masked_fill(~sees, -math.inf)
            y = torch.einsum("hij,jhd->ihd", scores.softmax(-1), v)
            x = x + layer.out(y.flatten(1))
        return self.head(x)

    @torch.no_grad()
    def step(self, tokens, caches, table, lens, cu):
        """Logits of a serving step's new tokens, which join the caches."""
        x = self.embed(tokens)
        for layer, (k_cache, v_cache) in zip(self.layers, caches):
            q, k, v = layer.rows(x)
            q = fap.append_paged_kv(q, k, v, layer.qk_weight, layer.scales, self.sin, self.cos, k_cache, v_cache, table,
                                    lens, cu)
            y = fap.paged_attention(q, k_cache, v_cache, table, lens, cu)
            x = x + layer.out(y.float().flatten(1))
        return self.head(x)


class Server:
    """Requests on a pool of pages: pages are handed out as requests grow."""

    def __init__(self, model, pages=256, page_size=16):
        self.model, self.page_size = model, page_size
        self.free = list(range(pages))
        shape = (pages, page_size, KV_HEADS, DIM)
        self.caches = [tuple(torch.empty(shape, dtype=torch.bfloat16, device="cuda") for _ in range(2))
                       for _ in model.layers]
        self.pages, self.lens = {}, {}

    def step(self, new):
        """{request: its new tokens} -> {request: logits of the last of them}."""
        names = list(new)
        for r in names:
            self.lens[r] = self.lens.get(r, 0) + len(new[r])
            held = self.pages.setdefault(r, [])
            while len(held) * self.page_size < self.lens[r]:
                held.append(self.free.pop())
        width = max(len(self.pages[r]) for r in names)
        table = torch.tensor([self.pages[r] + [0] * (width - len(self.pages[r])) for r in names], dtype=torch.int32)
        lens = torch.tensor([self.lens[r] for r in names], dtype=torch.int32)
        ends = torch.tensor([0] + [len(new[r]) for r in names]).cumsum(0).to(torch.int32)
        cu = None if int(ends[-1]) == len(names) else ends.cuda()
        tokens = torch.tensor([t for r in names for t in new[r]])
        logits = self.model.step(tokens.cuda(), self.caches, table.cuda(), lens.cuda(), cu)
        return dict(zip(names, logits[(ends[1:] - 1).long().cuda()]))


def train(model, steps):
    """Documents that count in steps of their own; returns the first and the last loss."""
    optimizer = torch.optim.AdamW(model.parameters(), lr=2e-3)
    g = torch.Generator().manual_seed(0)
    losses = []
    for _ in range(steps):
        lengths = torch.randint(20, 60, (8,), generator=g)
        document = torch.repeat_interleave(torch.arange(8), lengths)
        positions = torch.cat([torch.arange(n) for n in lengths.tolist()])
        start, stride = (torch.randint(1, VOCAB, (8,), generator=g)[document] for _ in range(2))
        tokens = ((start + stride * positions) % VOCAB).cuda()
        logits = model(tokens, positions.cuda(), document.cuda())
        same = (document[1:] == document[:-1]).cuda()
        loss = nn.functional.cross_entropy(logits[:-1][same], tokens[1:][same])
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
    return float(losses[0]), float(losses[-1])


def serve(model, requests, new):
    """Greedy continuations; the largest difference of a step's logits from the whole text's."""
    g = torch.Generator().manual_seed(1)
    server = Server(model)
    texts = {r: torch.randint(0, VOCAB, (int(n),), generator=g).tolist()
             for r, n in enumerate(torch.randint(3, 120, (requests,), generator=g))}
    # prompts in chunks of up to 32 tokens, all requests together until each is read
    read, last = dict.fromkeys(texts, 0), {}
    while any(read[r] < len(t) for r, t in texts.items()):
        chunk = {r: t[read[r]:read[r] + 32] for r, t in texts.items() if read[r] < len(t)}
        for r, logits in server.step(chunk).items():
            read[r] += len(chunk[r])
            last[r] = logits
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(new):
        nxt = {r: [int(logits.argmax())] for r, logits in last.items()}
        for r, t in nxt.items():
            texts[r] += t
        last = server.step(nxt)
    torch.cuda.synchronize()
    rate = requests * new / (time.perf_counter() - began)
    worst = 0.0
    with torch.no_grad():
        for r, t in texts.items():
            at = torch.arange(len(t), device="cuda")
            whole = model(torch.tensor(t, device="cuda"), at, torch.zeros_like(at))[-1]
            worst = max(worst, float((whole - last[r]).abs().max()))
    return worst, rate


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--requests", type=int, default=6)
    ap.add_argument("--new", type=int, default=24)
    args = ap.parse_args(argv)
    torch.manual_seed(0)
    model = Model().cuda()
    first, final = train(model, args.steps)
    print(f"trained {args.steps} steps: loss {first:.3f} -> {final:.3f}")
    worst, rate = serve(model, args.requests, args.new)
    print(f"served {args.requests} requests: {rate:.0f} tokens/s, logits within {worst:.4f} of the whole text's")
    return first, final, worst


if __name__ == "__main__":
    main()
