"""Plain 64-bit forms and builders shared by the grouped-query and paged tests."""
import random

import torch

# Largest relative rounding error of one cast, and the smallest step near zero.
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
# FP32 arithmetic before the cast: under 16 roundings of the terms' magnitude.
BAND = 2.0 ** -20


def tables(rows, dim, device="cuda"):
    inv = 10000.0 ** (-torch.arange(0, dim, 2, device=device, dtype=torch.float64) / dim)
    angle = torch.arange(rows, device=device, dtype=torch.float64)[:, None] * inv
    return angle.sin().float(), angle.cos().float()


def rotate64(x, w, sin, cos, gain, eps=1e-5):
    """(rows, magnitude of the rotation's terms) of the prologue in 64 bits; sin/cos broadcast to x[..., :D/2]."""
    x, sin, cos = x.double(), sin.double(), cos.double()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    a, b = x.chunk(2, -1)
    out = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    size = torch.cat(((a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()), -1)
    return out * gain, size * gain


def assert_within(got, exact, size, name=""):
    """|got - exact| is at most half an ulp of the cast and BAND of the terms' size."""
    bound = HALF_ULP[got.dtype] * exact.abs() + BAND * size + TINY[got.dtype]
    got, exact, size = got.detach(), exact.detach(), size.detach()
    off = (got.double() - exact).abs()
    # NaN where and only where the exact value is NaN
    assert torch.equal(got.isnan(), exact.isnan()), name
    worst = torch.where(exact.isnan(), 0, off / bound)
    assert not worst.numel() or float(worst.max()) <= 1, f"{name}: {float(worst.max())} of the bound"


class Requests:
    """Requests with `news` new tokens of `totals`, a paged cache of random K/V and shuffled pages.

    Slots that hold no token are NaN. `share`: request 1 has request 0's first page."""

    def __init__(self, news, totals, heads, kv_heads, dim, page, dtype, hnd=False, seed=0, spare=2, share=False):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rng = random.Random(seed)
        self.news, self.totals, self.page = news, totals, page
        counts = [-(-t // page) for t in totals]
        pool = list(range(sum(counts) + spare))
        rng.shuffle(pool)
        width = max([1] + counts)
        table = torch.full((len(news), width), -1, dtype=torch.int32)
        for r, n in enumerate(counts):
            table[r, :n] = torch.tensor([pool.pop() for _ in range(n)], dtype=torch.int32)
        if share:
            table[1, 0] = table[0, 0]
        self.table = table.cuda()
        self.seq_lens = torch.tensor(totals, dtype=torch.int32, device="cuda")
        self.cu = torch.tensor([0] + news).cumsum(0).to(torch.int32).cuda()
        pages = sum(counts) + spare
        shape = (pages, kv_heads, page, dim) if hnd else (pages, page, kv_heads, dim)
        self.k, self.v = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
        if hnd:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        held = torch.zeros(pages, page, dtype=torch.bool)
        for r, t in enumerate(totals):
            at = torch.arange(t)
            held[table[r].long()[at // page], at % page] = True
        self.k[~held.cuda()] = float("nan")
        self.v[~held.cuda()] = float("nan")
        self.q = torch.randn(sum(news), heads, dim, generator=g, device="cuda")

    def places(self, r, first, last):
        at = torch.arange(first, last, device="cuda")
        return self.table[r].long()[at // self.page], at % self.page
