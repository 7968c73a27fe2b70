"""The 4-bit format in 64 bits, channel by channel from its definition, and a cache of it for the tests."""
import torch

from tests._paged import Requests


def groups(dim, device="cuda"):
    return torch.arange(dim, device=device) // 8 % (dim // 32)


def cut(e, half):
    """-e / 8 with five significant bits, inside the range of the rows' type."""
    e = e.double() / 8
    power = torch.exp2(torch.floor(torch.log2(e.abs().clamp(min=2.0 ** -140))) - 4)
    s = -e.sign() * torch.floor(e.abs() / power) * power
    least, most = (2.0 ** -20, 7936.0) if half else (2.0 ** -100, 2.0 ** 122)
    return torch.where(s == 0, 0, s.sign() * s.abs().clamp(least, most))


def encode64(x, half):
    """(codes [..., D] in -8 .. 7, scales [..., D / 32]) of rows x in 64 bits."""
    x = x.double()
    of = groups(x.shape[-1], x.device)
    codes, scales = torch.zeros_like(x), []
    for g in range(x.shape[-1] // 32):
        part = x[..., of == g]
        high, low = part.amax(-1), part.amin(-1)
        s = cut(torch.where(high >= -low, high, low), half)
        s = torch.where(part.isfinite().all(-1), s, float("nan"))
        whole = torch.clamp(torch.round(part / torch.where(s == 0, 1, s)[..., None]), -8, 7)
        codes[..., of == g] = torch.where(((s == 0) | s.isnan())[..., None], 0, whole)
        scales.append(s)
    return codes, torch.stack(scales, -1)


def codes_of(packed):
    """Codes [..., D] in -8 .. 7 of packed bytes [..., D / 2]."""
    dim = 2 * packed.shape[-1]
    c = torch.arange(dim, device=packed.device)
    byte, shift = c // 8 * 4 + c % 2 * 2 + c % 8 // 4, c % 4 // 2 * 4
    return (packed.long()[..., byte] >> shift & 15) - 8


def pack(codes):
    """Packed bytes [..., D / 2] of codes [..., D] in -8 .. 7."""
    dim = codes.shape[-1]
    c = torch.arange(dim, device=codes.device)
    byte, shift = c // 8 * 4 + c % 2 * 2 + c % 8 // 4, c % 4 // 2 * 4
    out = torch.zeros(*codes.shape[:-1], dim // 2, dtype=torch.long, device=codes.device)
    out.index_add_(-1, byte, (codes.long() + 8) << shift)
    return out.to(torch.uint8)


def values64(packed, scales):
    return codes_of(packed).double() * scales.double()[..., groups(2 * packed.shape[-1], packed.device)]


class Requests4(Requests):
    """Requests whose cache is held in 4 bits; k and v stay the values it stands for (NaN where no token is)."""

    def __init__(self, news, totals, heads, kv_heads, dim, page, dtype, hnd=False, seed=0, **more):
        super().__init__(news, totals, heads, kv_heads, dim, page, dtype, hnd, seed, **more)
        g = torch.Generator(device="cuda").manual_seed(seed + 1000)
        self.codes, self.scales = [], []
        for name in ("k", "v"):
            rows = getattr(self, name)
            held = ~rows[..., 0].isnan()
            codes, scale = encode64(rows.nan_to_num(0.0), dtype is torch.float16)
            packed = pack(codes)
            # slots that hold no token: any codes, scales that are NaN
            packed[~held] = torch.randint(0, 256, packed.shape, generator=g, device="cuda").to(torch.uint8)[~held]
            scale[~held] = float("nan")
            if hnd:  # memory [pages, heads, slots, ...], passed transposed
                packed, scale = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (packed, scale))
            self.codes.append(packed)
            self.scales.append(scale.to(torch.bfloat16))
            setattr(self, name, values64(packed, self.scales[-1]))

    @property
    def cache(self):
        return (*self.codes, *self.scales)
