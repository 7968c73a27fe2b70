"""Positions with several axes (axes=): forward, backward and append against the formula in 64 bits."""
import math

import pytest
import torch

import flash_attn_prologue_b200 as fap
from flash_attn_prologue_b200 import _lib
from tests._paged import Requests, assert_within, rotate64, tables

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _axes(D, count, pattern):
    half = D // 2
    if pattern == "blocks":  # uneven: borders inside groups of four pairs
        return tuple(min(j * count // half + (j % 5 == 4), count - 1) if j > half // 3 else 0 for j in range(half))
    if pattern == "interleaved":
        return tuple(j % count for j in range(half))
    return tuple(j // 4 % count for j in range(half))  # whole groups of four


def _angles(sin, cos, pos, axes):
    """sin/cos [..., D/2] of each token, pos [axes, ...]."""
    pairs = range(len(axes))
    return (torch.stack([t[pos[axes[j]].long(), j] for j in pairs], -1) for t in (sin, cos))


def _problem(layout, B, N, Hq, Hk, D, dtype, count, pattern, ids=torch.int32, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    dense = layout.startswith("dense")
    if layout == "dense":
        q, k = (rand(B, h, N, D).to(dtype) for h in (Hq, Hk))
    elif layout == "dense view":
        q, k = (rand(B, N, h, D).to(dtype).transpose(1, 2) for h in (Hq, Hk))
    elif layout == "packed":
        buf = rand(N, Hq + 2 * Hk, D).to(dtype)
        q, k = buf[:, :Hq], buf[:, Hq:Hq + Hk]
    else:  # rows that start at an odd element
        q, k = (rand(N * h * D + 1).to(dtype)[1:].view(N, h, D) for h in (Hq, Hk))
    w, s = 1 + 0.2 * rand(2, 1, D), math.log(D ** -0.5) + 0.3 * rand(Hq, 1, 1)
    rows = 2 * N + 3
    sin, cos = tables(rows, D)
    shape = (B, N) if dense and ids is torch.int32 else (N,)
    pos = torch.randint(0, rows, (count, *shape), generator=g, device="cuda").to(ids)
    return q, k, w, s, sin, cos, pos, _axes(D, count, pattern), [rand(*t.shape).to(dtype) for t in (q, k)]


def _check(problem):
    q, k, w, s, sin, cos, pos, axes, up = problem
    args = [t.detach().requires_grad_() for t in (q, k, w, s)]
    got = fap.qknorm_rope_scale_gqa(*args, sin, cos, pos, axes=axes)
    grads = torch.autograd.grad(got, args, up)
    sn, cs = _angles(sin, cos, pos, axes)
    if q.ndim == 3 or sn.ndim == 3:
        sn, cs = sn[:, None], cs[:, None]
    gains = (s.double().exp().view(-1, 1) if q.ndim == 3 else s.double().exp(), 1.0)
    dw = []
    for t, (x, u) in enumerate(zip((q, k), up)):
        assert_within(got[t], *rotate64(x, w[t], sn, cs, gains[t]), "qk"[t])
        ga, gb = (u.double() * gains[t]).chunk(2, -1)
        dy = torch.cat((ga * cs + gb * sn, gb * cs - ga * sn), -1)
        size = torch.cat(((ga * cs).abs() + (gb * sn).abs(), (gb * cs).abs() + (ga * sn).abs()), -1)
        x = x.double()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)
        n, v, size_v = x * r, dy * w[t].double(), size * w[t].double().abs()
        # the row's mean adds log2(D) roundings of its terms: within 2 BAND in all
        assert_within(grads[t], r * (v - n * (v * n).mean(-1, keepdim=True)),
                      2 * r * (size_v + n.abs() * (size_v * n.abs()).mean(-1, keepdim=True)), "d" + "qk"[t])
        rest = tuple(range(x.ndim - 1))
        dw.append(((dy * n).sum(rest), (size * n.abs()).sum(rest)))
        if t == 0:
            others = tuple(i for i in range(x.ndim) if i != 1)
            ds = ((v * n).sum(others).view(-1, 1, 1), (size_v * n.abs()).sum(others).view(-1, 1, 1))
    dw = tuple(torch.stack([d[i] for d in dw])[:, None] for i in range(2))
    # fixed-order sums: no lane, warp or CTA adds over 128 values in sequence at these sizes
    for got_sum, (exact, size) in ((grads[2], dw), (grads[3], ds)):
        assert ((got_sum.double() - exact).abs() <= (128 + 16) * 2.0 ** -24 * size).all()
    return (*got, *grads)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("layout,B,N,Hq,Hk,count,pattern,ids", [
    ("packed", 1, 67, 8, 2, 3, "blocks", torch.int32),
    ("packed", 1, 130, 15, 5, 3, "interleaved", torch.int64),
    ("dense", 3, 33, 12, 4, 2, "fours", torch.int32),
    ("dense view", 2, 41, 8, 8, 4, "interleaved", torch.int64),
    ("odd", 1, 19, 6, 1, 4, "blocks", torch.int32),
    ("odd", 1, 1, 7, 7, 1, "interleaved", torch.int64),
])
def test_against_the_formula(layout, B, N, Hq, Hk, count, pattern, ids, D, dtype):
    _check(_problem(layout, B, N, Hq, Hk, D, dtype, count, pattern, ids))


@pytest.mark.gpu
@pytest.mark.parametrize("N,Hq,Hk", [(1, 32, 8), (5, 512, 4), (4000, 32, 8)])
def test_sizes(N, Hq, Hk):
    _check(_problem("packed", 1, N, Hq, Hk, 128, BF16, 3, "interleaved", seed=N))


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(4))
def test_gradient_against_differences(which):
    """As for one axis: 2e-3 covers the third derivative's share and the outputs' rounding at a step of 2^-8."""
    q, k, w, s, sin, cos, pos, axes, up = _problem("packed", 1, 50, 6, 2, 64, FP32, 3, "interleaved", seed=5)
    args = [t.detach().requires_grad_() for t in (q, k, w, s)]
    grad = torch.autograd.grad(fap.qknorm_rope_scale_gqa(*args, sin, cos, pos, axes=axes), args, up)[which].double()
    d = torch.randn(grad.shape, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda")

    def loss(sign):
        moved = [t.detach().clone() for t in args]
        moved[which] += sign * 2.0 ** -8 * d
        return sum((o.double() * u.double()).sum()
                   for o, u in zip(fap.qknorm_rope_scale_gqa(*moved, sin, cos, pos, axes=axes), up))

    slope = (loss(1) - loss(-1)) / 2.0 ** -7
    assert abs(slope - (grad * d).sum()) <= 2e-3 * grad.norm() * max(1.0, 1.0 if which < 2 else d.double().norm())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_axes_that_agree_are_one_position(dtype):
    q, k, w, s, sin, cos, pos, axes, up = _problem("packed", 1, 300, 8, 2, 128, dtype, 3, "interleaved")
    pos = pos[:1].expand(3, -1)  # one position for all axes, a broadcast view
    args = [t.detach().requires_grad_() for t in (q, k, w, s)]
    a = fap.qknorm_rope_scale_gqa(*args, sin, cos, pos, axes=axes)
    b = fap.qknorm_rope_scale_gqa(*args, sin, cos, pos[0].contiguous())
    for x, y in zip((*a, *torch.autograd.grad(a, args, up)), (*b, *torch.autograd.grad(b, args, up))):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_positions_out_of_range_give_nan_rows():
    q, k, w, s, sin, cos, pos, axes, up = _problem("packed", 1, 20, 8, 2, 64, BF16, 3, "blocks")
    good = fap.qknorm_rope_scale_gqa(q, k, w, s, sin, cos, pos, axes=axes)
    assert _lib.device_error() == 0
    pos = pos.clone()
    pos[1, 3], pos[2, 7], pos[0, 11] = -1, sin.shape[0], 2 ** 31 - 1
    args = [t.detach().requires_grad_() for t in (q, k, w, s)]
    got = fap.qknorm_rope_scale_gqa(*args, sin, cos, pos, axes=axes)
    assert _lib.device_error() == 2
    lost = torch.tensor([i in (3, 7, 11) for i in range(20)], device="cuda")
    for x, y in zip(got, good):
        assert x[lost].isnan().all() and torch.equal(x[~lost], y[~lost])
    dq = torch.autograd.grad(got, args, up)[0]
    assert _lib.device_error() == 2 and dq[lost].isnan().all() and dq[~lost].isfinite().all()


@pytest.mark.gpu
def test_eager_and_registered_calls_agree():
    q, k, w, s, sin, cos, pos, axes, up = _problem("packed", 1, 90, 8, 2, 64, BF16, 3, "interleaved")
    leaves = [t.detach().requires_grad_() for t in (q, k, w, s)]
    call = lambda *a: fap.qknorm_rope_scale_gqa(*a, sin, cos, pos, axes=axes)  # noqa: E731
    eager = call(*leaves)
    first = (*eager, *torch.autograd.grad(eager, leaves, up))
    compiled = torch.compile(call, fullgraph=True)(*leaves)
    for x, y in zip(first, (*compiled, *torch.autograd.grad(compiled, leaves, up))):
        assert torch.equal(x, y)
    with pytest.raises((NotImplementedError, RuntimeError)):
        out = torch.autograd.grad(call(*leaves)[0].float().sum(), leaves[0], create_graph=True)[0]
        torch.autograd.grad(out.float().square().sum(), leaves[0])
    result = torch.library.opcheck(torch.ops.flash_prologue.qknorm_rope_scale_gqa.default,
                                   (*(t.detach().requires_grad_() for t in (q, k, w, s)), sin, cos, pos, 1e-5, list(axes)),
                                   test_utils=("test_schema", "test_autograd_registration", "test_faketensor"))
    assert set(result.values()) == {"SUCCESS"}, result


@pytest.mark.gpu
def test_captured_forward_and_backward():
    q, k, w, s, sin, cos, pos, axes, up = _problem("packed", 1, 200, 8, 2, 64, BF16, 3, "interleaved")
    leaves = [t.detach().requires_grad_() for t in (q, k, w, s)]

    def step():
        return torch.autograd.grad(fap.qknorm_rope_scale_gqa(*leaves, sin, cos, pos, axes=axes), leaves, up)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    pos.copy_(pos.flip(1))
    graph.replay()
    replayed = [t.clone() for t in captured]
    for x, y in zip(replayed, step()):
        assert torch.equal(x, y)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("count,axes", [(1, None), (3, "blocks"), (2, "interleaved")])
def test_append_turns_by_other_positions(count, axes, dtype):
    D, req = 128, Requests([3, 0, 40, 1, 17], [3, 9, 140, 1, 64], 8, 2, 128, 16, dtype)
    g = torch.Generator(device="cuda").manual_seed(1)
    buf = torch.randn(61, 12, D, generator=g, device="cuda").to(dtype)
    q, k, v = buf[:, :8], buf[:, 8:10], buf[:, 10:]
    w, s = 1 + 0.2 * torch.randn(2, 1, D, generator=g, device="cuda"), 0.3 * torch.randn(8, 1, 1, generator=g, device="cuda")
    sin, cos = tables(50, D)  # fewer rows than the longest request has tokens
    names = None if axes is None else _axes(D, count, axes)
    pos = torch.randint(0, 50, (count, 61), generator=g, device="cuda")
    _lib.device_error()
    got = fap.append_paged_kv(q, k, v, w, s, sin, cos, req.k, req.v, req.table, req.seq_lens, req.cu,
                              positions=pos[0] if names is None else pos, axes=names)
    assert _lib.device_error() == 0
    sn, cs = (sin[pos[0]], cos[pos[0]]) if names is None else _angles(sin, cos, pos, names)
    assert_within(got, *rotate64(q, w[0], sn[:, None], cs[:, None], s.double().exp().view(-1, 1)), "q")
    rows, size = rotate64(k, w[1], sn[:, None], cs[:, None], 1.0)
    begin = 0
    for r, (n, t) in enumerate(zip(req.news, req.totals)):
        where = req.places(r, t - n, t)
        assert_within(req.k[where], rows[begin:begin + n], size[begin:begin + n], "k")
        assert torch.equal(req.v[where], v[begin:begin + n])
        begin += n


@pytest.mark.gpu
def test_append_leaves_out_tokens_that_cannot_be_turned():
    req = Requests([4, 3], [20, 3], 8, 2, 64, 8, BF16)
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(9, h, 64, generator=g, device="cuda").to(BF16) for h in (8, 2, 2))
    pos = torch.zeros(2, 9, dtype=torch.int32, device="cuda")
    pos[1, 5] = 8
    pos[:, 7:] = -1  # padding behind the requests: not read
    k0 = req.k.clone()
    _lib.device_error()
    got = fap.append_paged_kv(q, k, v, None, None, *tables(8, 64), req.k, req.v, req.table, req.seq_lens, req.cu,
                              positions=pos, axes=_axes(64, 2, "interleaved"))
    assert _lib.device_error() == 2
    assert (got == 0).flatten(1).all(1).tolist() == [i in (5, 7, 8) for i in range(9)]
    assert int((req.k.nan_to_num(77.0) != k0.nan_to_num(77.0)).flatten(2).any(2).sum()) == 6


def test_patterns():
    assert fap.rotary_axes((2, 1, 3)) == (0, 0, 1, 2, 2, 2)
    assert fap.rotary_axes((3, 1, 2), interleaved=True) == (0, 1, 2, 0, 2, 0)
    assert fap.rotary_axes((4,)) == (0,) * 4
    for bad in ((), (1, 1, 1, 1, 1), (3, -1)):
        with pytest.raises(ValueError, match="sections"):
            fap.rotary_axes(bad)


@pytest.mark.parametrize("positions,axes,text", [
    (None, (0,) * 32, "axes take positions"),
    (torch.zeros(3, 5, dtype=torch.int32), (0,) * 31, "each of the D / 2"),
    (torch.zeros(3, 5, dtype=torch.int32), (0,) * 31 + (4,), "in 0 .. 3"),
    (torch.zeros(3, 5, dtype=torch.int32), (0,) * 31 + (-1,), "in 0 .. 3"),
    (torch.zeros(2, 5, dtype=torch.int32), (0, 1, 2, 0) * 8, "positions must be"),
    (torch.zeros(5, 5, dtype=torch.int32), (0, 1, 2, 0) * 8, "positions must be"),
    (torch.zeros(3, 4, dtype=torch.int32), (0, 1, 2, 0) * 8, "positions must be"),
    (torch.zeros(5, dtype=torch.int32), (0,) * 32, "positions must be"),
    (torch.zeros(3, 5), (0,) * 32, "int32 or int64"),
])
def test_refusals(positions, axes, text):
    from flash_attn_prologue_b200.gqa import axes_of
    with pytest.raises(ValueError, match=text):
        axes_of(axes, positions, torch.zeros(5, 8, 64), 10)


@pytest.mark.gpu
def test_expanded_and_strided_positions():
    q, k, w, s, sin, cos, pos, axes, up = _problem("packed", 1, 60, 8, 2, 64, BF16, 3, "interleaved")
    same = fap.qknorm_rope_scale_gqa(q, k, w, s, sin, cos, pos[1])
    for p in (pos[1].expand(3, -1), pos[1].long().expand(3, -1)):
        assert all(torch.equal(x, y) for x, y in zip(fap.qknorm_rope_scale_gqa(q, k, w, s, sin, cos, p, axes=axes), same))
    first = fap.qknorm_rope_scale_gqa(q, k, w, s, sin, cos, pos, axes=axes)
    by_token = pos.t().contiguous().t()  # [axes, T], tokens outside
    again = fap.qknorm_rope_scale_gqa(q, k, w, s, sin, cos, by_token, axes=list(axes))
    assert all(torch.equal(x, y) for x, y in zip(again, first))
    none = fap.qknorm_rope_scale_gqa(q[:0], k[:0], w, s, sin, cos, pos[:, :0], axes=axes)
    assert [t.shape for t in none] == [q[:0].shape, k[:0].shape]
