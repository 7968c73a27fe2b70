"""Grouped-query prologue (qknorm_rope_scale_gqa): forward and backward against the formula in 64 bits."""
import math

import pytest
import torch

import flash_attn_prologue_b200 as fap
from flash_attn_prologue_b200 import _lib
from tests._paged import assert_within, rotate64, tables
from tests._paged import BAND, HALF_ULP, TINY

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _problem(layout, B, N, Hq, Hk, D, dtype, ids, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if layout == "dense":
        q, k = (rand(B, h, N, D).to(dtype) for h in (Hq, Hk))
    elif layout == "dense view":  # [B, N, H, D] memory
        q, k = (rand(B, N, h, D).to(dtype).transpose(1, 2) for h in (Hq, Hk))
    elif layout == "packed":
        q, k = (rand(N, h, D).to(dtype) for h in (Hq, Hk))
    elif layout == "fused":  # views of one projection
        buf = rand(N, Hq + 2 * Hk, D).to(dtype)
        q, k = buf[:, :Hq], buf[:, Hq:Hq + Hk]
    else:  # rows that start at an odd element
        q, k = (rand(N * h * D + 1).to(dtype)[1:].view(N, h, D) for h in (Hq, Hk))
    w = 1 + 0.2 * rand(2, 1, D)
    s = math.log(D ** -0.5) + 0.3 * rand(Hq, 1, 1)
    dense = q.ndim == 4
    rows = N if ids is None else 2 * N + 3
    sin, cos = tables(rows, D)
    pos = None
    if ids is not None:
        pos = torch.randint(0, rows, (B, N) if dense and ids[1] == "bn" else (N,), generator=g, device="cuda").to(ids[0])
    up = [rand(*t.shape).to(dtype) for t in (q, k)]
    return q, k, w, s, sin, cos, pos, up


def _exact(q, k, w, s, sin, cos, pos, up):
    """Outputs, gradients and each one's error scale in 64 bits."""
    D = q.shape[-1]
    at = torch.arange(q.shape[-2] if q.ndim == 4 else q.shape[0], device=q.device) if pos is None else pos
    sn, cs = sin[at], cos[at]
    if q.ndim == 3:
        sn, cs = sn[:, None], cs[:, None]
    elif sn.ndim == 3:
        sn, cs = sn[:, None], cs[:, None]
    gains = (s.double().exp().view(-1, 1) if q.ndim == 3 else s.double().exp(), 1.0)
    outs, grads, dws = [], [], []
    for t, (x, g) in enumerate(zip((q, k), up)):
        outs.append(rotate64(x, w[t], sn, cs, gains[t]))
        ga, gb = (g.double() * gains[t]).chunk(2, -1)
        dy = torch.cat((ga * cs + gb * sn, gb * cs - ga * sn), -1)
        size_dy = torch.cat(((ga * cs).abs() + (gb * sn).abs(), (gb * cs).abs() + (ga * sn).abs()), -1)
        x = x.double()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)
        n, u, size_u = x * r, dy * w[t].double(), size_dy * w[t].double().abs()
        grads.append((r * (u - n * (u * n).mean(-1, keepdim=True)),
                      r * (size_u + n.abs() * (size_u * n.abs()).mean(-1, keepdim=True))))
        rest = tuple(i for i in range(x.ndim - 1))
        dws.append(((dy * n).sum(rest), (size_dy * n.abs()).sum(rest)))
        if t == 0:
            heads = tuple(i for i in range(x.ndim) if i != 1)
            ds = ((u * n).sum(heads).view(-1, 1, 1), (size_u * n.abs()).sum(heads).view(-1, 1, 1))
    dw = tuple(torch.stack([d[i] for d in dws])[:, None] for i in range(2))
    return outs, grads, dw, ds


def _check(problem):
    q, k, w, s, sin, cos, pos, up = problem
    args = [t.detach().requires_grad_() for t in (q, k, w, s)]
    got = fap.qknorm_rope_scale_gqa(*args, sin, cos, pos)
    grads = torch.autograd.grad(got, args, up)
    outs, dx, dw, ds = _exact(*problem)
    for i, name in enumerate("qk"):
        assert_within(got[i], *outs[i], name)
        # the row's mean adds log2(D) roundings of its terms: within 2 BAND in all
        assert_within(grads[i], dx[i][0], 2 * dx[i][1], "d" + name)
    # fixed-order sums: no lane, warp or CTA adds over 128 values in sequence at these sizes
    for got_sum, (exact, size) in ((grads[2], dw), (grads[3], ds)):
        bound = (128 + 16) * 2.0 ** -24 * size
        assert ((got_sum.double() - exact).abs() <= bound).all()
    return got, grads


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("layout,B,N,Hq,Hk,ids", [
    ("packed", 1, 67, 8, 2, None),
    ("fused", 1, 130, 15, 5, (torch.int64, "n")),
    ("dense", 3, 33, 12, 4, (torch.int32, "bn")),
    ("dense view", 2, 41, 8, 8, (torch.int64, "n")),
    ("odd", 1, 19, 6, 1, None),
])
def test_against_the_formula(layout, B, N, Hq, Hk, ids, D, dtype):
    _check(_problem(layout, B, N, Hq, Hk, D, dtype, ids))


@pytest.mark.gpu
@pytest.mark.parametrize("N,Hq,Hk", [(1, 1, 1), (1, 32, 8), (2, 7, 7), (5, 512, 4), (1500, 32, 8), (9000, 4, 1)])
def test_sizes(N, Hq, Hk):
    _check(_problem("packed", 1, N, Hq, Hk, 128, BF16, (torch.int32, "n"), seed=N))


@pytest.mark.gpu
def test_equal_heads_match_the_existing_prologue():
    q, k, w, s, sin, cos, _, _ = _problem("packed", 1, 77, 8, 8, 64, BF16, None)
    for a, b in zip(fap.qknorm_rope_scale_gqa(q, k, w, s, sin, cos),
                    fap.qknorm_rope_scale(q, k, w, s, sin, cos, backend="cute")):
        assert (a.double() - b.double()).abs().max() <= 2.0 ** -8 * b.double().abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(4))
def test_gradient_against_differences(which):
    """FP32 rows: <grad, d> against the central difference of sum(up * out) along a random d.

    Step 2^-8: the third derivative's share is under 2^-16 times a small constant and the
    outputs' rounding under 2^-24 * 4 / 2^-8, both of the gradient's norm: 2e-3 covers them."""
    problem = _problem("packed", 1, 50, 6, 2, 64, FP32, (torch.int64, "n"), seed=5)
    q, k, w, s, sin, cos, pos, up = problem
    args = [t.detach().requires_grad_() for t in (q, k, w, s)]
    grad = torch.autograd.grad(fap.qknorm_rope_scale_gqa(*args, sin, cos, pos), args, up)[which].double()
    d = torch.randn(grad.shape, generator=torch.Generator(device="cuda").manual_seed(9), device="cuda")

    def loss(sign):
        moved = [t.detach().clone() for t in args]
        moved[which] += sign * 2.0 ** -8 * d
        out = fap.qknorm_rope_scale_gqa(*moved, sin, cos, pos)
        return sum((o.double() * u.double()).sum() for o, u in zip(out, up))

    slope = (loss(1) - loss(-1)) / 2.0 ** -7
    assert abs(slope - (grad * d).sum()) <= 2e-3 * grad.norm() * max(1.0, 1.0 if which < 2 else d.double().norm())


@pytest.mark.gpu
def test_repeats_bit_for_bit_and_on_another_stream():
    problem = _problem("packed", 1, 3000, 16, 4, 64, BF16, None)
    first = _check(problem)
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        again = _check(problem)
    torch.cuda.synchronize()
    for a, b in zip((*first[0], *first[1]), (*again[0], *again[1])):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_very_small_query_scales():
    """exp(scale) underflows: zero rows and zero gradients, no NaN."""
    q, k, w, s, sin, cos, _, up = _problem("packed", 1, 9, 4, 2, 64, FP32, None)
    s = torch.tensor([-200.0, -85.0, -60.0, 0.0], device="cuda").view(4, 1, 1)
    args = [t.detach().requires_grad_() for t in (q, k, w, s)]
    got = fap.qknorm_rope_scale_gqa(*args, sin, cos)
    grads = torch.autograd.grad(got, args, up)
    assert all(t.isfinite().all() for t in (*got, *grads))
    assert not got[0][:, 0].any() and not grads[0][:, 0].any() and grads[0][:, 3].any()


@pytest.mark.gpu
@pytest.mark.parametrize("layout,D", [("packed", 64), ("odd", 128), ("packed", 256)])
def test_gradients_of_small_query_scales(layout, D):
    """exp(scale) far below 1: FP32 gradients are right to their last bits down to 2^-126, and to a few of FP32's
    smallest steps below."""
    q, k, w, _, sin, cos, _, up = _problem(layout, 1, 11, 6, 2, D, FP32, None)
    s = torch.tensor([-95.0, -86.0, -84.0, -80.5, -79.0, -1.0], device="cuda").view(6, 1, 1)
    args = [t.detach().requires_grad_() for t in (q, k, w, s)]
    grads = torch.autograd.grad(fap.qknorm_rope_scale_gqa(*args, sin, cos), args, up)
    _, dx, _, (ds, ds_size) = _exact(q, k, w, s, sin, cos, None, up)
    for i, name in enumerate("qk"):
        # as elsewhere, and 64 half steps of FP32's subnormal numbers for the products of the terms (|x|, |u| < 8)
        off = (grads[i].double() - dx[i][0]).abs()
        bound = HALF_ULP[FP32] * dx[i][0].abs() + 2 * BAND * dx[i][1] + 64 * TINY[FP32]
        assert (off <= bound).all(), f"d{name}: {float((off / bound).max())}"
    assert ((grads[3].double() - ds).abs() <= (128 + 16) * 2.0 ** -24 * ds_size + 2 * D * 11 * 64 * TINY[FP32]).all()


@pytest.mark.gpu
def test_sums_over_a_peer_group_of_one_rank():
    """Inside reducing() the backward takes the group's reduction: one epoch a call, the plain call's bits."""
    import ctypes
    from types import SimpleNamespace
    from flash_attn_prologue_b200 import distributed
    nd, nf = ctypes.c_size_t(), ctypes.c_size_t()
    assert _lib.load().flash_prologue_peer_buffer_bytes(1, 160, ctypes.byref(nd), ctypes.byref(nf)) == 0
    data = torch.zeros(nd.value // 4, device="cuda")
    flags = torch.zeros(nf.value // 4, dtype=torch.int32, device="cuda")
    desc = _lib.PeersDesc()
    desc.world, desc.rank, desc.max_cols, desc.wait_ms = 1, 0, 160, 1000
    desc.data[0], desc.flags[0] = data.data_ptr(), flags.data_ptr()
    epochs = iter(range(1, 10))
    group = SimpleNamespace(desc=desc, next_epoch=lambda: next(epochs))
    q, k, w, s, sin, cos, _, up = _problem("packed", 1, 300, 16, 4, 64, BF16, None)
    args = [t.detach().requires_grad_() for t in (q, k, w, s)]
    plain = torch.autograd.grad(fap.qknorm_rope_scale_gqa(*args, sin, cos), args, up)
    index = torch.cuda.current_device()
    distributed._ACTIVE_PEER_GROUPS[index] = group
    try:
        for _ in range(2):
            grads = torch.autograd.grad(fap.qknorm_rope_scale_gqa(*args, sin, cos), args, up)
            assert all(torch.equal(a, b) for a, b in zip(plain, grads))
    finally:
        distributed._ACTIVE_PEER_GROUPS.pop(index)
    torch.cuda.synchronize()
    assert next(epochs) == 3 and _lib.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 8, 64), (2, 8, 0, 64)])
def test_no_tokens(shape):
    q = torch.randn(shape, device="cuda", requires_grad=True)
    k = torch.randn((*shape[:1], 4, *shape[2:]) if len(shape) == 4 else (0, 4, 64), device="cuda", requires_grad=True)
    w, s = torch.ones(2, 1, 64, device="cuda", requires_grad=True), torch.ones(8, 1, 1, device="cuda", requires_grad=True)
    out = fap.qknorm_rope_scale_gqa(q, k, w, s, *tables(4, 64))
    assert out[0].shape == q.shape and out[1].shape == k.shape
    dw, ds = torch.autograd.grad(out, (w, s), [torch.ones_like(t) for t in out])
    assert not dw.any() and not ds.any()


@pytest.mark.gpu
def test_broadcast_gradient_and_expanded_rows():
    q, k, w, s, sin, cos, _, _ = _problem("packed", 1, 21, 4, 2, 64, BF16, None)
    args = [t.detach().requires_grad_() for t in (q, k, w, s)]
    out = fap.qknorm_rope_scale_gqa(*args, sin, cos)
    summed = torch.autograd.grad(out[0].sum(), args[:1])[0]
    out = fap.qknorm_rope_scale_gqa(*args, sin, cos)
    written = torch.autograd.grad(out[0], args[:1], torch.ones_like(out[0]))[0]
    assert torch.equal(summed, written)
    wide = k[:, :1].expand(-1, 2, -1)
    a = fap.qknorm_rope_scale_gqa(q, wide, w, s, sin, cos)[1]
    assert torch.equal(a, fap.qknorm_rope_scale_gqa(q, wide.contiguous(), w, s, sin, cos)[1])


@pytest.mark.gpu
def test_rows_of_infinity_nan_and_zero_stay_alone():
    q, k, w, s, sin, cos, _, up = _problem("packed", 1, 16, 4, 2, 64, BF16, None)
    clean = fap.qknorm_rope_scale_gqa(q, k, w, s, sin, cos)
    q, k = q.clone(), k.clone()
    q[3, 1, 5], q[4, 2, 0], k[5, 0] = float("inf"), float("nan"), 0
    got = fap.qknorm_rope_scale_gqa(q, k, w, s, sin, cos)
    assert got[0][4, 2].isnan().all() and got[0][3, 1].isnan().any() and not got[1][5, 0].any()
    for t in range(2):
        same = torch.ones(got[t].shape[:2], dtype=torch.bool, device="cuda")
        if t == 0:
            same[3, 1] = same[4, 2] = False
        else:
            same[5, 0] = False
        assert torch.equal(got[t][same], clean[t][same])


@pytest.mark.gpu
def test_position_out_of_range_gives_nan_and_the_error_word():
    q, k, w, s, sin, cos, _, _ = _problem("packed", 1, 6, 4, 2, 64, BF16, None)
    _lib.device_error()
    pos = torch.tensor([0, 1, -1, 3, 6, 5], device="cuda")
    out = fap.qknorm_rope_scale_gqa(q, k, w, s, sin, cos, pos)
    assert _lib.device_error() == 2 and _lib.device_error() == 0
    for t in out:
        assert t.isnan().flatten(1).all(1).tolist() == [False, False, True, False, True, False]


@pytest.mark.gpu
def test_compiled_and_opcheck():
    q, k, w, s, sin, cos, pos, up = _problem("packed", 1, 40, 8, 2, 64, BF16, (torch.int64, "n"))
    args = [t.detach().requires_grad_() for t in (q, k, w, s)]

    def step(q, k, w, s):
        return fap.qknorm_rope_scale_gqa(q, k, w, s, sin, cos, pos)

    eager = torch.autograd.grad(step(*args), args, up)
    graph = torch.autograd.grad(torch.compile(step, fullgraph=True)(*args), args, up)
    assert all(torch.equal(a, b) for a, b in zip(eager, graph))
    checks = ("test_schema", "test_autograd_registration", "test_faketensor")
    ops = torch.ops.flash_prologue
    for result in (torch.library.opcheck(ops.qknorm_rope_scale_gqa.default, (*args, sin, cos, pos, 1e-5), test_utils=checks),
                   torch.library.opcheck(ops.qknorm_rope_scale_gqa_backward.default,
                                         (q, k, w, s, sin, cos, None, *up, 1e-5), test_utils=checks)):
        assert set(result.values()) == {"SUCCESS"}, result


def _cpu_args(Hq=8, Hk=2, D=64, N=5, dtype=BF16):
    sin, cos = tables(N, D, "cpu")
    return dict(q=torch.zeros(N, Hq, D, dtype=dtype), k=torch.zeros(N, Hk, D, dtype=dtype),
                rmsnorm_weight=torch.ones(2, 1, D), scales=torch.zeros(Hq, 1, 1), sin=sin, cos=cos)


@pytest.mark.parametrize("change,text", [
    (lambda a: a.update(k=a["k"][:4]), "head count only"),
    (lambda a: a.update(k=a["k"][None]), "packed .* or dense"),
    (lambda a: a.update(k=a["k"].float()), "share BF16"),
    (lambda a: a.update(k=torch.zeros(5, 3, 64, dtype=BF16)), "multiple of the key heads"),
    (lambda a: a.update(_cpu_args(Hq=1024)), "at most 512"),
    (lambda a: a.update(_cpu_args(D=96)), "head dimension"),
    (lambda a: a.update(rmsnorm_weight=torch.ones(2, 64)), "weight must be"),
    (lambda a: a.update(scales=torch.zeros(2, 1, 1)), "log-scales"),
    (lambda a: a.update(sin=a["sin"][:, :4]), "matching tables"),
    (lambda a: a.update(scales=a["scales"].double()), "must be FP32"),
    (lambda a: a.update(sin=a["sin"].clone().requires_grad_()), "not implemented"),
    (lambda a: a.update(eps=0.0), "eps"),
    (lambda a: a.update(eps=float("nan")), "eps"),
    (lambda a: None, "CUDA devices only"),
])
def test_refusals(change, text):
    args = _cpu_args()
    change(args)
    with pytest.raises(ValueError, match=text):
        fap.qknorm_rope_scale_gqa(**args)


@pytest.mark.gpu
@pytest.mark.parametrize("positions,text", [
    (torch.zeros(5, dtype=torch.int16), "int32 or int64"),
    (torch.zeros(4, dtype=torch.int64), "positions must be"),
    (torch.zeros(1, 5, dtype=torch.int64), "positions must be"),
])
def test_refused_positions(positions, text):
    args = {n: t.cuda() for n, t in _cpu_args().items()}
    with pytest.raises(ValueError, match=text):
        fap.qknorm_rope_scale_gqa(**args, positions=positions.cuda())
    with pytest.raises(ValueError, match="fewer rows"):
        fap.qknorm_rope_scale_gqa(**{**args, "sin": args["sin"][:4], "cos": args["cos"][:4]})
    with pytest.raises(ValueError, match="share a device"):
        fap.qknorm_rope_scale_gqa(**args, positions=torch.zeros(5, dtype=torch.int64))


def test_c_abi_refusals():
    """Arguments that the library turns away before it touches the device."""
    lib = _lib.load()

    def call(name="flash_prologue_gqa_fwd", B=1, N=4, Hq=8, Hk=2, D=64, dtype=0, eps=1e-5, ptr=64, w=64, rows=4, pos=0,
             bits=64, hs=64, out=64):
        r = (ptr, 0, hs, 512)
        o = (out, 0, 64, 512)
        return getattr(lib, name)(_lib.GQA_ARGS.pack(
            *r, *r, *o, *o, *r, *r, *o, *o, w, 64, 64, 32, 1, 64, 32, 1, rows, pos, 0, 1, bits, 64, 64, 64, 0, 0, 0,
            B, N, Hq, Hk, D, dtype, eps), None)

    assert call(N=0, ptr=0) == _lib.OK
    for wrong, status in ((dict(B=-1), 1), (dict(eps=0.0), 1), (dict(Hk=3), 1), (dict(Hk=0), 1), (dict(D=48), 2),
                          (dict(dtype=3), 2), (dict(Hq=1024), 2), (dict(ptr=0), 1), (dict(rows=3), 1),
                          (dict(pos=64, bits=16), 1), (dict(w=72), _lib.ERR_ALIGNMENT), (dict(hs=0), _lib.ERR_EXPANDED),
                          (dict(out=0), 1)):
        assert call(**wrong) == status, wrong
        assert call("flash_prologue_gqa_bwd", **wrong) == status, wrong
