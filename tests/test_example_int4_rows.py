"""The serving example with its cache in 4 bits: each step writes the rows that a 16-bit cache would hold, to the format's
precision and at the right slots, and attends to exactly those."""
import pytest
import torch

import flash_attn_prologue_b200 as fap
from tests._int4 import groups
from tests._paged import HALF_ULP
from tests.test_paged_attention import SCORE


@pytest.mark.gpu
def test_serves_from_the_rows_of_its_requests(monkeypatch):
    from examples.serve_paged import main
    for name in fap.__all__:  # names that load later would bring the functions back
        getattr(fap, name)
    append, attend = fap.append_paged_kv_int4, fap.paged_attention_int4
    beside, checked = {}, []

    def rows_of(tensor, table, r, n):
        page = tensor.shape[1]
        at = torch.arange(n, device="cuda")
        return tensor[table[r].long()[at // page], at % page]

    def append_both(q, k, v, w, s, sin, cos, k_cache, v_cache, k_scale, v_scale, table, lens, cu):
        """Into a 16-bit cache too, which is what the 4-bit one is held against."""
        held = beside.setdefault(k_cache.data_ptr(), [torch.zeros(*k_cache.shape[:3], 2 * k_cache.shape[3], dtype=q.dtype,
                                                                  device="cuda") for _ in range(2)])
        q16 = fap.append_paged_kv(q, k, v, w, s, sin, cos, *held, table, lens, cu)
        out = append(q, k, v, w, s, sin, cos, k_cache, v_cache, k_scale, v_scale, table, lens, cu)
        assert torch.equal(out, q16)
        for r, n in enumerate(lens.tolist()):
            for codes, scale, rows in ((k_cache, k_scale, held[0]), (v_cache, v_scale, held[1])):
                got = fap.unpack_int4(rows_of(codes, table, r, n), rows_of(scale, table, r, n), q.dtype).double()
                exact = rows_of(rows, table, r, n).double()
                size = rows_of(scale, table, r, n).double().abs()[..., groups(exact.shape[-1])]
                # half a step; or a code cut to 7 (value below 8.5 s, the scale being cut by up to 1/16); the 16-bit row's cast
                assert ((got - exact).abs() <= 1.5 * size + HALF_ULP[q.dtype] * exact.abs()).all()
                assert float((got - exact).abs().mean()) <= 0.35 * float(size.mean())  # a step's mean error is s / 4
        return out

    def attend_checked(q, k_cache, v_cache, k_scale, v_scale, table, lens, cu):
        out = attend(q, k_cache, v_cache, k_scale, v_scale, table, lens, cu)
        starts = list(range(len(lens) + 1)) if cu is None else cu.tolist()
        for r, n in enumerate(lens.tolist()):
            rows = slice(starts[r], starts[r + 1])
            new = rows.stop - rows.start
            if not new:
                continue
            k, v = (fap.unpack_int4(rows_of(c, table, r, n), rows_of(s, table, r, n), q.dtype).double()
                    .repeat_interleave(q.shape[1] // c.shape[2], 1) for c, s in ((k_cache, k_scale), (v_cache, v_scale)))
            sees = torch.arange(n, device="cuda") <= torch.arange(n - new, n, device="cuda")[:, None]
            p = torch.einsum("ihd,jhd->hij", q[rows].double(), k).masked_fill(~sees, -torch.inf).softmax(-1)
            exact, size = (torch.einsum("hij,jhd->ihd", p, x) for x in (v, v.abs()))
            u = HALF_ULP[q.dtype]
            # as in the operator's own tests; 8 |s|, the largest value of a group, stands for the lifted sums
            bound = u * exact.abs() + (u + SCORE) * size + 2.0 ** -16 * 17 / 16 * v.abs().amax() + 1e-30
            assert ((out[rows].double() - exact).abs() <= bound).all()
            checked.append(new)
        return out

    monkeypatch.setattr(fap, "append_paged_kv_int4", append_both)
    monkeypatch.setattr(fap, "paged_attention_int4", attend_checked)
    main(["--steps", "3", "--requests", "4", "--new", "6", "--int4"])
    assert len(checked) > 40 and max(checked) > 1 and min(checked) == 1
