"""Tensors of one row, column, token or slot, whose strides along that extent may be anything, and
logits whose rows repeat or overlap."""
import pytest
import torch

from table_moe.ops import Fp8Experts, Fp8Linear, route_experts, route_for_lookup

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


@pytest.mark.parametrize("m", [1, 5, 200, 3000])
def test_linear_into_an_output_of_one_column(m):
    lin = Fp8Linear.quantize(torch.randn(1, 300, generator=gen(1), device=DEV))
    x = torch.randn(m, 300, generator=gen(2), device=DEV, dtype=torch.bfloat16)
    want = lin(x)
    buf = torch.full((3, m), 7.0, dtype=torch.bfloat16, device=DEV)
    out = buf.t()[:, 1:2]  # strides (1, m)
    assert lin(x, out=out) is out and torch.equal(out, want)
    assert (buf[0] == 7).all() and (buf[2] == 7).all()
    wide = torch.full((m, 6), 7.0, dtype=torch.bfloat16, device=DEV)
    lin(x, out=wide[:, 2:3])
    lin(x, out=wide[:, 3:6:3])
    assert torch.equal(wide[:, 2:4], want.expand(m, 2)) and (wide[:, :2] == 7).all() and (wide[:, 4:] == 7).all()


def test_linear_refuses_rows_that_overlap():
    lin = Fp8Linear.quantize(torch.randn(8, 64, generator=gen(1), device=DEV))
    x = torch.randn(4, 64, generator=gen(2), device=DEV)
    with pytest.raises(ValueError):
        lin(x, out=torch.empty(8, device=DEV).expand(4, 8))
    with pytest.raises(ValueError):
        lin(x, out=torch.empty(8, 4, device=DEV).t())
    one = Fp8Linear.quantize(torch.randn(1, 64, generator=gen(1), device=DEV))
    with pytest.raises(ValueError):
        one(x, out=torch.empty(1, 1, device=DEV).expand(4, 1))


@pytest.mark.parametrize("q,s", [(1, 1), (1, 4), (1, 30), (6, 1), (40, 1)])
def test_experts_into_rows_of_one_token_or_slot(q, s):
    e, h, i = 5, 200, 96
    ex = Fp8Experts.quantize(torch.randn(e, 2, i, h, generator=gen(3), device=DEV), torch.randn(e, h, i, generator=gen(4), device=DEV))
    x = torch.randn(q, h, generator=gen(5), device=DEV, dtype=torch.bfloat16)
    sel = torch.randint(0, e, (q, s), generator=gen(6), device=DEV)
    comp = torch.rand(q, s, generator=gen(7), device=DEV) < 0.8
    comp[0, 0] = True
    want = ex(x, sel, comp)
    for t, u in ((1, 1), (0, 0), (h + 8, h + 8), (s * h + 16, h)):
        strides = (t if q == 1 else max(t, h + 8), u if s == 1 else h + 8, 1)
        buf = torch.full((q * s * (h + 8) + 8 * s * h,), 3.0, dtype=torch.bfloat16, device=DEV)
        out = torch.as_strided(buf, (q, s, h), strides)
        ex(x, sel, comp, out)
        assert torch.equal(out[comp], want[comp]) and (out[~comp] == 3).all()
    if q > 1:
        with pytest.raises(ValueError):
            ex(x, sel, comp, torch.empty(1, s, h, dtype=torch.bfloat16, device=DEV).expand(q, s, h))


@pytest.mark.parametrize("q", [3, 50])
def test_experts_of_one_column(q):
    e, i = 3, 40
    ex = Fp8Experts.quantize(torch.randn(e, 2, i, 1, generator=gen(8), device=DEV), torch.randn(e, 1, i, generator=gen(9), device=DEV))
    x = torch.randn(q, 1, generator=gen(10), device=DEV)
    sel = torch.randint(0, e, (q, 2), generator=gen(11), device=DEV)
    want = ex(x, sel)
    buf = torch.full((q, 2, 3), 7.0, device=DEV)
    out = torch.as_strided(buf, (q, 2, 1), (6, 3, 5))
    ex(x, sel, None, out)
    assert torch.equal(out, want) and (buf[:, :, 1:] == 7).all()


@pytest.mark.parametrize("route", [lambda x: route_for_lookup(x, 4), lambda x: route_experts(x, 4, scoring="sigmoid")])
def test_logits_of_any_strides(route):
    x = torch.randn(5, 16, generator=gen(7), device=DEV)
    want = route(x)
    one = route(x[:1].clone())
    for y in (x.t().contiguous().t(), torch.cat([x, x], 1)[:, :16], x.repeat(2, 1)[::2], x[:, None, :].expand(5, 3, 16)[:, 1]):
        if y.shape == x.shape and torch.equal(y, x):
            assert all(torch.equal(a, b) for a, b in zip(route(y), want))
    column = x[0].clone()[:, None]
    assert column.t().stride() == (1, 1)
    for y in (column.t(), x[0][None], torch.as_strided(x, (1, 16), (0, 1))):
        assert all(torch.equal(a, b) for a, b in zip(route(y), one))
    for y in (x[0].expand(3, 16), x[:1].expand(3, -1)):
        assert all(torch.equal(a, b.expand(3, -1)) for a, b in zip(route(y), one))
    narrow = torch.as_strided(torch.arange(40.0, device=DEV), (4, 16), (5, 1))  # rows that overlap
    assert all(torch.equal(a, b) for a, b in zip(route(narrow), route(narrow.clone())))
