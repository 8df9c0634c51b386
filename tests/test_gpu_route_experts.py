"""route_experts against a plain 64-bit loop (tests/fp8_reference.py route). Expert ids must be equal
except where the 64-bit keys (or group sums) of the two choices are within 1e-6 of each other; weights
within 1e-5 relative (fp32 exp and division: a few 2^-24 each, sums of up to 4096 terms rounded once)."""
import pytest
import torch

import fp8_reference as ref
from table_moe.ops import qwen_topk_softmax, route_experts, route_for_lookup

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def logits_of(q, e, dtype, seed):
    return (torch.randn(q, e, generator=torch.Generator().manual_seed(seed)) * 2).to(dtype).to(DEV)


@pytest.mark.parametrize("q,e,k,groups,keep", [
    (1, 1, 1, 1, 1), (1, 8, 8, 1, 1), (5, 72, 6, 1, 1), (33, 64, 6, 8, 3), (64, 128, 8, 1, 1), (40, 256, 8, 8, 4),
    (17, 160, 6, 32, 7), (9, 96, 12, 4, 4), (21, 500, 64, 5, 2), (7, 513, 9, 3, 2), (3, 4096, 8, 32, 4),
    (6, 24, 4, 24, 5), (11, 33, 33, 1, 1),
])
@pytest.mark.parametrize("scoring,use_bias,rule", [("softmax", False, "max"), ("sigmoid", True, "top2"),
                                                  ("softmax", True, "max"), ("sigmoid", False, "top2")])
def test_routing_matches_64_bits(q, e, k, groups, keep, scoring, use_bias, rule):
    for dtype, normalize, scale in ((torch.float32, True, 2.5), (torch.bfloat16, False, 1.0)):
        x = logits_of(q, e, dtype, q * e + k)
        bias = torch.randn(e, generator=torch.Generator().manual_seed(e)).mul(0.1).to(DEV) if use_bias else None
        w, sel, comp, reuse = route_experts(x, k, scoring=scoring, bias=bias, n_group=groups, topk_group=keep,
                                            group_rule=rule, normalize_topk=normalize, scale=scale, keep_k=k // 2)
        rw, rsel = ref.route(x, k, scoring, bias, groups, keep, rule, normalize, scale)
        p = torch.softmax(x.double(), -1).cpu() if scoring == "softmax" else torch.sigmoid(x.double()).cpu()
        key = p + (0 if bias is None else bias.double().cpu())
        for t in range(q):
            if sel[t].cpu().equal(rsel[t]):
                assert torch.allclose(w[t].double().cpu(), rw[t], rtol=1e-5, atol=0)
                continue
            gap = (key[t][sel[t].cpu()] - key[t][rsel[t]]).abs().max()
            assert gap < 1e-6 and dtype == torch.float32, (t, sel[t], rsel[t])
        assert (sel.sort(-1).values.diff() != 0).all()
        assert torch.equal(comp, (torch.arange(k, device=DEV) < k // 2).expand(q, k)) and torch.equal(reuse, ~comp)


def test_plain_softmax_is_the_drop_in_router():
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = logits_of(50, 128, dtype, 3)
        for normalize in (False, True):
            w, sel = qwen_topk_softmax(x.float() + torch.arange(128, device=DEV) * 1e-4, 8, normalize_topk=normalize)
            w2, sel2, _, _ = route_experts(x.float() + torch.arange(128, device=DEV) * 1e-4, 8, normalize_topk=normalize)
            assert torch.equal(sel, sel2) and torch.allclose(w, w2, rtol=1e-5, atol=0)


def test_equal_keys_go_to_the_lowest_expert():
    x = torch.zeros(3, 40, device=DEV)
    x[1, 20:] = 1.0
    x[2] = -0.0
    x[2, ::2] = 0.0
    for kw in (dict(), dict(scoring="sigmoid"), dict(bias=torch.zeros(40, device=DEV)),
               dict(scoring="sigmoid", n_group=4, topk_group=4, group_rule="top2")):
        _, sel, _, _ = route_experts(x, 5, **kw)
        assert sel[0].tolist() == [0, 1, 2, 3, 4]
        assert sel[1].tolist() == [20, 21, 22, 23, 24]
        assert sel[2].tolist() == [0, 1, 2, 3, 4]
    _, sel, _, _ = route_experts(x[:1], 4, n_group=10, topk_group=2)  # equal groups too
    assert sel[0].tolist() == [0, 1, 2, 3]
    big = torch.zeros(1, 4096, device=DEV)
    assert route_experts(big, 6)[1][0].tolist() == list(range(6))


def test_masked_and_non_finite_logits():
    inf, nan = float("inf"), float("nan")
    x = torch.randn(6, 16, generator=torch.Generator().manual_seed(1)).to(DEV)
    x[0, 4:] = -inf        # four experts left for a top 6
    x[1] = -inf            # a row with nothing left
    x[2, 3] = nan
    x[3, 5] = inf
    x[4, :] = torch.finfo(torch.float32).min
    bias = torch.full((16,), 5.0, device=DEV)
    bias[:8] = 0.0
    for kw in (dict(), dict(bias=bias), dict(scoring="sigmoid"), dict(scoring="sigmoid", bias=bias)):
        w, sel, comp, reuse = route_experts(x, 6, keep_k=3, **kw)
        assert ((sel >= 0) & (sel < 16)).all() and (sel.sort(-1).values.diff() > 0).all()
        assert sorted(sel[0, :4].tolist()) == [0, 1, 2, 3] and sel[0, 4:].tolist() == [4, 5] and (w[0, 4:] == 0).all()
        assert sel[1].tolist() == list(range(6)) and (w[1] == 0).all()
        assert w[5].isfinite().all() and w[4].isfinite().all()
        if kw.get("scoring") == "sigmoid":
            assert 3 not in sel[2].tolist() and w[2].isfinite().all()
            assert 5 in sel[3].tolist() or kw.get("bias") is not None
        else:
            assert w[2].isnan().all() and w[3].isnan().all()
    w, sel, _, _ = route_experts(x[:2], 6, normalize_topk=True)
    assert abs(float(w[0].sum()) - 1) < 1e-6 and (w[1] == 0).all()
    w, sel, _, _ = route_experts(x[:2], 4, n_group=4, topk_group=2, group_rule="top2", scoring="sigmoid")
    assert sel[1].tolist() == [0, 1, 2, 3]


def test_importance_mask_is_the_one_of_route_for_lookup():
    x = logits_of(300, 64, torch.float32, 9)
    attn = torch.rand(300, generator=torch.Generator().manual_seed(2)).to(DEV)
    for a in (None, attn):
        want = route_for_lookup(x, 6, keep="importance", keep_rate=0.5, attn_scores=a)
        got = route_experts(x, 6, keep="importance", keep_rate=0.5, attn_scores=a)
        assert torch.equal(want[1], got[1])
        assert (want[2] != got[2]).float().mean() < 0.02  # an expert on the boundary at most
    assert torch.equal(got[3], ~got[2])


def test_strides_streams_and_empty_batches():
    wide = logits_of(20, 90, torch.float16, 4)
    x = wide[:, 11:83]
    want = route_experts(x.contiguous(), 6, scoring="sigmoid")
    got = route_experts(x, 6, scoring="sigmoid")
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        got = route_experts(x.t().contiguous().t(), 6, scoring="sigmoid")
    st.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    assert route_experts(x[:0], 6)[0].shape == (0, 6)


@pytest.mark.parametrize("kw", [dict(top_k=0), dict(top_k=17), dict(n_group=3), dict(n_group=4, topk_group=5),
                                dict(n_group=8, topk_group=1, top_k=3), dict(n_group=0), dict(n_group=16, topk_group=0),
                                dict(scoring="tanh"), dict(group_rule="sum"), dict(keep="none"),
                                dict(bias=torch.zeros(15)), dict(keep="importance", keep_rate=-1.0)])
def test_refusals(kw):
    x = torch.zeros(2, 16, device=DEV)
    kw = dict(kw)
    if "bias" in kw:
        kw["bias"] = kw["bias"].to(DEV)
    with pytest.raises(ValueError):
        route_experts(x, kw.pop("top_k", 4), **kw)
