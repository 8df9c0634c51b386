"""The routers on rows that are not ordinary numbers, on inputs of unusual strides, and on several
streams and in graphs: ``route_for_lookup`` / ``qwen_topk_softmax`` (softmax top-k) and
``route_experts``."""
import pytest
import torch

from table_moe.ops import qwen_topk_softmax, route_for_lookup

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
INF, NAN = float("inf"), float("nan")


def logits_of(q, e, seed):
    return (torch.randn(q, e, generator=torch.Generator().manual_seed(seed)) * 2).to(DEV)


@pytest.mark.parametrize("e,k", [(6, 6), (16, 6), (72, 6), (128, 8), (1000, 64), (33, 1)])
@pytest.mark.parametrize("normalize", [False, True])
def test_softmax_router_on_rows_without_an_order(e, k, normalize):
    """Every row names k different experts; a bad row's weights are NaN (a NaN or +inf logit) or 0 (no
    expert left), and the other rows are what they are without it."""
    x = logits_of(8, e, e + k)
    good = qwen_topk_softmax(x, k, normalize_topk=normalize)
    x[0] = NAN
    x[1, e // 2] = NAN
    x[2, e - 1] = INF
    x[3] = -INF
    x[4, 1:] = -INF  # one expert left
    x[5] = torch.finfo(torch.float32).min
    w, sel = qwen_topk_softmax(x, k, normalize_topk=normalize)
    assert ((sel >= 0) & (sel < e)).all()
    assert all(len(set(r)) == k for r in sel.tolist())
    assert w[:3].isnan().all()
    first = list(range(k))
    assert sel[0].tolist() == first and sel[1].tolist() == first and sel[2].tolist() == first
    assert (w[3] == 0).all() and sel[3].tolist() == first
    assert w[4, 0] == 1 and (w[4, 1:] == 0).all() and sel[4].tolist() == first
    assert sel[5].tolist() == first
    want = torch.full((k,), 1.0 / (k if normalize else e), device=DEV)
    assert torch.allclose(w[5], want, rtol=1e-5, atol=0)  # 1000 additions of 1 and two divisions
    assert torch.equal(w[6:], good[0][6:]) and torch.equal(sel[6:], good[1][6:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_softmax_router_masks_hold_on_such_rows(dtype):
    x = logits_of(40, 64, 5).to(dtype)
    x[7], x[9, 3], x[11] = NAN, INF, -INF
    for kw in (dict(keep="fixed", keep_k=2), dict(keep="importance", keep_rate=0.5)):
        w, sel, comp, reuse = route_for_lookup(x, 6, **kw)
        assert ((sel >= 0) & (sel < 64)).all() and torch.equal(reuse, ~comp)
    assert torch.equal(route_for_lookup(x, 6, keep_k=2)[2], (torch.arange(6, device=DEV) < 2).expand(40, 6))
