"""The routers on rows that are not ordinary numbers, and on several streams and in graphs: ``route_for_lookup`` / ``qwen_topk_softmax`` (softmax top-k) and
``route_experts``."""
import pytest
import torch

from table_moe.ops import qwen_topk_softmax, route_experts, route_for_lookup
from table_moe.skip import build_prefill_keep_mask

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


def _importance(kind):
    """A call of importance mode on logits, and the masks that it returns."""
    if kind == "softmax":
        return lambda x: route_for_lookup(x, 6, keep="importance", keep_rate=0.4)[2:]
    if kind == "experts":
        return lambda x: route_experts(x, 6, scoring="sigmoid", keep="importance", keep_rate=0.4)[2:]

    def mask(x):
        w, sel = x.topk(6, dim=-1)
        keep = build_prefill_keep_mask(sel, w.sigmoid(), None, x.shape[1], 0.4)
        return keep, ~keep
    return mask


@pytest.mark.parametrize("kind", ["softmax", "experts", "mask"])
def test_importance_masks_of_calls_on_two_streams(kind):
    """Each call's sums are its own: calls with other experts in favour, at the same time on other
    streams, return what they return alone."""
    call, e, n = _importance(kind), 96, 40
    xs = [logits_of(3000, e, s) + torch.linspace(-2, 2, e, device=DEV).roll(31 * s) for s in (1, 2, 3)]
    want = [call(x) for x in xs]
    assert not torch.equal(want[0][0], want[1][0])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[] for _ in xs]
    for _ in range(n):
        for x, st, g in zip(xs, streams, got):
            with torch.cuda.stream(st):
                g.append(call(x))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, w[0]) and torch.equal(b, w[1]) for a, b in g)


@pytest.mark.parametrize("kind,e", [("softmax", 37), ("experts", 41), ("mask", 43)])
def test_importance_masks_whose_first_call_is_captured(kind, e):
    """Expert counts that no other test uses: the first call is recorded, then an eager call runs before
    the first replay, and both are right."""
    call = _importance(kind)
    _importance(kind)(logits_of(50, 64, 0))  # (the kernels are loaded)
    x, y = logits_of(500, e, 1), logits_of(700, e, 2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(x)
    other = torch.empty(1 << 20, dtype=torch.uint8, device=DEV).fill_(255)  # memory that is not zero
    del other
    eager = call(y)
    graph.replay()
    again = call(y)
    x0 = x.clone()
    x.copy_(logits_of(500, e, 3))
    graph.replay()
    torch.cuda.synchronize()
    second = [t.clone() for t in out]
    x.copy_(x0)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, again))
    assert all(torch.equal(a, b) for a, b in zip(out, call(x0)))
    assert all(torch.equal(a, b) for a, b in zip(second, call(logits_of(500, e, 3))))
    want = call(torch.cat([y]))
    assert all(torch.equal(a, b) for a, b in zip(eager, want))


@pytest.mark.parametrize("bad", [1, 2, 5])
def test_a_nan_token_does_not_decide_the_others_masks(bad):
    """Its score adds nothing to its experts' sums: the mask is the one of weights with 0 in its place."""
    e, k = 48, 4
    x = logits_of(200, e, bad)
    x[:, :k] += 3.0  # the experts that a NaN row names are the batch's most important
    rows = torch.arange(bad, device=DEV) * 7
    x[rows] = NAN
    for route in (lambda **kw: route_for_lookup(x, k, **kw), lambda **kw: route_experts(x, k, scoring="softmax", **kw)):
        for attn in (None, torch.rand(200, generator=torch.Generator().manual_seed(1)).to(DEV)):
            w, sel, comp, _ = route(keep="importance", keep_rate=0.2, attn_scores=attn)
            assert w[rows].isnan().all()
            want = build_prefill_keep_mask(sel, w.nan_to_num(0.0), attn, e, 0.2)
            assert torch.equal(comp, want) and comp[rows].all()
            assert torch.equal(build_prefill_keep_mask(sel, w, attn, e, 0.2), want)
