"""The cached MoE layer with its routed experts, shared expert and router on the new kernels:
table_moe.models.ALUTCachedMoE with Fp8Experts as run_experts, Fp8SharedExpert, and grouped sigmoid
routing with a bias, against a restatement of the combine (cached rows, computed outputs, weights
renormalised over the survivors) on 64-bit expert outputs. Tolerance: tests/parity.py check_combined
(1e-2 of the value and of the largest value), which covers the 8-bit form's rounding flips."""
import pytest
import torch

import fp8_reference as ref
import oracle.oracle as orc
from parity import check_combined, check_search
from table_moe.cache_engine import HybridStorageManager
from table_moe.models import ALUTCachedMoE, Fp8SharedExpert
from table_moe.ops import Fp8Experts, quantize_fp8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
E, H, I, L, K, S = 16, 256, 192, 32, 64, 4


def layer(seed):
    g = torch.Generator().manual_seed(seed)
    raw = torch.randn(E, 2, K, L, generator=g)
    proj = torch.stack([torch.linalg.qr(torch.randn(H, L, generator=g))[0] for _ in range(2)]).contiguous()
    values = (torch.randn(E, 2, K, H, generator=g) * 0.5).to(torch.bfloat16)
    pca = {m: {"proj": proj[i].to(DEV), "bias": torch.zeros(L, device=DEV)} for i, m in enumerate(("vision", "text"))}
    mgr = HybridStorageManager.from_tables(0, raw.to(DEV), values.to(DEV), pca, enable_online=False)
    gate_up = (torch.randn(E, 2, I, H, generator=g) * H ** -0.5).to(DEV)
    down = (torch.randn(E, H, I, generator=g) * I ** -0.5).to(DEV)
    shared = (torch.randn(2 * I, H, generator=g) * H ** -0.5).to(DEV), (torch.randn(H, I, generator=g) * I ** -0.5).to(DEV)
    return mgr, raw, proj, values, gate_up, down, shared


@pytest.mark.parametrize("Q,prefill,with_shared", [(1, False, False), (12, False, True), (200, True, True),
                                                   (300, True, False)])
def test_cached_layer_with_8_bit_experts(Q, prefill, with_shared):
    mgr, raw, proj, values, gate_up, down, sh = layer(Q)
    g = torch.Generator().manual_seed(100 + Q)
    x = torch.randn(Q, H, generator=g).to(torch.bfloat16).to(DEV)
    vis = (torch.rand(Q, generator=g) < 0.3).to(DEV)
    logits = torch.randn(Q, E, generator=g).to(DEV)
    bias = (torch.randn(E, generator=g) * 0.05).to(DEV)
    experts = Fp8Experts.quantize(gate_up, down)
    shared = Fp8SharedExpert.quantize(*sh) if with_shared else None
    router = dict(scoring="sigmoid", bias=bias, n_group=4, topk_group=2, group_rule="top2", scale=2.0)
    moe = ALUTCachedMoE(mgr, S, normalize_topk=True, decode_keep_k=2, keep_rate=0.5, router=router, shared=shared)
    out, r = moe(x, logits, vis, experts, is_prefill=prefill, return_routing=True)
    torch.cuda.synchronize()
    assert experts.device_errors() == 0
    sel, w, comp = r["selected_experts"], r["weights"], r["compute_mask"]
    rw, rsel = ref.route(logits, S, "sigmoid", bias, 4, 2, "top2", True, 2.0)
    assert torch.equal(sel.cpu(), rsel) and torch.allclose(w.double().cpu(), rw, rtol=1e-5, atol=0)
    sn, vn, hit, idx = sel.cpu().numpy(), vis.cpu().numpy(), r["hit"].cpu().numpy(), r["idx"].cpu().numpy()
    q = orc.project(x.float().cpu().numpy(), vn, proj.numpy(), torch.zeros(2, L).numpy())
    rh, ri, _, _ = orc.search(q, raw.numpy(), sn, vn, ~comp.cpu().numpy(), 0.0, 0.0, cmp_ge=False)
    check_search(hit, idx, rh, ri, q, raw.numpy(), sn, vn, (0.0, 0.0), "float32", what="lookups")
    # the combine on 64-bit expert outputs
    forms = lambda t: ref.values(*(v.view(-1, v.shape[-1]) for v in quantize_fp8(t, 128)), 128)  # noqa: E731
    rows = torch.zeros(Q, S, H, dtype=torch.float64, device=DEV)
    for e in range(E):
        t, s = torch.nonzero((sel == e) & comp, as_tuple=True)
        if t.numel():
            rows[t, s] = ref.expert(x[t], forms(gate_up[e, 0]), forms(gate_up[e, 1]), forms(down[e]))[0]
    hits = r["hit"] & ~comp
    t, s = torch.nonzero(hits, as_tuple=True)
    rows[t, s] = values.to(DEV)[sel[t, s], (~vis[t]).long(), r["idx"][t, s]].double()
    surv = (comp | hits).double()
    kept = (w.double() * surv).sum(-1, keepdim=True)
    wt = torch.where(kept > 0, w.double() * surv / torch.where(kept > 0, kept, torch.ones_like(kept)), torch.zeros_like(kept))
    want = torch.einsum("ts,tsh->th", wt, rows)
    if with_shared:
        both = forms(sh[0])  # one weight of 2 I rows: its blocks of 128 rows may straddle the halves
        want = want + ref.expert(x, both[:I], both[I:], forms(sh[1]))[0]
    check_combined(out.float().cpu().numpy(), want.cpu().numpy(), what=f"layer Q{Q}")


def test_shared_expert_refuses_what_does_not_fit():
    with pytest.raises(ValueError):
        Fp8SharedExpert.quantize(torch.zeros(64, 32, device=DEV), torch.zeros(32, 48, device=DEV))
