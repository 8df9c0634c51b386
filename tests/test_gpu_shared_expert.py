"""ALUTCachedMoE with a shared expert of the caller's: the layer adds to what it returns, whatever that
is, and changes none of the caller's tensors."""
import pytest
import torch

from table_moe.cache_engine import HybridStorageManager
from table_moe.models import ALUTCachedMoE

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
E, H, L, K, S = 8, 64, 16, 32, 4


def manager():
    g = torch.Generator(device=DEV).manual_seed(1)
    pca = {m: {"proj": torch.randn(H, L, generator=g, device=DEV), "bias": torch.zeros(L, device=DEV)} for m in ("vision", "text")}
    return HybridStorageManager.from_tables(0, torch.randn(E, 2, K, L, generator=g, device=DEV),
                                            torch.randn(E, 2, K, H, generator=g, device=DEV).to(torch.bfloat16), pca,
                                            enable_online=False)


@pytest.mark.parametrize("q", [1, 6, 300])
def test_a_shared_expert_may_return_any_tensor(q):
    mgr = manager()
    g = torch.Generator(device=DEV).manual_seed(q)
    x = torch.randn(q, H, generator=g, device=DEV).to(torch.bfloat16)
    logits = torch.randn(q, E, generator=g, device=DEV)
    vis = torch.zeros(q, dtype=torch.bool, device=DEV)

    def zeros(x, sel, comp, collected):
        collected.zero_()

    def layer(shared):
        moe = ALUTCachedMoE(mgr, S, decode_keep_k=1, shared=shared)
        return moe(x, logits, vis, zeros, is_prefill=False)

    before = x.clone()
    row = torch.randn(1, H, generator=g, device=DEV).to(torch.bfloat16)
    wide = torch.zeros(q, 2 * H, dtype=torch.bfloat16, device=DEV)
    wide[:, ::2] = x
    kept = x.clone()
    want = layer(lambda x, out_dtype: x.to(out_dtype, copy=True))
    assert not torch.equal(want, layer(None))
    for what, shared in {"its input": lambda x, out_dtype: x, "a buffer of its own": lambda x, out_dtype: kept,
                         "every second column": lambda x, out_dtype: wide[:, ::2],
                         "columns first": lambda x, out_dtype: x.t().contiguous().t(),
                         "another type": lambda x, out_dtype: x.float()}.items():
        for _ in range(2):
            assert torch.equal(layer(shared), want), what
    assert torch.equal(layer(lambda x, out_dtype: row.expand(q, H)), layer(lambda x, out_dtype: row.repeat(q, 1)))
    assert torch.equal(x, before) and torch.equal(kept, before) and (wide[:, 1::2] == 0).all()
    with pytest.raises((ValueError, RuntimeError)):
        layer(lambda x, out_dtype: torch.zeros(q + 1, H, dtype=out_dtype, device=DEV))
