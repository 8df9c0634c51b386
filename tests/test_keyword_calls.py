"""The public functions keep their arguments' names: called by keyword they do what they do by position,
and a call without its tensor is Python's own TypeError. On the host, no GPU call is made."""
import inspect

import pytest
import torch

from table_moe.cache_engine.manager import normalize_rows
from table_moe.ops import qwen_topk_softmax, quantize_fp8, route_experts, route_for_lookup
from table_moe.skip import build_prefill_keep_mask


def test_keywords_reach_the_functions():
    x = torch.zeros(2, 8)
    for fn in (route_experts, route_for_lookup, qwen_topk_softmax):
        with pytest.raises(ValueError, match="CUDA"):
            fn(router_logits=x, top_k=2)
    with pytest.raises(ValueError, match="CUDA"):
        quantize_fp8(x=x, block_rows=1)
    kw = dict(routing_weights=x, attn_scores=None, num_experts=8, keep_rate=0.5)
    with pytest.raises(ValueError, match="CUDA"):
        build_prefill_keep_mask(selected_experts=x.long(), **kw)
    assert build_prefill_keep_mask(selected_experts=x.long()[:0], **kw).shape == (0, 8)
    y = torch.randn(3, 5)
    assert torch.equal(normalize_rows(x=y, eps=1e-6), normalize_rows(y, 1e-6))


@pytest.mark.parametrize("fn,first", [(route_experts, "router_logits"), (route_for_lookup, "router_logits"),
                                      (quantize_fp8, "x"), (build_prefill_keep_mask, "selected_experts"),
                                      (normalize_rows, "x")])
def test_signatures(fn, first):
    assert next(iter(inspect.signature(fn).parameters)) == first
    with pytest.raises(TypeError, match=first):
        fn()
