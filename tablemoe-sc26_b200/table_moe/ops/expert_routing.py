"""Expert routing on the ``alut_route_experts`` kernel of ``libalut.so``: softmax or sigmoid
scores, a balance bias, expert groups, top-k, renormalised and scaled weights, and the keep
mask of the layer. New: the reference routes by a plain softmax
(``table_moe/ops/qwen_topk_softmax.py:122-153``, here ``qwen_topk_softmax``).

The four results are the inputs of ``VectorSearchEngine.lookup_combine``, as
``route_for_lookup``'s are. There is no torch fallback.
"""
from __future__ import annotations

import torch

from ..cache_engine import _alut
from .qwen_topk_softmax import _check_logits, _workspace

_SCORING = {"softmax": 0, "sigmoid": 1}
_GROUP_RULE = {"max": 0, "top2": 1}
_KEEP = {"fixed": 0, "importance": 1}


def _choice(table, value, name):
    try:
        return table[value]
    except (KeyError, TypeError):
        raise ValueError(f"{name} must be one of {sorted(table)}, got {value!r}") from None


@_alut.on_device_of_first
def route_experts(router_logits, top_k, *, scoring="softmax", bias=None, n_group=1, topk_group=None, group_rule="max",
                  normalize_topk=False, scale=1.0, keep="fixed", keep_k=None, keep_rate=0.6, attn_scores=None):
    """(weights [Q,k] f32, selected_experts [Q,k] int64, compute_mask [Q,k] bool, reuse_mask
    [Q,k] bool) of router logits [Q,E] (f32, bf16 or f16).

    ``scoring``: "softmax" or "sigmoid". ``bias`` [E] fp32 is added to the scores for the choice
    only; the weights are the scores themselves. With ``n_group`` > 1 the experts form that many
    groups of consecutive ones, and only those of the ``topk_group`` best groups (default: all) may
    be chosen; a group counts by its largest biased score (``group_rule`` "max") or by the sum of
    its two largest ("top2"). Equal scores go to the lowest expert id; logits of -inf and NaN
    come last. ``normalize_topk`` divides the weights by their sum (clamped at 1e-20), then
    ``scale`` multiplies them. ``keep``, ``keep_k``, ``keep_rate``, ``attn_scores``: the keep
    mask, as in ``route_for_lookup``."""
    x, stride = _check_logits(router_logits)
    q, e = x.shape
    dev = x.device
    top_k, n_group = int(top_k), int(n_group)
    if top_k <= 0:
        raise ValueError(f"top_k must be positive, got {top_k}")
    if bias is not None and (bias.shape != (e,) or bias.dtype != torch.float32 or bias.device != dev
                             or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous fp32 tensor of shape ({e},) on {dev}")
    r = _alut.Router(e, top_k, _choice(_SCORING, scoring, "scoring"), n_group,
                     n_group if topk_group is None else int(topk_group), _choice(_GROUP_RULE, group_rule, "group_rule"),
                     1 if normalize_topk else 0, scale, None if bias is None else bias.data_ptr())
    mode = _choice(_KEEP, keep, "keep")
    shape, rows = (q, top_k), (top_k, 1)  # empty_strided: 0.9 us less than empty, four times
    w = torch.empty_strided(shape, rows, dtype=torch.float32, device=dev)
    sel = torch.empty_strided(shape, rows, dtype=torch.int64, device=dev)
    comp = torch.empty_strided(shape, rows, dtype=torch.bool, device=dev)
    reuse = torch.empty_strided(shape, rows, dtype=torch.bool, device=dev)
    attn, ws, ws_bytes = None, None, 0
    if mode == 1:
        if attn_scores is not None and attn_scores.numel() == q:
            attn = attn_scores.reshape(-1).to(device=dev, dtype=torch.float32).contiguous()
        ws = _workspace(dev, e)
        ws_bytes = ws.numel()
    rc = _alut.load().alut_route_experts(r, q, x.data_ptr(), _alut.dtype_code(x.dtype), stride, mode,
                                         -1 if keep_k is None else max(int(keep_k), 0), keep_rate, _alut.ptr(attn),
                                         w.data_ptr(), sel.data_ptr(), comp.data_ptr(), reuse.data_ptr(), top_k,
                                         _alut.ptr(ws), ws_bytes, _alut.stream_ptr(dev))
    if rc:
        _alut.check(rc, "alut_route_experts")
    return w, sel, comp, reuse
