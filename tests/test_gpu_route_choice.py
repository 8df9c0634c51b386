"""What route_experts chooses, held against the 64-bit keys that the choice goes by. A choice by logits
is exact: the expert ids are those of the plain form. A choice by scores may differ from it only where
the 64-bit keys, or group keys, are as near to each other as fp32 scores can be wrong; the weights
always belong to the ids that were chosen.

Errors of an fp32 score p, in units of u = 2^-24: softmax p = expf(x - m) / sum: the difference is off by
u |x - m|, expf by 4 u, the sum by the same again, the rounding of the sum and the division by 2 u; a
sigmoid has expf by 4 u, an addition and a division. So |dp| <= (2 max|x - m| + 16) u p; a key adds one
rounding for its bias, a group key one more for its sum. Weights: the normalisation adds the error of the sum, k
additions and a division, the scale one rounding."""
import pytest
import torch

import fp8_reference as ref
from table_moe.ops import route_experts

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
U = 2.0 ** -24


def keys_of(x, scoring, bias):
    """(scores, keys, error of each score) in 64 bits."""
    x = x.double().cpu()
    p = torch.softmax(x, -1) if scoring == "softmax" else torch.sigmoid(x)
    spread = (x.amax(-1) - x.amin(-1)).amax() if scoring == "softmax" else 0.0
    b = torch.zeros(x.shape[1], dtype=torch.float64) if bias is None else bias.double().cpu()
    return p, p + b, (2 * spread + 16) * U * p


@pytest.mark.parametrize("q,e,k,groups,keep", [
    (33, 64, 6, 8, 3), (64, 128, 8, 1, 1), (200, 256, 8, 8, 4), (17, 160, 6, 32, 7), (50, 500, 64, 5, 2), (7, 513, 9, 3, 2),
    (30, 4096, 8, 32, 4), (6, 24, 4, 24, 5), (20, 2000, 64, 1, 1),
])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("use_bias,rule", [(False, "max"), (True, "max"), (False, "top2"), (True, "top2")])
def test_the_choice_follows_its_keys(q, e, k, groups, keep, scoring, use_bias, rule):
    g = torch.Generator().manual_seed(q * e + k)
    x = (torch.randn(q, e, generator=g) * 2).to(DEV)
    bias = (torch.randn(e, generator=g) * 0.05).to(DEV) if use_bias else None
    per = e // groups
    for normalize, scale in ((False, 1.0), (True, 2.5)):
        w, sel, _, _ = (t.cpu() for t in route_experts(x, k, scoring=scoring, bias=bias, n_group=groups, topk_group=keep,
                                                       group_rule=rule, normalize_topk=normalize, scale=scale))
        p, key, dp = keys_of(x, scoring, bias)
        if not use_bias and rule == "max":  # by the logit itself
            assert torch.equal(sel, ref.route(x, k, scoring, bias, groups, keep, rule, normalize, scale)[1])
        else:
            err = dp + U * key.abs()
            top = key.view(q, groups, per).sort(-1, descending=True).values[..., :2 if rule == "top2" else 1]
            gkey = top.sum(-1)
            gerr = err.view(q, groups, per).amax(-1) * 2 + U * gkey.abs()
            last = gkey.sort(-1, descending=True).values[:, keep - 1:keep]  # the last group that stays
            slack = gerr + gerr.amax(-1, keepdim=True)
            may = (gkey >= last - slack).repeat_interleave(per, 1)
            must = (gkey > last + slack).repeat_interleave(per, 1)
            assert may.gather(1, sel).all()
            assert all(len(set((r // per).tolist())) <= keep and len(set(r.tolist())) == k for r in sel)
            ks, es = key.gather(1, sel), err.gather(1, sel)
            assert (ks[:, :-1] - ks[:, 1:] >= -(es[:, :-1] + es[:, 1:])).all()  # descending
            chosen = torch.zeros_like(must).scatter_(1, sel, True)
            ahead = key - ks[:, -1:] > err + es[:, -1:]  # surely larger than the last one chosen
            assert not (must & ~chosen & ahead).any()
        want, dw = p.gather(1, sel), dp.gather(1, sel)
        if normalize:
            total = want.sum(-1, keepdim=True)
            dw = (dw + want * (dw.sum(-1, keepdim=True) / total + (k + 1) * U)) / total
            want = want / total
        assert ((w.double() - want * scale).abs() <= scale * (dw + 2 * U * want)).all()
