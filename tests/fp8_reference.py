"""Plain 64-bit forms of the 8-bit products and of expert routing, with the error bounds the GPU
tests use.

The 8-bit form of a row (and of a weight block) is defined bit by bit in fp32: a = max(max|x|,
2^-100), scale a / 448, q = e4m3(x * (448 / a)). Given the same bits, a product of two e4m3 numbers
is exact in fp32, so a kernel's dot product differs from the exact one only by fp32 additions:
at most 128 inside a block and one per block outside, plus the two scale products, each off by at
most 2^-24 of the running magnitude: |error| <= (128 + blocks + 4) 2^-24 sum |x^ w^|. On top comes
the rounding of the output type (unit roundoff of 8, 11 and 24 significant bits: 2^-8 bf16, 2^-11
fp16, 2^-24 fp32, relative, and half of the smallest subnormal)."""
import torch

BLOCK = 128
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
HALF_TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def blocks(n):
    return -(-n // BLOCK)


def e4m3_form(x, block_rows=1):
    """(q e4m3, scale fp32) of a 2D fp32 tensor."""
    x = x.float()
    rows, cols = x.shape
    rb, cb = -(-rows // block_rows), blocks(cols)
    p = torch.zeros(rb * block_rows, cb * BLOCK, device=x.device)
    p[:rows, :cols] = x
    p = p.view(rb, block_rows, cb, BLOCK)
    a = p.abs().amax((1, 3), keepdim=True).clamp_min(2.0 ** -100)
    top = torch.full_like(a, 448.0)
    q = (p * (top / a)).to(torch.float8_e4m3fn)
    scale = (a / top)[:, 0, :, 0]
    return q.view(rb * block_rows, cb * BLOCK)[:rows, :cols].contiguous(), scale.contiguous()


def values(q, scale, block_rows):
    """What (q, scale) stands for, in 64 bits."""
    rows, cols = q.shape
    s = scale.double().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
    return q.double() * s


def product(xv, wv):
    """(xv wv^T, bound of the fp32 error) for 64-bit values of 8-bit forms."""
    k = xv.shape[1]
    return xv @ wv.T, (128 + blocks(k) + 4) * 2.0 ** -24 * (xv.abs() @ wv.abs().T)


def with_output(y, bound, dtype):
    """The bound after rounding to the output type."""
    return bound * (1 + HALF_ULP[dtype]) + HALF_ULP[dtype] * y.abs() + HALF_TINY[dtype]


def expert(x, gate, up, down):
    """(y, bound before the output rounding) of down(silu(gate x) * (up x)); x: 2D input of any float
    type; gate, up, down: 64-bit weight values. Hidden elements whose fp32 error interval straddles
    an e4m3 rounding boundary may land on either side: their whole step is in the bound."""
    q, s = e4m3_form(x)
    xv = values(q, s, 1)
    g, dg = product(xv, gate)
    u, du = product(xv, up)
    sg = g * torch.sigmoid(g)
    h = sg * u
    # |silu'| <= 1.1; exp, the division and the products in fp32: below 2^-20 in all
    dh = 1.1 * dg * u.abs() + (sg.abs() + 1.1 * dg) * du + 2.0 ** -20 * h.abs()
    k = h.shape[1]
    pad = blocks(k) * BLOCK - k
    hp = torch.nn.functional.pad(h, (0, pad)).view(h.shape[0], -1, BLOCK)
    dp = torch.nn.functional.pad(dh, (0, pad)).view(h.shape[0], -1, BLOCK)
    a = hp.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100)
    da = dp.amax(-1, keepdim=True) / a  # relative error of the scale
    z, dz = hp * (448.0 / a), dp * (448.0 / a) + (hp * (448.0 / a)).abs() * (da + 2.0 ** -22)
    r = lambda v: v.clamp(-448, 448).to(torch.float8_e4m3fn).double()  # noqa: E731
    qv = r(z)
    step = torch.maximum((r(z + dz) - qv).abs(), (r(z - dz) - qv).abs())
    hv = (qv * (a / 448.0)).flatten(1)[:, :k]
    slack = ((step + qv.abs() * (da + 2.0 ** -22)) * (a / 448.0)).flatten(1)[:, :k]
    y, dy = product(hv, down)
    return y, dy + slack @ down.abs().T


def route(logits, top_k, scoring, bias, n_group, topk_group, rule, normalize, scale):
    """(weights, sel) of one definition in 64 bits, by a plain loop over the tokens. Keys as in the
    header: the logits without a bias when groups go by their largest key."""
    x = logits.double().cpu()
    q, e = x.shape
    m = x.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m) & (m < 0), torch.zeros_like(m), m)
    if scoring == "softmax":
        ex = torch.exp(x - m)
        tot = ex.sum(-1, keepdim=True)
        p = torch.where(tot == 0, torch.zeros_like(ex), ex / tot)
    else:
        p = torch.sigmoid(x)
    key = x.clone() if bias is None and rule == "max" else p + (0 if bias is None else bias.double().cpu())
    key[(x == -float("inf")) | key.isnan()] = -float("inf")
    w, sel = torch.zeros(q, top_k, dtype=torch.float64), torch.zeros(q, top_k, dtype=torch.int64)
    per = e // n_group
    for t in range(q):
        row = key[t].tolist()
        groups = []
        for g in range(n_group):
            best = sorted(row[g * per:(g + 1) * per], reverse=True)[:2 if rule == "top2" else 1]
            groups.append((-sum(best), g))
        kept = {g for _, g in sorted(groups)[:topk_group]}
        order = sorted((j for j in range(e) if j // per in kept), key=lambda j: (-row[j], j))[:top_k]
        sel[t] = torch.tensor(order)
        w[t] = p[t, sel[t]]
    if normalize:
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-20)
    return w * scale, sel
