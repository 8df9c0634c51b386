"""The routed-expert operators as timed workloads: expert routing, the 8-bit linear product and
the routed experts' products, each in a plain form (elementary torch operations in 32 bits)
and through the package's public calls."""
import math
import sys
from pathlib import Path

import torch

own = False

BLOCK = 128          # columns (and weight rows) that share one scale
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _package():
    root = str(Path(__file__).resolve().parents[1] / "tablemoe-sc26_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from table_moe import ops

    return ops


# ---- cases ---------------------------------------------------------------------------------


def _route(name, q, e, k, dtype, scoring, bias, groups, keep_groups, rule, normalize, scale, keep_k):
    return dict(name=name, op="route", q=q, e=e, k=k, dtype=dtype, scoring=scoring, bias=bias, groups=groups,
                keep_groups=keep_groups, rule=rule, normalize=normalize, scale=scale, keep_k=keep_k)


def _linear(name, m, n, k, dtype):
    return dict(name=name, op="linear", m=m, n=n, k=k, dtype=dtype)


def _experts(name, q, s, e, h, i, dtype, keep, skew):
    return dict(name=name, op="experts", q=q, s=s, e=e, h=h, i=i, dtype=dtype, keep=keep, skew=skew)


def listed():
    return [
        # one decoded token of the 128-expert model (top 8, softmax, renormalised): pure latency
        _route("route_token", 1, 128, 8, "bf16", "softmax", False, 1, 1, "max", True, 1.0, 5),
        # a 4096-token prompt, sigmoid scores with a balance bias, 8 groups of 32 experts of which 4 stay
        _route("route_prompt_groups", 4096, 256, 8, "f32", "sigmoid", True, 8, 4, "top2", True, 2.5, 5),
        # several prompts packed into one odd-sized batch of the 72-expert model (top 6), biased softmax
        _route("route_packed", 20011, 72, 6, "bf16", "softmax", True, 1, 1, "max", False, 1.0, 4),
        # one decoded token through a square projection of the 2048-wide model: weight-read latency
        _linear("linear_token", 1, 2048, 2048, "bf16"),
        # odd everything: 77 tokens, sizes that are no multiple of 16 or 128, fp16
        _linear("linear_odd", 77, 1111, 1000, "f16"),
        # a small prompt through a 2560-wide projection
        _linear("linear_prompt", 512, 2560, 2560, "bf16"),
        # the largest: packed prompts through a 4096-wide projection, bound by the tensor cores
        _linear("linear_packed", 8192, 4096, 4096, "bf16"),
        # one decoded token: 8 experts of 128, of which the first 5 or so are computed
        _experts("experts_token", 1, 8, 128, 2048, 768, "bf16", 0.6, 0.0),
        # a 16-token decode step of the 128-expert model, 60 % of the slots computed, the rest looked up
        _experts("experts_decode", 16, 8, 128, 2048, 768, "bf16", 0.6, 0.0),
        # a short prompt of a 72-expert, 2560-wide layer, every slot computed: weight reads with some reuse
        _experts("experts_short", 300, 6, 72, 2560, 1280, "bf16", 1.0, 0.5),
        # a few experts, odd widths, very uneven routing (experts without a token, tokens without a slot), fp16
        _experts("experts_odd", 333, 4, 24, 1000, 600, "f16", 0.5, 3.0),
        # a 4096-token prompt of the 128-expert model, 60 % computed: the largest
        _experts("experts_prompt", 4096, 8, 128, 2048, 768, "bf16", 0.6, 0.5),
    ]


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return v - 1 if v == 3072 else v  # a size kept free


def _width(rng, lo, hi):
    v = _log_int(rng, lo, hi)
    step = rng.choice((1, 8, 64, 128))
    v = max(lo, v // step * step)
    return v - step if v == 3072 else v


def draw(rng):
    op = rng.choice(("route", "linear", "experts"))
    if op == "route":
        groups = rng.choice((1, 1, 2, 4, 8))
        e = groups * rng.randint(max(2, 16 // groups), 320 // groups)
        keep_groups = rng.randint(max(1, groups // 2), groups)
        k = rng.randint(1, min(12, keep_groups * (e // groups)))
        q = _log_int(rng, 1, min(24000, 4000000 // e))
        return dict(op=op, q=q, e=e, k=k, dtype=rng.choice(("bf16", "f16", "f32")),
                    scoring=rng.choice(("softmax", "sigmoid")), bias=rng.random() < 0.5, groups=groups,
                    keep_groups=keep_groups, rule=rng.choice(("max", "top2")), normalize=rng.random() < 0.5,
                    scale=rng.choice((1.0, 2.5)), keep_k=rng.randint(0, k))
    if op == "linear":
        n, k = _width(rng, 64, 6000), _width(rng, 64, 6000)
        m = _log_int(rng, 1, min(8192, max(1, 8192 * 4096 * 4096 // (n * k))))
        return dict(op=op, m=m, n=n, k=k, dtype=rng.choice(("bf16", "f16")))
    h, i = _width(rng, 128, 2560), _width(rng, 64, 1400)
    e = rng.randint(4, min(128, max(5, 200000000 // (h * i))))
    s = rng.randint(1, min(8, e))
    q = _log_int(rng, 1, min(4096, max(1, 4096 * 8 * 2048 * 768 // (s * h * i))))
    return dict(op=op, q=q, s=s, e=e, h=h, i=i, dtype=rng.choice(("bf16", "f16")), keep=rng.choice((0.4, 0.6, 1.0)),
                skew=rng.choice((0.0, 0.5, 3.0)))


# ---- inputs --------------------------------------------------------------------------------


def _weight(gen, lead, n, k):
    """An e4m3 weight [*lead, n, k] with one fp32 scale per 128 x 128 block (short at the edges)."""
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    w = torch.randn(*lead, n, k, generator=gen, device="cuda", dtype=torch.float16).mul_(100.0)
    q = w.clamp_(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    scale = torch.rand(*lead, nb, kb, generator=gen, device="cuda").add_(0.5).mul_(0.01 / math.sqrt(k))
    return q, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case=dict(case))
    dt = DTYPES[case["dtype"]]
    if case["op"] == "route":
        st["logits"] = (torch.randn(case["q"], case["e"], generator=gen, device="cuda") * 1.5).to(dt)
        st["bias"] = torch.randn(case["e"], generator=gen, device="cuda") * 0.02 if case["bias"] else None
    elif case["op"] == "linear":
        # activations with a few large columns, as hidden states have
        x = torch.randn(case["m"], case["k"], generator=gen, device="cuda")
        x[:, ::97] *= 8.0
        st["x"] = x.to(dt)
        st["w"], st["ws"] = _weight(gen, (), case["n"], case["k"])
        if own:
            st["handle"] = _package().Fp8Linear(st["w"], st["ws"])
    else:
        q, s, e, h, i = (case[n] for n in ("q", "s", "e", "h", "i"))
        x = torch.randn(q, h, generator=gen, device="cuda")
        x[:, ::97] *= 8.0
        st["x"] = x.to(dt)
        pop = -case["skew"] * torch.log1p(torch.randperm(e, generator=gen, device="cuda").float())
        logits = torch.randn(q, e, generator=gen, device="cuda") + pop
        st["sel"] = torch.sort(logits, dim=-1, descending=True, stable=True).indices[:, :s].contiguous()
        keep = torch.rand(q, s, generator=gen, device="cuda") < case["keep"]
        if q == 1:
            keep = torch.arange(s, device="cuda")[None, :] < max(1, round(case["keep"] * s))
        st["compute"] = keep
        st["w13"], st["s13"] = _weight(gen, (e, 2), i, h)
        st["w2"], st["s2"] = _weight(gen, (e,), h, i)
        if own:
            st["handle"] = _package().Fp8Experts(st["w13"], st["s13"], st["w2"], st["s2"])
    return st


# ---- plain forms ---------------------------------------------------------------------------


def _round_rows(x):
    """x (fp32 [..., k]) as the values of its e4m3 form: one scale per row and 128 columns."""
    k = x.shape[-1]
    kb = -(-k // BLOCK)
    x = torch.nn.functional.pad(x, (0, kb * BLOCK - k)).unflatten(-1, (kb, BLOCK))
    a = x.abs().amax(-1, keepdim=True).clamp_min(AMAX_FLOOR)
    top = torch.full_like(a, E4M3_MAX)
    v = (x * (top / a)).to(torch.float8_e4m3fn).float() * (a / top)
    return v.flatten(-2)[..., :k]


def _values(q, scale):
    """An e4m3 weight [..., n, k] times its block scales, in fp32."""
    n, k = q.shape[-2:]
    s = scale.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]
    return q.float() * s


def _plain_route(st):
    c = st["case"]
    q, e = st["logits"].shape
    x = st["logits"].float()
    out = x == -math.inf
    if c["scoring"] == "softmax":
        m = x.amax(-1, keepdim=True)
        ex = torch.exp(x - torch.where(m == -math.inf, torch.zeros_like(m), m))
        total = ex.double().sum(-1, keepdim=True).float()  # the same 32 bits in whatever order it is summed
        score = torch.where(total == 0, torch.zeros_like(ex), ex / total)
    else:
        score = torch.ones_like(x) / (1.0 + torch.exp(-x))
    if st["bias"] is None and c["rule"] == "max":
        key = x
    else:
        key = score if st["bias"] is None else score + st["bias"]
    key = torch.where(out | key.isnan(), torch.full_like(key, -math.inf), key)
    allowed = torch.ones_like(out)
    if c["groups"] > 1:
        per = e // c["groups"]
        best = torch.sort(key.view(q, c["groups"], per), dim=-1, descending=True).values
        gkey = best[..., 0] + best[..., 1] if c["rule"] == "top2" and per > 1 else best[..., 0]
        gsel = torch.sort(gkey, dim=-1, descending=True, stable=True).indices[:, :c["keep_groups"]]
        gmask = torch.zeros(q, c["groups"], dtype=torch.bool, device=x.device).scatter_(1, gsel, True)
        allowed = gmask.repeat_interleave(per, 1)
    # allowed experts first, each part by key: a stable sort by key, then one by allowed
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.sort(allowed.gather(1, order).to(torch.int8), dim=-1, descending=True, stable=True).indices
    sel = order.gather(1, rank)[:, :c["k"]].contiguous()
    w = score.gather(1, sel)
    if c["normalize"]:
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-20)
    w = w * c["scale"]
    compute = (torch.arange(c["k"], device=x.device) < c["keep_k"]).expand(q, -1).contiguous()
    return dict(weights=w, sel=sel, compute=compute, reuse=~compute)


def _plain_linear(st):
    return torch.matmul(_round_rows(st["x"].float()), _values(st["w"], st["ws"]).T).to(st["x"].dtype)


def _plain_experts(st):
    """The computed slots sorted by expert and padded to the longest expert: three batched products
    over the experts that have a slot."""
    c, x, comp = st["case"], st["x"], st["compute"]
    out = torch.zeros(c["q"] * c["s"], c["h"], device=x.device)
    slots = comp.flatten().nonzero().squeeze(1)
    if slots.numel() == 0:
        return out.to(x.dtype).view(c["q"], c["s"], c["h"])
    active, which = torch.unique(st["sel"].flatten()[slots], return_inverse=True)
    order = torch.argsort(which, stable=True)
    slots, which = slots[order], which[order]
    count = torch.bincount(which, minlength=active.numel())
    place = torch.arange(slots.numel(), device=x.device) - (count.cumsum(0) - count)[which]
    rows = torch.zeros(active.numel(), int(count.max()), c["h"], device=x.device)
    rows[which, place] = _round_rows(x.float())[slots // c["s"]]
    pick = lambda w: w.view(torch.uint8)[active].view(torch.float8_e4m3fn)  # noqa: E731
    w13 = _values(pick(st["w13"]), st["s13"][active])
    g = torch.bmm(rows, w13[:, 0].transpose(1, 2))
    u = torch.bmm(rows, w13[:, 1].transpose(1, 2))
    hid = _round_rows(g / (1.0 + torch.exp(-g)) * u)
    y = torch.bmm(hid, _values(pick(st["w2"]), st["s2"][active]).transpose(1, 2))
    out[slots] = y[which, place]
    return out.to(x.dtype).view(c["q"], c["s"], c["h"])


def run(st):
    c = st["case"]
    if not own:
        return {"route": _plain_route, "linear": _plain_linear, "experts": _plain_experts}[c["op"]](st)
    if c["op"] == "route":
        w, sel, compute, reuse = _package().route_experts(
            st["logits"], c["k"], scoring=c["scoring"], bias=st["bias"], n_group=c["groups"],
            topk_group=c["keep_groups"], group_rule=c["rule"], normalize_topk=c["normalize"], scale=c["scale"],
            keep_k=c["keep_k"])
        return dict(weights=w, sel=sel, compute=compute, reuse=reuse)
    if c["op"] == "linear":
        return st["handle"](st["x"])
    return st["handle"](st["x"], st["sel"], st["compute"])


# ---- what a pass cannot do without -------------------------------------------------------------


def work(case):
    c, size = case, 4 if case["dtype"] == "f32" else 2
    if c["op"] == "route":
        return {"bytes": c["q"] * (c["e"] * size + c["k"] * (4 + 8 + 1 + 1)) + 4 * c["e"] * c["bias"],
                "flops": c["q"] * c["e"] * 8}
    kb = lambda n: -(-n // BLOCK)  # noqa: E731
    if c["op"] == "linear":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": size * m * (k + n) + n * k + 4 * kb(n) * kb(k), "flops": 2 * m * n * k}
    q, s, e, h, i = (c[n] for n in ("q", "s", "e", "h", "i"))
    slots = max(1, round(q * s * c["keep"]))
    active = min(slots, e * (1.0 - (1.0 - 1.0 / e) ** slots))  # expected experts with a slot (even routing)
    return {"bytes": size * q * h + q * s * (8 + 1) + active * (3 * h * i + 12 * kb(h) * kb(i)) + size * q * s * h,
            "flops": 6 * slots * h * i}


# ---- the definitions in 64 bits ----------------------------------------------------------------


def _e4m3_64(x):
    """The 8-bit form is defined bit by bit (its scale, its factor and the scaled value are 32-bit
    numbers, so that bf16 inputs on a rounding boundary have one answer); what it stands for is exact."""
    parts = []
    for b in torch.split(x, BLOCK, dim=-1):
        b = b.float()
        a = torch.clamp(b.abs().max(dim=-1, keepdim=True).values, min=AMAX_FLOOR)
        c = torch.tensor(E4M3_MAX, device=b.device)
        parts.append((b * c.div(a)).to(torch.float8_e4m3fn).double() * a.div(c).double())
    return torch.cat(parts, dim=-1)


def _weight_64(q, scale):
    w = q.double()
    for r in range(scale.shape[0]):
        for k in range(scale.shape[1]):
            w[r * BLOCK:(r + 1) * BLOCK, k * BLOCK:(k + 1) * BLOCK] *= scale[r, k].double()
    return w


def exact(case, seed):
    st = prepare(case, seed)
    c = case
    if c["op"] == "route":
        x = st["logits"].double()
        score = torch.softmax(x, -1) if c["scoring"] == "softmax" else torch.sigmoid(x)
        # the order of the keys is the same for logits and scores; the whole-number outputs are left to the plain form
        key = score + (0 if st["bias"] is None else st["bias"].double())
        if c["groups"] > 1:
            g = key.unflatten(1, (c["groups"], -1))
            top = g.topk(min(2, g.shape[-1]) if c["rule"] == "top2" else 1, -1).values.sum(-1)
            chosen = torch.argsort(top, dim=-1, descending=True, stable=True)[:, :c["keep_groups"]]
            mask = torch.full_like(top, -math.inf).scatter(1, chosen, 0.0)
            key = (g + mask[..., None]).flatten(1)
        w = score.gather(1, torch.argsort(key, dim=-1, descending=True, stable=True)[:, :c["k"]])
        if c["normalize"]:
            w = w / w.sum(-1, keepdim=True)
        return dict(weights=w * c["scale"], sel=None, compute=None, reuse=None)
    if c["op"] == "linear":
        return _e4m3_64(st["x"].double()) @ _weight_64(st["w"], st["ws"]).T
    out = torch.zeros(c["q"], c["s"], c["h"], dtype=torch.float64, device="cuda")
    x = _e4m3_64(st["x"].double())
    for e in range(c["e"]):
        t, s = torch.nonzero((st["sel"] == e) & st["compute"], as_tuple=True)
        if t.numel() == 0:
            continue
        g = x[t] @ _weight_64(st["w13"][e, 0], st["s13"][e, 0]).T
        u = x[t] @ _weight_64(st["w13"][e, 1], st["s13"][e, 1]).T
        h = _e4m3_64(g * torch.sigmoid(g) * u)
        out[t, s] = h @ _weight_64(st["w2"][e], st["s2"][e]).T
    return out
