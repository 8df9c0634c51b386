"""The 8-bit products on the GPU against plain 64-bit forms (tests/fp8_reference.py, which derives
the bounds): the quantisers bit for bit, Fp8Linear and Fp8Experts over the kernels' size ranges,
types, strides and masks."""
import pytest
import torch

import fp8_reference as ref
from table_moe.cache_engine import CacheConfig
from table_moe.ops import Fp8Experts, Fp8Linear, quantize_fp8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def activations(g, rows, cols, dtype):
    x = torch.randn(rows, cols, generator=g, device=DEV)
    x[:, ::37] *= 8.0
    return x.to(dtype)


def weight(g, lead, n, k):
    w = torch.randn(*lead, n, k, generator=g, device=DEV)
    w = w * torch.exp(torch.randn(*lead, n, 1, generator=g, device=DEV)) / k ** 0.5
    return quantize_fp8(w, 128)


def close(y, want, bound, what=""):
    got = y.double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst " \
        f"{float(((got - want).abs() / bound)[bad].max()):.3g} x the bound at {bad.nonzero()[0].tolist()}"


# ---- the form --------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 127), (5, 128), (130, 129), (64, 1000), (257, 300)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_is_the_form_bit_for_bit(rows, cols, dtype, block_rows):
    g = gen(rows * 1000 + cols)
    x = (torch.randn(rows, cols, generator=g, device=DEV) * torch.exp(4 * torch.randn(rows, 1, generator=g, device=DEV)))
    x[rows // 2] = 0.0  # an empty row: its scale is the floor's
    x = x.to(dtype)
    q, s = quantize_fp8(x, block_rows)
    wq, wsc = ref.e4m3_form(x, block_rows)
    assert torch.equal(s, wsc)
    assert torch.equal(q.view(torch.uint8) & 0x7F, wq.view(torch.uint8) & 0x7F)
    nz = (wq.float() != 0) & ~wq.float().isnan()  # (a NaN has no sign to compare)
    assert torch.equal(q.float()[nz], wq.float()[nz])


def test_quantize_batches_views_and_extremes():
    x = torch.randn(2, 3, 130, 200, generator=gen(1), device=DEV)
    q, s = quantize_fp8(x, 128)
    assert q.shape == x.shape and s.shape == (2, 3, 2, 2)
    for i in range(2):
        for j in range(3):
            wq, wsc = ref.e4m3_form(x[i, j], 128)
            assert torch.equal(q[i, j].float(), wq.float()) and torch.equal(s[i, j], wsc)
    wide = torch.randn(9, 400, generator=gen(2), device=DEV)
    q, s = quantize_fp8(wide[:, 5:205])  # rows of a wider tensor, an odd start
    wq, wsc = ref.e4m3_form(wide[:, 5:205])
    assert torch.equal(q.float(), wq.float()) and torch.equal(s, wsc)
    e = torch.zeros(4, 256, device=DEV)
    e[0, 3], e[1, 200], e[2, :] = float("nan"), float("inf"), 1e-38
    q, s = quantize_fp8(e)
    v = q.float() * s.repeat_interleave(128, 1)
    assert v[0, :128].isnan().all() and (v[0, 128:] == 0).all()
    assert v[1, 128:].isnan().all() and (v[1, :128] == 0).all()
    assert (v[2] == 0).all() and (v[3] == 0).all()  # far below the floor of 2^-100
    big = torch.tensor([[3.4e38, -3.4e38, 1.0, 3.4e38 / 448]], device=DEV)
    q, _ = quantize_fp8(big)
    assert q.float().tolist() == [[448.0, -448.0, 0.0, 1.0]]


# ---- linear ----------------------------------------------------------------------------------


@pytest.mark.parametrize("m,n,k", [
    (1, 1, 1), (1, 2048, 2048), (2, 33, 129), (7, 128, 127), (8, 100, 16), (9, 257, 1000), (16, 512, 2560),
    (31, 64, 4096), (64, 1111, 640), (65, 130, 8200), (127, 129, 128), (128, 256, 256), (129, 255, 272),
    (300, 1000, 1000), (513, 384, 2048), (1000, 700, 136),
])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_linear_matches_64_bits(m, n, k, dtype):
    g = gen(m + n + k)
    x = activations(g, m, k, dtype)
    w, s = weight(g, (), n, k)
    y = Fp8Linear(w, s)(x)
    assert y.dtype == dtype and y.shape == (m, n)
    want, bound = ref.product(ref.values(*ref.e4m3_form(x), 1), ref.values(w, s, 128))
    close(y, want, ref.with_output(want, bound, dtype), f"{m}x{n}x{k}")


@pytest.mark.parametrize("m", [3, 200])
def test_linear_strides_types_and_out(m):
    g = gen(m)
    n, k = 300, 520
    wide = activations(g, m, k + 24, BF16)
    w, s = weight(g, (), n, k)
    lin = Fp8Linear(w, s)
    for start in (0, 8, 3):  # rows aligned and not
        x = wide[:, start:start + k]
        want, bound = ref.product(ref.values(*ref.e4m3_form(x), 1), ref.values(w, s, 128))
        for od in (BF16, F16, F32):
            buf = torch.full((m, n + 13), 7.0, dtype=od, device=DEV)
            for off in (0, 5):
                out = buf[:, off:off + n]
                assert lin(x, out=out) is out
                close(out, want, ref.with_output(want, bound, od), f"start {start} {od} {off}")
                assert (buf[:, :off] == 7).all() and (buf[:, off + n:] == 7).all()
                buf.fill_(7.0)
            close(lin(x, out_dtype=od), want, ref.with_output(want, bound, od))
    row = wide[:1, :k]
    one = lin(row)
    assert torch.equal(lin(row.expand(m, k)), one.expand(m, n))           # a broadcast row
    assert torch.equal(lin(wide[:, :k].t().contiguous().t()), lin(wide[:, :k]))  # column-major x
    assert lin(wide[:, :k].reshape(1, m, k)).shape == (1, m, n)
    assert lin(wide[:0, :k]).shape == (0, n)
    view = Fp8Linear(torch.cat([w, w])[n:], s)  # a slice of a larger weight: not on 16 bytes for every n
    assert torch.equal(view(wide[:, :k]), lin(wide[:, :k]))


@pytest.mark.parametrize("m", [4, 150])
def test_linear_rows_are_independent_and_non_finite_rows_stay_apart(m):
    g = gen(11)
    n, k = 200, 384
    x = activations(g, m, k, BF16)
    w, s = weight(g, (), n, k)
    lin = Fp8Linear(w, s)
    clean = lin(x)
    x[1, 130] = float("nan")
    x[3, 5] = float("-inf")
    y = lin(x)
    assert y[1].isnan().all() and y[3].isnan().all()
    keep = [i for i in range(m) if i not in (1, 3)]
    assert torch.equal(y[keep], clean[keep])
    assert torch.equal(lin(x[:2])[0], clean[0]) or (lin(x[:2])[0].float() - clean[0].float()).abs().max() <= \
        2 * ref.HALF_ULP[BF16] * 2 * clean[0].float().abs().max()


def test_linear_ignores_what_pads_the_weight_rows():
    g = gen(12)
    n, k = 70, 100
    w, s = weight(g, (), n, k)
    wide = torch.full((n, 112), 0x7F, dtype=torch.uint8, device=DEV)  # NaN bytes past column k
    wide[:, :k] = w.view(torch.uint8)
    for m in (5, 140):
        x = activations(g, m, k, F16)
        assert torch.equal(Fp8Linear(wide.view(torch.float8_e4m3fn)[:, :k], s)(x), Fp8Linear(w, s)(x))


@pytest.mark.parametrize("m", [8, 256])
def test_linear_on_another_stream_and_in_a_graph(m):
    g = gen(13)
    x = activations(g, m, 512, BF16)
    w, s = weight(g, (), 384, 512)
    lin = Fp8Linear(w, s)
    want = lin(x)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        a = lin(x)
        out = torch.empty_like(a)
        lin(x, out=out)
    st.synchronize()
    assert torch.equal(a, want) and torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = lin(x)
    x2 = activations(g, m, 512, BF16)
    x.copy_(x2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, lin(x2))


def test_quantized_weight_constructors():
    g = gen(14)
    w = torch.randn(200, 300, generator=g, device=DEV, dtype=BF16)
    lin = Fp8Linear.quantize(w)
    q, s = ref.e4m3_form(w, 128)
    x = activations(g, 6, 300, F32)
    want, bound = ref.product(ref.values(*ref.e4m3_form(x), 1), ref.values(q, s, 128))
    close(lin(x), want, ref.with_output(want, bound, F32))
    ex = Fp8Experts.quantize(torch.randn(3, 2, 72, 300, generator=g, device=DEV),
                             torch.randn(3, 300, 72, generator=g, device=DEV))
    assert ex(x, torch.zeros(6, 2, dtype=torch.int64, device=DEV)).shape == (6, 2, 300)


# ---- experts ---------------------------------------------------------------------------------


def make_experts(g, e, h, i):
    w13, s13 = weight(g, (e, 2), i, h)
    w2, s2 = weight(g, (e,), h, i)
    return (w13, s13, w2, s2), Fp8Experts(w13, s13, w2, s2)


def check_experts(x, sel, comp, weights, out, dtype, skipped=0.0):
    w13, s13, w2, s2 = weights
    e = w13.shape[0]
    done = torch.zeros_like(sel, dtype=torch.bool)
    for ei in range(e):
        t, s = torch.nonzero((sel == ei) & comp, as_tuple=True)
        if t.numel() == 0:
            continue
        want, bound = ref.expert(x[t], ref.values(w13[ei, 0], s13[ei, 0], 128), ref.values(w13[ei, 1], s13[ei, 1], 128),
                                 ref.values(w2[ei], s2[ei], 128))
        close(out[t, s], want, ref.with_output(want, bound, dtype), f"expert {ei}")
        done[t, s] = True
    assert (out[~done] == skipped).all()


@pytest.mark.parametrize("q,s,e,h,i,keep,dtype", [
    (1, 1, 1, 16, 16, 1.0, BF16),
    (1, 8, 128, 256, 96, 0.6, BF16),
    (2, 3, 5, 100, 70, 1.0, F16),
    (16, 8, 16, 384, 128, 0.6, BF16),     # more than 8 slots of an expert: several leaders
    (64, 8, 4, 130, 200, 1.0, F32),       # 512 slots
    (65, 8, 4, 272, 136, 0.5, BF16),      # 520 slots: the planned path
    (300, 6, 7, 256, 384, 1.0, F16),
    (700, 2, 3, 520, 129, 0.7, BF16),     # several 128-row tiles per expert
    (129, 4, 64, 128, 256, 0.4, F32),
    (1000, 1, 2, 64, 40, 0.9, BF16),
])
def test_experts_match_64_bits(q, s, e, h, i, keep, dtype):
    g = gen(q + s + e + h + i)
    weights, ex = make_experts(g, e, h, i)
    x = activations(g, q, h, dtype)
    sel = torch.argsort(torch.rand(q, max(e, s), generator=g, device=DEV), dim=-1)[:, :s] % e
    comp = torch.rand(q, s, generator=g, device=DEV) < keep
    out = ex(x, sel, comp)
    assert out.dtype == dtype
    check_experts(x, sel, comp, weights, out, dtype)
    assert torch.equal(ex(x, sel, comp), out)  # the same on every run
    assert ex.device_errors() == 0


@pytest.mark.parametrize("q,s,e", [(1, 8, 8), (1, 8, 40), (2, 4, 3), (8, 1, 2), (4, 2, 1), (1, 1, 5), (3, 2, 4)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_experts_of_few_slots(q, s, e, dtype):
    g = gen(q + 10 * s + 100 * e)
    h, i = 328, 200
    weights, ex = make_experts(g, e, h, i)
    x = activations(g, q, h, dtype)
    sel = torch.randint(0, e, (q, s), generator=g, device=DEV)
    comp = torch.rand(q, s, generator=g, device=DEV) < 0.7
    out = ex(x, sel, comp)
    check_experts(x, sel, comp, weights, out, dtype)
    assert torch.equal(ex(x, sel)[comp], out[comp])  # whoever else shares the expert
    assert ex.device_errors() == 0


@pytest.mark.parametrize("m,n,k", [(128, 4096, 2688), (24, 4224, 4096), (16, 9000, 4480)])
def test_linear_of_few_rows_and_much_weight(m, n, k):
    g = gen(m)
    x = activations(g, m, k, BF16)
    w, s = weight(g, (), n, k)
    want, bound = ref.product(ref.values(*ref.e4m3_form(x), 1), ref.values(w, s, 128))
    close(Fp8Linear(w, s)(x), want, ref.with_output(want, bound, BF16), f"{m}x{n}x{k}")


@pytest.mark.parametrize("m,n,k", [(2600, 1100, 136), (1300, 1700, 264), (8200, 130, 1000), (1153, 1792, 640)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_linear_of_many_rows(m, n, k, dtype):
    g = gen(m + n)
    x = activations(g, m, k, dtype)
    w, s = weight(g, (), n, k)
    lin = Fp8Linear(w, s)
    y = lin(x)
    want, bound = ref.product(ref.values(*ref.e4m3_form(x), 1), ref.values(w, s, 128))
    close(y, want, ref.with_output(want, bound, dtype), f"{m}x{n}x{k}")
    buf = torch.full((m, n + 13), 7.0, dtype=dtype, device=DEV)
    for off in (0, 5):
        assert torch.equal(lin(x, out=buf[:, off:off + n]), y)
        assert (buf[:, :off] == 7).all() and (buf[:, off + n:] == 7).all()
        buf.fill_(7.0)
    x[m // 2, 3], x[m - 1, 0] = float("nan"), float("inf")
    z = lin(x)
    assert not z[[m // 2, m - 1]].isfinite().any()
    rest = torch.ones(m, dtype=torch.bool, device=DEV)
    rest[[m // 2, m - 1]] = False
    assert torch.equal(z[rest], y[rest]) and lin.device_errors() == 0


@pytest.mark.parametrize("h,i,dtype", [(256, 128, BF16), (200, 136, F16), (392, 260, F32)])
def test_experts_with_any_number_of_tokens(h, i, dtype):
    counts = [0, 1, 15, 16, 17, 33, 50, 64, 80, 96, 97, 112, 113, 127, 128, 129, 200, 257]
    q = sum(counts)
    g = gen(h)
    weights, ex = make_experts(g, len(counts), h, i)
    x = activations(g, q, h, dtype)
    sel = torch.repeat_interleave(torch.arange(len(counts), device=DEV), torch.tensor(counts, device=DEV))
    sel = sel[torch.randperm(q, generator=g, device=DEV)][:, None]
    comp = torch.ones(q, 1, dtype=torch.bool, device=DEV)
    out = ex(x, sel, comp)
    check_experts(x, sel, comp, weights, out, dtype)
    # a token's result does not depend on how many share its expert
    few = torch.arange(0, q, 2, device=DEV)
    assert torch.equal(out[few], ex(x[few], sel[few], comp[few]))
    assert ex.device_errors() == 0


@pytest.mark.parametrize("h,i,dtype", [(256, 128, F16), (200, 136, F32), (1160, 520, BF16)])
def test_experts_with_many_tokens_each(h, i, dtype):
    counts = [700, 97, 112, 113, 128, 241, 0, 131]
    q = sum(counts)
    g = gen(h + 1)
    weights, ex = make_experts(g, len(counts), h, i)
    x = activations(g, q, h, dtype)
    sel = torch.repeat_interleave(torch.arange(len(counts), device=DEV), torch.tensor(counts, device=DEV))
    sel = sel[torch.randperm(q, generator=g, device=DEV)][:, None]
    out = ex(x, sel)
    check_experts(x, sel, torch.ones(q, 1, dtype=torch.bool, device=DEV), weights, out, dtype)
    few = torch.arange(0, q, 4, device=DEV)  # other groups, the same results
    assert torch.equal(out[few], ex(x[few], sel[few]))
    assert ex.device_errors() == 0


@pytest.mark.parametrize("q", [12, 300])
def test_experts_uneven_routing_and_empty_masks(q):
    g = gen(q)
    s, e, h, i = 3, 6, 192, 160
    weights, ex = make_experts(g, e, h, i)
    x = activations(g, q, h, BF16)
    sel = torch.randint(0, 2, (q, s), generator=g, device=DEV) * 4  # experts 0 and 4 only, repeated within a token
    comp = torch.rand(q, s, generator=g, device=DEV) < 0.5
    comp[q // 3] = False  # a token without a slot
    check_experts(x, sel, comp, weights, ex(x, sel, comp), BF16)
    none = torch.zeros_like(comp)
    assert (ex(x, sel, none) == 0).all()
    full = ex(x, sel)
    assert torch.equal(full, ex(x, sel, torch.ones_like(comp)))
    assert ex(x[:0], sel[:0], comp[:0]).shape == (0, s, h)
    assert ex(x, sel[:, :0]).shape == (q, 0, h)


@pytest.mark.parametrize("q", [10, 260])
def test_experts_strides_and_given_rows(q):
    g = gen(q + 1)
    s, e, h, i = 4, 5, 150, 100
    weights, ex = make_experts(g, e, h, i)
    wide = activations(g, q, h + 9, F16)
    x = wide[:, 7:7 + h]
    selw = torch.randint(0, e, (q, s + 3), generator=g, device=DEV)
    sel = selw[:, 2:2 + s]
    comp = (torch.rand(q, s + 1, generator=g, device=DEV) < 0.6)[:, 1:]
    buf = torch.full((q, s + 1, h + 5), 3.0, dtype=BF16, device=DEV)
    out = buf[:, 1:, 2:2 + h]
    assert ex(x, sel, comp, out) is out
    check_experts(x, sel, comp, weights, out, BF16, skipped=3.0)
    assert (buf[:, 0] == 3).all() and (buf[:, :, :2] == 3).all() and (buf[:, :, 2 + h:] == 3).all()
    nan = x.clone()
    nan[1, 3] = float("nan")
    a, b = ex(nan, sel, comp), ex(x.contiguous(), sel, comp)
    assert a[1][comp[1]].isnan().all()
    rest = [t for t in range(q) if t != 1]
    assert torch.equal(a[rest], b[rest])


@pytest.mark.parametrize("q", [6, 300])
def test_experts_bad_ids_are_reported_and_skipped(q, monkeypatch):
    g = gen(q + 2)
    weights, ex = make_experts(g, 4, 128, 64)
    x = activations(g, q, 128, BF16)
    sel = torch.randint(0, 4, (q, 2), generator=g, device=DEV)
    comp = torch.ones(q, 2, dtype=torch.bool, device=DEV)
    want = ex(x, sel, comp)
    bad = sel.clone()
    bad[2, 1], bad[4, 0] = 4, -1
    out = ex(x, bad, comp)
    assert ex.device_errors() == 1 and ex.device_errors() == 0
    assert (out[2, 1] == 0).all() and (out[4, 0] == 0).all()
    ok = (bad == sel)
    assert torch.equal(out[ok], want[ok])
    masked = comp.clone()
    masked[2, 1] = masked[4, 0] = False
    ex(x, bad, masked)  # a slot that is not computed may name anything
    assert ex.device_errors() == 0
    cfg = CacheConfig.ALUT_CHECK_ERRORS
    CacheConfig.ALUT_CHECK_ERRORS = True
    try:
        with pytest.raises(IndexError):
            ex(x, bad, comp)
    finally:
        CacheConfig.ALUT_CHECK_ERRORS = cfg


def test_experts_in_a_graph_and_on_two_streams():
    g = gen(21)
    weights, ex = make_experts(g, 8, 256, 128)
    for q in (8, 200):
        x = activations(g, q, 256, BF16)
        sel = torch.argsort(torch.rand(q, 8, generator=g, device=DEV), dim=-1)[:, :4].contiguous()
        comp = torch.rand(q, 4, generator=g, device=DEV) < 0.6
        want = ex(x, sel, comp)
        torch.cuda.synchronize()
        a, b = torch.cuda.Stream(), torch.cuda.Stream()
        outs = []
        for st in (a, b):
            with torch.cuda.stream(st):
                outs.append([ex(x, sel, comp) for _ in range(3)])
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for os in outs for o in os)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ex(x, sel, comp)
        x2, sel2 = activations(g, q, 256, BF16), sel.flip(1).contiguous()
        x.copy_(x2)
        sel.copy_(sel2)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ex(x2, sel2, comp))
