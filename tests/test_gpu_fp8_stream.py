"""The weight-streaming product where its CTAs take several steps, a ragged last one among them, and
split K over fewer than all warps (launch_stream in alut_fp8_api.cu); and few rows past the K that it
takes. Bounds as in tests/fp8_reference.py."""
import pytest
import torch

import fp8_reference as ref
from table_moe.ops import Fp8Experts, Fp8Linear, quantize_fp8
from test_gpu_fp8 import BF16, DEV, F16, F32, activations, check_experts, close, gen

pytestmark = pytest.mark.gpu


def weight(g, lead, n, k):
    w = torch.randn(*lead, n, k, generator=g, device=DEV)
    w *= torch.exp(torch.randn(*lead, n, 1, generator=g, device=DEV)) / k ** 0.5
    return quantize_fp8(w, 128)


SIZES = [              # steps of a CTA x warps that split K
    (40001, 2048),     # 1 x 4
    (12010, 3190),     # 1 x 8, enough CTAs for two per SM
    (160001, 1000),    # 2 x 2
    (230003, 1000),    # 3 x 2
    (113701, 2048),    # 3 x 4
    (57001, 3190),     # 3 x 8
    (455003, 200),     # 3 x 1
    (303200, 256),     # 2 x 1
    (59000, 8192),     # 3 x 8, the longest K
]


@pytest.mark.parametrize("n,k", SIZES)
def test_linear_of_one_pass_over_many_weight_rows(n, k):
    g = gen(n)
    w, s = weight(g, (), n, k)
    lin = Fp8Linear(w, s)
    for m, dtype in ((1, BF16), (5, F16), (8, F32)):
        x = activations(g, m, k, dtype)
        y = lin(x)
        xv = ref.values(*ref.e4m3_form(x), 1)
        for r in range(0, n, 65536):  # (the 64-bit weight in parts: they start on a block's first row)
            want, bound = ref.product(xv, ref.values(w[r:r + 65536], s[r // 128:(r + 65536) // 128], 128))
            close(y[:, r:r + 65536], want, ref.with_output(want, bound, dtype), f"{m}x{n}x{k} from {r}")
        assert torch.equal(lin(x[m - 1:])[0], y[m - 1])  # a row's result does not depend on the others
    assert lin.device_errors() == 0


@pytest.mark.parametrize("m,n,k", [(40, 4000, 200), (128, 2500, 130), (100, 1500, 256)])
def test_linear_of_several_passes_over_many_ctas(m, n, k):
    g = gen(m + n)
    w, s = weight(g, (), n, k)
    x = activations(g, m, k, BF16)
    want, bound = ref.product(ref.values(*ref.e4m3_form(x), 1), ref.values(w, s, 128))
    close(Fp8Linear(w, s)(x), want, ref.with_output(want, bound, BF16), f"{m}x{n}x{k}")


@pytest.mark.parametrize("e,h,i,dtype", [
    (2, 8100, 3190, BF16),   # GateUp two steps, Down three
    (3, 3200, 8000, F16),    # GateUp three steps, Down one
    (2, 500, 8190, F32),     # few k-blocks: K over one warp and two
])
@pytest.mark.parametrize("q,s", [(8, 1), (1, 8), (2, 3)])
def test_experts_of_few_slots_and_wide_layers(e, h, i, dtype, q, s):
    g = gen(h + q)
    w13, s13 = weight(g, (e, 2), i, h)
    w2, s2 = weight(g, (e,), h, i)
    ex = Fp8Experts(w13, s13, w2, s2)
    x = activations(g, q, h, dtype)
    sel = torch.randint(0, e, (q, s), generator=g, device=DEV)
    comp = torch.rand(q, s, generator=g, device=DEV) < 0.8
    comp[0, 0] = True
    out = ex(x, sel, comp)
    check_experts(x, sel, comp, (w13, s13, w2, s2), out, dtype)
    assert torch.equal(ex(x, sel, comp), out) and ex.device_errors() == 0


@pytest.mark.parametrize("m", [1, 5, 8, 20])
@pytest.mark.parametrize("n,k", [(300, 8300), (2048, 12288), (129, 20001)])
def test_linear_of_few_rows_and_a_long_k(m, n, k):
    g = gen(n + k)
    w, s = weight(g, (), n, k)
    x = activations(g, m, k, BF16)
    want, bound = ref.product(ref.values(*ref.e4m3_form(x), 1), ref.values(w, s, 128))
    close(Fp8Linear(w, s)(x), want, ref.with_output(want, bound, BF16), f"{m}x{n}x{k}")
