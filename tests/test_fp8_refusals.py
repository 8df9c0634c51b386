"""What the expert routing and the 8-bit products refuse, on the host: no GPU call is made."""
import pytest
import torch

from table_moe.cache_engine import _alut
from table_moe.ops import Fp8Experts, Fp8Linear, quantize_fp8, route_experts

E4M3 = torch.float8_e4m3fn
PTR = 4096  # a 16-byte aligned address that nothing reads


def code(rc, text):
    assert text in _alut.load().alut_last_error().decode(), _alut.load().alut_last_error()
    return rc


def test_cpu_tensors_are_refused():
    with pytest.raises(ValueError):
        route_experts(torch.zeros(2, 8), 2)
    with pytest.raises(ValueError):
        quantize_fp8(torch.zeros(2, 8))
    with pytest.raises(ValueError):
        Fp8Linear(torch.zeros(4, 16, dtype=E4M3), torch.ones(1, 1))
    with pytest.raises(ValueError):
        Fp8Experts(torch.zeros(2, 2, 8, 16, dtype=E4M3), torch.ones(2, 2, 1, 1), torch.zeros(2, 16, 8, dtype=E4M3),
                   torch.ones(2, 1, 1))


def test_weights_of_other_types_and_shapes_are_refused():
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        Fp8Linear(torch.zeros(4, 16), torch.ones(1, 1))
    with pytest.raises(ValueError):
        quantize_fp8(torch.zeros(8), 1)


def quantize(batch=1, rows=2, cols=64, block_rows=1, src=PTR, dtype=1, ss=64, out=PTR, os=64, scale=PTR):
    return _alut.load().alut_quantize_fp8(batch, rows, cols, block_rows, src, dtype, 128, ss, out, 128, os, scale, None)


def test_quantize_arguments():
    assert code(quantize(block_rows=64), "block_rows") == _alut.ALUT_EINVAL
    assert code(quantize(rows=-1), "negative") == _alut.ALUT_EINVAL
    assert code(quantize(src=None), "NULL") == _alut.ALUT_EINVAL
    assert code(quantize(dtype=9), "dtype") == _alut.ALUT_EDTYPE
    assert code(quantize(ss=63), "strides") == _alut.ALUT_ESHAPE
    assert quantize(rows=0, src=None) == _alut.ALUT_OK


def linear(m=2, n=32, k=40, x=PTR, xd=1, xs=40, w=PTR, wstride=48, ws=PTR, out=PTR, od=1, os=32, work=PTR, nbytes=1 << 30):
    return _alut.load().alut_linear_fp8(m, n, k, x, xd, xs, w, wstride, ws, out, od, os, None, work, nbytes, None)


def test_linear_arguments():
    assert code(linear(k=0), "k=0") == _alut.ALUT_EINVAL
    assert code(linear(m=-1), "m=-1") == _alut.ALUT_EINVAL
    assert code(linear(x=None), "NULL") == _alut.ALUT_EINVAL
    assert code(linear(ws=None), "NULL weight") == _alut.ALUT_EINVAL
    assert code(linear(xd=3), "dtype") == _alut.ALUT_EDTYPE
    assert code(linear(xs=39), "strides") == _alut.ALUT_ESHAPE
    assert code(linear(os=31), "strides") == _alut.ALUT_ESHAPE
    assert code(linear(w=PTR + 8), "16-byte") == _alut.ALUT_ESHAPE
    assert code(linear(wstride=40), "16-byte") == _alut.ALUT_ESHAPE
    assert code(linear(wstride=32), "< 48") == _alut.ALUT_ESHAPE
    assert code(linear(m=300, nbytes=16), "workspace") == _alut.ALUT_EWORKSPACE
    assert code(linear(m=300, work=None), "workspace") == _alut.ALUT_EWORKSPACE
    assert linear(m=0, x=None) == _alut.ALUT_OK
    assert _alut.load().alut_linear_fp8_workspace_size(4, 0, 8) == 0


def weights(**kw):
    w = _alut.Fp8ExpertWeights()
    w.num_experts, w.h, w.i = 4, 64, 32
    w.gate_up = w.gate_up_scale = w.down = w.down_scale = PTR
    w.gate_up_stride[:] = [2 * 32 * 64, 32 * 64, 64]
    w.down_stride[:] = [64 * 32, 32]
    for k, v in kw.items():
        setattr(w, k, v)
    return w


def experts(w, q=2, s=2, x=PTR, xd=1, xs=64, sel=PTR, ss=2, cs=2, out=PTR, od=1, ot=128, os=64, work=PTR,
            nbytes=1 << 30):
    return _alut.load().alut_experts_fp8(w, q, s, x, xd, xs, sel, ss, PTR, cs, 1, out, od, ot, os, None, work, nbytes, None)


def test_experts_arguments():
    w = weights()
    lib = _alut.load()
    assert lib.alut_experts_fp8(None, 1, 1, PTR, 1, 64, PTR, 1, None, 1, 1, PTR, 1, 64, 64, None, PTR, 1 << 30,
                                None) == _alut.ALUT_EINVAL
    assert code(experts(weights(i=0)), "positive") == _alut.ALUT_EINVAL
    assert code(experts(weights(num_experts=5000)), "exceeds") == _alut.ALUT_ERANGE
    assert code(experts(weights(down=None)), "down") == _alut.ALUT_EINVAL
    assert code(experts(weights(gate_up=PTR + 1)), "gate_up") == _alut.ALUT_ESHAPE
    odd = weights()
    odd.gate_up_stride[1] = 32 * 64 + 8
    assert code(experts(odd), "multiples of 16") == _alut.ALUT_ESHAPE
    assert code(experts(w, s=65, ss=65, cs=65), "exceeds") == _alut.ALUT_ERANGE
    assert code(experts(w, q=1 << 30), "too large") == _alut.ALUT_ERANGE
    assert code(experts(w, sel=None), "NULL") == _alut.ALUT_EINVAL
    assert code(experts(w, od=7), "dtype") == _alut.ALUT_EDTYPE
    for bad in (dict(xs=63), dict(ss=1), dict(cs=1), dict(ot=63), dict(os=63)):
        assert code(experts(w, **bad), "strides") == _alut.ALUT_ESHAPE
    assert code(experts(w, nbytes=64), "workspace") == _alut.ALUT_EWORKSPACE
    assert experts(w, q=0, x=None) == _alut.ALUT_OK and experts(w, s=0, x=None) == _alut.ALUT_OK
    assert lib.alut_experts_fp8_workspace_size(w, -1, 2) == 0
    assert 0 < lib.alut_experts_fp8_workspace_size(w, 2, 2) <= lib.alut_experts_fp8_workspace_size(w, 5000, 8)


def router(**kw):
    r = _alut.Router()
    r.num_experts, r.top_k, r.n_group, r.topk_group, r.scale = 16, 4, 1, 1, 1.0
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def route(r, q=3, x=PTR, xd=0, xs=16, mode=0, rate=0.5, w=PTR, os=4, work=None, nbytes=0):
    return _alut.load().alut_route_experts(r, q, x, xd, xs, mode, -1, rate, None, w, PTR, PTR, PTR, os, work, nbytes, None)


def test_route_arguments():
    for kw in (dict(num_experts=0), dict(top_k=0), dict(n_group=0), dict(topk_group=0), dict(scoring=2),
               dict(group_rule=2)):
        assert route(router(**kw)) == _alut.ALUT_EINVAL, kw
    for kw in (dict(top_k=17), dict(num_experts=5000), dict(n_group=3), dict(n_group=4, topk_group=5),
               dict(n_group=8, topk_group=1), dict(num_experts=64, n_group=64, topk_group=64)):
        assert route(router(**kw)) == _alut.ALUT_ERANGE, kw
    assert route(router(), x=None) == _alut.ALUT_EINVAL
    assert route(router(), xd=5) == _alut.ALUT_EDTYPE
    assert route(router(), xs=15) == _alut.ALUT_ESHAPE and route(router(), os=3) == _alut.ALUT_ESHAPE
    assert route(router(), mode=2) == _alut.ALUT_EINVAL
    assert route(router(), mode=1) == _alut.ALUT_EWORKSPACE
    assert route(router(), mode=1, work=PTR, nbytes=1 << 20, rate=-1.0) == _alut.ALUT_EINVAL
    assert route(router(), q=0, x=None) == _alut.ALUT_OK
