"""Waits that run out inside the 8-bit products' tensor-core kernels: the call returns with
ALUT_ERR_MMA_TIMEOUT, and the next call is as if nothing had been."""
import contextlib

import pytest
import torch

from table_moe.cache_engine import CacheConfig, _alut
from table_moe.ops import Fp8Experts, Fp8Linear

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


@contextlib.contextmanager
def wait_limit(ns):
    _alut.load().alut_set_wait_limit(ns)
    try:
        yield
    finally:
        _alut.load().alut_set_wait_limit(10 ** 9)


def linear_call(m, n, k):
    g = torch.Generator(device=DEV).manual_seed(m)
    lin = Fp8Linear.quantize(torch.randn(n, k, generator=g, device=DEV))
    x = torch.randn(m, k, generator=g, device=DEV, dtype=torch.bfloat16)
    return lin, lambda: lin(x)


def experts_call(q, s, e, h, i):
    g = torch.Generator(device=DEV).manual_seed(q)
    ex = Fp8Experts.quantize(torch.randn(e, 2, i, h, generator=g, device=DEV), torch.randn(e, h, i, generator=g, device=DEV))
    x = torch.randn(q, h, generator=g, device=DEV, dtype=torch.bfloat16)
    sel = torch.randint(0, e, (q, s), generator=g, device=DEV)
    return ex, lambda: ex(x, sel)


CALLS = {
    "one tile each": (linear_call, 70, 2000, 3200),     # tokens in groups, at most one tile per SM
    "groups": (linear_call, 300, 1000, 1000),
    "experts": (experts_call, 40, 2, 4, 256, 384),
    "experts, many tiles": (experts_call, 2000, 4, 8, 1024, 640),
    "pairs": (linear_call, 2600, 1100, 136),             # pairs of CTAs, a ragged last one
    "pairs, many tiles": (linear_call, 6000, 4000, 1536),
}


@pytest.mark.parametrize("name", CALLS)
def test_a_call_that_gives_up_ends_and_says_so(name):
    make, *sizes = CALLS[name]
    obj, call = make(*sizes)
    want = call()
    assert obj.device_errors() == 0
    with wait_limit(0):
        call()
        assert obj.device_errors() == _alut.ERR_MMA_TIMEOUT
    assert torch.equal(call(), want) and obj.device_errors() == 0


@pytest.mark.parametrize("name", CALLS)
def test_a_call_that_gives_up_on_its_way_ends(name):
    """A limit of 1 ns: any wait of more than a few hundred tries runs out, wherever the call is. Whether
    one does is up to the timing; the call ends, and a call without the error bit is right."""
    make, *sizes = CALLS[name]
    obj, call = make(*sizes)
    want = call()
    for _ in range(5):
        with wait_limit(1):
            out = call()
            bits = obj.device_errors()
        assert bits in (0, _alut.ERR_MMA_TIMEOUT)
        assert bits or torch.equal(out, want)
    assert torch.equal(call(), want) and obj.device_errors() == 0


def test_the_error_is_raised_where_errors_are_checked():
    lin, call = linear_call(200, 384, 512)
    want = call()
    checked = CacheConfig.ALUT_CHECK_ERRORS
    CacheConfig.ALUT_CHECK_ERRORS = True
    try:
        with wait_limit(0), pytest.raises(RuntimeError, match="timed out"):
            call()
    finally:
        CacheConfig.ALUT_CHECK_ERRORS = checked
    assert torch.equal(call(), want)
