"""Calls on tensors of a GPU that is not the current one run with theirs current. One GPU is enough to
see it: the current one is made to look like another until ``torch.cuda.device`` is entered."""
import pytest
import torch

from table_moe.cache_engine import HybridStorageManager, VectorSearchEngine, _alut
from table_moe.cache_engine.manager import normalize_rows
from table_moe.ops import Fp8Experts, Fp8Linear, quantize_fp8, route_experts, route_for_lookup
from table_moe.skip import build_prefill_keep_mask

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _calls():
    g = torch.Generator(device=DEV).manual_seed(1)
    x = torch.randn(12, 64, generator=g, device=DEV)
    lin = Fp8Linear.quantize(torch.randn(48, 64, generator=g, device=DEV))
    ex = Fp8Experts.quantize(torch.randn(4, 2, 32, 64, generator=g, device=DEV), torch.randn(4, 64, 32, generator=g, device=DEV))
    sel = torch.randint(0, 4, (12, 2), generator=g, device=DEV)
    w = torch.rand(12, 2, generator=g, device=DEV)
    keys = torch.randn(4, 2, 16, 8, generator=g, device=DEV)
    values = torch.randn(4, 2, 16, 64, generator=g, device=DEV).to(torch.bfloat16)
    pca = {m: {"proj": torch.randn(64, 8, generator=g, device=DEV), "bias": torch.zeros(8, device=DEV)} for m in ("vision", "text")}
    mgr = HybridStorageManager.from_tables(0, keys, values, pca)
    eng = VectorSearchEngine(mgr)
    vis, every = torch.zeros(12, dtype=torch.bool, device=DEV), torch.ones(12, 2, dtype=torch.bool, device=DEV)
    return {
        "route_experts": lambda: route_experts(x, 4),
        "route_experts importance": lambda: route_experts(x, 4, keep="importance"),
        "route_for_lookup": lambda: route_for_lookup(x, 4, keep="importance"),
        "build_prefill_keep_mask": lambda: build_prefill_keep_mask(sel, w, None, 4, 0.5),
        "quantize_fp8": lambda: quantize_fp8(x)[1],
        "Fp8Linear": lambda: lin(x),
        "Fp8Experts": lambda: ex(x, sel),
        "normalize_rows": lambda: normalize_rows(x, 1e-6),
        "search": lambda: eng.search_prefill_offline_dot(0, x, sel, vis, every),
        "lookup_combine": lambda: eng.lookup_combine(x, sel, vis, every, w),
        "gather_values": lambda: mgr.gather_values(sel[:, 0], vis.long(), sel[:, 1]),
        "device_errors": lambda: torch.tensor([ex.device_errors(), eng.device_errors()]),
    }


def _same(a, b):
    return all(map(_same, a, b)) if isinstance(a, tuple) else torch.equal(a, b)


def test_every_call_makes_its_tensors_gpu_current(monkeypatch):
    calls = _calls()
    want = {name: call() for name, call in calls.items()}
    current, entered = [0], []

    class Device:
        def __init__(self, device):
            self.index = torch.device(device).index if not isinstance(device, int) else device

        def __enter__(self):
            self.before, current[0] = current[0], self.index
            entered.append(self.index)

        def __exit__(self, *exc):
            current[0] = self.before

    lib = _alut.load()

    class Library:  # every launch finds its tensors' GPU current
        def __getattr__(self, name):
            fn = getattr(lib, name)

            def call(*args):
                if "_size" not in name and "_bytes" not in name and name not in ("alut_scan_kind", "alut_last_error"):
                    assert current[0] == 0, name
                    launched.append(name)
                return fn(*args)
            return call

    launched = []
    monkeypatch.setattr(_alut, "_lib", Library())
    calls = _calls()  # (its objects hold the library)
    monkeypatch.setattr(_alut, "_current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    for name, call in calls.items():
        current[0] = 7
        entered.clear()
        launched.clear()
        got = call()
        assert current[0] == 7 and entered and set(entered) == {0}, name
        assert launched or name == "device_errors", name
        assert _same(got, want[name]), name
        current[0] = 0  # and where theirs is current nothing is switched
        entered.clear()
        call()
        assert not entered, name
