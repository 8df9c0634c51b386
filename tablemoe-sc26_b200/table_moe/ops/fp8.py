"""Products in 8-bit floating point (e4m3) with a scale for each block of 128, on the
``alut_quantize_fp8``, ``alut_linear_fp8`` and ``alut_experts_fp8`` kernels of ``libalut.so``.

New: the reference computes the experts that are not looked up in a Python loop over the
routed experts (``qwen3_vl_moe/cached_layers.py:431-437``). ``Fp8Experts`` is that loop as one
call, with the signature of ``ALUTCachedMoE``'s ``run_experts``; ``Fp8Linear`` is the plain
product (shared experts, projections). Weights hold one fp32 scale per 128 x 128 block;
activations are taken in their 8-bit form inside the call, one scale per row and 128 columns.
Inference only; there is no torch fallback: CUDA tensors are required.
"""
from __future__ import annotations

import torch

from ..cache_engine import _alut
from ..cache_engine.config import CacheConfig

BLOCK = 128
_E4M3 = torch.float8_e4m3fn


def _blocks(n):
    return -(-n // BLOCK)


@_alut.on_device_of_first
def quantize_fp8(x, block_rows=1):
    """(e4m3 [..., rows, cols], fp32 scales [..., ceil(rows / block_rows), ceil(cols / 128)]) of x
    (f32, bf16 or f16; at least 2D): block_rows 1 for activations, 128 for weights."""
    if x.device.type != "cuda":
        raise ValueError("quantize_fp8: CUDA tensors only")
    if x.dim() < 2:
        raise ValueError(f"quantize_fp8 expects at least 2 dimensions, got {tuple(x.shape)}")
    if block_rows not in (1, BLOCK):
        raise ValueError(f"block_rows must be 1 or {BLOCK}, got {block_rows}")
    lead, (rows, cols) = x.shape[:-2], x.shape[-2:]
    code = _alut.dtype_code(x.dtype)
    v = x if x.dim() == 2 and x.stride(-1) == 1 and x.stride(0) >= cols else x.contiguous()
    q = torch.empty(x.shape, dtype=_E4M3, device=x.device)
    s = torch.empty(*lead, -(-rows // block_rows), _blocks(cols), dtype=torch.float32, device=x.device)
    batch = lead.numel()
    stride = v.stride(0) if v.dim() == 2 else cols
    rc = _alut.load().alut_quantize_fp8(batch, rows, cols, block_rows, v.data_ptr(), code, rows * cols, max(stride, cols),
                                        q.data_ptr(), rows * cols, cols, s.data_ptr(), _alut.stream_ptr(x.device))
    _alut.check(rc, "alut_quantize_fp8")
    return q, s


def _padded(w):
    """w (e4m3 [..., n, k]) with rows that start on 16 bytes: itself where it is so already."""
    k = w.shape[-1]
    ok = w.stride(-1) == 1 and w.stride(-2) >= -(-k // 16) * 16 and all(s % 16 == 0 for s in w.stride()[:-1])
    if ok and w.data_ptr() % 16 == 0:
        return w
    out = torch.zeros(*w.shape[:-1], -(-k // 16) * 16, dtype=torch.uint8, device=w.device)
    out[..., :k] = w.view(torch.uint8)
    return out.view(_E4M3)[..., :k]


def _check_weight(w, scale, name, dims):
    if w.dtype != _E4M3:
        raise ValueError(f"{name} must be torch.float8_e4m3fn, got {w.dtype}")
    if w.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor (the 8-bit products have no CPU path)")
    if w.dim() != dims or 0 in w.shape:
        raise ValueError(f"{name} must be a non-empty {dims}D tensor, got {tuple(w.shape)}")
    want = (*w.shape[:-2], _blocks(w.shape[-2]), _blocks(w.shape[-1]))
    if tuple(scale.shape) != want or scale.dtype != torch.float32 or scale.device != w.device:
        raise ValueError(f"{name}'s scales must be fp32 {want} on {w.device}, got {scale.dtype} {tuple(scale.shape)}")


class _Fp8Module:
    def _init_device(self, device):
        self.device = device
        self._lib = _alut.load()
        self._errors = torch.zeros(1, dtype=torch.int32, device=device)
        self._err = self._errors.data_ptr()

    def _check_x(self, x, width):
        """x as rows (2D, unit innermost stride), its row stride and dtype code."""
        if x.device != self.device:
            raise ValueError(f"x is on {x.device}, the weights on {self.device}")
        if x.dim() < 1 or x.shape[-1] != width:
            raise ValueError(f"x must have {width} columns, got {tuple(x.shape)}")
        if x.dim() != 2:
            x = x.reshape(-1, width)
        stride, inner = x.stride()
        if inner != 1 or stride < width:  # also a broadcast row
            x = x.contiguous()
            stride = width
        return x, stride, _alut.dtype_code(x.dtype)

    def device_errors(self, clear=True):
        """Error bits (ALUT_ERR_*) that this object's calls have set; waits for the current stream."""
        bits = int(self._errors.item())
        if clear and bits:
            self._errors.zero_()
        return bits

    def _raise_errors(self, what):
        _alut.raise_device_errors(self.device_errors(), what)


class Fp8Linear(_Fp8Module):
    """y = x W^T with W e4m3 [N, K] and its fp32 block scales [ceil(N/128), ceil(K/128)].

    The weights are kept as given when K % 16 == 0 and they are contiguous; otherwise one
    padded copy is made here."""

    def __init__(self, weight, scale):
        _check_weight(weight, scale, "weight", 2)
        self._init_device(weight.device)
        self.n, self.k = weight.shape
        self.weight, self.scale = _padded(weight), scale.contiguous()
        self._w, self._w_stride, self._s = self.weight.data_ptr(), self.weight.stride(0), self.scale.data_ptr()

    @classmethod
    def quantize(cls, weight):
        """From a weight [N, K] in f32, bf16 or f16."""
        return cls(*quantize_fp8(weight, BLOCK))

    @_alut.on_own_device
    def __call__(self, x, out=None, *, out_dtype=None):
        """x [..., K] (f32, bf16 or f16) -> [..., N] in ``out_dtype`` (default x's), or into ``out``
        (a 2D tensor [rows, N] with unit innermost stride)."""
        v, xs, xd = self._check_x(x, self.k)
        m, n, k = v.shape[0], self.n, self.k
        if out is None:
            # (empty_strided takes 0.9 us less than empty)
            y = torch.empty_strided((m, n), (n, 1), dtype=out_dtype or x.dtype, device=self.device)
            if x.dim() != 2:
                y = y.view(*x.shape[:-1], n)
            stride = n
        else:
            if out.shape != (m, n) or out.device != x.device or (n > 1 and out.stride(-1) != 1):
                raise ValueError(f"out must be a [{m}, {n}] tensor on {x.device} with unit innermost stride")
            if out_dtype is not None and out_dtype != out.dtype:
                raise ValueError(f"out is {out.dtype}, out_dtype {out_dtype}")
            y, stride = out, out.stride(0) if m > 1 else max(out.stride(0), n)
        lib = self._lib
        nbytes = lib.alut_linear_fp8_workspace_size(m, n, k)
        ws = torch.empty_strided((nbytes,), (1,), dtype=torch.uint8, device=self.device) if nbytes else None
        rc = lib.alut_linear_fp8(m, n, k, v.data_ptr(), xd, xs, self._w, self._w_stride, self._s, y.data_ptr(),
                                 _alut.dtype_code(y.dtype), stride, self._err, _alut.ptr(ws), nbytes,
                                 _alut.stream_ptr(self.device))
        if rc:
            _alut.check(rc, "alut_linear_fp8")
        if CacheConfig.ALUT_CHECK_ERRORS:
            self._raise_errors("alut_linear_fp8")
        return y


class Fp8Experts(_Fp8Module):
    """The routed experts of a layer, down(silu(gate x) * (up x)).

    ``gate_up`` e4m3 [E, 2, I, H] (gate rows, then up rows) with scales [E, 2, ceil(I/128),
    ceil(H/128)]; ``down`` e4m3 [E, H, I] with scales [E, ceil(H/128), ceil(I/128)]. Kept as given
    when H and I are multiples of 16 and they are contiguous; otherwise one padded copy."""

    def __init__(self, gate_up, gate_up_scale, down, down_scale):
        _check_weight(gate_up, gate_up_scale, "gate_up", 4)
        _check_weight(down, down_scale, "down", 3)
        e, two, i, h = gate_up.shape
        if two != 2 or tuple(down.shape) != (e, h, i) or down.device != gate_up.device:
            raise ValueError(f"gate_up [E, 2, I, H] and down [E, H, I] do not fit: {tuple(gate_up.shape)}, "
                             f"{tuple(down.shape)}")
        self._init_device(gate_up.device)
        self.num_experts, self.inner, self.hidden = e, i, h
        self.gate_up, self.down = _padded(gate_up), _padded(down)
        self.gate_up_scale, self.down_scale = gate_up_scale.contiguous(), down_scale.contiguous()
        w = _alut.Fp8ExpertWeights()
        w.num_experts, w.h, w.i = e, h, i
        w.gate_up, w.gate_up_scale = self.gate_up.data_ptr(), self.gate_up_scale.data_ptr()
        w.gate_up_stride[:] = list(self.gate_up.stride()[:3])
        w.down, w.down_scale = self.down.data_ptr(), self.down_scale.data_ptr()
        w.down_stride[:] = list(self.down.stride()[:2])
        self._weights = w

    @classmethod
    def quantize(cls, gate_up, down):
        """From weights [E, 2, I, H] and [E, H, I] in f32, bf16 or f16."""
        return cls(*quantize_fp8(gate_up, BLOCK), *quantize_fp8(down, BLOCK))

    @_alut.on_own_device
    def __call__(self, x, selected_experts, compute_mask=None, collected=None):
        """Outputs [Q, S, H] of the experts ``selected_experts`` [Q, S] on the tokens x [Q, H], for
        the slots of ``compute_mask`` [Q, S] (None: all). Without ``collected`` a new tensor of x's
        dtype, 0 at the other slots; otherwise written into it (f32, bf16 or f16, unit innermost
        stride), its other rows untouched: the form of ``ALUTCachedMoE``'s ``run_experts``."""
        v, xs, xd = self._check_x(x, self.hidden)
        dev, h, sel = self.device, self.hidden, selected_experts
        if sel.dim() != 2 or sel.shape[0] != v.shape[0]:
            raise ValueError(f"selected_experts must be [{v.shape[0]}, S], got {tuple(sel.shape)}")
        if sel.dtype != torch.int64 or sel.device != dev:
            raise ValueError("selected_experts must be int64 on x's device")
        q, s = sel.shape
        sel_stride, inner = sel.stride()
        if inner != 1 or sel_stride < s:
            sel, sel_stride = sel.contiguous(), s
        comp, comp_stride = compute_mask, s
        if comp is not None:
            if comp.shape != (q, s) or comp.dtype not in (torch.bool, torch.uint8) or comp.device != dev:
                raise ValueError(f"compute_mask must be bool [{q}, {s}] on x's device")
            comp_stride, inner = comp.stride()
            if inner != 1 or comp_stride < s:
                comp, comp_stride = comp.contiguous(), s
        out = collected
        if out is None:
            out = torch.empty_strided((q, s, h), (s * h, h, 1), dtype=x.dtype, device=dev)
        elif out.shape != (q, s, h) or out.device != dev or (h > 1 and out.stride(-1) != 1):
            raise ValueError(f"collected must be [{q}, {s}, {h}] on {dev} with unit innermost stride")
        out_t, out_s, _ = out.stride()
        if q == 1:  # (the stride of one token, or slot, means nothing)
            out_t = max(out_t, h)
        if s == 1:
            out_s = max(out_s, h)
        lib = self._lib
        nbytes = lib.alut_experts_fp8_workspace_size(self._weights, q, s)
        ws = torch.empty_strided((nbytes,), (1,), dtype=torch.uint8, device=dev)
        rc = lib.alut_experts_fp8(self._weights, q, s, v.data_ptr(), xd, xs, sel.data_ptr(), sel_stride, _alut.ptr(comp),
                                  comp_stride, 1 if collected is None else 0, out.data_ptr(),
                                  _alut.dtype_code(out.dtype), out_t, out_s, self._err, ws.data_ptr(), nbytes,
                                  _alut.stream_ptr(dev))
        if rc:
            _alut.check(rc, "alut_experts_fp8")
        if CacheConfig.ALUT_CHECK_ERRORS:
            self._raise_errors("alut_experts_fp8")
        return out
