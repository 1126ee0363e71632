"""8-bit serving operators: rows to codes and back, RMS norm with 8-bit output, int8 product, int8 policy network.

A quantised row holds codes ``q`` in ``[-127, 127]`` and one fp32 scale ``s = max |row| / 127``; it stands for ``q * s``.
Activations are quantised per row (token, state), weights per output channel (the rows of ``weight[out, in]``)::

    wq, ws = quantize_rows(layer.weight)                              # once
    q, s, h = add_rms_norm_int8(x, norm_weight, residual)             # per call
    y = linear_int8(q, s, wq, ws, layer.bias, "relu", torch.bfloat16)

On a ROCm tensor the functions launch the kernels of ``csrc/int8.hip`` on the current stream of the tensors' device; on a
CPU tensor they evaluate ``ops/ref.py``.  They serve: no gradient flows through codes, and what they make requires none
(``add_rms_norm_int8`` without a residual hands back ``x`` itself as ``h``, which requires what ``x`` requires).

Code matrices are handed out with rows padded to 16 bytes (a view of ``[..., K]`` codes whose row stride is the next
multiple of 16), which is what the product reads directly; codes laid out differently are copied once per call.

A row with a NaN or an infinity gets scale NaN and codes 0, so everything computed from it is NaN; a row of zeros gets
scale 0 and codes 0.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence, Tuple

import torch

from . import hip as H
from . import ref

_FLOATS = {torch.float32: H.F_FP32, torch.bfloat16: H.F_BF16, torch.float16: H.F_FP16}
_ACTS = {"none": H.ACT_NONE, "relu": H.ACT_RELU, "tanh": H.ACT_TANH}
#: products of two codes are at most 128^2 in magnitude: sums of this many fit 32 bits
MAX_K = 131071
_F32, _I8 = torch.float32, torch.int8
_MOST = 2 ** 31 - 1


#: the plain case of every operator in C++ (``csrc/int8_bind.cpp``; loaded with the first GPU tensor).  What it returns
#: None for - other layouts, types and devices, mistakes - takes the way through the functions below.
_plain = None


def _binding():
    global _plain
    if _plain is None:
        _plain = H.int8_binding()
    return _plain


def _float_code(t: torch.Tensor, what: str) -> int:
    code = _FLOATS.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, not {t.dtype}")
    return code


def _out_code(dtype: torch.dtype) -> int:
    code = _FLOATS.get(dtype)
    if code is None:
        raise TypeError(f"dtype must be torch.float32, torch.bfloat16 or torch.float16, not {dtype}")
    return code


def _act_code(activation: str) -> int:
    code = _ACTS.get(activation)
    if code is None:
        raise ValueError(f"activation must be one of {sorted(_ACTS)}, not {activation!r}")
    return code


def _on(device: torch.device, what: str, t: torch.Tensor) -> None:
    if t.device != device:
        raise ValueError(f"{what} is on {t.device}, not on {device}")


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """``x[..., K]`` as ``[M, K]`` with neighbouring elements side by side, in memory as they read (a view whose sign is
    pending, such as ``z.conj().imag``, is copied)."""
    x = x.resolve_neg()
    if x.ndim != 2:
        if x.ndim < 1 or x.shape[-1] < 1:
            raise ValueError(f"{what} needs at least one column, not shape {tuple(x.shape)}")
        x = x.reshape(-1, x.shape[-1])
    K = x.shape[1]
    if K < 1:
        raise ValueError(f"{what} needs at least one column, not shape {tuple(x.shape)}")
    if x.shape[0] > _MOST or K > _MOST:
        raise ValueError(f"{what}: {x.shape[0]} rows of {K} elements are more than 2^31 - 1 of either")
    return x if K == 1 or x.stride(1) == 1 else x.contiguous()


def _code_rows(q: torch.Tensor, what: str) -> Tuple[torch.Tensor, int]:
    """Codes as ``[M, K]`` in rows the product can read 16 bytes at a time, and the row stride."""
    q = _rows(q, what)
    M, K = q.shape
    kp = (K + 15) & ~15
    ld = q.stride(0) if M > 1 else kp
    fits = ld >= kp and ld % 16 == 0 and q.data_ptr() % 16 == 0
    if fits and kp != K:      # the bytes that fill the last row up must belong to the tensor's memory too
        fits = q.storage_offset() + (M - 1) * ld + kp <= q.untyped_storage().nbytes()
    if fits:
        return q, ld
    buf = torch.empty(M, kp, dtype=_I8, device=q.device)
    buf[:, :K] = q
    return buf, kp


def _new_codes(M: int, K: int, device) -> Tuple[torch.Tensor, int]:
    kp = (K + 15) & ~15
    buf = torch.empty(M, kp, dtype=_I8, device=device)
    return (buf if kp == K else buf[:, :K]), kp


def _padded_codes(q: torch.Tensor) -> torch.Tensor:
    K = q.shape[1]
    return q if K % 16 == 0 else torch.nn.functional.pad(q, (0, -K % 16))[:, :K]


def _vector(device: torch.device, what: str, s: torch.Tensor, shape) -> torch.Tensor:
    """Scales or biases of ``shape`` as contiguous fp32 (their shape may stay that of several dimensions)."""
    if s.shape != shape:
        raise ValueError(f"{what} has shape {tuple(s.shape)}, expected {tuple(shape)}")
    if s.device != device:
        raise ValueError(f"{what} is on {s.device}, not on {device}")
    if s.dtype is not _F32:
        if not s.is_floating_point():
            raise TypeError(f"{what} must be a floating tensor, not {s.dtype}")
        s = s.float()
    return s.resolve_neg().contiguous()


def _codes_given(q: torch.Tensor, what: str) -> None:
    if q.dtype is not _I8:
        raise TypeError(f"{what} must be int8, not {q.dtype}")


def _launch(name: str, args, device: torch.device) -> None:
    rc = H.launch_on(name, args, device.index)
    if rc:
        H._check(rc, name)


def _shaped(t: torch.Tensor, x: torch.Tensor, *last: int) -> torch.Tensor:
    """``t[M, ...]`` with the leading dimensions of ``x``."""
    return t if x.ndim == 2 else t.view((*x.shape[:-1], *last))


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x[..., K]`` (fp32 / bf16 / fp16) -> ``(codes[..., K] int8, scale[...] fp32)``:
    ``scale = max |row| / 127``, ``code = round(x * 127 / max |row|)``, the quotient rounded to fp32 and then to the nearest
    whole number, halves to even."""
    if x.is_cuda:
        out = _binding().quantize(x)
        if out is not None:
            return out
    dt = _float_code(x, "x")
    x2 = _rows(x, "x")
    M, K = x2.shape
    if not x.is_cuda:
        with torch.no_grad():
            q, scale = ref.quantize_rows(x2)
            return _shaped(_padded_codes(q), x, K), _shaped(scale, x)
    device = x.device
    q, ld = _new_codes(M, K, device)
    scale = torch.empty(M, dtype=_F32, device=device)
    if M:
        _launch("d4pg_quant_rows", H.QuantRowsArgs(x2.data_ptr(), None, None, None, q.data_ptr(), scale.data_ptr(), M, K,
                                                   x2.stride(0), 0, 0, ld, dt, H.F_NONE, 0, 0.0), device)
    return (q, scale) if x.ndim == 2 else (_shaped(q, x, K), _shaped(scale, x))


def dequantize_rows(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``codes[..., K]``, ``scale[...]`` -> ``codes * scale`` in ``dtype``."""
    if q.is_cuda:
        out = _binding().dequantize(q, scale, _FLOATS.get(dtype, -1))
        if out is not None:
            return out
    dt = _out_code(dtype)
    _codes_given(q, "q")
    device = q.device
    q2 = _rows(q, "q")
    M, K = q2.shape
    s = _vector(device, "scale", scale, q.shape[:-1])
    if not q.is_cuda:
        with torch.no_grad():
            return _shaped(ref.dequantize_rows(q2, s.reshape(-1), dtype), q, K)
    out = torch.empty(M, K, dtype=dtype, device=device)
    if M:
        _launch("d4pg_dequant_rows", H.DequantRowsArgs(q2.data_ptr(), s.data_ptr(), out.data_ptr(), M, K, q2.stride(0), dt, 0), device)
    return out if q.ndim == 2 else _shaped(out, q, K)


def add_rms_norm_int8(x: torch.Tensor, weight: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                      eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``h = x + residual``; ``y = h * weight / sqrt(mean(h^2) + eps)``; returns ``(codes of y, scales of y, h)``.

    ``x[..., K]`` and ``residual`` (same shape and type, or ``None``: then ``h`` is ``x`` itself) are fp32, bf16 or fp16;
    ``weight[K]`` any of them, or ``None`` for ones.  The norm is of the fp32 sum; ``h`` is that sum rounded to the type
    of ``x``.  ``mean`` and everything up to the codes is fp32, ``eps`` too (what fp32 does not hold is refused)."""
    if x.is_cuda:
        out = _binding().quantize(x, weight, residual, eps)
        if out is not None:
            return out
    dt = _float_code(x, "x")
    given, eps = eps, C.c_float(eps).value
    if not (given >= 0.0 and eps < float("inf")):
        raise ValueError(f"eps must be a number >= 0 that fp32 holds, not {given}")
    device = x.device
    x2 = _rows(x, "x")
    M, K = x2.shape
    r2, wt = None, H.F_NONE
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"residual is {tuple(residual.shape)} {residual.dtype}, x is {tuple(x.shape)} {x.dtype}")
        _on(device, "residual", residual)
        r2 = _rows(residual, "residual")
    if weight is not None:
        if weight.shape != (K,):
            raise ValueError(f"weight has shape {tuple(weight.shape)}, expected ({K},)")
        wt = _float_code(weight, "weight")
        _on(device, "weight", weight)
        weight = weight.resolve_neg().contiguous()
    if not x.is_cuda:
        with torch.no_grad():
            q, scale, h = ref.add_rms_norm_int8(x2, weight, r2, eps)
            return _shaped(_padded_codes(q), x, K), _shaped(scale, x), (x if residual is None else _shaped(h, x, K))
    q, ld = _new_codes(M, K, device)
    scale = torch.empty(M, dtype=_F32, device=device)
    h = x if r2 is None else torch.empty(M, K, dtype=x.dtype, device=device)
    if M:
        _launch("d4pg_quant_rows", H.QuantRowsArgs(
            x2.data_ptr(), None if r2 is None else r2.data_ptr(), None if weight is None else weight.data_ptr(),
            None if r2 is None else h.data_ptr(), q.data_ptr(), scale.data_ptr(), M, K, x2.stride(0),
            0 if r2 is None else r2.stride(0), K, ld, dt, wt, 1, eps), device)
    if x.ndim == 2:
        return q, scale, h
    return _shaped(q, x, K), _shaped(scale, x), (x if r2 is None else _shaped(h, x, K))


def _layer(device: torch.device, K: int, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor]):
    """``(weight scales, bias)`` of a layer with ``K`` inputs, as the kernels read them."""
    _codes_given(weight, "weight")
    if weight.ndim != 2 or weight.shape[1] != K:
        raise ValueError(f"weight has shape {tuple(weight.shape)}, expected (out, {K})")
    if K > MAX_K:
        raise ValueError(f"{K} columns: sums of more than {MAX_K} products can leave 32 bits")
    if weight.shape[0] > 1 << 29:
        raise ValueError(f"{weight.shape[0]} outputs: at most 2^29 are supported")
    _on(device, "weight", weight)
    outs = weight.shape[:1]
    return _vector(device, "weight_scale", weight_scale, outs), None if bias is None else _vector(device, "bias", bias, outs)


def linear_int8(q: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, activation: str = "none",
                dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``act((q @ weight.T) * scale * weight_scale + bias)`` in ``dtype``, the sums exact in 32-bit integers.

    ``q[..., K]`` int8 with ``scale[...]``; ``weight[N, K]`` int8 with ``weight_scale[N]``; ``bias[N]`` or ``None``;
    ``activation`` in {none, relu, tanh}; ``dtype`` fp32, bf16 or fp16."""
    if q.is_cuda:
        out = _binding().linear(q, scale, weight, weight_scale, bias, _ACTS.get(activation, -1), _FLOATS.get(dtype, -1))
        if out is not None:
            return out
    dt = _out_code(dtype)
    act = _act_code(activation)
    _codes_given(q, "q")
    device = q.device
    if q.ndim < 1 or q.shape[-1] < 1:
        raise ValueError(f"q needs at least one column, not shape {tuple(q.shape)}")
    K = q.shape[-1]
    ws, b = _layer(device, K, weight, weight_scale, bias)
    s = _vector(device, "scale", scale, q.shape[:-1])
    N = weight.shape[0]
    if not q.is_cuda:
        with torch.no_grad():
            return _shaped(ref.linear_int8(_rows(q, "q"), s.reshape(-1), weight, ws, b, activation, dtype), q, N)
    q2, ldq = _code_rows(q, "q")
    M = q2.shape[0]
    out = torch.empty(M, N, dtype=dtype, device=device)
    if M and N:
        w2, ldw = _code_rows(weight, "weight")
        _launch("d4pg_linear_int8", H.LinearInt8Args(
            q2.data_ptr(), s.data_ptr(), w2.data_ptr(), ws.data_ptr(), None if b is None else b.data_ptr(), out.data_ptr(),
            ldq, ldw, N, M, N, K, act, dt, 0), device)
    return out if q.ndim == 2 else _shaped(out, q, N)


_FINAL = ("none", "relu", "softmax", "tanh")


def mlp3_int8(x: torch.Tensor, layers: Sequence[Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]],
              final: str = "none", dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Three-layer MLP of the actor / critic on 8-bit codes (ReLU, ReLU, ``final`` in {none, relu, tanh, softmax}).

    ``x[..., S]`` fp32, bf16 or fp16; ``layers``: three ``(weight[out, in] int8, weight_scale[out], bias[out] or None)``.
    The input of every layer is quantised per row; what the layers hand on is fp32; the result is in ``dtype``.  On the GPU
    the network is one launch (``mlp3_int8_kernel``) where no layer has more than 1024 outputs and the LDS holds it: always up
    to 1024 columns, except for a layer of 113 - 128 outputs beside one of more than 960 inputs with up to 4096 states.
    Otherwise it is a quantisation and a product a layer (``d4pg_mlp3_int8_launches`` says which)."""
    if x.is_cuda and len(layers) == 3:
        out = _binding().mlp3(x, *layers[0], *layers[1], *layers[2], _ACTS.get(final, -1), _FLOATS.get(dtype, -1))
        if out is not None:
            return out
    dt = _out_code(dtype)
    if len(layers) != 3:
        raise ValueError(f"three layers are expected, not {len(layers)}")
    if final not in _FINAL:
        raise ValueError(f"final must be one of {_FINAL}, not {final!r}")
    if final == "softmax":
        return torch.softmax(mlp3_int8(x, layers), dim=-1).to(dtype)
    if x.is_cuda:
        out = _mlp3_fused(x, layers, final, dtype, dt)
        if out is not None:
            return out
    h = x
    for weight, weight_scale, bias in layers[:2]:
        h = linear_int8(*quantize_rows(h), weight, weight_scale, bias, "relu")
    return linear_int8(*quantize_rows(h), *layers[2], activation=final, dtype=dtype)


def _mlp3_fused(x: torch.Tensor, layers, final: str, dtype: torch.dtype, dt: int) -> Optional[torch.Tensor]:
    xdt = _float_code(x, "x")
    x2 = _rows(x, "x")
    device = x.device
    M, K = x2.shape
    a = H.Mlp3Int8Args()
    held, width = [], [K]
    for i, (weight, weight_scale, bias) in enumerate(layers):
        ws, b = _layer(device, K, weight, weight_scale, bias)
        K = weight.shape[0]
        if K < 1:
            return None
        w2, a.ld_w[i] = _code_rows(weight, "weight")
        a.w[i], a.wscale[i] = w2.data_ptr(), ws.data_ptr()
        if b is not None:
            a.bias[i] = b.data_ptr()
        held.append((w2, ws, b))
        width.append(K)
    out = torch.empty(M, K, dtype=dtype, device=device)
    if M:
        a.width[:] = width
        a.x, a.ld_x, a.out, a.ld_out, a.M = x2.data_ptr(), x2.stride(0), out.data_ptr(), K, M
        a.xdtype, a.dtype, a.act = xdt, dt, _ACTS[final]
        rc = H.launch_on("d4pg_mlp3_int8", a, device.index)
        if rc == H.NOT_TAKEN:    # too wide for one workgroup's LDS
            return None
        if rc:
            H._check(rc, "d4pg_mlp3_int8")
    return out if x.ndim == 2 else _shaped(out, x, K)
