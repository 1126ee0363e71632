"""8-bit serving operators: rows to codes and back, RMS norm with 8-bit output, int8 product, int8 policy network.

A quantised row holds codes ``q`` in ``[-127, 127]`` and one fp32 scale ``s = max |row| / 127``; it stands for ``q * s``.
Activations are quantised per row (token, state), weights per output channel (the rows of ``weight[out, in]``)::

    wq, ws = quantize_rows(layer.weight)                              # once
    q, s, h = add_rms_norm_int8(x, norm_weight, residual)             # per call
    y = linear_int8(q, s, wq, ws, layer.bias, "relu", torch.bfloat16)

On a ROCm tensor the functions launch the kernels of ``csrc/int8.hip`` on the current stream of the tensors' device; on a
CPU tensor they evaluate ``ops/ref.py``.  They serve: no gradient flows through codes, and what they return requires none.

Code matrices are handed out with rows padded to 16 bytes (a view of ``[..., K]`` codes whose row stride is the next
multiple of 16), which is what the product reads directly; codes laid out differently are copied once per call.

A row with a NaN or an infinity gets scale NaN and codes 0, so everything computed from it is NaN; a row of zeros gets
scale 0 and codes 0.
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch

from . import hip as H
from . import ref

_FLOATS = {torch.float32: H.F_FP32, torch.bfloat16: H.F_BF16, torch.float16: H.F_FP16}
_ACTS = {"none": H.ACT_NONE, "relu": H.ACT_RELU, "tanh": H.ACT_TANH}
#: products of two codes are at most 128^2 in magnitude: sums of this many fit 32 bits
MAX_K = 131071


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


def _same_device(a: torch.Tensor, what: str, b: Optional[torch.Tensor]) -> None:
    if b is not None and b.device != a.device:
        raise ValueError(f"{what} is on {b.device}, not on {a.device}")


def _rows(x: torch.Tensor, what: str) -> Tuple[torch.Tensor, int, int]:
    """``x[..., K]`` as ``[M, K]`` with neighbouring elements side by side, and ``M``, ``K``."""
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError(f"{what} needs at least one column, not shape {tuple(x.shape)}")
    K = x.shape[-1]
    x2 = x if x.ndim == 2 else x.reshape(-1, K)
    if K > 1 and x2.stride(1) != 1:
        x2 = x2.contiguous()
    return x2, x2.shape[0], K


def _code_rows(q: torch.Tensor, what: str) -> Tuple[torch.Tensor, int, int, int]:
    """Codes as ``[M, K]`` in rows the product can read 16 bytes at a time, with ``M``, ``K`` and the row stride."""
    q2, M, K = _rows(q, what)
    kp = (K + 15) & ~15
    ld = q2.stride(0) if M > 1 else kp
    fits = q2.data_ptr() % 16 == 0 and ld % 16 == 0 and ld >= kp
    if fits and kp != K:      # the bytes that fill the last row up must belong to the tensor's memory too
        fits = q2.storage_offset() + (M - 1) * ld + kp <= q2.untyped_storage().nbytes()
    if not fits:
        buf = torch.empty(M, kp, dtype=torch.int8, device=q.device)
        buf[:, :K] = q2
        q2, ld = buf, kp
    return q2, M, K, ld


def _new_codes(M: int, K: int, device) -> Tuple[torch.Tensor, int]:
    kp = (K + 15) & ~15
    buf = torch.empty(M, kp, dtype=torch.int8, device=device)
    return (buf if kp == K else buf[:, :K]), kp


def _padded_codes(q: torch.Tensor) -> torch.Tensor:
    K = q.shape[1]
    return q if K % 16 == 0 else torch.nn.functional.pad(q, (0, -K % 16))[:, :K]


def _launch(name: str, args, t: torch.Tensor) -> None:
    if t.device.index == torch.cuda.current_device():
        H.launch(name, args)
    else:
        with torch.cuda.device(t.device):
            H.launch(name, args)


def _shaped(t: torch.Tensor, x: torch.Tensor, *last: int) -> torch.Tensor:
    """``t[M, ...]`` with the leading dimensions of ``x``."""
    return t if x.ndim == 2 else t.view((*x.shape[:-1], *last))


@torch.no_grad()
def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``x[..., K]`` (fp32 / bf16 / fp16) -> ``(codes[..., K] int8, scale[...] fp32)``:
    ``scale = max |row| / 127``, ``code = round(x * 127 / max |row|)``, halves to even."""
    dt = _float_code(x, "x")
    x2, M, K = _rows(x, "x")
    if not x.is_cuda:
        q, scale = ref.quantize_rows(x2)
        return _shaped(_padded_codes(q), x, K), _shaped(scale, x)
    q, ld = _new_codes(M, K, x.device)
    scale = torch.empty(M, dtype=torch.float32, device=x.device)
    if M:
        a = H.QuantRowsArgs()
        a.x, a.q, a.scale = x2.data_ptr(), q.data_ptr(), scale.data_ptr()
        a.M, a.K, a.ld_x, a.ld_q = M, K, x2.stride(0), ld
        a.dtype, a.wdtype = dt, H.F_NONE
        _launch("d4pg_quant_rows", a, x)
    return _shaped(q, x, K), _shaped(scale, x)


@torch.no_grad()
def dequantize_rows(q: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``codes[..., K]``, ``scale[...]`` -> ``codes * scale`` in ``dtype``."""
    dt = _out_code(dtype)
    if q.dtype != torch.int8:
        raise TypeError(f"q must be int8, not {q.dtype}")
    q2, M, K = _rows(q, "q")
    s = _scales(q, "scale", scale, q.shape[:-1])
    if not q.is_cuda:
        return _shaped(ref.dequantize_rows(q2, s, dtype), q, K)
    out = torch.empty(M, K, dtype=dtype, device=q.device)
    if M:
        a = H.DequantRowsArgs()
        a.q, a.scale, a.out = q2.data_ptr(), s.data_ptr(), out.data_ptr()
        a.M, a.K, a.ld_q, a.dtype = M, K, q2.stride(0), dt
        _launch("d4pg_dequant_rows", a, q)
    return _shaped(out, q, K)


def _scales(near: torch.Tensor, what: str, s: torch.Tensor, shape) -> torch.Tensor:
    if s.shape != shape:
        raise ValueError(f"{what} has shape {tuple(s.shape)}, expected {tuple(shape)}")
    _same_device(near, what, s)
    if s.dtype != torch.float32:
        if not s.is_floating_point():
            raise TypeError(f"{what} must be a floating tensor, not {s.dtype}")
        s = s.float()
    return s if s.is_contiguous() and s.ndim == 1 else s.reshape(-1).contiguous()


@torch.no_grad()
def add_rms_norm_int8(x: torch.Tensor, weight: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                      eps: float = 1e-6) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``h = x + residual``; ``y = h * weight / sqrt(mean(h^2) + eps)``; returns ``(codes of y, scales of y, h)``.

    ``x[..., K]`` and ``residual`` (same shape and type, or ``None``: then ``h`` is ``x`` itself) are fp32, bf16 or fp16;
    ``weight[K]`` any of them, or ``None`` for ones.  The norm is of the fp32 sum; ``h`` is that sum rounded to the type
    of ``x``.  ``mean`` and everything up to the codes is fp32."""
    dt = _float_code(x, "x")
    eps = float(eps)
    if not 0.0 <= eps < float("inf"):
        raise ValueError(f"eps must be a finite number >= 0, not {eps}")
    x2, M, K = _rows(x, "x")
    r2 = None
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype:
            raise ValueError(f"residual is {tuple(residual.shape)} {residual.dtype}, x is {tuple(x.shape)} {x.dtype}")
        _same_device(x, "residual", residual)
        r2 = _rows(residual, "residual")[0]
    wt = H.F_NONE
    if weight is not None:
        if weight.shape != (K,):
            raise ValueError(f"weight has shape {tuple(weight.shape)}, expected ({K},)")
        wt = _float_code(weight, "weight")
        _same_device(x, "weight", weight)
        weight = weight.contiguous()
    if not x.is_cuda:
        q, scale, h = ref.add_rms_norm_int8(x2, weight, r2, eps)
        return _shaped(_padded_codes(q), x, K), _shaped(scale, x), (x if residual is None else _shaped(h, x, K))
    q, ld = _new_codes(M, K, x.device)
    scale = torch.empty(M, dtype=torch.float32, device=x.device)
    h = None if r2 is None else torch.empty(M, K, dtype=x.dtype, device=x.device)
    if M:
        a = H.QuantRowsArgs()
        a.x, a.q, a.scale = x2.data_ptr(), q.data_ptr(), scale.data_ptr()
        a.M, a.K, a.ld_x, a.ld_q = M, K, x2.stride(0), ld
        a.dtype, a.wdtype, a.norm, a.eps = dt, wt, 1, eps
        if weight is not None:
            a.weight = weight.data_ptr()
        if r2 is not None:
            a.residual, a.ld_r, a.h, a.ld_h = r2.data_ptr(), r2.stride(0), h.data_ptr(), K
        _launch("d4pg_quant_rows", a, x)
    return _shaped(q, x, K), _shaped(scale, x), (x if h is None else _shaped(h, x, K))


def _layer_checks(K: int, near: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                  bias: Optional[torch.Tensor]):
    """``(weight scales, bias)`` as the kernels read them."""
    if weight.dtype != torch.int8:
        raise TypeError(f"weight must be int8, not {weight.dtype}")
    if weight.ndim != 2 or weight.shape[1] != K:
        raise ValueError(f"weight has shape {tuple(weight.shape)}, expected (out, {K})")
    if K > MAX_K:
        raise ValueError(f"{K} columns: sums of more than {MAX_K} products can leave 32 bits")
    _same_device(near, "weight", weight)
    ws = _scales(near, "weight_scale", weight_scale, weight.shape[:1])
    return ws, None if bias is None else _scales(near, "bias", bias, weight.shape[:1])


@torch.no_grad()
def linear_int8(q: torch.Tensor, scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, activation: str = "none",
                dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``act((q @ weight.T) * scale * weight_scale + bias)`` in ``dtype``, the sums exact in 32-bit integers.

    ``q[..., K]`` int8 with ``scale[...]``; ``weight[N, K]`` int8 with ``weight_scale[N]``; ``bias[N]`` or ``None``;
    ``activation`` in {none, relu, tanh}; ``dtype`` fp32, bf16 or fp16."""
    dt = _out_code(dtype)
    if activation not in _ACTS:
        raise ValueError(f"activation must be one of {sorted(_ACTS)}, not {activation!r}")
    if q.dtype != torch.int8:
        raise TypeError(f"q must be int8, not {q.dtype}")
    if q.ndim < 1 or q.shape[-1] < 1:
        raise ValueError(f"q needs at least one column, not shape {tuple(q.shape)}")
    ws, b = _layer_checks(q.shape[-1], q, weight, weight_scale, bias)
    s = _scales(q, "scale", scale, q.shape[:-1])
    N = weight.shape[0]
    if not q.is_cuda:
        y = ref.linear_int8(_rows(q, "q")[0], s, weight, ws, b, activation, dtype)
        return _shaped(y, q, N)
    q2, M, K, ldq = _code_rows(q, "q")
    out = torch.empty(M, N, dtype=dtype, device=q.device)
    if M and N:
        w2, _, _, ldw = _code_rows(weight, "weight")
        a = H.LinearInt8Args()
        a.q, a.scale, a.w, a.wscale, a.out = q2.data_ptr(), s.data_ptr(), w2.data_ptr(), ws.data_ptr(), out.data_ptr()
        if b is not None:
            a.bias = b.data_ptr()
        a.ld_q, a.ld_w, a.ld_out = ldq, ldw, N
        a.M, a.N, a.K, a.act, a.dtype = M, N, K, _ACTS[activation], dt
        _launch("d4pg_linear_int8", a, q)
    return _shaped(out, q, N)


def mlp3_int8(x: torch.Tensor, layers: Sequence[Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]],
              final: str = "none", dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Three-layer MLP of the actor / critic on 8-bit codes (ReLU, ReLU, ``final`` in {none, relu, tanh, softmax}).

    ``layers``: three ``(weight[out, in] int8, weight_scale[out], bias[out] or None)``.  The input of every layer is
    quantised per row; what the layers hand on is fp32; the result is in ``dtype``."""
    if len(layers) != 3:
        raise ValueError(f"three layers are expected, not {len(layers)}")
    _out_code(dtype)
    if final not in ("none", "relu", "tanh", "softmax"):
        raise ValueError(f"final must be none, relu, tanh or softmax, not {final!r}")
    h = x
    for weight, weight_scale, bias in layers[:2]:
        h = linear_int8(*quantize_rows(h), weight, weight_scale, bias, "relu")
    if final == "softmax":
        return torch.softmax(linear_int8(*quantize_rows(h), *layers[2]), dim=-1).to(dtype)
    return linear_int8(*quantize_rows(h), *layers[2], activation=final, dtype=dtype)
