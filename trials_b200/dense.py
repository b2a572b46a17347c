"""Dense FP8 block-scaled products: the parts of a MoE block around the routed
experts (projections, the shared expert, dense feed-forward layers) in the
layer's number formats.

  * fp8_block_linear  x . w^T with 1x128 activation and 128x128 weight scales
  * fp8_gate_up       gate/up projection, silu(gate) * up, re-quantised 1x128
  * fp8_mlp           fp8_gate_up then fp8_block_linear, optionally added to a
                      residual (the routed experts' output)

The reference has no counterpart: its serving framework fuses the shared expert
as one more routed slot (runner.fuse_shared_expert), which needs the routed
experts' intermediate size. Every op runs the CUDA kernels of libb200moe.so on
the current torch stream of its tensors' device; there is no fallback path.
"""
from __future__ import annotations

import contextlib
from typing import Optional

import torch

from . import _lib
from .moe import FP8, _ptr, _require_cuda, _stream, _workspaces


def _on_device(dev: torch.device):
    """Kernels launch on the current device: make it the tensors' device."""
    if torch.cuda.current_device() == dev.index:
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


def _rows(t: torch.Tensor, what: str) -> int:
    """Row stride in elements of a 2-D tensor whose rows are contiguous."""
    if t.shape[1] > 1 and t.stride(1) != 1:
        raise ValueError(f"{what}: elements of a row must be contiguous")
    if t.shape[0] <= 1:
        return t.shape[1]  # the stride of a single row says nothing
    if t.stride(0) < t.shape[1]:
        raise ValueError(f"{what}: rows must not overlap")
    return t.stride(0)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy whose rows are contiguous and start 16-byte aligned."""
    size = t.element_size()
    ok = (t.stride(1) == 1 and (t.shape[0] <= 1 or (t.stride(0) * size % 16 == 0 and t.stride(0) >= t.shape[1]))
          and t.data_ptr() % 16 == 0)
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _input(x: torch.Tensor, x_scale: Optional[torch.Tensor]):
    """Checked activation rows and scales, copied only where their layout asks for it."""
    if x.dim() != 2:
        raise ValueError("x must be (M, K)")
    if x.dtype == FP8:
        if x_scale is None or x_scale.dim() != 2 or tuple(x_scale.shape) != (x.shape[0], x.shape[1] // 128):
            raise ValueError("fp8 x needs x_scale of shape (M, K/128) (1x128 per-token-group scales)")
        if x_scale.dtype != torch.float32:
            raise NotImplementedError("x_scale must be float32")
        if x_scale.stride(1) != 1 or (x_scale.shape[0] > 1 and x_scale.stride(0) < x_scale.shape[1]):
            x_scale = x_scale.contiguous()
    elif x.dtype == torch.bfloat16:
        if x_scale is not None:
            raise ValueError("x_scale is only meaningful with fp8 x")
    else:
        raise NotImplementedError("x must be bf16, or fp8 e4m3 with (M, K/128) x_scale")
    if x.shape[1] == 0 or x.shape[1] % 128:
        raise NotImplementedError("K must be a multiple of 128")
    return _aligned(x), x_scale


def _weight(w: torch.Tensor, scale: torch.Tensor, K: int, what: str):
    if w.dtype != FP8:
        raise NotImplementedError(f"{what} must be float8_e4m3fn with 128x128 block scales")
    if w.dim() != 2 or w.shape[1] != K or w.shape[0] == 0:
        raise ValueError(f"{what} must be (N, {K}), got {tuple(w.shape)}")
    if scale.dtype != torch.float32:
        raise NotImplementedError(f"{what}_scale must be float32")
    if tuple(scale.shape) != ((w.shape[0] + 127) // 128, K // 128):
        raise ValueError(f"{what}_scale must be (ceil(N/128), K/128), got {tuple(scale.shape)}")
    return _rows(w, what), scale.contiguous()


def _output(out: Optional[torch.Tensor], residual: Optional[torch.Tensor], M: int, N: int, dtype: torch.dtype,
            dev: torch.device):
    if out is None:
        out = torch.empty(M, N, dtype=dtype, device=dev)
    elif tuple(out.shape) != (M, N) or out.dtype != dtype:
        raise ValueError(f"out must be ({M}, {N}) {dtype}")
    if residual is not None:
        if residual.dtype != torch.bfloat16:
            raise NotImplementedError("residual must be bf16")
        if tuple(residual.shape) != (M, N):
            raise ValueError(f"residual must be ({M}, {N})")
    return out, residual


def _call_state(dev: torch.device, nbytes: int):
    """(stream, error word pointer, workspace) of one call. The workspace is
    this call's own, from torch's allocator on the current stream; the error
    word is the cached one of (device, stream) (moe.layer_error_word)."""
    stream = _stream(dev)
    err = _workspaces.get_for(dev, stream, 256).data_ptr()
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    return stream, err, ws


def fp8_block_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                     x_scale: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """(M, N) = x . weight^T (+ residual): x (M, K) bf16 (quantised 1x128 first)
    or fp8 e4m3 with x_scale (M, K/128); weight (N, K) fp8 e4m3 with
    weight_scale (ceil(N/128), K/128) f32; residual (M, N) bf16, added in fp32.
    Accumulated in fp32 and rounded once to out_dtype (bf16 or f32). Any M and
    N; K % 128 == 0. out may be residual itself. See b200moe_linear."""
    dev = _require_cuda(x, weight, weight_scale, x_scale, residual, out)
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise NotImplementedError("out_dtype must be bf16 or float32")
    x, x_scale = _input(x, x_scale)
    M, K = x.shape
    N = weight.shape[0]
    ld_w, weight_scale = _weight(weight, weight_scale, K, "weight")
    out, residual = _output(out, residual, M, N, out_dtype, dev)
    if M == 0:
        return out
    L = _lib.lib()
    quantised = x_scale is not None
    with _on_device(dev):
        stream, err, ws = _call_state(dev, 0 if quantised else L.b200moe_linear_workspace_size(M, K))
        _lib.check(L.b200moe_linear(
            None if quantised else x.data_ptr(), x.data_ptr() if quantised else None, _ptr(x_scale), _rows(x, "x"),
            _rows(x_scale, "x_scale") if quantised else 0, M, N, K, weight.data_ptr(), ld_w, weight_scale.data_ptr(),
            _ptr(residual), 0 if residual is None else _rows(residual, "residual"), out.data_ptr(),
            _rows(out, "out"), int(out_dtype == torch.float32), _ptr(ws), 0 if ws is None else ws.numel(), err,
            stream), "fp8_block_linear")
    return out


def fp8_gate_up(x: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor, x_scale: Optional[torch.Tensor] = None):
    """(q e4m3 (M, I), s f32 (M, I/128)) = 1x128 quantisation of silu(gate) * up,
    (gate, up) = x . w13^T with gate/up rows interleaved (row 2j = gate j, 2j+1 =
    up j). x as in fp8_block_linear; w13 (2I, H) fp8 e4m3, w13_scale (2I/128,
    H/128) f32; I % 128 == 0. See b200moe_gate_up."""
    dev = _require_cuda(x, w13, w13_scale, x_scale)
    x, x_scale = _input(x, x_scale)
    M, H = x.shape
    ld_w, w13_scale = _weight(w13, w13_scale, H, "w13")
    if w13.shape[0] % 256:
        raise NotImplementedError("w13 must have 2I rows with I a multiple of 128")
    I = w13.shape[0] // 2
    q = torch.empty(M, I, dtype=FP8, device=dev)
    s = torch.empty(M, I // 128, dtype=torch.float32, device=dev)
    if M == 0:
        return q, s
    L = _lib.lib()
    quantised = x_scale is not None
    with _on_device(dev):
        stream, err, ws = _call_state(dev, 0 if quantised else L.b200moe_linear_workspace_size(M, H))
        _lib.check(L.b200moe_gate_up(
            None if quantised else x.data_ptr(), x.data_ptr() if quantised else None, _ptr(x_scale), _rows(x, "x"),
            _rows(x_scale, "x_scale") if quantised else 0, M, H, I, w13.data_ptr(), ld_w, w13_scale.data_ptr(),
            q.data_ptr(), I, s.data_ptr(), I // 128, _ptr(ws), 0 if ws is None else ws.numel(), err, stream),
            "fp8_gate_up")
    return q, s


def fp8_mlp(x: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor, w2_scale: torch.Tensor,
            x_scale: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(M, H) bf16 = w2 . (silu(gate) * up) (+ residual): fp8_gate_up with w13
    (2I, H), then fp8_block_linear with w2 (H, I), in one call (same bits).
    out may be residual itself. See b200moe_mlp."""
    dev = _require_cuda(x, w13, w13_scale, w2, w2_scale, x_scale, residual, out)
    x, x_scale = _input(x, x_scale)
    M, H = x.shape
    ld13, w13_scale = _weight(w13, w13_scale, H, "w13")
    if w13.shape[0] % 256:
        raise NotImplementedError("w13 must have 2I rows with I a multiple of 128")
    I = w13.shape[0] // 2
    ld2, w2_scale = _weight(w2, w2_scale, I, "w2")
    if w2.shape[0] != H:
        raise ValueError(f"w2 must be ({H}, {I}), got {tuple(w2.shape)}")
    if ld13 != H or ld2 != I:
        raise ValueError("w13 and w2 must be contiguous")
    out, residual = _output(out, residual, M, H, torch.bfloat16, dev)
    if M == 0:
        return out
    L = _lib.lib()
    quantised = x_scale is not None
    with _on_device(dev):
        stream, err, ws = _call_state(dev, L.b200moe_mlp_workspace_size(M, H, I))
        _lib.check(L.b200moe_mlp(
            None if quantised else x.data_ptr(), x.data_ptr() if quantised else None, _ptr(x_scale), _rows(x, "x"),
            _rows(x_scale, "x_scale") if quantised else 0, M, H, I, w13.data_ptr(), w13_scale.data_ptr(),
            w2.data_ptr(), w2_scale.data_ptr(), _ptr(residual),
            0 if residual is None else _rows(residual, "residual"), out.data_ptr(), _rows(out, "out"), ws.data_ptr(),
            ws.numel(), err, stream), "fp8_mlp")
    return out
