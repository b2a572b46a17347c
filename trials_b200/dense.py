"""Dense FP8 block-scaled products: the parts of a MoE block around the routed
experts (projections, the shared expert, dense feed-forward layers) in the
layer's number formats.

  * fp8_block_linear  x . w^T with 1x128 activation and 128x128 weight scales
  * fp8_gate_up       gate/up projection, silu(gate) * up, re-quantised 1x128
  * fp8_mlp           fp8_gate_up then fp8_block_linear, optionally added to a
                      residual (the routed experts' output)

The reference has no counterpart: its serving framework fuses the shared expert
as one more routed slot (runner.fuse_shared_expert), which needs the routed
experts' intermediate size. A NaN in a token's row, or in silu(gate) * up, is kept:
it makes its 128-group and the outputs behind it NaN (per_token_group_quant_fp8 and
the routed layer code it as -448). Every op runs the CUDA kernels of libb200moe.so on
the current torch stream of its tensors' device; there is no fallback path.
"""
from __future__ import annotations

import functools
import struct
from typing import Optional

import torch

from . import _lib
from .moe import FP8, _require_cuda, _stream, _workspaces

# These calls take a few microseconds on the GPU for a few tokens, so the checks
# below read each attribute once and build no intermediate objects, and the C
# entries get their arguments packed as one struct of 8-byte members (0 = NULL).
_PACK = {n: struct.Struct(f"{n}q").pack for n in (19, 20)}
_F32, _BF16 = torch.float32, torch.bfloat16


def _device_of(x: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """Index of the one CUDA device all tensors are on."""
    index = x.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            _require_cuda(x, *others)  # says what is wrong
    if index < 0:
        _require_cuda(x)
    return index


def _call(fn, where: str, index: int, *args: int) -> None:
    """Calls a C entry on the current stream of device `index`, the current one; args
    are its arguments up to the error word and the stream. The error word is the one
    of (device, stream), moe.layer_error_word."""
    stream = torch._C._cuda_getCurrentRawStream(index)
    status = fn(_PACK[len(args) + 2](*args, _workspaces.header_ptr(index, stream), stream))
    if status:
        _lib.check(status, where)


def _rows(t: torch.Tensor, what: str) -> int:
    """Row stride in elements of a 2-D tensor whose rows are contiguous."""
    if t.is_contiguous():
        return t.shape[1]
    s0, s1 = t.stride()
    n, m = t.shape
    if m > 1 and s1 != 1:
        raise ValueError(f"{what}: elements of a row must be contiguous")
    if n <= 1:
        return m  # the stride of a single row says nothing
    if s0 < m:
        raise ValueError(f"{what}: rows must not overlap")
    return s0


def _input(x: torch.Tensor, x_scale: Optional[torch.Tensor]):
    """Checked activation rows and scales, copied only where their layout asks for
    it: (x, x_scale, M, K, stride of x, stride of x_scale)."""
    shape = x.shape
    if len(shape) != 2:
        raise ValueError("x must be (M, K)")
    M, K = shape
    dtype = x.dtype
    ld_s = 0
    if dtype is FP8:
        align = 16
        if x_scale is None or x_scale.shape != (M, K // 128):
            raise ValueError("fp8 x needs x_scale of shape (M, K/128) (1x128 per-token-group scales)")
        if x_scale.dtype is not _F32:
            raise NotImplementedError("x_scale must be float32")
        ld_s, s1 = x_scale.stride()
        if s1 != 1 or (M > 1 and ld_s < K // 128):
            x_scale = x_scale.contiguous()
            ld_s = K // 128
        elif M <= 1:
            ld_s = K // 128
    elif dtype is _BF16:
        align = 8
        if x_scale is not None:
            raise ValueError("x_scale is only meaningful with fp8 x")
    else:
        raise NotImplementedError("x must be bf16, or fp8 e4m3 with (M, K/128) x_scale")
    if K == 0 or K % 128:
        raise NotImplementedError("K must be a multiple of 128")
    s0, s1 = x.stride()
    if M <= 1:
        s0 = K
    if s1 != 1 or s0 < K or s0 % align or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        s0 = K
    return x, x_scale, M, K, s0, ld_s


def _weight(w: torch.Tensor, scale: torch.Tensor, K: int, what: str):
    """(row stride of the weight, contiguous scales, rows), checked."""
    if w.dtype is not FP8:
        raise NotImplementedError(f"{what} must be float8_e4m3fn with 128x128 block scales")
    shape = w.shape
    if len(shape) != 2 or shape[1] != K or shape[0] == 0:
        raise ValueError(f"{what} must be (N, {K}), got {tuple(shape)}")
    N = shape[0]
    if scale.dtype is not _F32:
        raise NotImplementedError(f"{what}_scale must be float32")
    if scale.shape != ((N + 127) >> 7, K >> 7):
        raise ValueError(f"{what}_scale must be (ceil(N/128), K/128), got {tuple(scale.shape)}")
    if w.is_contiguous():
        ld = K
    else:
        ld = _rows(w, what)
    return ld, scale if scale.is_contiguous() else scale.contiguous(), N


def _output(out: Optional[torch.Tensor], residual: Optional[torch.Tensor], M: int, N: int, dtype: torch.dtype,
            dev: torch.device):
    """(out, its row stride, the residual's row stride), checked."""
    if out is None:
        out = torch.empty((M, N), dtype=dtype, device=dev)
        ld = N
    else:
        if out.shape != (M, N) or out.dtype is not dtype:
            raise ValueError(f"out must be ({M}, {N}) {dtype}")
        ld = _rows(out, "out")
    if residual is None:
        return out, ld, 0
    if residual.dtype is not _BF16:
        raise NotImplementedError("residual must be bf16")
    if residual.shape != (M, N):
        raise ValueError(f"residual must be ({M}, {N})")
    return out, ld, _rows(residual, "residual")


# Sizes of workspaces by sizes of the call and its device, which is the current one:
# asking the library each time is a tenth of a one-token call.
@functools.lru_cache(maxsize=4096)
def _linear_bytes(index: int, M: int, N: int, K: int, gate_up: int) -> int:
    return _lib.lib().b200moe_linear_workspace_size(M, N, K, 1, gate_up)


@functools.lru_cache(maxsize=4096)
def _mlp_bytes(index: int, M: int, H: int, I: int, bf16: bool) -> int:
    return _lib.lib().b200moe_mlp_workspace_size(M, H, I, bf16)


def _workspace(nbytes: int, dev: torch.device):
    """(tensor to hold until the call returns, pointer, size): this call's own, from
    torch's allocator on the current stream, so calls on other streams and captured
    graphs have theirs."""
    if nbytes == 0:
        return None, 0, 0
    ws = torch.empty((nbytes,), dtype=torch.uint8, device=dev)
    return ws, ws.data_ptr(), nbytes


def fp8_block_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                     x_scale: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """(M, N) = x . weight^T (+ residual): x (M, K) bf16 (quantised 1x128 first)
    or fp8 e4m3 with x_scale (M, K/128); weight (N, K) fp8 e4m3 with
    weight_scale (ceil(N/128), K/128) f32; residual (M, N) bf16, added in fp32.
    Accumulated in fp32 and rounded once to out_dtype (bf16 or f32). Any M and
    N; K % 128 == 0. out may be residual itself and overlaps no other input. See
    b200moe_linear."""
    index = _device_of(x, weight, weight_scale, x_scale, residual, out)
    if torch.cuda.current_device() != index:  # plans, sizes and launches go by the current device
        with torch.cuda.device(index):
            return fp8_block_linear(x, weight, weight_scale, x_scale, residual, out, out_dtype)
    if out_dtype is not _BF16 and out_dtype is not _F32:
        raise NotImplementedError("out_dtype must be bf16 or float32")
    x, x_scale, M, K, ld_x, ld_s = _input(x, x_scale)
    dev = x.device
    ld_w, weight_scale, N = _weight(weight, weight_scale, K, "weight")
    out, ld_out, ld_res = _output(out, residual, M, N, out_dtype, dev)
    if M == 0:
        return out
    L = _lib.lib()
    if x_scale is None:
        ws, ws_ptr, ws_bytes = _workspace(_linear_bytes(index, M, N, K, 0), dev)
        rows = (x.data_ptr(), 0, 0)
    else:
        ws_ptr, ws_bytes = 0, 0
        rows = (0, x.data_ptr(), x_scale.data_ptr())
    _call(L.b200moe_linear, "fp8_block_linear", index,
          *rows, ld_x, ld_s, M, N, K, weight.data_ptr(), ld_w, weight_scale.data_ptr(),
          0 if residual is None else residual.data_ptr(), ld_res, out.data_ptr(), ld_out,
          out_dtype is _F32, ws_ptr, ws_bytes)
    return out


def fp8_gate_up(x: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor, x_scale: Optional[torch.Tensor] = None):
    """(q e4m3 (M, I), s f32 (M, I/128)) = 1x128 quantisation of silu(gate) * up,
    (gate, up) = x . w13^T with gate/up rows interleaved (row 2j = gate j, 2j+1 =
    up j). x as in fp8_block_linear; w13 (2I, H) fp8 e4m3, w13_scale (2I/128,
    H/128) f32; I % 128 == 0. See b200moe_gate_up."""
    index = _device_of(x, w13, w13_scale, x_scale)
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return fp8_gate_up(x, w13, w13_scale, x_scale)
    x, x_scale, M, H, ld_x, ld_s = _input(x, x_scale)
    dev = x.device
    ld_w, w13_scale, N = _weight(w13, w13_scale, H, "w13")
    if N % 256:
        raise NotImplementedError("w13 must have 2I rows with I a multiple of 128")
    I = N // 2
    q = torch.empty((M, I), dtype=FP8, device=dev)
    s = torch.empty((M, I // 128), dtype=_F32, device=dev)
    if M == 0:
        return q, s
    L = _lib.lib()
    if x_scale is None:
        ws, ws_ptr, ws_bytes = _workspace(_linear_bytes(index, M, 2 * I, H, 1), dev)
        rows = (x.data_ptr(), 0, 0)
    else:
        ws_ptr, ws_bytes = 0, 0
        rows = (0, x.data_ptr(), x_scale.data_ptr())
    _call(L.b200moe_gate_up, "fp8_gate_up", index,
          *rows, ld_x, ld_s, M, H, I, w13.data_ptr(), ld_w, w13_scale.data_ptr(), q.data_ptr(), I, s.data_ptr(),
          I // 128, ws_ptr, ws_bytes)
    return q, s


def fp8_mlp(x: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor, w2_scale: torch.Tensor,
            x_scale: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """(M, H) bf16 = w2 . (silu(gate) * up) (+ residual): fp8_gate_up with w13
    (2I, H), then fp8_block_linear with w2 (H, I), in one call (same bits).
    out may be residual or x itself. See b200moe_mlp."""
    index = _device_of(x, w13, w13_scale, w2, w2_scale, x_scale, residual, out)
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            return fp8_mlp(x, w13, w13_scale, w2, w2_scale, x_scale, residual, out)
    x, x_scale, M, H, ld_x, ld_s = _input(x, x_scale)
    dev = x.device
    ld13, w13_scale, N = _weight(w13, w13_scale, H, "w13")
    if N % 256:
        raise NotImplementedError("w13 must have 2I rows with I a multiple of 128")
    I = N // 2
    ld2, w2_scale, rows2 = _weight(w2, w2_scale, I, "w2")
    if rows2 != H:
        raise ValueError(f"w2 must be ({H}, {I}), got {tuple(w2.shape)}")
    if ld13 != H or ld2 != I:
        raise ValueError("w13 and w2 must be contiguous")
    out, ld_out, ld_res = _output(out, residual, M, H, _BF16, dev)
    if M == 0:
        return out
    L = _lib.lib()
    ws, ws_ptr, ws_bytes = _workspace(_mlp_bytes(index, M, H, I, x_scale is None), dev)
    rows = (x.data_ptr(), 0, 0) if x_scale is None else (0, x.data_ptr(), x_scale.data_ptr())
    _call(L.b200moe_mlp, "fp8_mlp", index,
          *rows, ld_x, ld_s, M, H, I, w13.data_ptr(), w13_scale.data_ptr(), w2.data_ptr(), w2_scale.data_ptr(),
          0 if residual is None else residual.data_ptr(), ld_res, out.data_ptr(), ld_out, ws_ptr, ws_bytes)
    return out
