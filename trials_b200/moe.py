"""Drop-in host API of the FP8 block-scaled MoE layer.

Mirrors the reference's operator surface for this path:
  * moe_decode_megakernel_full / _moe_decode_megakernel_full
      <- sglang_integration/aiter.py:74-177
  * fused_moe (per_128x128 / Silu / interleaved gate-up subset)
      <- the aiter fused_moe call at sglang_integration/aiter.py:459-478
  * moe_align_block_size        <- sglang op called at aiter.py:113-115
  * per_token_group_quant_fp8   <- sglang op called at aiter.py:132-133, 151-152
  * per_block_quant_fp8         <- phase5_orchestrator.py:35-41
Every op runs the CUDA kernels of libb200moe.so through its C ABI on the
current torch stream. Unsupported options raise NotImplementedError; there is
no fallback path.
"""
from __future__ import annotations

import ctypes
import struct
import threading
from enum import Enum
from typing import Optional

import torch

from . import _lib

FP8 = torch.float8_e4m3fn


# ----------------------------------------------------------------------------
# helpers
# ----------------------------------------------------------------------------
def _ptr(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _stream(device: torch.device) -> int:
    """Handle of the device's current stream (the raw form of
    torch.cuda.current_stream(device).cuda_stream, 0.1 us instead of 2.2)."""
    index = device.index
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if index is None else index)


def _require_cuda(*tensors: torch.Tensor) -> torch.device:
    dev = tensors[0].device
    for t in tensors:
        if t is None:
            continue
        if t.device.type != "cuda":
            raise ValueError("b200moe ops take CUDA tensors; there is no CPU implementation")
        if t.device != dev:
            raise ValueError("all tensors must be on the same device")
    return dev


class _Workspaces:
    """What calls on one (device, stream) share: a header of 256 zeroed bytes (the
    device error word, int 0, then the router's CTA counter and the whole-layer
    launch's sync words, ints 1..3, left at zero by every call) and the layer's
    grow-only scratch. A header is there until the process exits, since captured
    graphs keep its address, and is zeroed outside any capture, or a graph's replay
    would clear it. A scratch that a captured graph may use is kept when a larger
    one takes its place."""

    def __init__(self):
        self._headers = {}
        self._bufs = {}
        self._captured = set()  # keys whose scratch a captured call was given
        self._kept = []
        self._lock = threading.Lock()

    def get(self, device: torch.device, nbytes: int) -> torch.Tensor:
        """The scratch of (device, its current stream)."""
        key = (device.index, _stream(device))
        capturing = torch.cuda.is_current_stream_capturing()
        with self._lock:
            buf = self._bufs.get(key)
            if buf is None or buf.numel() < nbytes:
                if key in self._captured:
                    self._kept.append(buf)
                    self._captured.discard(key)
                buf = torch.empty(nbytes, dtype=torch.uint8, device=device)
                self._bufs[key] = buf
            if capturing:
                self._captured.add(key)
            return buf

    def header_ptr(self, index: int, stream: int) -> int:
        """Address of the header of (device index, its current stream)."""
        ptr = self._headers.get((index, stream))
        return self._new_header(index, stream) if ptr is None else ptr

    def is_header(self, ptr: int) -> bool:
        with self._lock:
            return ptr in self._headers.values()

    def _new_header(self, index: int, stream: int) -> int:
        with self._lock:
            if (index, stream) not in self._headers:
                out = ctypes.c_void_p()
                with torch.cuda.device(index):
                    _lib.check(_lib.lib().b200moe_header_create(ctypes.byref(out)), "header_create")
                self._headers[index, stream] = out.value
            return self._headers[index, stream]


class _DeviceInts:
    """Device memory as the CUDA array interface describes it."""

    def __init__(self, ptr: int, n: int):
        self.__cuda_array_interface__ = {"shape": (n,), "typestr": "<i4", "data": (ptr, False), "version": 2}


_workspaces = _Workspaces()
_SCORING = {"softmax": 0, "sigmoid": 1}
_PACK_GROUPED = struct.Struct("10qd3q").pack  # b200moe_router_grouped_args
_PACK_LAYER = struct.Struct("15qd13q").pack  # b200moe_layer_args


def read_device_error(err_word: torch.Tensor, clear: bool = True) -> int:
    """Returns the device error word (B200MOE_DEVERR_* bits) after the stream ran. When
    layer_error_word() reports a timeout, clearing it puts the counters behind it back
    to zero too, which a call that gave up may have left in between."""
    val = ctypes.c_int32()
    _lib.check(_lib.lib().b200moe_read_error(err_word.data_ptr(), ctypes.byref(val), int(clear),
                                             _stream(err_word.device)), "read_error")
    if clear and val.value & _lib.DEVERR_TIMEOUT and _workspaces.is_header(err_word.data_ptr()):
        torch.as_tensor(_DeviceInts(err_word.data_ptr(), 64), device=err_word.device).zero_()
    return int(val.value)


def layer_error_word(device: Optional[torch.device] = None) -> torch.Tensor:
    """The error word of the calls on (device, its current stream), graphs captured
    on that stream among them; the same word until the process exits."""
    index = torch.cuda.current_device() if device is None or device.index is None else device.index
    ptr = _workspaces.header_ptr(index, torch._C._cuda_getCurrentRawStream(index))
    return torch.as_tensor(_DeviceInts(ptr, 1), device=torch.device("cuda", index))


# ----------------------------------------------------------------------------
# routing and quantisation ops
# ----------------------------------------------------------------------------
def moe_align_block_size(topk_ids: torch.Tensor, block_size: int, num_experts: int,
                         expert_map: Optional[torch.Tensor] = None, num_local_experts: Optional[int] = None,
                         err_word: Optional[torch.Tensor] = None):
    """Returns (sorted_token_ids, expert_ids, num_tokens_post_padded) with the
    reference's layout; see include/b200moe.h b200moe_align."""
    dev = _require_cuda(topk_ids)
    ids = topk_ids.to(torch.int32).contiguous()
    M, topk = ids.shape
    L = _lib.lib()
    E = num_local_experts if expert_map is not None else num_experts
    if expert_map is not None:
        expert_map = expert_map.to(device=dev, dtype=torch.int32).contiguous()
        if E is None:
            raise ValueError("num_local_experts is required with expert_map")
    cap = L.b200moe_align_capacity_rows(M * topk, E, block_size)
    cap_b = L.b200moe_align_capacity_blocks(M * topk, E, block_size)
    sorted_ids = torch.empty(cap, dtype=torch.int32, device=dev)
    expert_ids = torch.empty(cap_b, dtype=torch.int32, device=dev)
    ntp = torch.empty(1, dtype=torch.int32, device=dev)
    stream = _stream(dev)
    err = _workspaces.header_ptr(ids.get_device(), stream) if err_word is None else _ptr(err_word)
    _lib.check(L.b200moe_align(_ptr(ids), M, topk, num_experts, block_size, _ptr(expert_map), E or 0,
                               _ptr(sorted_ids), cap, _ptr(expert_ids), cap_b, _ptr(ntp), err, stream),
               "moe_align_block_size")
    return sorted_ids, expert_ids, ntp


def _check_groups(num_expert_group: Optional[int], topk_group: Optional[int]) -> bool:
    if (num_expert_group is None) != (topk_group is None):
        raise ValueError("num_expert_group and topk_group go together")
    if num_expert_group is not None and num_expert_group < 1:
        raise ValueError("num_expert_group must be positive")
    return num_expert_group is not None


def _router_bias(bias: Optional[torch.Tensor], dev: torch.device, index: Optional[int],
                 E: int) -> Optional[torch.Tensor]:
    """The correction bias as the kernels read it: E contiguous f32 on the device, or
    more, of which the first E count (index: the device's, None if unknown)."""
    if bias is None:
        return None
    if bias.numel() < E:
        raise ValueError(f"correction_bias must have {E} entries, got {tuple(bias.shape)}")
    if bias.dtype is torch.float32 and bias.get_device() == index and bias.is_contiguous():
        return bias
    return bias.to(device=dev, dtype=torch.float32).contiguous()


def select_experts(router_logits: torch.Tensor, top_k: int, scoring_func: str = "softmax",
                   correction_bias: Optional[torch.Tensor] = None, renormalize: bool = True,
                   routed_scaling_factor: float = 1.0, num_expert_group: Optional[int] = None,
                   topk_group: Optional[int] = None):
    """Router: (M, E) f32/bf16 logits -> (topk_weights (M, k) f32, topk_ids (M, k) int32).
    softmax: top-k softmax probabilities; sigmoid: top-k of sigmoid + correction_bias
    with the unbiased sigmoid as weights (GLM's routing). See b200moe_router_topk.
    num_expert_group, topk_group: group-limited routing, only the experts of the
    topk_group best of num_expert_group equal groups can be selected (a group's
    score is its largest value, with correction_bias the sum of its two largest).
    See b200moe_router_topk_grouped."""
    dev = router_logits.device
    index = router_logits.get_device()
    if index < 0:
        _require_cuda(router_logits)
    if torch.cuda.current_device() != index:  # kernels launch on the current device
        with torch.cuda.device(index):
            return select_experts(router_logits, top_k, scoring_func, correction_bias, renormalize,
                                  routed_scaling_factor, num_expert_group, topk_group)
    bf16 = router_logits.dtype is torch.bfloat16
    if not bf16 and router_logits.dtype is not torch.float32:
        raise NotImplementedError("router logits must be float32 or bfloat16")
    scoring = _SCORING.get(scoring_func)
    if scoring is None:
        raise NotImplementedError(f"scoring_func {scoring_func!r}")
    grouped = _check_groups(num_expert_group, topk_group)
    logits = router_logits.contiguous()
    M, E = logits.shape
    bias = _router_bias(correction_bias, dev, index, E)
    w = torch.empty(M, top_k, dtype=torch.float32, device=dev)
    ids = torch.empty(M, top_k, dtype=torch.int32, device=dev)
    if grouped:
        # one packed struct: fourteen converted arguments cost 1.3 us more
        status = _lib.lib().b200moe_router_topk_grouped(_PACK_GROUPED(
            logits.data_ptr(), bf16, M, E, num_expert_group, topk_group, top_k, scoring,
            0 if bias is None else bias.data_ptr(), bool(renormalize), routed_scaling_factor, w.data_ptr(),
            ids.data_ptr(), torch._C._cuda_getCurrentRawStream(index)))
        if status:
            _lib.check(status, "select_experts")
        return w, ids
    _lib.check(_lib.lib().b200moe_router_topk(_ptr(logits), int(logits.dtype == torch.bfloat16), M, E, top_k,
                                              scoring, _ptr(bias), int(renormalize), float(routed_scaling_factor),
                                              _ptr(w), _ptr(ids), _stream(dev)), "select_experts")
    return w, ids


def per_token_group_quant_fp8(x: torch.Tensor, group_size: int = 128):
    """(M, K) bf16 -> (q e4m3 (M, K), s f32 (M, K/128))."""
    if group_size != 128:
        raise NotImplementedError("only 128-wide groups are supported")
    dev = _require_cuda(x)
    if x.dtype != torch.bfloat16:
        raise NotImplementedError("per_token_group_quant_fp8 takes bf16 input")
    if x.dim() != 2 or x.stride(1) != 1:
        x = x.reshape(-1, x.shape[-1]).contiguous()
    M, K = x.shape
    q = torch.empty(M, K, dtype=FP8, device=dev)
    s = torch.empty(M, K // 128, dtype=torch.float32, device=dev)
    _lib.check(_lib.lib().b200moe_quant_1x128(_ptr(x), M, K, x.stride(0), _ptr(q), K, _ptr(s), K // 128, 1,
                                              _stream(dev)), "per_token_group_quant_fp8")
    return q, s


def per_block_quant_fp8(w: torch.Tensor, bn: int = 128, bk: int = 128):
    """(E, N, K) bf16 -> (q e4m3 (E, N, K), s f32 (E, ceil(N/128), K/128)); a 2-D
    (N, K) weight -> 2-D q and s. The last block of an N that is no multiple of
    128 covers the rows that exist."""
    if bn != 128 or bk != 128:
        raise NotImplementedError("only 128x128 blocks are supported")
    dev = _require_cuda(w)
    if w.dtype != torch.bfloat16:
        raise NotImplementedError("per_block_quant_fp8 takes bf16 input")
    if w.dim() == 2:
        q, s = per_block_quant_fp8(w.unsqueeze(0), bn, bk)
        return q[0], s[0]
    w = w.contiguous()
    E, N, K = w.shape
    q = torch.empty(E, N, K, dtype=FP8, device=dev)
    s = torch.empty(E, (N + 127) // 128, K // 128, dtype=torch.float32, device=dev)
    _lib.check(_lib.lib().b200moe_quant_block128(_ptr(w), E, N, K, _ptr(q), _ptr(s), _stream(dev)),
               "per_block_quant_fp8")
    return q, s


# ----------------------------------------------------------------------------
# the layer
# ----------------------------------------------------------------------------
def _check_layer_args(hidden, w13, w13_scale, w2, w2_scale, topk_weights, topk_ids, a1_scale=None):
    dev = _require_cuda(hidden, w13, w13_scale, w2, w2_scale, topk_weights, topk_ids)
    if hidden.dtype == FP8:
        if a1_scale is None or a1_scale.dim() != 2 or tuple(a1_scale.shape) != (hidden.shape[0], hidden.shape[1] // 128):
            raise NotImplementedError("fp8 hidden_states need a1_scale of shape (M, H/128) (1x128 per-token-group "
                                      "scales); per-token (M,) scales are not supported")
    elif hidden.dtype != torch.bfloat16:
        raise NotImplementedError("hidden_states must be bf16, or fp8 e4m3 with (M, H/128) a1_scale")
    if w13.dtype != FP8 or w2.dtype != FP8:
        raise NotImplementedError("weights must be float8_e4m3fn with 128x128 block scales")
    if w13_scale is None or w2_scale is None:
        raise ValueError("w13_scale and w2_scale are required")
    M, H = hidden.shape
    E, N2, H2 = w13.shape
    I = w2.shape[2]
    if H2 != H or N2 != 2 * I or w2.shape[:2] != (E, H):
        raise ValueError(f"shape mismatch: hidden {tuple(hidden.shape)}, w13 {tuple(w13.shape)}, "
                         f"w2 {tuple(w2.shape)}")
    if tuple(w13_scale.shape) != (E, N2 // 128, H // 128) or tuple(w2_scale.shape) != (E, H // 128, I // 128):
        raise ValueError("block scale shapes must be (E, N/128, K/128)")
    if topk_ids.shape != topk_weights.shape or topk_ids.shape[0] != M:
        raise ValueError("topk_ids and topk_weights must both be (M, topk)")
    return dev, M, H, I, E


_NO_ROUTER = (0, 0, 0, 0, 0, 0, 0, 0.0)


def _layer_call(where: str, dev: torch.device, ws_bytes: int, rows, sizes, router, tensors, n_local: int,
                out: torch.Tensor) -> None:
    """b200moe_layer_call on the current stream of `dev`, with its header and scratch."""
    ws = _workspaces.get(dev, ws_bytes)
    stream = _stream(dev)
    index = torch.cuda.current_device() if dev.index is None else dev.index
    _lib.check(_lib.lib().b200moe_layer_call(_PACK_LAYER(
        *rows, *sizes, *router, *(_ptr(t) or 0 for t in tensors), n_local, _ptr(out),
        _workspaces.header_ptr(index, stream), _ptr(ws), ws.numel(), stream)), where)


def _run_layer(hidden, w13, w13_scale, w2, w2_scale, topk_weights, topk_ids, expert_map, num_experts, out=None,
               a1_scale=None):
    dev = _require_cuda(hidden)
    if torch.cuda.current_device() != dev.index:  # kernels launch on the current device
        with torch.cuda.device(dev):
            return _run_layer(hidden, w13, w13_scale, w2, w2_scale, topk_weights, topk_ids, expert_map, num_experts,
                              out, a1_scale)
    dev, M, H, I, E_w = _check_layer_args(hidden, w13, w13_scale, w2, w2_scale, topk_weights, topk_ids, a1_scale)
    topk = topk_ids.shape[1]
    if out is None:
        out = torch.empty(M, H, dtype=torch.bfloat16, device=dev)
    if M == 0:
        return out
    hidden = hidden.contiguous()
    ids = topk_ids.to(torch.int32).contiguous()
    tw = topk_weights.to(torch.float32).contiguous()
    L = _lib.lib()
    n_local = E_w
    ws_bytes = L.b200moe_layer_workspace_size(M, H, I, num_experts, n_local, topk)
    # Contiguous copies are bound to names so that they live until the call
    # returns: a copy whose pointer alone were passed could be freed, and its
    # memory reused by the next copy, before the kernels read it.
    w13_scale, w2_scale = w13_scale.contiguous(), w2_scale.contiguous()
    fp8 = hidden.dtype == FP8
    a1 = a1_scale.to(torch.float32).contiguous() if fp8 else None
    _layer_call("b200moe_layer_quantized" if fp8 else "b200moe_layer", dev, ws_bytes,
                (0, _ptr(hidden), _ptr(a1)) if fp8 else (_ptr(hidden), 0, 0), (M, H, I, num_experts, topk), _NO_ROUTER,
                (w13, w13_scale, w2, w2_scale, tw, ids, expert_map), n_local, out)
    return out


def moe_decode_megakernel_full(hidden_states: torch.Tensor, w13_fp8: torch.Tensor, w13_scale: torch.Tensor,
                               w2_fp8: torch.Tensor, w2_scale: torch.Tensor, topk_weights: torch.Tensor,
                               topk_ids: torch.Tensor, a1_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Full MoE layer, same arguments and result as the reference
    `_moe_decode_megakernel_full` (sglang_integration/aiter.py:74-177):
    (M, H) bf16 = sum_j topk_weights[:, j] * W2[e] . silu_mul(W13[e] . h).
    hidden_states may be bf16, or fp8 e4m3 already quantised 1x128 with
    a1_scale (M, H/128); the reference's per-token (M,) a1_scale form
    (aiter.py:126-130) cannot run there either and is rejected."""
    if hidden_states.dtype != FP8 and a1_scale is not None:
        raise ValueError("a1_scale is only meaningful with fp8 hidden_states")
    return _run_layer(hidden_states, w13_fp8, w13_scale, w2_fp8, w2_scale, topk_weights, topk_ids, None,
                      w13_fp8.shape[0], a1_scale=a1_scale)


_moe_decode_megakernel_full = moe_decode_megakernel_full


class QuantType(str, Enum):
    """aiter QuantType names (sglang_integration/aiter.py:180-184)."""
    No = "No"
    per_Token = "per_Token"
    per_128x128 = "per_128x128"
    per_1x32 = "per_1x32"


class ActivationType(str, Enum):
    Silu = "Silu"
    Gelu = "Gelu"
    Swiglu = "Swiglu"
    Situv2 = "Situv2"


def _enum_value(x) -> str:
    return x.value if isinstance(x, Enum) else (x.name if hasattr(x, "name") else str(x))


def expert_map_from_mask(expert_mask: torch.Tensor) -> torch.Tensor:
    """expert_mask (E_global,) of 0/1 -> map global id -> local weight index or -1."""
    m = expert_mask.to(torch.int32)
    local = torch.cumsum(m, 0, dtype=torch.int32) - 1
    return torch.where(m > 0, local, torch.full_like(local, -1)).contiguous()


def fused_moe(hidden_states: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor, topk_weight: torch.Tensor,
              topk_ids: torch.Tensor, quant_type=QuantType.per_128x128, activation=ActivationType.Silu,
              w1_scale: Optional[torch.Tensor] = None, w2_scale: Optional[torch.Tensor] = None,
              a1_scale: Optional[torch.Tensor] = None, a2_scale: Optional[torch.Tensor] = None,
              bias1: Optional[torch.Tensor] = None, bias2: Optional[torch.Tensor] = None,
              expert_mask: Optional[torch.Tensor] = None, doweight_stage1: bool = False, hidden_pad: int = 0,
              intermediate_pad: int = 0, gate_mode: str = "interleave", num_local_tokens=None, dtype=None,
              no_combine: bool = False, **extra) -> torch.Tensor:
    """The aiter fused_moe call of sglang_integration/aiter.py:459-478 for the
    block-scaled FP8 configuration (per_128x128, Silu, gate/up interleaved).

    expert_mask (E_global,) marks the experts whose weights w1/w2 hold (in
    ascending id order); slots routed elsewhere contribute nothing."""
    if _enum_value(quant_type) != QuantType.per_128x128.value:
        raise NotImplementedError(f"quant_type {quant_type!r}: only per_128x128 is supported")
    if _enum_value(activation) != ActivationType.Silu.value:
        raise NotImplementedError(f"activation {activation!r}: only Silu is supported")
    if str(_enum_value(gate_mode)).lower() not in ("interleave", "0"):
        raise NotImplementedError("only the interleaved gate/up weight layout is supported")
    if bias1 is not None or bias2 is not None:
        raise NotImplementedError("bias is not supported")
    if a2_scale is not None:
        raise NotImplementedError("static a2_scale is not supported (stage-2 activations are quantised per group)")
    if doweight_stage1 or hidden_pad or intermediate_pad:
        raise NotImplementedError("doweight_stage1 / hidden_pad / intermediate_pad are not supported")
    if no_combine:
        raise NotImplementedError("no_combine is not supported")
    if dtype not in (None, torch.bfloat16):
        raise NotImplementedError("output dtype must be bf16")
    if num_local_tokens is not None:
        raise NotImplementedError("num_local_tokens is not supported")
    if extra.pop("swiglu_limit", 0.0):
        raise NotImplementedError("swiglu_limit is not supported")
    if extra:
        raise NotImplementedError(f"unsupported arguments: {sorted(extra)}")
    if hidden_states.dtype != FP8 and a1_scale is not None:
        raise NotImplementedError("static a1_scale with bf16 hidden_states is not supported (activations are "
                                  "quantised per 1x128 group)")
    if hidden_states.shape[0] == 0:
        return hidden_states.new_empty((0, hidden_states.shape[1]), dtype=torch.bfloat16)
    if expert_mask is not None:
        emap = expert_map_from_mask(expert_mask.to(hidden_states.device))
        return _run_layer(hidden_states, w1, w1_scale, w2, w2_scale, topk_weight, topk_ids, emap,
                          int(expert_mask.numel()), a1_scale=a1_scale)
    return _run_layer(hidden_states, w1, w1_scale, w2, w2_scale, topk_weight, topk_ids, None, w1.shape[0],
                      a1_scale=a1_scale)


def moe_layer_from_logits(hidden_states: torch.Tensor, router_logits: torch.Tensor, w13_fp8: torch.Tensor,
                          w13_scale: torch.Tensor, w2_fp8: torch.Tensor, w2_scale: torch.Tensor, top_k: int,
                          scoring_func: str = "sigmoid", correction_bias: Optional[torch.Tensor] = None,
                          renormalize: bool = True, routed_scaling_factor: float = 1.0,
                          expert_map: Optional[torch.Tensor] = None, num_expert_group: Optional[int] = None,
                          topk_group: Optional[int] = None, shared_expert: Optional[tuple] = None):
    """Router + layer: select_experts(router_logits, ...) followed by
    moe_decode_megakernel_full, with the router inside routing's first launch
    (b200moe_layer_logits). Returns (out (M, H) bf16, topk_weights (M, k) f32,
    topk_ids (M, k) int32), bit-identical to the two calls. expert_map
    (num_experts,) maps a global id to a local weight index or -1 (the weights
    then hold only the mapped experts). num_expert_group, topk_group: as in
    select_experts. shared_expert: (w13, w13_scale, w2, w2_scale) of a dense
    expert that every token passes through; dense.fp8_mlp adds it to out."""
    dev = _require_cuda(hidden_states, router_logits, w13_fp8, w2_fp8)
    if torch.cuda.current_device() != dev.index:  # kernels launch on the current device
        with torch.cuda.device(dev):
            return moe_layer_from_logits(hidden_states, router_logits, w13_fp8, w13_scale, w2_fp8, w2_scale, top_k,
                                         scoring_func, correction_bias, renormalize, routed_scaling_factor,
                                         expert_map, num_expert_group, topk_group, shared_expert)
    grouped = _check_groups(num_expert_group, topk_group)
    if hidden_states.dtype != torch.bfloat16:
        raise NotImplementedError("moe_layer_from_logits takes bf16 hidden_states")
    if router_logits.dtype not in (torch.float32, torch.bfloat16):
        raise NotImplementedError("router logits must be float32 or bfloat16")
    scoring = {"softmax": 0, "sigmoid": 1}.get(scoring_func)
    if scoring is None:
        raise NotImplementedError(f"scoring_func {scoring_func!r}")
    M, E_router = router_logits.shape
    tw = torch.empty(M, top_k, dtype=torch.float32, device=dev)
    ids = torch.empty(M, top_k, dtype=torch.int32, device=dev)
    _, _, H, I, E_w = _check_layer_args(hidden_states, w13_fp8, w13_scale, w2_fp8, w2_scale, tw, ids)
    out = torch.empty(M, H, dtype=torch.bfloat16, device=dev)
    if M == 0:
        return out, tw, ids
    if expert_map is not None:
        expert_map = expert_map.to(device=dev, dtype=torch.int32).contiguous()
    elif E_w != E_router:
        raise ValueError("without expert_map the weights must hold every routed expert")
    bias = _router_bias(correction_bias, dev, router_logits.get_device(), E_router)
    logits = router_logits.contiguous()
    hidden = hidden_states.contiguous()
    w13_scale, w2_scale = w13_scale.contiguous(), w2_scale.contiguous()  # held through the call
    L = _lib.lib()
    _layer_call("b200moe_layer_logits_grouped" if grouped else "b200moe_layer_logits", dev,
                L.b200moe_layer_workspace_size(M, H, I, E_router, E_w, top_k), (_ptr(hidden), 0, 0),
                (M, H, I, E_router, top_k),
                (_ptr(logits), logits.dtype == torch.bfloat16, num_expert_group if grouped else 0,
                 topk_group if grouped else 0, scoring, _ptr(bias) or 0, bool(renormalize),
                 float(routed_scaling_factor)),
                (w13_fp8, w13_scale, w2_fp8, w2_scale, tw, ids, expert_map), E_w, out)
    if shared_expert is not None:
        from .dense import fp8_mlp

        fp8_mlp(hidden, *shared_expert, residual=out, out=out)
    return out, tw, ids


def moe_layer_ep_local(hidden_states, w13, w13_scale, w2, w2_scale, topk_weights, topk_ids, expert_map,
                       num_experts: int, out=None):
    """Layer over the experts this rank holds: ids are global, expert_map maps
    them to local weight rows (-1 = elsewhere). Used by the expert-parallel path."""
    return _run_layer(hidden_states, w13, w13_scale, w2, w2_scale, topk_weights, topk_ids, expert_map,
                      num_experts, out=out)
