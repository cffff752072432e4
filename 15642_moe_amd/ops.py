"""Host-side mirror of the reference's ``ops`` module (pybind11 ``moe_fused``,
kernels/moe.cu:902-909): ``pack_w13``, ``pack_w2`` and ``moe_forward`` with the
reference's argument order, shape/dtype checks and RuntimeError behaviour,
implemented over the C ABI (include/moe_fp8.h).

Every function runs asynchronously on the current HIP stream of the input's
device.  There is no CPU path: CPU tensors raise RuntimeError.
"""

from __future__ import annotations

import ctypes
import functools

import numpy as np
import torch

from . import capi
from .geometry import (
    E_GLOBAL,
    G1_BLOCKS,
    H,
    H_BLOCKS,
    I_BLOCKS,
    I_DIM,
    MAX_E_LOCAL,
    N_GROUP,
    TOP_K,
    TOPK_GROUP,
    W13_PACKED_SHAPE,
    W2_PACKED_SHAPE,
)


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _ptr(t: torch.Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(t.data_ptr())


def _stream(device: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _require_device(name: str, t: torch.Tensor, device: torch.device | None = None) -> None:
    # The messages are formatted only for the error: those of every check of a
    # forward cost 9 us (validation 19 -> 10 us).
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a HIP device tensor (no CPU path)")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name} must be on {device}, got {t.device}")


# --------------------------------------------------------------------------- packs
def _check_out(out: torch.Tensor | None, shape: tuple, like: torch.Tensor, name: str) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=torch.int32, device=like.device)
    _check(out.dtype == torch.int32 and tuple(out.shape) == shape and out.is_contiguous(),
           f"{name} out must be int32 {list(shape)} contiguous")
    _require_device(f"{name} out", out, like.device)
    return out


def pack_w13(W13: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """W13 e4m3 [E_local, 4096, 7168] -> int32 packed MFMA operand tiles
    (kernels/moe.cu:700-720).  `out` (optional) receives them in place, e.g.
    one expert's slot ``packed[e:e+1]`` of a larger packed buffer."""
    _require_device("W13", W13)
    _check(W13.dim() == 3, "W13 must be [E_local, 4096, 7168]")
    _check(W13.element_size() == 1, "W13 must be an FP8 tensor")
    _check(W13.is_contiguous(), "W13 must be contiguous")
    E = int(W13.size(0))
    _check(W13.size(1) == 2 * I_DIM and W13.size(2) == H, "W13 must be [E_local, 4096, 7168]")
    out = _check_out(out, (E, *W13_PACKED_SHAPE), W13, "pack_w13")
    if E == 0:
        return out
    with torch.cuda.device(W13.device):
        capi.check(capi.load().moe_pack_w13(_ptr(W13), _ptr(out), E, _stream(W13.device)), "pack_w13")
    return out


def pack_w2(W2: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """W2 e4m3 [E_local, 7168, 2048] -> int32 packed MFMA operand tiles
    (kernels/moe.cu:722-742); `out` as for pack_w13."""
    _require_device("W2", W2)
    _check(W2.dim() == 3, "W2 must be [E_local, 7168, 2048]")
    _check(W2.element_size() == 1, "W2 must be an FP8 tensor")
    _check(W2.is_contiguous(), "W2 must be contiguous")
    E = int(W2.size(0))
    _check(W2.size(1) == H and W2.size(2) == I_DIM, "W2 must be [E_local, 7168, 2048]")
    out = _check_out(out, (E, *W2_PACKED_SHAPE), W2, "pack_w2")
    if E == 0:
        return out
    with torch.cuda.device(W2.device):
        capi.check(capi.load().moe_pack_w2(_ptr(W2), _ptr(out), E, _stream(W2.device)), "pack_w2")
    return out


def unpack_w13(packed: torch.Tensor) -> torch.Tensor:
    """Inverse of pack_w13, returned as uint8 [E, 4096, 7168]."""
    _require_device("W13_packed", packed)
    _check(packed.dim() == 7 and tuple(packed.shape[1:]) == W13_PACKED_SHAPE and packed.is_contiguous(),
           "W13_packed must be [E_local, 16, 56, 16, 2, 64, 4] contiguous")
    E = int(packed.size(0))
    out = torch.empty((E, 2 * I_DIM, H), dtype=torch.uint8, device=packed.device)
    with torch.cuda.device(packed.device):
        capi.check(capi.load().moe_unpack_w13(_ptr(packed), _ptr(out), E, _stream(packed.device)), "unpack_w13")
    return out


def unpack_w2(packed: torch.Tensor) -> torch.Tensor:
    """Inverse of pack_w2, returned as uint8 [E, 7168, 2048]."""
    _require_device("W2_packed", packed)
    _check(packed.dim() == 7 and tuple(packed.shape[1:]) == W2_PACKED_SHAPE and packed.is_contiguous(),
           "W2_packed must be [E_local, 56, 16, 8, 2, 64, 4] contiguous")
    E = int(packed.size(0))
    out = torch.empty((E, H, I_DIM), dtype=torch.uint8, device=packed.device)
    with torch.cuda.device(packed.device):
        capi.check(capi.load().moe_unpack_w2(_ptr(packed), _ptr(out), E, _stream(packed.device)), "unpack_w2")
    return out


# --------------------------------------------------------------------------- upstream producer
ROUTER_PACKED_SHAPE = (56, 4, 16, 64, 8)  # [kb, ks, expert tile, lane, bf16]


def pack_router(router_w: torch.Tensor) -> torch.Tensor:
    """Router weight bf16 [256, 7168] -> packed bf16 MFMA operand fragments
    (ROUTER_PACKED_SHAPE), for router_quant."""
    _require_device("router_w", router_w)
    _check(router_w.dtype == torch.bfloat16, "router_w must be bfloat16")
    _check(tuple(router_w.shape) == (E_GLOBAL, H) and router_w.is_contiguous(),
           "router_w must be [256, 7168] contiguous")
    out = torch.empty(ROUTER_PACKED_SHAPE, dtype=torch.bfloat16, device=router_w.device)
    with torch.cuda.device(router_w.device):
        capi.check(capi.load().moe_pack_router(_ptr(router_w), _ptr(out), _stream(router_w.device)), "pack_router")
    return out


def unpack_router(packed: torch.Tensor) -> torch.Tensor:
    """Inverse of pack_router."""
    _require_device("router_packed", packed)
    _check(tuple(packed.shape) == ROUTER_PACKED_SHAPE and packed.is_contiguous() and packed.dtype == torch.bfloat16,
           "router_packed must be a pack_router result")
    out = torch.empty((E_GLOBAL, H), dtype=torch.bfloat16, device=packed.device)
    with torch.cuda.device(packed.device):
        capi.check(capi.load().moe_unpack_router(_ptr(packed), _ptr(out), _stream(packed.device)), "unpack_router")
    return out


def router_quant(hidden: torch.Tensor, router_packed: torch.Tensor):
    """bf16 hidden states [T, 7168] -> (routing_logits f32 [T, 256],
    hidden_states e4m3 [T, 7168], hidden_states_scale f32 [56, T]): the
    router GEMM and the dynamic FP8 quantisation in front of moe_forward,
    in one pass over the hidden states (moe_router_quant)."""
    _require_device("hidden", hidden)
    dev = hidden.device
    _check(hidden.dtype == torch.bfloat16, "hidden must be bfloat16")
    _check(hidden.dim() == 2 and hidden.size(1) == H and hidden.is_contiguous(), "hidden must be [T, 7168] contiguous")
    _require_device("router_packed", router_packed, dev)
    _check(tuple(router_packed.shape) == ROUTER_PACKED_SHAPE and router_packed.dtype == torch.bfloat16,
           "router_packed must be a pack_router result")
    T = int(hidden.size(0))
    _check(T <= capi.MAX_T, f"T must be <= {capi.MAX_T}")
    lib = capi.load()
    logits = torch.empty((T, E_GLOBAL), dtype=torch.float32, device=dev)
    hq = torch.empty((T, H), dtype=torch.float8_e4m3fn, device=dev)
    hs = torch.empty((H_BLOCKS, T), dtype=torch.float32, device=dev)
    ws_bytes = int(lib.moe_router_workspace_bytes(T))
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        capi.check(lib.moe_router_quant(_ptr(hidden), _ptr(router_packed), T, _ptr(ws), ws_bytes, _ptr(logits),
                                        _ptr(hq), _ptr(hs), _stream(dev)), "router_quant")
    return logits, hq, hs


# --------------------------------------------------------------------------- forward
def _validate_forward(hidden, hidden_scale, W13_packed, W13_scale, W2_packed, W2_scale, logits, bias):
    """The checks of kernels/moe.cu:759-817, for this build's packed layout."""
    _check(hidden.dim() == 2, "hidden must be [T, 7168]")
    _check(hidden_scale.dim() == 2, "hidden_scale must be [56, T]")
    _check(W13_packed.dim() == 7, "W13_packed must be [E_local, 16, 56, 16, 2, 64, 4]")
    _check(W13_scale.dim() == 3, "W13_scale must be [E_local, 32, 56]")
    _check(W2_packed.dim() == 7, "W2_packed must be [E_local, 56, 16, 8, 2, 64, 4]")
    _check(W2_scale.dim() == 3, "W2_scale must be [E_local, 56, 16]")
    _check(logits.dim() == 2, "logits must be [T, 256]")
    _check(hidden.element_size() == 1, "hidden must be an FP8 tensor")
    _check(hidden_scale.dtype == torch.float32, "hidden_scale must be float32")
    _check(W13_packed.dtype == torch.int32, "W13_packed must be int32-packed FP8 fragments")
    _check(W13_scale.dtype == torch.float32, "W13_scale must be float32")
    _check(W2_packed.dtype == torch.int32, "W2_packed must be int32-packed FP8 fragments")
    _check(W2_scale.dtype == torch.float32, "W2_scale must be float32")
    _check(logits.dtype == torch.float32, "logits must be float32")
    _check(bias.dtype == torch.float32, "bias must be float32")
    T, H_dim = int(hidden.size(0)), int(hidden.size(1))
    E = int(W13_packed.size(0))
    _check(H_dim == H, "hidden must have hidden dim 7168")
    _check(hidden_scale.size(0) == H_BLOCKS and hidden_scale.size(1) == T, "hidden_scale must be [56, T]")
    _check(logits.size(0) == T and logits.size(1) == E_GLOBAL, "logits must be [T, 256]")
    _check(bias.numel() == E_GLOBAL, "bias must have 256 elements")
    _check(tuple(W13_packed.shape[1:]) == W13_PACKED_SHAPE, "W13_packed must be [E_local, 16, 56, 16, 2, 64, 4]")
    _check(tuple(W13_scale.shape) == (E, G1_BLOCKS, H_BLOCKS), "W13_scale must be [E_local, 32, 56]")
    _check(W2_packed.size(0) == E and tuple(W2_packed.shape[1:]) == W2_PACKED_SHAPE,
           "W2_packed must be [E_local, 56, 16, 8, 2, 64, 4]")
    _check(tuple(W2_scale.shape) == (E, H_BLOCKS, I_BLOCKS), "W2_scale must be [E_local, 56, 16]")
    if not 1 <= E <= MAX_E_LOCAL:
        raise RuntimeError(f"E_local must be in [1, {MAX_E_LOCAL}], got {E}")
    dev = hidden.device
    for name, t in (("hidden", hidden), ("hidden_scale", hidden_scale), ("W13_packed", W13_packed),
                    ("W13_scale", W13_scale), ("W2_packed", W2_packed), ("W2_scale", W2_scale),
                    ("logits", logits), ("bias", bias)):
        if not t.is_contiguous():
            raise RuntimeError(f"{name} must be contiguous")
        _require_device(name, t, dev)
    return T, E


def moe_forward_workspace(hidden, hidden_scale, W13_packed, W13_scale, W2_packed, W2_scale, logits, bias,
                          rsf: float, local_offset: int):
    """moe_forward that also returns its workspace tensor (for inspection)."""
    _require_device("hidden", hidden)
    T, E = _validate_forward(hidden, hidden_scale, W13_packed, W13_scale, W2_packed, W2_scale, logits, bias)
    lib = capi.load()
    dev = hidden.device
    out = torch.empty((T, H), dtype=torch.bfloat16, device=dev)
    ws_bytes = int(lib.moe_workspace_bytes(T, E))
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    if T == 0:
        return out, ws
    with torch.cuda.device(dev):
        rc = lib.moe_forward(_ptr(hidden), _ptr(hidden_scale), _ptr(W13_packed), _ptr(W13_scale), _ptr(W2_packed),
                             _ptr(W2_scale), _ptr(logits), _ptr(bias), float(rsf), int(local_offset), T, E,
                             _ptr(ws), ws_bytes, _ptr(out), _stream(dev))
    capi.check(rc, "moe_forward")
    return out, ws


def moe_forward(hidden, hidden_scale, W13_packed, W13_scale, W2_packed, W2_scale, logits, bias, rsf: float,
                local_offset: int) -> torch.Tensor:
    """bf16 [T, 7168] MoE forward; argument order of kernels/moe.cu:744-754."""
    return moe_forward_workspace(hidden, hidden_scale, W13_packed, W13_scale, W2_packed, W2_scale, logits, bias,
                                 rsf, local_offset)[0]


# --------------------------------------------------------------------------- general router
# A call of these operators may take the GPU 3 us, so the host's share counts: one C call on plain integers, devices
# compared by their numbers, the device switched only where another one is current, and the stream read as a raw handle.
# route_topk took the host 14 us at T = 1 with wrapped pointers, device and stream objects.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice  # a tensor on a device is there: the runtime is up
_F32, _BF16, _F16, _I32, _U8, _E4M3 = (torch.float32, torch.bfloat16, torch.float16, torch.int32, torch.uint8,
                                       torch.float8_e4m3fn)


def _index(name: str, t: torch.Tensor) -> int:
    """The number of the HIP device that t is on."""
    i = t.get_device()
    if i < 0:
        _require_device(name, t)
    return i


def _on(name: str, t: torch.Tensor, like: torch.Tensor, i: int) -> None:
    """t is on the device of `like`, whose number is i."""
    if t.get_device() != i:
        _require_device(name, t, like.device)


def _call(what: str, fn, i: int, *args) -> None:
    """fn(*args, stream) with device i current, on its current stream; RuntimeError for a non-zero status."""
    if i == _current_device():
        rc = fn(*args, _raw_stream(i))
    else:
        with torch.cuda.device(i):
            rc = fn(*args, _raw_stream(i))
    if rc:
        capi.check(rc, what)


def _empty(rows: int, cols: int, dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    # 1.3 us, where torch.empty with its keywords takes 1.7
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=dev)


_DTYPES = {_F32: capi.DTYPE_F32, _BF16: capi.DTYPE_BF16, _F16: capi.DTYPE_F16}


def _rows(name: str, x: torch.Tensor) -> tuple:
    """Checks a [T, n] float input and returns T, n, its row stride in elements, its type and its device's number."""
    i = _index(name, x)
    dtype = _DTYPES.get(x.dtype)
    if dtype is None:
        raise RuntimeError(f"{name} must be float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() != 2:
        raise RuntimeError(f"{name} must be two-dimensional")
    T, n = x.shape
    stride, step = x.stride()
    if step != 1 and n != 1:
        raise RuntimeError(f"{name} must be contiguous along its last dimension")
    return T, n, stride if T > 1 else n, dtype, i


def _check_router(logits, top_k, scoring):
    T, E, stride, dtype, i = _rows("logits", logits)
    score = capi.SCORING.get(scoring)
    if score is None:
        raise RuntimeError(f"scoring must be one of {sorted(capi.SCORING)}, got {scoring!r}")
    if T > capi.MAX_ROUTE_T:
        raise RuntimeError(f"T must be <= {capi.MAX_ROUTE_T}, got {T}")
    if not 1 <= E <= capi.MAX_EXPERTS:
        raise RuntimeError(f"logits must have 1 to {capi.MAX_EXPERTS} experts, got {E}")
    if not 1 <= top_k <= min(capi.MAX_TOP_K, E):
        raise RuntimeError(f"top_k must be in [1, {min(capi.MAX_TOP_K, E)}], got {top_k}")
    return T, E, stride, dtype, i, score


def _route_topk(logits, bias, top_k, scoring, n_group, topk_group, group_top, renormalize, scale):
    T, E, stride, dtype, i, score = _check_router(logits, top_k, scoring)
    # here, where numbers past 32 bits are still what they are
    if not 1 <= topk_group <= n_group <= 64 or not 1 <= group_top <= 2:
        raise RuntimeError(f"n_group must be in [1, 64], topk_group in [1, n_group], group_top 1 or 2, got {n_group}, "
                           f"{topk_group}, {group_top}")
    dev = logits.device
    if bias is not None:
        if bias.dtype != _F32 or bias.shape != (E,) or not bias.is_contiguous():
            raise RuntimeError(f"bias must be float32 [{E}] contiguous")
        _on("bias", bias, logits, i)
    weights = _empty(T, top_k, _F32, dev)
    ids = _empty(T, top_k, _I32, dev)
    _call("route_topk", capi.load().moe_route_topk, i, logits.data_ptr(), dtype, stride,
          None if bias is None else bias.data_ptr(), T, E, top_k, score, n_group, topk_group, group_top, renormalize,
          scale, weights.data_ptr(), ids.data_ptr())
    return weights, ids


def route_topk_backward(grad_weights: torch.Tensor, logits: torch.Tensor, ids: torch.Tensor, scoring: str = "sigmoid",
                        renormalize: bool = True, scale: float = 1.0) -> torch.Tensor:
    """The gradient of route_topk's logits [T, n_experts], in their type, from that of its weights (f32 [T, top_k])
    and its picks.  Picks outside [0, n_experts) (an unfilled slot's -1) take no part."""
    if ids.dim() != 2 or ids.dtype != _I32 or not ids.is_contiguous():
        raise RuntimeError("ids must be int32 [T, top_k] contiguous")
    rows, top_k = ids.shape
    T, E, stride, dtype, i, score = _check_router(logits, top_k, scoring)
    if rows != T:
        raise RuntimeError("ids must have a row per token")
    if grad_weights.dtype != _F32 or grad_weights.shape != ids.shape or not grad_weights.is_contiguous():
        raise RuntimeError("grad_weights must be float32 [T, top_k] contiguous")
    _on("ids", ids, logits, i)
    _on("grad_weights", grad_weights, logits, i)
    out = _empty(T, E, logits.dtype, logits.device)
    _call("route_topk_backward", capi.load().moe_route_topk_backward, i, grad_weights.data_ptr(), logits.data_ptr(), dtype,
          stride, ids.data_ptr(), T, E, top_k, score, renormalize, scale, out.data_ptr())
    return out


class _RouteTopK(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, top_k, scoring, n_group, topk_group, group_top, renormalize, scale):
        weights, ids = _route_topk(logits, bias, top_k, scoring, n_group, topk_group, group_top, renormalize, scale)
        ctx.save_for_backward(logits, ids)
        ctx.form = (scoring, renormalize, scale)
        ctx.mark_non_differentiable(ids)
        return weights, ids

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_weights, _):
        logits, ids = ctx.saved_tensors
        return (route_topk_backward(grad_weights.contiguous(), logits, ids, *ctx.form),) + (None,) * 8


def route_topk(logits: torch.Tensor, bias: torch.Tensor | None, top_k: int, scoring: str = "sigmoid",
               n_group: int = 1, topk_group: int | None = None, group_top: int = 2, renormalize: bool = True,
               scale: float = 1.0):
    """(weights f32 [T, top_k], ids int32 [T, top_k]) of the experts that each token goes to.

    Scores are sigmoid or softmax of the logits [T, n_experts] (float32, bfloat16 or float16; rows may be strided).
    Picks go by score + bias: of the `topk_group` best of `n_group` equal groups (a group counts the sum of its
    `group_top` largest), the `top_k` best experts, ties to the lower index, listed in ascending order.  Weights are the
    picks' scores, divided by their sum with `renormalize`, times `scale`.

    An expert whose logit (or logit's score + bias) is -inf or NaN is never picked; a slot that no expert fills holds
    id -1 and weight 0.  The weights are differentiable in the logits; the bias only balances load and takes no
    gradient.  `experts_w4` takes the result as it is (under no_grad, where the logits are a parameter's).  A captured
    backward pass calls for what every captured one does: no eager graph of the same leaves alive beside it;
    route_topk_backward has no such condition."""
    topk_group = n_group if topk_group is None else topk_group
    if logits.requires_grad and torch.is_grad_enabled():
        return _RouteTopK.apply(logits, None if bias is None else bias.detach(), top_k, scoring, n_group, topk_group,
                                group_top, renormalize, scale)
    return _route_topk(logits, bias, top_k, scoring, n_group, topk_group, group_top, renormalize, scale)


# --------------------------------------------------------------------------- 4-bit weights
W4_GROUP = 32            # elements of K that share an e8m0 scale
W4_CHUNK_BYTES = 4352    # 16 rows x 512 elements of K, codes and scales
W4_CHUNK_K = 512


def _check_size(T: int, K: int) -> None:
    if not 0 < K <= capi.MAX_W4_DIM or K % 128:
        raise RuntimeError(f"x must have a multiple of 128 columns, got {K}")
    if T > capi.MAX_T:
        raise RuntimeError(f"T must be <= {capi.MAX_T}")


def quant_act(x: torch.Tensor):
    """[T, K] float32, bfloat16 or float16 (K a multiple of 128) -> (e4m3 [T, K], scale f32 [K / 128, T]): the
    quantisation that router_quant does on its way, for the input of linear_w4 and experts_w4 or moe_forward."""
    T, K, stride, dtype, i = _rows("x", x)
    _check_size(T, K)
    at, dev = x.data_ptr(), x.device
    if stride * x.element_size() % 16 or at % 16:
        raise RuntimeError("x must have 16-byte aligned rows")
    codes = _empty(T, K, _E4M3, dev)
    scale = _empty(K // 128, T, _F32, dev)
    _call("quant_act", capi.load().moe_quant_act, i, at, dtype, stride, T, K, codes.data_ptr(), scale.data_ptr())
    return codes, scale


def quantize_w4(w: torch.Tensor):
    """A weight [..., N, K] (float32, bfloat16 or float16; K a multiple of 128) to OCP MXFP4: codes uint8
    [..., N, K / 2] (two e2m1 elements a byte, the lower index in the low half) and e8m0 scales uint8 [..., N, K / 32],
    for pack_w4.  Round to nearest, ties to even, saturating; a group with an infinity or NaN gets the NaN scale."""
    _require_device("w", w)
    if w.dtype not in _DTYPES:
        raise RuntimeError(f"w must be float32, bfloat16 or float16, got {w.dtype}")
    _check(w.dim() >= 2 and w.is_contiguous() and w.data_ptr() % 16 == 0, "w must be [..., N, K] contiguous, 16-byte aligned")
    K = int(w.size(-1))
    _check(0 < K <= capi.MAX_W4_DIM and K % 128 == 0, f"w must have a multiple of 128 columns, got {K}")
    codes = torch.empty((*w.shape[:-1], K // 2), dtype=torch.uint8, device=w.device)
    scales = torch.empty((*w.shape[:-1], K // W4_GROUP), dtype=torch.uint8, device=w.device)
    _call("quantize_w4", capi.load().moe_quantize_w4, w.get_device(), w.data_ptr(), _DTYPES[w.dtype], w.numel() // W4_GROUP,
          codes.data_ptr(), scales.data_ptr())
    return codes, scales


def _w4_shape(N: int, K: int) -> tuple:
    return (-(-N // 16), -(-K // W4_CHUNK_K), W4_CHUNK_BYTES)


def pack_w4(codes: torch.Tensor, scales: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """MXFP4 codes uint8 [N, K / 2] and scales uint8 [N, K / 32], or e of them [e, N, ...], in the MFMA operand layout:
    uint8 [ceil(N / 16), ceil(K / 512), 4352], or [e, ...].  `out` (optional) receives them in place, e.g. one
    expert's slot ``packed[e:e+1]`` of a larger buffer."""
    _require_device("codes", codes)
    _require_device("scales", scales, codes.device)
    _check(codes.dtype == torch.uint8 and scales.dtype == torch.uint8, "codes and scales must be uint8")
    _check(codes.dim() in (2, 3) and codes.is_contiguous() and scales.is_contiguous(),
           "codes and scales must be [N, ...] or [e, N, ...] contiguous")
    N, K = int(codes.size(-2)), 2 * int(codes.size(-1))
    _check(0 < K <= capi.MAX_W4_DIM and K % 128 == 0, f"K must be a multiple of 128, got {K}")
    _check(0 < N <= capi.MAX_W4_DIM, f"N must be in [1, {capi.MAX_W4_DIM}], got {N}")
    _check(tuple(scales.shape) == (*codes.shape[:-1], K // W4_GROUP), "scales must be [..., N, K / 32] beside codes")
    _check(codes.data_ptr() % 16 == 0 and scales.data_ptr() % 16 == 0, "codes and scales must be 16-byte aligned")
    n = int(codes.size(0)) if codes.dim() == 3 else 1
    shape = (*codes.shape[:-2], *_w4_shape(N, K))
    if out is None:
        out = torch.empty(shape, dtype=torch.uint8, device=codes.device)
    else:
        _check(out.dtype == torch.uint8 and tuple(out.shape) == shape and out.is_contiguous(),
               f"pack_w4 out must be uint8 {list(shape)} contiguous")
        _require_device("pack_w4 out", out, codes.device)
    _call("pack_w4", capi.load().moe_pack_w4, codes.get_device(), codes.data_ptr(), scales.data_ptr(), out.data_ptr(), n, N, K)
    return out


def unpack_w4(packed: torch.Tensor, N: int, K: int):
    """Inverse of pack_w4: (codes uint8 [.., N, K / 2], scales uint8 [.., N, K / 32])."""
    _require_device("packed", packed)
    _check_packed("packed", packed, N, K, batched=packed.dim() == 4)
    lead = packed.shape[:-3]
    codes = torch.empty((*lead, N, K // 2), dtype=torch.uint8, device=packed.device)
    scales = torch.empty((*lead, N, K // W4_GROUP), dtype=torch.uint8, device=packed.device)
    n = int(packed.size(0)) if packed.dim() == 4 else 1
    _call("unpack_w4", capi.load().moe_unpack_w4, packed.get_device(), packed.data_ptr(), codes.data_ptr(), scales.data_ptr(),
          n, N, K)
    return codes, scales


def _check_packed(name, packed, N, K, batched):
    want = _w4_shape(N, K)
    if packed.dtype != _U8 or packed.dim() != 3 + batched or packed.shape[-3:] != want or not packed.is_contiguous():
        lead = "[e_local, " if batched else "["
        raise RuntimeError(f"{name} must be a pack_w4 result uint8 {lead}{want[0]}, {want[1]}, {want[2]}] contiguous, "
                           f"got {packed.dtype} {list(packed.shape)}")


def _check_act(x, x_scale):
    i = _index("x", x)
    _on("x_scale", x_scale, x, i)
    if x.dtype != _E4M3 or x.dim() != 2 or not x.is_contiguous():
        raise RuntimeError("x must be e4m3 [T, K] contiguous")
    T, K = x.shape
    _check_size(T, K)
    if x_scale.dtype != _F32 or x_scale.shape != (K // 128, T) or not x_scale.is_contiguous():
        raise RuntimeError(f"x_scale must be float32 [{K // 128}, {T}] contiguous")
    return T, K, i


def linear_w4(x: torch.Tensor, x_scale: torch.Tensor, packed: torch.Tensor, n_out: int | None = None) -> torch.Tensor:
    """bf16 [T, N] = x W^T for a dense layer in 4 bits: x and x_scale from quant_act (or router_quant), `packed` from
    pack_w4.  `n_out` is N where it is not a multiple of 16."""
    T, K, i = _check_act(x, x_scale)
    if packed.dim() != 3:
        raise RuntimeError("packed must be a pack_w4 result [row tiles, chunks, 4352]")
    tiles = packed.size(0)
    N = 16 * tiles if n_out is None else int(n_out)
    if not 16 * (tiles - 1) < N <= 16 * tiles:
        raise RuntimeError(f"n_out must be in [{16 * tiles - 15}, {16 * tiles}] for {tiles} packed row tiles, got {N}")
    _on("packed", packed, x, i)
    _check_packed("packed", packed, N, K, False)
    out = _empty(T, N, _BF16, x.device)
    _call("linear_w4", capi.load().moe_linear_w4, i, x.data_ptr(), x_scale.data_ptr(), packed.data_ptr(), T, N, K,
          out.data_ptr())
    return out


@functools.lru_cache(256)  # of sizes alone: 0.1 us, where the call takes 0.5
def _experts_w4_workspace(T: int, hidden: int, inter: int, e_local: int, top_k: int) -> int:
    return capi.load().moe_experts_w4_workspace_bytes(T, hidden, inter, e_local, top_k)


def experts_w4(x: torch.Tensor, x_scale: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, ids: torch.Tensor,
               weights: torch.Tensor, local_offset: int = 0) -> torch.Tensor:
    """bf16 [T, hidden]: the routed experts of moe_forward with 4-bit weights, on the picks of any router.

    x e4m3 [T, hidden] and x_scale as for linear_w4; w13 and w2 are pack_w4 results of [e_local, 2 * inter, hidden]
    (rows [0, inter) multiply, SiLU takes rows [inter, 2 * inter), as in moe_forward) and [e_local, hidden, inter]; ids
    int32 [T, top_k] and weights f32 [T, top_k] as route_topk gives them.  Picks outside [local_offset, local_offset +
    e_local) are another rank's, or none, and add nothing; a token without local picks gets zeros.  hidden and inter
    are multiples of 128.  For serving: it has no gradient, and refuses weights that would lose theirs."""
    T, K, i = _check_act(x, x_scale)
    if w13.dim() != 4 or w2.dim() != 4:
        raise RuntimeError("w13 and w2 must be pack_w4 results [e_local, row tiles, chunks, 4352]")
    E, inter = w13.size(0), 8 * w13.size(1)
    _check(inter % 128 == 0, "w13 must have 2 * inter rows, inter a multiple of 128")
    _on("w13", w13, x, i)
    _on("w2", w2, x, i)
    _check_packed("w13", w13, 2 * inter, K, True)
    _check_packed("w2", w2, K, inter, True)
    if w2.size(0) != E:
        raise RuntimeError("w13 and w2 must have the same experts")
    if ids.dim() != 2 or ids.dtype != _I32 or ids.size(0) != T or not ids.is_contiguous():
        raise RuntimeError("ids must be int32 [T, top_k] contiguous")
    if weights.dtype != _F32 or weights.shape != ids.shape or not weights.is_contiguous():
        raise RuntimeError("weights must be float32 [T, top_k] contiguous")
    _on("ids", ids, x, i)
    _on("weights", weights, x, i)
    if weights.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("experts_w4 has no gradient: call it under torch.no_grad(), or with weights.detach()")
    if not 0 <= local_offset <= 1 << 30:
        raise RuntimeError(f"local_expert_offset must be in [0, 2^30], got {local_offset}")
    k, dev = ids.size(1), x.device
    ws_bytes = _experts_w4_workspace(T, K, inter, E, k)
    out = _empty(T, K, _BF16, dev)
    ws = _empty(1, max(ws_bytes, 1), _U8, dev)
    _call("experts_w4", capi.load().moe_experts_w4, i, x.data_ptr(), x_scale.data_ptr(), w13.data_ptr(), w2.data_ptr(),
          ids.data_ptr(), weights.data_ptr(), T, K, inter, E, k, local_offset, ws.data_ptr(), ws_bytes, out.data_ptr())
    return out


def moe_forward_w4(hidden, hidden_scale, w13: torch.Tensor, w2: torch.Tensor, logits, bias, rsf: float,
                   local_offset: int) -> torch.Tensor:
    """moe_forward with 4-bit weights: the layer's router (no-aux-loss, 8 groups, top 4, top 8 of 256) and experts_w4.
    Arguments as moe_forward's, with pack_w4 results in the place of the packed FP8 weights and their scales."""
    _check(logits.dim() == 2 and logits.size(1) == E_GLOBAL, "logits must be [T, 256]")
    weights, ids = _route_topk(logits, bias, TOP_K, "sigmoid", N_GROUP, TOPK_GROUP, 2, True, rsf)
    return experts_w4(hidden, hidden_scale, w13, w2, ids, weights, local_offset)


# --------------------------------------------------------------------------- inspection
def workspace_views(ws: torch.Tensor, T: int, E: int) -> dict:
    """Typed views of the MOE_WS_* buffers inside a forward/route workspace.

    ``Y`` rows of routes whose ``route_token`` entry has bit 31 set (the
    token's only local route) are not written by the forward: GEMM2 writes
    that token's bf16 output row directly, so those Y rows hold stale data.
    """
    off = capi.workspace_offsets(T, E)
    R = T * min(TOP_K, E)

    def view(idx, dtype, shape):
        n = int(np.prod(shape)) * torch.empty((), dtype=dtype).element_size()
        return ws[off[idx]:off[idx] + n].view(dtype).view(shape)

    return {
        "topk_ids": view(capi.WS_TOPK_IDS, torch.int32, (T, TOP_K)),
        "topk_w": view(capi.WS_TOPK_W, torch.float32, (T, TOP_K)),
        "counts": view(capi.WS_COUNTS, torch.int32, (E,)),
        "offsets": view(capi.WS_OFFSETS, torch.int32, (E + 1,)),
        "route_token": view(capi.WS_ROUTE_TOKEN, torch.int32, (R,)),
        "route_weight": view(capi.WS_ROUTE_WEIGHT, torch.float32, (R,)),
        "token_route": view(capi.WS_TOKEN_ROUTE, torch.int32, (T, TOP_K)),
        "Cq": view(capi.WS_CQ, torch.uint8, (R, I_DIM)),
        "Cs": view(capi.WS_CS, torch.float32, (R, I_BLOCKS)),
        "Y": view(capi.WS_Y, torch.float32, (R, H)),
    }


def route(logits: torch.Tensor, bias: torch.Tensor, rsf: float, local_offset: int, e_local: int = 32) -> dict:
    """Routing + local dispatch only; returns the dispatch buffers (cloned)."""
    _require_device("logits", logits)
    _check(logits.dim() == 2 and logits.size(1) == E_GLOBAL, "logits must be [T, 256]")
    _check(logits.dtype == torch.float32 and bias.dtype == torch.float32, "logits and bias must be float32")
    _check(bias.numel() == E_GLOBAL, "bias must have 256 elements")
    _check(logits.is_contiguous() and bias.is_contiguous(), "logits and bias must be contiguous")
    _require_device("bias", bias, logits.device)
    lib = capi.load()
    T = int(logits.size(0))
    dev = logits.device
    ws_bytes = int(lib.moe_workspace_bytes(T, e_local))
    _check(ws_bytes > 0 or T == 0, f"invalid e_local {e_local}")
    ws = torch.empty(max(ws_bytes, 1), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        rc = lib.moe_route(_ptr(logits), _ptr(bias), float(rsf), int(local_offset), T, int(e_local), _ptr(ws),
                           ws_bytes, _stream(dev))
    capi.check(rc, "moe_route")
    views = workspace_views(ws, T, e_local)
    keep = ("topk_ids", "topk_w", "counts", "offsets", "route_token", "route_weight", "token_route")
    return {k: views[k].clone() for k in keep}


# --------------------------------------------------------------------------- synthesis
def fill_normal_e4m3_(t: torch.Tensor, seed: int, stream_id: int) -> torch.Tensor:
    """In-place device fill with the counter-based ~N(0,1) e4m3 sequence."""
    _require_device("t", t)
    _check(t.element_size() == 1 and t.is_contiguous(), "t must be a contiguous 1-byte tensor")
    with torch.cuda.device(t.device):
        capi.check(capi.load().moe_fill_normal_e4m3(_ptr(t), t.numel(), int(seed), int(stream_id), _stream(t.device)),
                   "moe_fill_normal_e4m3")
    return t


def host_normal_e4m3(n: int, seed: int, stream_id: int, first_index: int = 0, threads: int = 0) -> np.ndarray:
    """Elements [first_index, first_index+n) of the same sequence, on the CPU."""
    out = np.empty(n, dtype=np.uint8)
    if n:
        rc = capi.load().moe_host_fill_normal_e4m3(out.ctypes.data_as(ctypes.c_void_p), n, int(seed), int(stream_id),
                                                   int(first_index), int(threads))
        capi.check(rc, "moe_host_fill_normal_e4m3")
    return out
