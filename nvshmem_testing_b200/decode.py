"""The gated MoE layer for a few tokens, in one kernel.

``combine.moe_layer`` and ``mlp.moe_mlp`` route, pack, exchange and multiply
in separate launches and read the largest bucket on the host; with a handful
of tokens (a decode step) their fixed costs and padded tiles outweigh the
work, which is one pass over the weights of the experts that were chosen.
``moe_layer`` is that pass for tokens whose routing is known, and
``routed_layer`` includes the router (reference: utils.py:17-25 for the
router, utils.py:28-75 and baseline.py:18-50 for routing and products).

    y[t] = sum_k v[t, k] * (silu(x_t W_gate,e) * (x_t W_up,e)) W_down,e

with e = ids[t, k] - first_expert.  Ids outside the experts held here are
skipped and a token without any gets a zero row: a rank that holds experts
[first_expert, first_expert + El) of a replicated batch computes its part of
the sum, and the ranks' parts add up.  Sums are fp32, silu(gate) * up keeps 16
bits between the products, and y is rounded once.  Nothing is read on the
host, and a call may be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from . import _native as N
from . import utils


@functools.lru_cache(maxsize=512)  # a decode step repeats its shapes
def _dims(x, w13, w2) -> tuple[int, int, int, int]:
    if len(x) != 2 or len(w13) != 3 or len(w2) != 3:
        raise ValueError("x [T, H], w13 [El, H, 2F] and w2 [El, F, H] are required")
    T, H = x
    El, F2 = w13[0], w13[2]
    F = F2 // 2
    if w13[1] != H or F2 % 2 or tuple(w2) != (El, F, H):
        raise ValueError(f"x {tuple(x)}, w13 {tuple(w13)} and w2 {tuple(w2)} do not form an MLP")
    if H % 8 or F % 8 or not 0 < H <= 32768 or F == 0:
        raise ValueError(f"H = {H} and F = {F} must be positive multiples of 8, H 32768 at most")
    if not 1 <= El <= 1024:
        raise ValueError(f"{El} experts: 1 to 1024")
    if T > N.DECODE_MAX_TOKENS:
        raise ValueError(f"{T} tokens: this form takes {N.DECODE_MAX_TOKENS} at most (mlp.moe_mlp has no limit)")
    return T, H, F, El


def _check(x, w13, w2, first_expert, out, status):
    dims = _dims(x.shape, w13.shape, w2.shape)
    if not (x.dtype == w13.dtype == w2.dtype == torch.bfloat16):
        raise TypeError("x, w13 and w2 must be bfloat16")
    if not x.is_cuda or w13.device != x.device or w2.device != x.device:
        raise ValueError("x, w13 and w2 must be CUDA tensors on one device")
    if not w13.is_contiguous() or not w2.is_contiguous():
        raise ValueError("w13 and w2 must be contiguous")
    if out is not None and (out.shape != x.shape or out.dtype != torch.bfloat16 or out.device != x.device
                            or not out.is_contiguous()):
        raise ValueError(f"out must be a contiguous bfloat16 tensor of shape {tuple(x.shape)} on the tokens' device")
    if not 0 <= first_expert < 1 << 31:
        raise ValueError(f"first_expert = {first_expert} must be an expert's id")
    if status is not None and (status.dtype != torch.int32 or status.numel() != 1 or not status.is_pinned()):
        raise ValueError("status must be one pinned int32")
    return dims


@functools.lru_cache(maxsize=256)
def _scratch_bytes(*sizes) -> int:
    need = ctypes.c_size_t()
    N.check(N.lib().moe_decode_scratch_bytes(*sizes, ctypes.byref(need)), "moe_decode_scratch_bytes")
    return need.value


def _launch(x, ids, vals, w13, w2, router_w, K, first_expert, renormalize, out, status, dims):
    T, H, F, El = dims
    if out is None:
        out = torch.empty((T, H), dtype=torch.bfloat16, device=x.device)
    if T == 0:
        return out
    Er = 0 if router_w is None else router_w.shape[1]
    need = _scratch_bytes(T, H, F, El, K, Er, x.device.index)
    scratch = torch.empty(need, dtype=torch.uint8, device=x.device)
    p = N.DecodeParams(T, H, F, El, K, first_expert, Er, renormalize, ids.dtype == torch.int64,
                       vals.dtype == torch.bfloat16, 0, x.data_ptr(), w13.data_ptr(), w2.data_ptr(),
                       None if router_w is None else router_w.data_ptr(), ids.data_ptr(), vals.data_ptr(),
                       out.data_ptr(), scratch.data_ptr(), need, None if status is None else status.data_ptr())
    with utils.on_device(x.device) as stream:
        N.check(N.lib().moe_decode_layer(ctypes.byref(p), stream), "moe_decode_layer")
    return out


def moe_layer(x: torch.Tensor, top_idxs: torch.Tensor, top_vals: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor,
              *, first_expert: int = 0, out: torch.Tensor | None = None,
              status: torch.Tensor | None = None) -> torch.Tensor:
    """``y [T, H]`` bf16 for tokens whose routing is known.

    x         [T, H] bf16, T <= 64
    top_idxs  [T, K] int32/int64 expert ids, T * K <= 1024, K <= 32
    top_vals  [T, K] float32 or bfloat16 routing weights
    w13       [El, H, 2F] bf16: gate columns [0, F), up columns [F, 2F)
    w2        [El, F, H] bf16
    first_expert: id of the first expert held here.  ``out`` optionally
    supplies y; ``status`` (one pinned int32) receives a device-side error
    word, if any."""
    dims = _check(x, w13, w2, first_expert, out, status)
    if top_idxs.dim() == 1:
        top_idxs = top_idxs[:, None]
    if top_vals.dim() == 1:
        top_vals = top_vals[:, None]
    if top_idxs.dim() != 2 or top_idxs.shape[0] != dims[0] or top_vals.shape != top_idxs.shape:
        raise ValueError(f"top_idxs {tuple(top_idxs.shape)} and top_vals {tuple(top_vals.shape)} must be [T, K]")
    if top_idxs.dtype not in (torch.int32, torch.int64):
        raise TypeError("top_idxs must be int32 or int64")
    if top_vals.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("top_vals must be float32 or bfloat16")
    if top_idxs.device != x.device or top_vals.device != x.device:
        raise ValueError("top_idxs and top_vals must be on the tokens' device")
    K = top_idxs.shape[1]
    if not 1 <= K <= 32 or dims[0] * K > N.DECODE_MAX_ROWS:
        raise ValueError(f"{dims[0]} tokens with {K} ids each: 1 to 32 ids, {N.DECODE_MAX_ROWS} in all at most")
    return _launch(x.contiguous(), top_idxs.contiguous(), top_vals.contiguous(), w13, w2, None, K, int(first_expert),
                   False, out, status, dims)


def routed_layer(x: torch.Tensor, router_w: torch.Tensor, topk: int, w13: torch.Tensor, w2: torch.Tensor, *,
                 renormalize: bool = False, first_expert: int = 0, ids_dtype=torch.int64,
                 out: torch.Tensor | None = None,
                 status: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The whole layer from activations: ``(y [T, H], top_vals [T, K] float32,
    top_idxs [T, K])``.

    router_w [H, E] bf16.  The logits ``x @ router_w`` stay in fp32 (unlike
    ``utils.router``, which rounds logits and probabilities to bf16 as the
    reference does), top_vals are the K largest of their softmax in
    descending order, equal ones by ascending id, divided by their sum with
    ``renormalize``.  The other arguments are those of ``moe_layer``; w13 and
    w2 may hold a part of the E experts."""
    dims = _check(x, w13, w2, first_expert, out, status)
    T, H = dims[0], dims[1]
    if router_w.dim() != 2 or router_w.shape[0] != H:
        raise ValueError(f"router_w {tuple(router_w.shape)} does not match x {tuple(x.shape)}")
    if router_w.dtype != torch.bfloat16:
        raise TypeError("router_w must be bfloat16")
    if router_w.device != x.device:
        raise ValueError("router_w must be on the tokens' device")
    if ids_dtype not in (torch.int32, torch.int64):
        raise TypeError("ids_dtype must be int32 or int64")
    E = router_w.shape[1]
    if E % 4 or not 4 <= E <= 1024:
        raise ValueError(f"{E} experts: a multiple of 4, 1024 at most")
    if not 1 <= topk <= min(32, E) or T * topk > N.DECODE_MAX_ROWS:
        raise ValueError(f"{T} tokens with {topk} of {E} experts each: 1 to 32, {N.DECODE_MAX_ROWS} in all at most")
    vals = torch.empty((T, topk), dtype=torch.float32, device=x.device)
    ids = torch.empty((T, topk), dtype=ids_dtype, device=x.device)
    y = _launch(x.contiguous(), ids, vals, w13, w2, router_w.contiguous(), topk, int(first_expert), renormalize, out,
                status, dims)
    return y, vals, ids
