"""Expert products in 8-bit integers (8-bit weights, 8-bit activations).

The reference's expert product is bf16 (baseline.py:50).  Here rows are
quantised with one scale each and weights with one scale per output channel,

    x[r, k] ~ xs[r] * xq[r, k],      w[e, k, n] ~ ws[e, n] * wq[e, n, k]
    out[r, n] = xs[r] * ws[e, n] * sum_k xq[r, k] * wq[e, n, k]

with the integer sum exact.  Half the bytes of bf16 weights and twice the
tensor-core rate.

* ``quantize_weights`` — once, when a model is loaded;
* ``quantize_rows`` — rows of activations, optionally gathered by the
  dispatch permutation of ``utils.route`` on the way;
* ``grouped_gemm`` — one product per expert over rows in expert order, with
  SwiGLU in its epilogue on request; ``linear`` — the dense form from bf16;
* ``moe_layer`` — the gated layer on one rank's experts, the 8-bit sibling of
  ``combine.moe_layer`` over ``mlp``: route, gather and quantise, gate/up
  product with SwiGLU, quantise, down product, weighted sum per token (for a
  few tokens two launches, which route, quantise and add for themselves).

Nothing is read on the host and every call may be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes
import functools
from dataclasses import dataclass

import torch

from . import _native as N
from . import utils


@dataclass(frozen=True)
class QuantWeights:
    """``q [El, N, K]`` int8 (K contiguous) and ``scale [El, N]`` float32."""
    q: torch.Tensor
    scale: torch.Tensor


# Checks of shapes are remembered (a decode step repeats them); the error of a
# failed one is raised anew each time.
@functools.lru_cache(maxsize=512)
def _weights_dims(q, scale, name: str) -> tuple[int, int, int]:
    if len(q) != 3 or scale != q[:2]:
        raise ValueError(f"{name}: q [El, N, K] and scale [El, N] are required, got {tuple(q)} and {tuple(scale)}")
    return tuple(q)


def _check_weights(w: QuantWeights, name: str, device) -> tuple[int, int, int]:
    q, scale = w.q, w.scale
    dims = _weights_dims(q.shape, scale.shape, name)
    if q.dtype != torch.int8 or scale.dtype != torch.float32:
        raise TypeError(f"{name}: q must be int8 and scale float32")
    if not q.is_contiguous() or not scale.is_contiguous():
        raise ValueError(f"{name}: q and scale must be contiguous")
    if q.device != device or scale.device != device:
        raise ValueError(f"{name}: q and scale must be on {device}")
    return dims


def _check_product(K: int, Nw: int, El: int, swiglu: bool):
    if K % 16 or not 0 < K <= 131056:
        raise ValueError(f"K = {K} must be a multiple of 16, 131056 at most")
    if Nw % (16 if swiglu else 8) or Nw == 0:
        raise ValueError(f"{Nw} channels: a multiple of {16 if swiglu else 8} is needed")
    if not 1 <= El <= 1024:
        raise ValueError(f"{El} experts: 1 to 1024")


def _on_gpu(device, **tensors):
    if device.type != "cuda":
        raise ValueError(f"CUDA tensors are required, not {device}")
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} must be on {device}")


def _check_status(status):
    if status is not None and (status.dtype != torch.int32 or status.numel() != 1 or not status.is_pinned()):
        raise ValueError("status must be one pinned int32")


def quantize_rows(x: torch.Tensor, perm: torch.Tensor | None = None,
                  live_rows: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q [rows, K] int8, scale [rows] float32)`` of x [n, K], bf16 or fp32.

    scale = max|row| * (1/127) in fp32 and q the exact quotient, rounded half to
    even.  With ``perm`` [rows] int32, row r is x[perm[r]] (``Routing.perm``:
    the send buffer of ``utils.pack_compact``, quantised on the way); rows
    from ``live_rows`` (one int32 on the device, e.g. ``Routing.offsets[-1:]``)
    on are not written.  A row of zeros gets scale 0; a row that holds an
    infinity or a NaN gets a NaN scale and zeros."""
    if x.dim() != 2 or x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("x [n, K] in bfloat16 or float32 is required")
    K = x.shape[1]
    if K % 8 or K == 0:
        raise ValueError(f"K = {K} must be a positive multiple of 8")
    if perm is not None and (perm.dtype != torch.int32 or perm.dim() != 1 or not perm.is_contiguous()):
        raise TypeError("perm must be a contiguous int32 vector")
    if live_rows is not None and (live_rows.dtype != torch.int32 or live_rows.numel() != 1):
        raise TypeError("live_rows must be one int32")
    _on_gpu(x.device, perm=perm, live_rows=live_rows)
    rows = x.shape[0] if perm is None else perm.shape[0]
    x = x.contiguous()
    q = torch.empty((rows, K), dtype=torch.int8, device=x.device)
    scale = torch.empty(rows, dtype=torch.float32, device=x.device)
    with utils.on_device(x.device) as stream:
        N.check(N.lib().moe_quant_rows(x.data_ptr(), x.dtype == torch.float32, rows, K,
                                       None if perm is None else perm.data_ptr(),
                                       None if live_rows is None else live_rows.data_ptr(), q.data_ptr(),
                                       scale.data_ptr(), stream), "moe_quant_rows")
    return q, scale


def quantize_weights(w: torch.Tensor) -> QuantWeights:
    """[El, K, N] (bf16 or fp32) -> one scale per output channel, laid out with
    K contiguous.  One expert's transposed copy at a time."""
    if w.dim() != 3:
        raise ValueError("w [El, K, N] is required")
    El, K, Nout = w.shape
    _on_gpu(w.device)
    q = torch.empty((El, Nout, K), dtype=torch.int8, device=w.device)
    scale = torch.empty((El, Nout), dtype=torch.float32, device=w.device)
    for e in range(El):
        q[e], scale[e] = quantize_rows(w[e].t().contiguous())
    return QuantWeights(q, scale)


@functools.lru_cache(maxsize=256)
def _scratch_bytes(*sizes) -> int:
    need = ctypes.c_size_t()
    N.check(N.lib().moe_w8a8_scratch_bytes(*sizes, ctypes.byref(need)), "moe_w8a8_scratch_bytes")
    return need.value


def grouped_gemm(xq: torch.Tensor, xs: torch.Tensor, w: QuantWeights, counts: torch.Tensor | None = None, *,
                 swiglu: bool = False, out_dtype=torch.bfloat16, out: torch.Tensor | None = None,
                 status: torch.Tensor | None = None) -> torch.Tensor:
    """``out [rows, N]`` of one 8-bit product per expert.

    xq [rows, K] int8 and xs [rows] float32: rows in expert order, counts [El]
    int32 of them per expert, on the device (None: one expert for all).  K a
    multiple of 16.  With ``swiglu`` w's channels are gate [0, N/2) and up
    [N/2, N) and ``out [rows, N/2] = silu(gate) * up``.  Rows behind the last
    expert's are left as they were (``out`` supplies the buffer).
    ``out_dtype`` is bfloat16 or float32; ``status`` (one pinned int32)
    receives a device-side error word, if any."""
    El, Nw, K = _check_weights(w, "w", xq.device)
    if xq.dim() != 2 or xq.shape[1] != K or tuple(xs.shape) != (xq.shape[0],):
        raise ValueError(f"xq {tuple(xq.shape)} and xs {tuple(xs.shape)} do not match w {tuple(w.q.shape)}")
    if xq.dtype != torch.int8 or xs.dtype != torch.float32:
        raise TypeError("xq must be int8 and xs float32")
    _check_product(K, Nw, El, swiglu)
    if counts is None:
        if El != 1:
            raise ValueError("counts may be left out for one expert only")
    elif counts.dtype != torch.int32 or tuple(counts.shape) != (El,) or not counts.is_contiguous():
        raise ValueError(f"counts must be a contiguous int32 vector of {El}")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("out_dtype must be bfloat16 or float32")
    rows, cols = xq.shape[0], Nw // 2 if swiglu else Nw
    if out is None:
        out = torch.empty((rows, cols), dtype=out_dtype, device=xq.device)
    elif tuple(out.shape) != (rows, cols) or out.dtype != out_dtype or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous {out_dtype} tensor of shape {(rows, cols)}")
    _check_status(status)
    _on_gpu(xq.device, xs=xs, counts=counts, out=out)
    if rows == 0:
        return out
    with utils.on_device(xq.device) as stream:
        _gemm(xq.contiguous(), xs.contiguous(), None, w, counts, rows, K, Nw, El, swiglu, out, status, stream)
    return out


def _gemm(xq, xs, x, w, counts, rows, K, Nw, El, swiglu, out, status, stream):
    """The checked call, for quantised rows (xq, xs) or rows x that are still
    to be."""
    need = _scratch_bytes(rows, K, Nw, El, int(swiglu), int(x is not None), out.device.index)
    scratch = torch.empty(need, dtype=torch.uint8, device=out.device) if need else None
    p = N.W8A8Params(rows, K, Nw, El, swiglu, out.dtype == torch.float32, x is not None and x.dtype == torch.float32,
                     None if xq is None else xq.data_ptr(), None if xs is None else xs.data_ptr(), w.q.data_ptr(),
                     w.scale.data_ptr(), None if counts is None else counts.data_ptr(), out.data_ptr(),
                     None if scratch is None else scratch.data_ptr(), need,
                     None if status is None else status.data_ptr(), None if x is None else x.data_ptr(), None, None)
    N.check(N.lib().moe_w8a8_gemm(ctypes.byref(p), stream), "moe_w8a8_gemm")


def linear(x: torch.Tensor, w: QuantWeights, *, out_dtype=torch.bfloat16,
           status: torch.Tensor | None = None) -> torch.Tensor:
    """``x [rows, K] @ w`` for one weight matrix (w.q [1, N, K]): quantises the
    rows and multiplies.  ``status`` is grouped_gemm's."""
    El, Nw, K = _check_weights(w, "w", x.device)
    if El != 1:
        raise ValueError(f"one weight matrix [1, N, K] is required, got {tuple(w.q.shape)}")
    if x.dim() != 2 or x.shape[1] != K or x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"x [rows, {K}] in bfloat16 or float32 is required")
    _check_product(K, Nw, El, False)
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("out_dtype must be bfloat16 or float32")
    _check_status(status)
    _on_gpu(x.device)
    rows = x.shape[0]
    out = torch.empty((rows, Nw), dtype=out_dtype, device=x.device)
    if rows:
        with utils.on_device(x.device) as stream:
            _gemm(None, None, x.contiguous(), w, None, rows, K, Nw, 1, False, out, status, stream)
    return out


@functools.lru_cache(maxsize=512)
def _layer_dims(x, ids, vals, q13, q2) -> tuple[int, int]:
    """(T, ids per token)."""
    El, F2, H = q13
    F = F2 // 2
    if F2 % 2 or tuple(q2) != (El, H, F):
        raise ValueError(f"w13 {tuple(q13)} and w2 {tuple(q2)} do not form an MLP")
    if len(x) != 2 or x[1] != H:
        raise ValueError(f"x {tuple(x)} does not match w13 {tuple(q13)}")
    if H % 16 or F % 16:
        raise ValueError(f"H = {H} and F = {F} must be multiples of 16")
    _check_product(H, F2, El, True)
    _check_product(F, H, El, False)
    T = x[0]
    if len(ids) != 2 or ids[0] != T or vals != ids:
        raise ValueError(f"top_idxs {tuple(ids)} and top_vals {tuple(vals)} must be [T, K]")
    K = ids[1]
    if not 1 <= K <= 32:
        raise ValueError(f"{K} ids per token: 1 to 32")
    return T, K


@functools.lru_cache(maxsize=256)
def _layer_scratch_bytes(*sizes) -> int:
    need = ctypes.c_size_t()
    N.check(N.lib().moe_w8a8_layer_scratch_bytes(*sizes, ctypes.byref(need)), "moe_w8a8_layer_scratch_bytes")
    return need.value


def moe_layer(x: torch.Tensor, top_idxs: torch.Tensor, top_vals: torch.Tensor, w13: QuantWeights, w2: QuantWeights,
              *, first_expert: int = 0, status: torch.Tensor | None = None) -> torch.Tensor:
    """``y [T, H]`` bf16 of the gated layer on this rank's experts:

        y[t] = sum_k v[t, k] * down_e(silu(gate_e(x_t)) * up_e(x_t))

    with e = top_idxs[t, k] - first_expert; other ids are skipped and an id
    repeated within a row counts once, so that ranks holding parts of the
    experts add their y's.

    x [T, H] bf16, top_idxs [T, K] int32/int64, top_vals [T, K] float32 or
    bfloat16; w13.q [El, 2F, H] (gate channels [0, F), up after them) and w2.q
    [El, H, F].  H and F multiples of 16.  ``status`` is grouped_gemm's."""
    dev = x.device
    El, F2, H = _check_weights(w13, "w13", dev)
    _check_weights(w2, "w2", dev)
    F = F2 // 2
    if top_idxs.dim() == 1:
        top_idxs = top_idxs[:, None]
    if top_vals.dim() == 1:
        top_vals = top_vals[:, None]
    T, K = _layer_dims(x.shape, top_idxs.shape, top_vals.shape, w13.q.shape, w2.q.shape)
    if x.dtype != torch.bfloat16:
        raise TypeError("x must be bfloat16")
    if top_idxs.dtype not in (torch.int32, torch.int64):
        raise TypeError("top_idxs must be int32 or int64")
    if top_vals.dtype not in (torch.float32, torch.bfloat16):
        raise TypeError("top_vals must be float32 or bfloat16")
    _check_status(status)
    if not 0 <= first_expert < 1 << 31:
        raise ValueError(f"first_expert = {first_expert} must be an expert's id")
    _on_gpu(dev, top_idxs=top_idxs, top_vals=top_vals)
    y = torch.empty((T, H), dtype=torch.bfloat16, device=x.device)
    if T == 0:
        return y
    ids, vals = top_idxs.contiguous(), top_vals.contiguous()
    x = x.contiguous()
    need = _layer_scratch_bytes(T, H, F, El, K, dev.index)
    scratch = torch.empty(need, dtype=torch.uint8, device=dev)
    p = N.W8A8LayerParams(T, H, F, El, K, first_expert, ids.dtype == torch.int64, vals.dtype == torch.bfloat16, 0,
                          x.data_ptr(), w13.q.data_ptr(), w13.scale.data_ptr(), w2.q.data_ptr(),
                          w2.scale.data_ptr(), ids.data_ptr(), vals.data_ptr(), y.data_ptr(), scratch.data_ptr(),
                          need, None if status is None else status.data_ptr())
    with utils.on_device(dev) as stream:
        N.check(N.lib().moe_w8a8_layer(ctypes.byref(p), stream), "moe_w8a8_layer")
    return y
