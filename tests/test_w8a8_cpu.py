"""Argument checks of the 8-bit operators, which need no GPU."""
import ctypes

import pytest
import torch

from nvshmem_testing_b200 import _native as N
from nvshmem_testing_b200 import w8a8


def weights(E=2, Nn=32, K=64, q=torch.int8, s=torch.float32):
    return w8a8.QuantWeights(torch.zeros(E, Nn, K, dtype=q), torch.zeros(E, Nn, dtype=s))


def rows(n=3, K=64):
    return torch.zeros(n, K, dtype=torch.int8), torch.zeros(n)


C = torch.zeros(2, dtype=torch.int32)


@pytest.mark.parametrize("call,error", [
    (lambda: w8a8.quantize_rows(torch.zeros(2, 64, dtype=torch.float16)), TypeError),
    (lambda: w8a8.quantize_rows(torch.zeros(2, 60)), ValueError),
    (lambda: w8a8.quantize_rows(torch.zeros(2, 64), perm=torch.zeros(4, dtype=torch.int64)), TypeError),
    (lambda: w8a8.quantize_rows(torch.zeros(2, 64), live_rows=torch.zeros(2, dtype=torch.int32)), TypeError),
    (lambda: w8a8.quantize_rows(torch.zeros(2, 64)), ValueError),  # not on a GPU
    (lambda: w8a8.quantize_weights(torch.zeros(4, 4)), ValueError),
    (lambda: w8a8.grouped_gemm(*rows(K=48), weights(), C), ValueError),
    (lambda: w8a8.grouped_gemm(*rows(K=72), weights(K=72), C), ValueError),
    (lambda: w8a8.grouped_gemm(*rows(), weights(Nn=36), C), ValueError),
    (lambda: w8a8.grouped_gemm(*rows(), weights(Nn=24), C, swiglu=True), ValueError),
    (lambda: w8a8.grouped_gemm(*rows(), weights()), ValueError),  # two experts without counts
    (lambda: w8a8.grouped_gemm(*rows(), weights(), C.long()), ValueError),
    (lambda: w8a8.grouped_gemm(*rows(), weights(q=torch.uint8), C), TypeError),
    (lambda: w8a8.grouped_gemm(*rows(), weights(s=torch.float64), C), TypeError),
    (lambda: w8a8.grouped_gemm(*rows(), weights(), C, out_dtype=torch.float16), TypeError),
    (lambda: w8a8.grouped_gemm(*rows(), weights(), C, out=torch.zeros(3, 16, dtype=torch.bfloat16)), ValueError),
    (lambda: w8a8.grouped_gemm(*rows(), weights(), C), ValueError),  # not on a GPU
    (lambda: w8a8.linear(torch.zeros(2, 64), weights()), ValueError),
    (lambda: w8a8.moe_layer(torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, 1, dtype=torch.int64),
                            torch.zeros(2, 1), weights(Nn=32), weights(Nn=64, K=32)), ValueError),
    (lambda: w8a8.moe_layer(torch.zeros(2, 64), torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1),
                            weights(Nn=32), weights(Nn=64, K=16)), TypeError),
])
def test_refusals(call, error):
    with pytest.raises(error):
        call()


def test_c_entries_refuse_before_any_device_call():
    lib = N.lib()
    assert lib.moe_w8a8_gemm(None, None) == N.BAD_ARG
    need = ctypes.c_size_t()

    def scratch(*a):
        return lib.moe_w8a8_scratch_bytes(*a, ctypes.byref(need))

    #              rows, K, N, E, swiglu, with_x, device
    assert scratch(-1, 64, 64, 1, 0, 0, 0) == N.BAD_ARG
    assert scratch(4, 60, 64, 1, 0, 0, 0) == N.BAD_ARG
    assert scratch(4, 131072, 64, 1, 0, 0, 0) == N.BAD_ARG
    assert scratch(4, 64, 60, 1, 0, 0, 0) == N.BAD_ARG
    assert scratch(4, 64, 24, 1, 1, 0, 0) == N.BAD_ARG
    assert scratch(4, 64, 64, 1025, 0, 0, 0) == N.BAD_ARG
    p = N.W8A8Params()
    p.rows, p.K, p.N, p.experts = 4, 64, 64, 2
    assert lib.moe_w8a8_gemm(ctypes.byref(p), None) == N.BAD_ARG  # null pointers
    p.rows = 0
    assert lib.moe_w8a8_gemm(ctypes.byref(p), None) == N.OK
    assert lib.moe_quant_rows(None, 0, 4, 64, None, None, None, None, None) == N.BAD_ARG
    assert lib.moe_quant_rows(None, 0, 4, 63, None, None, None, None, None) == N.BAD_ARG
    assert lib.moe_quant_rows(None, 0, 0, 64, None, None, None, None, None) == N.OK
    assert lib.moe_weighted_sum(None, 0, None, 1, 0, None, 0, None, None, 4, 2, 64, 2, None, None) == N.BAD_ARG
    assert lib.moe_weighted_sum(None, 0, None, 1, 0, None, 0, None, None, 4, 33, 64, 2, None, None) == N.BAD_ARG
    assert lib.moe_weighted_sum(None, 0, None, 1, 0, None, 0, None, None, 0, 2, 64, 2, None, None) == N.OK


def test_c_entries_refuse_scales_that_are_no_floats():
    buf = ctypes.create_string_buffer(64)
    at = (ctypes.addressof(buf) + 15) // 16 * 16
    lib = N.lib()
    for bad in ("xs", "ws"):
        p = N.W8A8Params()
        p.rows, p.K, p.N, p.experts = 4, 64, 64, 1
        for f in ("xq", "xs", "wq", "ws", "out", "scratch"):
            setattr(p, f, at + 2 * (f == bad))
        assert lib.moe_w8a8_gemm(ctypes.byref(p), None) == N.BAD_ARG
    for bad in ("w13_scale", "w2_scale"):
        p = N.W8A8LayerParams()
        p.T, p.hidden, p.ffn, p.experts, p.K = 4, 64, 64, 2, 1
        for f in ("x", "w13", "w13_scale", "w2", "w2_scale", "top_idxs", "top_vals", "y", "scratch"):
            setattr(p, f, at + 2 * (f == bad))
        assert lib.moe_w8a8_layer(ctypes.byref(p), None) == N.BAD_ARG


@pytest.mark.parametrize("status", [torch.zeros(1), torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)])
def test_every_product_takes_a_pinned_status_word(status):
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    for call in (lambda: w8a8.linear(x, weights(E=1), status=status),
                 lambda: w8a8.grouped_gemm(*rows(), weights(), C, status=status),
                 lambda: w8a8.moe_layer(x, torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1), weights(Nn=32),
                                        weights(Nn=64, K=16), status=status)):
        with pytest.raises(ValueError, match="status"):
            call()
