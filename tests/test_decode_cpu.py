"""Argument checks of the one-kernel layer, which need no GPU."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

from nvshmem_testing_b200 import _native as N
from nvshmem_testing_b200 import decode


def args(T=4, H=64, E=4, K=2, F=32):
    bf = torch.bfloat16
    return dict(x=torch.zeros(T, H, dtype=bf), top_idxs=torch.zeros(T, K, dtype=torch.int64),
                top_vals=torch.zeros(T, K), w13=torch.zeros(E, H, 2 * F, dtype=bf), w2=torch.zeros(E, F, H, dtype=bf))


@pytest.mark.parametrize("change,error", [
    (dict(x=torch.zeros(4, 64)), TypeError),
    (dict(x=torch.zeros(4, 72, dtype=torch.bfloat16)), ValueError),
    (dict(x=torch.zeros(2, 2, 64, dtype=torch.bfloat16)), ValueError),
    (dict(w13=torch.zeros(4, 64, 63, dtype=torch.bfloat16)), ValueError),
    (dict(w2=torch.zeros(4, 64, 32, dtype=torch.bfloat16)), ValueError),
    (dict(w2=torch.zeros(3, 32, 64, dtype=torch.bfloat16)), ValueError),
    (dict(), ValueError),  # not on a GPU
])
def test_refusals(change, error):
    with pytest.raises(error):
        decode.moe_layer(**{**args(), **change})


def test_router_refusals():
    a = args()
    for bad in (torch.zeros(63, 8, dtype=torch.bfloat16), torch.zeros(64, 8)):
        with pytest.raises((ValueError, TypeError)):
            decode.routed_layer(a["x"], bad, 2, a["w13"], a["w2"])


def test_c_entry_refuses_before_any_device_call():
    lib = N.lib()
    assert lib.moe_decode_layer(None, None) == N.BAD_ARG
    need = ctypes.c_size_t()

    def scratch(*a):
        return lib.moe_decode_scratch_bytes(*a, ctypes.byref(need))

    #              T, H, F, E, K, Er, device
    assert scratch(65, 64, 64, 4, 2, 0, 0) == N.BAD_ARG
    assert scratch(-1, 64, 64, 4, 2, 0, 0) == N.BAD_ARG
    assert scratch(4, 60, 64, 4, 2, 0, 0) == N.BAD_ARG
    assert scratch(4, 64, 4, 4, 2, 0, 0) == N.BAD_ARG
    assert scratch(4, 64, 64, 0, 2, 0, 0) == N.BAD_ARG
    assert scratch(4, 64, 64, 1025, 2, 0, 0) == N.BAD_ARG
    assert scratch(64, 64, 64, 64, 17, 0, 0) == N.BAD_ARG  # 1088 rows
    assert scratch(4, 64, 64, 4, 33, 0, 0) == N.BAD_ARG
    assert scratch(4, 64, 64, 4, 3, 2, 0) == N.BAD_ARG     # K > router experts
    assert scratch(4, 64, 64, 4, 1, 6, 0) == N.BAD_ARG     # router experts not a multiple of 4
    p = N.DecodeParams()
    p.T, p.hidden, p.ffn, p.experts, p.K = 4, 64, 64, 4, 2
    assert lib.moe_decode_layer(ctypes.byref(p), None) == N.BAD_ARG  # null pointers
    buf = ctypes.create_string_buffer(64)
    at = (ctypes.addressof(buf) + 15) // 16 * 16
    for f in ("x", "w13", "w2", "y", "top_idxs", "top_vals", "scratch"):
        setattr(p, f, at)
    p.x = at + 2  # misaligned
    assert lib.moe_decode_layer(ctypes.byref(p), None) == N.BAD_ARG
    p.x, p.T = at, 0
    assert lib.moe_decode_layer(ctypes.byref(p), None) == N.OK  # nothing to do


def test_every_unit_belongs_to_one_part(tmp_path):
    """The kernel's division of its work, an empty rank's included, on the host."""
    exe = tmp_path / "check"
    here = Path(__file__).resolve().parent
    subprocess.run(["g++", "-std=c++17", "-O1", "-I", str(here.parent / "nvshmem_testing_b200" / "csrc"),
                    str(here / "native" / "decode_parts_check.cpp"), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, f"status {done.returncode}: {done.stdout}"


def test_c_entry_refuses_a_misaligned_router():
    buf = ctypes.create_string_buffer(64)
    at = (ctypes.addressof(buf) + 15) // 16 * 16
    p = N.DecodeParams()
    p.T, p.hidden, p.ffn, p.experts, p.K, p.router_experts = 4, 64, 64, 4, 2, 4
    for f in ("x", "w13", "w2", "y", "top_idxs", "top_vals", "scratch"):
        setattr(p, f, at)
    p.router_w = at + 2
    assert N.lib().moe_decode_layer(ctypes.byref(p), None) == N.BAD_ARG
