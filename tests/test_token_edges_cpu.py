"""Refusals of the token operators' C entries at the ends of their ranges, and what their Python side does without a GPU (nothing is launched)."""
import ctypes
import subprocess
import sys

import pytest

from diffusionmodelscustom_amd import hip_engine
from tests.test_token_ops_cpu import EINVAL, attention


@pytest.mark.parametrize("dtype,head_dim,rows", [(1, 32, 64), (2, 128, 64), (0, 64, 64), (0, 128, 32)])
@pytest.mark.parametrize("group", [1, 2, 3, 7])
def test_attention_backward_refuses_tiles_of_rows_past_32_bit_offsets(dtype, head_dim, rows, group):
    """a tile is `rows` (token, head) rows: with few heads to a key head the more tokens; past 2^31 bytes they would read as zero"""
    lib = hip_engine.load_library()
    p, size = ctypes.c_void_p(16), 4 if dtype == 0 else 2
    spanned = -(-(rows - 1) // group)                       # the last row's token, where the tile starts with a token's first head
    step = -(-(1 << 31) // (spanned * size * 8)) * 8        # that many tokens further: 2^31 bytes and a little
    near = dict(k_stride=(1 << 20, head_dim, head_dim), v_stride=(1 << 20, head_dim, head_dim), dout_stride=(1 << 20, group * head_dim, head_dim),
                q_stride=(1 << 20, group * head_dim, head_dim))
    for far in ("q_stride", "dout_stride"):
        d = attention(**{**dict(dtype=dtype, batch=1, heads=group, kv_heads=1, head_dim=head_dim, q_len=100, kv_len=100), **near, far: (1 << 40, step, head_dim)})
        assert lib.danra_token_attention_bwd(ctypes.byref(d), *[p] * 11, None) == EINVAL
        assert b"2^31" in lib.danra_last_error()


@pytest.mark.parametrize("sizes", [dict(q_len=1, kv_len=(1 << 31) - 60), dict(q_len=(1 << 31) - 60, kv_len=0), dict(q_len=(1 << 30) - 60, kv_len=1, heads=2, kv_heads=1)])
def test_attention_refuses_lengths_whose_last_tile_passes_31_bits(sizes):
    """places are counted up to the end of the last tile of up to 256 rows or keys, with 32-bit integers"""
    lib = hip_engine.load_library()
    d, p = attention(**{**dict(batch=1, heads=1, kv_heads=1, head_dim=8, q_docs=16, k_docs=16), **sizes}), ctypes.c_void_p(16)
    assert lib.danra_token_attention_fwd_workspace(ctypes.byref(d)) == 0 and lib.danra_token_attention_bwd_workspace(ctypes.byref(d)) == 0
    assert lib.danra_token_attention_fwd(ctypes.byref(d), p, p, p, p, None, None, p, None) == EINVAL
    assert lib.danra_token_attention_bwd(ctypes.byref(d), *[p] * 11, None) == EINVAL


def test_imports_in_a_torch_without_gpu_bindings():
    """a torch that is built without a GPU lacks the bindings that only the calls need"""
    code = ("import torch\nfor n in ('_cuda_getCurrentRawStream', '_cuda_getDevice'):\n    if hasattr(torch._C, n): delattr(torch._C, n)\n"
            "import diffusionmodelscustom_amd.training, diffusionmodelscustom_amd.token_ops\n")
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr


@pytest.mark.parametrize("scale", [1e38, -3e38])
def test_attention_refuses_scales_that_leave_float32_in_units_of_log2(scale):
    lib = hip_engine.load_library()
    d, p = attention(scale=scale), ctypes.c_void_p(16)
    assert lib.danra_token_attention_fwd(ctypes.byref(d), p, p, p, p, None, None, p, None) == EINVAL
    assert lib.danra_token_attention_bwd(ctypes.byref(d), *[p] * 11, None) == EINVAL
