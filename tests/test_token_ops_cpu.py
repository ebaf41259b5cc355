"""Refusals and workspaces of the token operators at the C entries (no GPU: nothing is launched), and the float64 definitions that the
GPU tests hold the kernels to, against autograd."""
import ctypes
import math

import pytest
import torch

from diffusionmodelscustom_amd import hip_engine
from tests.token_util import attention_reference, rotary_reference

EINVAL = -1


def attention(**kw):
    d = hip_engine.TokenAttention()
    given = dict(dtype=1, batch=2, q_len=8, kv_len=16, heads=4, kv_heads=2, head_dim=32, scale=0.2, softcap=0.0,
                 q_stride=(1024, 128, 32), k_stride=(1024, 64, 32), v_stride=(1024, 64, 32), dout_stride=(1024, 128, 32))
    given.update(kw)
    for n, v in given.items():
        if n.endswith("_stride"):
            at = 3 * ("q_stride", "k_stride", "v_stride", "dout_stride").index(n)
            d.strides[at:at + 3] = v
        else:
            setattr(d, n, v)
    return d


def rotary(**kw):
    d = hip_engine.QkNormRotary()
    given = dict(dtype=1, weight_dtype=1, batch=2, length=8, q_heads=4, k_heads=2, head_dim=32, rotated=32, table=8, eps=1e-6, cos=16, sin=16)
    given.update(kw)
    for n, v in given.items():
        setattr(d, n, v)
    return d


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(dtype=-1), dict(batch=-1), dict(q_len=-1), dict(kv_len=-1), dict(heads=0), dict(kv_heads=0), dict(heads=3),
                                 dict(head_dim=0), dict(head_dim=12), dict(head_dim=136), dict(scale=math.inf), dict(scale=math.nan), dict(softcap=-1.0),
                                 dict(softcap=math.inf), dict(prefix=16), dict(q_docs=16), dict(k_docs=16), dict(q_len=1 << 30, kv_len=1 << 30),
                                 dict(batch=1 << 20, heads=1 << 14, kv_heads=1 << 14)])
def test_attention_descriptions_refused(bad):
    lib = hip_engine.load_library()
    d = attention(**bad)
    p = ctypes.c_void_p(16)
    assert lib.danra_token_attention_fwd_workspace(ctypes.byref(d)) == 0
    assert lib.danra_token_attention_bwd_workspace(ctypes.byref(d)) == 0
    assert lib.danra_token_attention_fwd(ctypes.byref(d), p, p, p, p, None, None, p, None) == EINVAL
    assert lib.danra_token_attention_bwd(ctypes.byref(d), *[p] * 11, None) == EINVAL
    assert lib.danra_last_error()


def test_attention_pointers_refused():
    lib = hip_engine.load_library()
    d = attention()
    p, odd = ctypes.c_void_p(16), ctypes.c_void_p(24)
    for args in ((None, p, p, p), (p, None, p, p), (p, p, None, p), (p, p, p, None), (odd, p, p, p), (p, odd, p, p), (p, p, odd, p), (p, p, p, odd)):
        assert lib.danra_token_attention_fwd(ctypes.byref(d), *args, None, None, p, None) == EINVAL
    for bad in (dict(q_stride=(4, 128, 32)), dict(k_stride=(1024, 68, 32)), dict(v_stride=(1024, 64, 33)), dict(k_stride=(1024, 24, 32)), dict(v_stride=(1024, 0, 32)),
                dict(k_stride=(1024, 1 << 23, 32)), dict(v_stride=(1024, -64, 32))):
        assert lib.danra_token_attention_fwd(ctypes.byref(attention(**bad)), p, p, p, p, None, None, p, None) == EINVAL
    assert lib.danra_token_attention_fwd(None, p, p, p, p, None, None, p, None) == EINVAL
    docs = attention(q_docs=16, k_docs=16)
    assert lib.danra_token_attention_fwd_workspace(ctypes.byref(docs)) > 0
    assert lib.danra_token_attention_fwd(ctypes.byref(docs), p, p, p, p, None, None, None, None) == EINVAL
    for n in range(11):   # q, k, v, out, out_rest, dout, stats, dq, dk, dv, workspace
        args = [p] * 11
        args[n] = ctypes.c_void_p(20)
        assert lib.danra_token_attention_bwd(ctypes.byref(d), *args, None) == EINVAL, n
        args[n] = None
        if n not in (4, 7):   # (out_rest and dq alone may be left out)
            assert lib.danra_token_attention_bwd(ctypes.byref(d), *args, None) == EINVAL, n
    for bad in (dict(dout_stride=(1024, 128, 4)), dict(q_stride=(1024, 1 << 25, 32)), dict(dout_stride=(1024, 128, 1 << 30)), dict(q_stride=(1024, -128, 32)),
                dict(k_stride=(1024, 0, 32))):
        assert lib.danra_token_attention_bwd(ctypes.byref(attention(**bad)), *[p] * 11, None) == EINVAL, bad


def test_attention_without_work_touches_nothing():
    lib = hip_engine.load_library()
    for empty in (dict(batch=0), dict(q_len=0), dict(batch=0, q_len=0, kv_len=0)):
        d = attention(**empty)
        lib.danra_token_attention_fwd_workspace(ctypes.byref(d))
        lib.danra_token_attention_bwd_workspace(ctypes.byref(d))
        assert lib.danra_token_attention_fwd(ctypes.byref(d), *[None] * 8) == 0
    d = attention(batch=0)
    assert lib.danra_token_attention_bwd(ctypes.byref(d), *[None] * 12) == 0


def test_attention_workspace_covers_the_longest_split():
    """as many bytes as the kernels of the call index: partial sums and {maximum, sum} of each split, 16 bytes per 32 keys of documents"""
    lib = hip_engine.load_library()
    d = attention(batch=1, q_len=1, kv_len=1 << 20, heads=8, kv_heads=2, head_dim=128)
    size = lib.danra_token_attention_fwd_workspace(ctypes.byref(d))
    assert size % (8 * (128 * 4 + 16)) == 0 and 2 <= size // (8 * (128 * 4 + 16)) <= 128
    d.q_docs = d.k_docs = 16
    assert lib.danra_token_attention_fwd_workspace(ctypes.byref(d)) == size + (1 << 20) // 32 * 16
    assert lib.danra_token_attention_bwd_workspace(ctypes.byref(d)) >= (1 << 20) // 32 * 16 + 1024 + 2 * 16


@pytest.mark.parametrize("bad", [dict(dtype=5), dict(weight_dtype=2), dict(batch=-1), dict(length=-1), dict(q_heads=0),
                                 dict(k_heads=0), dict(q_heads=65535, k_heads=1), dict(head_dim=20), dict(head_dim=256),
                                 dict(rotated=0), dict(rotated=3), dict(rotated=34), dict(cos=None), dict(sin=None), dict(table=0), dict(table=7), dict(eps=-1.0),
                                 dict(eps=math.nan), dict(batch=1 << 20, length=1 << 20)])
def test_rotary_descriptions_refused(bad):
    lib = hip_engine.load_library()
    d, p = rotary(**bad), ctypes.c_void_p(16)
    assert lib.danra_qk_norm_rotary_fwd(ctypes.byref(d), *[p] * 6, None) == EINVAL
    assert lib.danra_qk_norm_rotary_bwd(ctypes.byref(d), *[p] * 11, None) == EINVAL
    assert lib.danra_qk_norm_rotary_bwd_workspace(ctypes.byref(d)) == 0


def test_rotary_pointers_refused():
    lib = hip_engine.load_library()
    d, p, odd = rotary(), ctypes.c_void_p(16), ctypes.c_void_p(18)
    for n in (0, 1, 4, 5):   # q, k, weights (may be left out), results
        for value in (None, odd):
            args = [p] * 6
            args[n] = value
            assert lib.danra_qk_norm_rotary_fwd(ctypes.byref(d), *args, None) == EINVAL
    for n in (0, 1, 4, 5, 6, 7, 10):
        for value in (None, odd):
            args = [p] * 11
            args[n] = value
            assert lib.danra_qk_norm_rotary_bwd(ctypes.byref(d), *args, None) == EINVAL
    d.batch = 0
    assert lib.danra_qk_norm_rotary_fwd(ctypes.byref(d), *[None] * 7) == 0


def test_clip_refused():
    lib = hip_engine.load_library()
    p = ctypes.c_void_p(16)

    def call(pointer=16, out=16, numel=5, kind=0, out_kind=0, count=1, limit=1.0, eps=1e-6, norm=p, workspace=p):
        return lib.danra_clip_gradients((ctypes.c_void_p * 1)(pointer), (ctypes.c_void_p * 1)(out), (ctypes.c_size_t * 1)(numel), (ctypes.c_int * 1)(kind),
                                        (ctypes.c_int * 1)(out_kind), count, limit, eps, norm, workspace, None)
    for bad in (dict(pointer=None), dict(out=None), dict(kind=3), dict(kind=-1), dict(out_kind=7), dict(out_kind=1), dict(count=-1), dict(limit=-1.0), dict(limit=math.nan),
                dict(eps=-1.0), dict(norm=None), dict(workspace=None), dict(workspace=ctypes.c_void_p(20)), dict(numel=1 << 41)):
        assert call(**bad) == EINVAL, bad
    assert lib.danra_clip_gradients(None, None, None, None, None, 1, 1.0, 0.0, p, p, None) == EINVAL

    def two(pointers, outs, numel=(8, 8), kinds=(0, 0), out_kinds=(0, 0)):
        return lib.danra_clip_gradients((ctypes.c_void_p * 2)(*pointers), (ctypes.c_void_p * 2)(*outs), (ctypes.c_size_t * 2)(*numel), (ctypes.c_int * 2)(*kinds),
                                        (ctypes.c_int * 2)(*out_kinds), 2, 1.0, 1e-6, p, p, None)
    assert two((64, 64), (64, 64)) == EINVAL             # the same tensor twice, in place
    assert two((64, 80), (64, 80)) == EINVAL             # parts of one memory, in place
    assert two((64, 96), (96, 64)) == EINVAL             # each into the other
    assert two((64, 512), (128, 144)) == EINVAL          # overlapping results
    assert two((64, 512), (72, 1024), kinds=(1, 0)) == EINVAL and b"overlaps" in lib.danra_last_error()   # into its own end
    assert lib.danra_clip_gradients_workspace(-1) == 0 and lib.danra_clip_gradients_workspace(5000) >= 8 * 2048


def test_attention_definition_against_autograd():
    g = torch.Generator().manual_seed(0)
    B, Lq, Lk, H, Hk, D = 2, 7, 11, 4, 2, 8
    q, k, v, dout = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((B, Lq, H, D), (B, Lk, Hk, D), (B, Lk, Hk, D), (B, Lq, H, D)))
    slopes, prefix, lens = torch.rand(H, generator=g), torch.tensor([0, 6]), torch.tensor([11, 9])
    qd, kd = torch.randint(-1, 2, (B, Lq), generator=g), torch.randint(-1, 2, (B, Lk), generator=g)
    xs = [t.clone().requires_grad_(True) for t in (q, k, v)]
    outs = []
    for b in range(B):
        for i in range(Lq):
            pos = i + int(lens[b]) - Lq
            seen = [j for j in range(int(lens[b])) if (j <= pos or j < int(prefix[b])) and qd[b, i] == kd[b, j] and qd[b, i] >= 0]
            for h in range(H):
                if not seen:
                    outs.append(xs[0].new_zeros(D))
                    continue
                s = torch.stack([3.0 * torch.tanh(0.7 * xs[0][b, i, h].dot(xs[1][b, j, h // 2]) / 3.0) - slopes[h].double() * abs(pos - j) for j in seen])
                outs.append(s.softmax(0) @ torch.stack([xs[2][b, j, h // 2] for j in seen]))
    out = torch.stack(outs).view(B, Lq, H, D)
    want = [out.detach(), *torch.autograd.grad(out, xs, dout)]

    got, _ = attention_reference(q, k, v, dout, scale=0.7, softcap=3.0, slopes=slopes, causal=True, prefix=prefix, kv_lens=lens, q_docs=qd, k_docs=kd)
    assert all(torch.allclose(a, b, rtol=1e-10, atol=1e-12) for a, b in zip(got, want))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_definition_against_autograd(interleaved):
    g = torch.Generator().manual_seed(1)
    q, k, dq, dk = (torch.randn(2, 5, h, 16, generator=g, dtype=torch.float64) for h in (3, 1, 3, 1))
    qw, kw = (1 + torch.randn(16, generator=g, dtype=torch.float64) for _ in range(2))
    from diffusionmodelscustom_amd.token_ops import rotary_tables
    cos, sin = rotary_tables(5, 12)
    angle = torch.arange(5, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(6, dtype=torch.float64) / 6)
    assert torch.equal(cos, angle.cos().float()) and torch.equal(sin, angle.sin().float())
    want, grads = [], []
    for x, w, dy in ((q, qw, dq), (k, kw, dk)):
        x, w = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        y = x / (x.square().mean(-1, keepdim=True) + 1e-4).sqrt() * w
        pairs = [(2 * p, 2 * p + 1) if interleaved else (p, 6 + p) for p in range(6)]
        cols = list(y.unbind(-1))
        for p, (a, b) in enumerate(pairs):
            c, s = cos[:, p, None].double(), sin[:, p, None].double()
            cols[a], cols[b] = cols[a] * c - cols[b] * s, cols[b] * c + cols[a] * s
        y = torch.stack(cols, -1)
        want.append(y.detach())
        grads.append(torch.autograd.grad(y, (x, w), dy))
    want += [grads[0][0], grads[1][0], grads[0][1], grads[1][1]]
    got, _ = rotary_reference(q, k, qw, kw, cos, sin, None, 1e-4, interleaved, dq, dk)
    assert all(torch.allclose(a, b, rtol=1e-10, atol=1e-12) for a, b in zip(got, want))


def test_token_operators_refuse_cpu_tensors():
    from diffusionmodelscustom_amd import token_ops
    x = torch.zeros(1, 2, 1, 8)
    with pytest.raises(RuntimeError):
        token_ops.token_attention(x, x, x)
    with pytest.raises(RuntimeError):
        token_ops.qk_norm_rotary(x, x, None, None, torch.ones(2, 4), torch.ones(2, 4))
    with pytest.raises(RuntimeError):
        token_ops.clip_gradients([x], 1.0)
