"""Token operators of the native library: attention with capped scores, a distance bias and masks; the norms of queries and keys with the
position rotation; clipping of a list of gradients.

They stand beside the attention core and the token LayerNorm of ``hip_engine`` for attention blocks that the reference's networks
do not have: sequences packed from several documents, a bidirectional prefix, one new token over a cache, half-precision tensors.
``training.GraphedTrainStep`` and ``training.eager_train_step`` clip through ``clip_gradients``.

All of them take CUDA tensors in float32, bfloat16 or float16, run on the current stream of the tensors' device, allocate nothing
outside torch's allocator, never synchronise, and may be captured into a graph.  There is no fallback: a call that the library does
not take raises.
"""
import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from .hip_engine import QkNormRotary, TokenAttention, _check, _ptr, _stream, load_library

__all__ = ["token_attention", "qk_norm_rotary", "rotary_tables", "clip_gradients"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _tokens(t, name, like=None):
    """[batch, length, heads, head_dim] on the GPU in one of the three types"""
    if not torch.is_tensor(t) or not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.dtype not in _TYPES:
        raise ValueError(f"{name} is {t.dtype}: float32, bfloat16 or float16")
    if t.dim() != 4:
        raise ValueError(f"{name} has shape {tuple(t.shape)}: [batch, length, heads, head_dim]")
    if t.shape[3] % 8 or not 8 <= t.shape[3] <= 128:
        raise ValueError(f"{name} has head_dim {t.shape[3]}: a multiple of 8, at most 128")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} is {t.dtype} on {t.device}, the other tensors are {like.dtype} on {like.device}")
    return t


def _beside(t, name, like, dtype, shape):
    """a further argument: the given type and shape, on the same device, contiguous"""
    if t is None:
        return None
    if not torch.is_tensor(t) or t.device != like.device:
        raise RuntimeError(f"{name} must be a tensor on {like.device}")
    if t.dtype != dtype or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} is {t.dtype} {tuple(t.shape)}: {dtype} {tuple(shape)}")
    return t.contiguous()


def _rows(t):
    """`t` where the kernels can read it as it lies - consecutive channels, every row on 16 bytes -, else a contiguous copy"""
    per = 16 // t.element_size()
    n = t.shape
    if (t.stride(3) == 1 and t.data_ptr() % 16 == 0
            and all(n[i] <= 1 or t.stride(i) % per == 0 for i in range(3))):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t):
    return (ctypes.c_int64 * 3)(*(t.stride(i) if t.shape[i] > 1 else 0 for i in range(3)))


def _describe(q, k, v, beside, scale, softcap, causal, dout=None):
    slopes, prefix, kv_lens, q_docs, k_docs = beside
    d = TokenAttention(_TYPES[q.dtype], q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3], int(causal), scale,
                       softcap, _ptr(slopes), _ptr(prefix), _ptr(kv_lens), _ptr(q_docs), _ptr(k_docs), _strides(q), _strides(k),
                       _strides(v))
    if dout is not None:
        d.dout_stride = _strides(dout)
    return d


def _workspace(size, device):
    return torch.empty(size, device=device, dtype=torch.uint8) if size else None


def _attention_forward(q, k, v, beside, scale, softcap, causal, keep):
    """(out, lse2 or None) of tensors that _rows returned"""
    lib = load_library()
    B, Lq, H, D = q.shape
    out = torch.empty((B, Lq, H, D), device=q.device, dtype=q.dtype)
    lse2 = torch.empty((B, k.shape[2], Lq * (H // k.shape[2])), device=q.device, dtype=torch.float32) if keep else None
    d = _describe(q, k, v, beside, scale, softcap, causal)
    with torch.cuda.device(q.device):
        workspace = _workspace(lib.danra_token_attention_fwd_workspace(ctypes.byref(d)), q.device)
        _check(lib, lib.danra_token_attention_fwd(ctypes.byref(d), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse2), _ptr(workspace),
                                                  _stream()), "danra_token_attention_fwd")
    return out, lse2


class _TokenAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, prefix, kv_lens, q_docs, k_docs, scale, softcap, causal):
        q, k, v = _rows(q), _rows(k), _rows(v)
        beside = (slopes, prefix, kv_lens, q_docs, k_docs)
        out, lse2 = _attention_forward(q, k, v, beside, scale, softcap, causal, True)
        ctx.save_for_backward(q, k, v, out, lse2, *beside)
        ctx.call = (scale, softcap, causal)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        lib = load_library()
        q, k, v, out, lse2, *beside = ctx.saved_tensors
        dout = _rows(dout)
        d = _describe(q, k, v, beside, *ctx.call, dout=dout)

        def like(t):
            return torch.empty(t.shape, device=t.device, dtype=t.dtype)
        dq = like(q) if ctx.needs_input_grad[0] else None
        dk, dv = (like(k), like(v)) if ctx.needs_input_grad[1] or ctx.needs_input_grad[2] else (None, None)
        with torch.cuda.device(q.device):
            workspace = _workspace(lib.danra_token_attention_bwd_workspace(ctypes.byref(d)), q.device)
            _check(lib, lib.danra_token_attention_bwd(ctypes.byref(d), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(dout), _ptr(lse2),
                                                      _ptr(dq), _ptr(dk), _ptr(dv), _ptr(workspace), _stream()),
                   "danra_token_attention_bwd")
        return (dq, dk if ctx.needs_input_grad[1] else None, dv if ctx.needs_input_grad[2] else None) + (None,) * 8


def token_attention(q, k, v, scale=None, softcap=0.0, slopes=None, causal=False, prefix=None, kv_lens=None, q_docs=None, k_docs=None):
    """Softmax attention of ``q [B, Lq, H, D]`` over ``k, v [B, Lk, Hk, D]`` -> ``[B, Lq, H, D]``, differentiable in q, k and v.

    Query head h reads key head ``h // (H // Hk)``.  The queries are the last Lq of their sequence: query i stands at
    ``pos_i = i + n_b - Lq`` among the ``n_b`` keys of sequence b, so a new token over a cache is ``Lq = 1``.

    * ``scale``: of the products, ``D ** -0.5`` by default.
    * ``softcap`` > 0: scores become ``softcap * tanh(score / softcap)``.
    * ``slopes [H]`` float32: ``- slopes[h] * |pos_i - j|`` is added to the (capped) score.  Not differentiable.
    * ``kv_lens [B]`` int32: n_b, the keys of each sequence that count (Lk without it; clamped to 0 .. Lk).
    * ``causal``: query i sees the keys j <= pos_i; with ``prefix [B]`` int32 also every j < prefix[b].
    * ``q_docs [B, Lq]``, ``k_docs [B, Lk]`` int32: query i sees the keys of its own document; a negative id is padding, which
      sees nothing and is seen by nothing.

    A query that sees no key gives zeros and takes no part in any gradient, whatever it holds; keys and values that are padding or lie
    past ``n_b`` may hold anything.  A non-finite value in a key that some query may see can reach every query of its head.

    D is a multiple of 8, at most 128.  Tensors are read in place where channels are consecutive and rows start on 16 bytes (parts of a
    fused projection's output do), else copied first.  Scores, softmax and sums are float32; the probabilities, and the score gradients, are
    rounded to the tensors' type for their products.  Results are the same bits for the same inputs.
    """
    _tokens(q, "q")
    _tokens(k, "k", q)
    _tokens(v, "v", q)
    B, Lq, H, D = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != D:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)}: [B, Lq, H, D] and twice [B, Lk, Hk, D]")
    Lk, Hk = k.shape[1], k.shape[2]
    if Hk == 0 or H == 0 or H % Hk:
        raise ValueError(f"{H} query heads over {Hk} key heads: a positive multiple")
    if prefix is not None and not causal:
        raise ValueError("prefix needs causal=True")
    if (q_docs is None) != (k_docs is None):
        raise ValueError("q_docs and k_docs come together")
    if slopes is not None and slopes.requires_grad:
        raise ValueError("slopes are not differentiable: pass slopes.detach()")
    scale, softcap = float(D ** -0.5 if scale is None else scale), float(softcap)
    if not math.isfinite(scale) or not math.isfinite(softcap) or softcap < 0:
        raise ValueError(f"scale {scale}, softcap {softcap}: finite, softcap not negative")
    beside = (_beside(slopes, "slopes", q, torch.float32, (H,)), _beside(prefix, "prefix", q, torch.int32, (B,)),
              _beside(kv_lens, "kv_lens", q, torch.int32, (B,)), _beside(q_docs, "q_docs", q, torch.int32, (B, Lq)),
              _beside(k_docs, "k_docs", q, torch.int32, (B, Lk)))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _TokenAttention.apply(q, k, v, *beside, scale, softcap, bool(causal))
    return _attention_forward(_rows(q), _rows(k), _rows(v), beside, scale, softcap, bool(causal), False)[0]


def rotary_tables(length, rotated, base=10000.0, device=None):
    """(cos, sin) of position * base^(-2 p / rotated) for positions 0 .. length - 1 and pairs p, [length, rotated / 2] float32.
    The angles are formed in float64: far positions keep their place in the circle."""
    if rotated < 2 or rotated % 2:
        raise ValueError(f"rotated {rotated}: even and positive")
    rate = float(base) ** (-torch.arange(0, rotated, 2, dtype=torch.float64, device=device) / rotated)
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * rate
    return angle.cos().float(), angle.sin().float()


def _describe_rotary(q, k, weight, cos, sin, positions, eps, interleaved):
    d = QkNormRotary(_TYPES[q.dtype], _TYPES[weight.dtype] if weight is not None else _TYPES[q.dtype], q.shape[0], q.shape[1],
                     (ctypes.c_int * 2)(q.shape[2], k.shape[2]), q.shape[3], 2 * cos.shape[1], cos.shape[0], int(interleaved), eps,
                     _ptr(cos), _ptr(sin), _ptr(positions))
    d.x_stride[0], d.x_stride[1] = _strides(q), _strides(k)
    return d


def _rotary_forward(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
    lib = load_library()
    q_out, k_out = (torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k))
    d = _describe_rotary(q, k, q_weight if q_weight is not None else k_weight, cos, sin, positions, eps, interleaved)
    with torch.cuda.device(q.device):
        _check(lib, lib.danra_qk_norm_rotary_fwd(ctypes.byref(d), _ptr(q), _ptr(k), _ptr(q_weight), _ptr(k_weight), _ptr(q_out),
                                                 _ptr(k_out), _stream()), "danra_qk_norm_rotary_fwd")
    return q_out, k_out


class _QkNormRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
        q, k = _rows(q), _rows(k)
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.call = (eps, interleaved)
        return _rotary_forward(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq_out, dk_out):
        lib = load_library()
        q, k, q_weight, k_weight, cos, sin, positions = ctx.saved_tensors
        eps, interleaved = ctx.call
        dq_out, dk_out = _rows(dq_out), _rows(dk_out)
        d = _describe_rotary(q, k, q_weight if q_weight is not None else k_weight, cos, sin, positions, eps, interleaved)
        d.dy_stride[0], d.dy_stride[1] = _strides(dq_out), _strides(dk_out)
        dq, dk = (torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k))
        dqw = torch.empty_like(q_weight) if q_weight is not None and ctx.needs_input_grad[2] else None
        dkw = torch.empty_like(k_weight) if k_weight is not None and ctx.needs_input_grad[3] else None
        with torch.cuda.device(q.device):
            workspace = None
            if dqw is not None or dkw is not None:
                workspace = _workspace(lib.danra_qk_norm_rotary_bwd_workspace(ctypes.byref(d)), q.device)
            _check(lib, lib.danra_qk_norm_rotary_bwd(ctypes.byref(d), _ptr(q), _ptr(k), _ptr(q_weight), _ptr(k_weight), _ptr(dq_out),
                                                     _ptr(dk_out), _ptr(dq), _ptr(dk), _ptr(dqw), _ptr(dkw), _ptr(workspace),
                                                     _stream()), "danra_qk_norm_rotary_bwd")
        return dq, dk, dqw, dkw, None, None, None, None, None


def qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions=None, eps=1e-6, interleaved=False):
    """Root-mean-square norm of every head of ``q [B, L, H, D]`` and ``k [B, L, Hk, D]`` with a gain per channel, and the position
    rotation, in one pass -> (q, k) of the same shapes, contiguous; differentiable in q, k and the gains.

    ``y = rot(x / sqrt(mean(x^2) + eps) * weight)``; rot turns the pair (a, b) into ``(a cos - b sin, b cos + a sin)``.

    * ``q_weight, k_weight [D]``: in the tensors' type or float32 (both in the same), or None for ones.
    * ``cos, sin [P, R / 2]`` float32 (``rotary_tables``): the first R <= D channels are rotated, the others keep their normalised value.
      Pair p is channels (p, R / 2 + p), or with ``interleaved`` (2 p, 2 p + 1).
    * ``positions [B, L]`` int64: rows of the tables; without it a token's index in its sequence.  A position outside the tables
      turns the rotated channels into NaN (nothing is read back to check).

    Tensors are read in place where channels are consecutive and rows start on 16 bytes, else copied first.
    """
    _tokens(q, "q")
    _tokens(k, "k", q)
    B, L, H, D = q.shape
    if k.shape[:2] != q.shape[:2] or k.shape[3] != D or H == 0 or k.shape[2] == 0:
        raise ValueError(f"q {tuple(q.shape)}, k {tuple(k.shape)}: [B, L, H, D] and [B, L, Hk, D]")
    if not torch.is_tensor(cos) or cos.dim() != 2 or cos.shape[0] == 0 or not 2 <= 2 * cos.shape[1] <= D:
        raise ValueError("cos: [positions, R / 2] with R at most head_dim")
    cos = _beside(cos, "cos", q, torch.float32, cos.shape)
    sin = _beside(sin, "sin", q, torch.float32, cos.shape)
    positions = _beside(positions, "positions", q, torch.int64, (B, L))
    if positions is None and L > cos.shape[0]:
        raise ValueError(f"{L} tokens, the tables have {cos.shape[0]} rows")
    if cos.requires_grad or sin.requires_grad:
        raise ValueError("the tables are not differentiable")
    kind = None
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            continue
        if not torch.is_tensor(w) or w.device != q.device:
            raise RuntimeError(f"{name} must be a tensor on {q.device}")
        if w.dtype not in (q.dtype, torch.float32) or tuple(w.shape) != (D,) or kind not in (None, w.dtype):
            raise ValueError(f"{name} is {w.dtype} {tuple(w.shape)}: ({D},) in {q.dtype} or float32, the same for both")
        kind = w.dtype
    eps = float(eps)
    if not math.isfinite(eps) or eps < 0:
        raise ValueError(f"eps {eps}: finite, not negative")
    q_weight, k_weight = (w if w is None else w.contiguous() for w in (q_weight, k_weight))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _QkNormRotary.apply(q, k, q_weight, k_weight, cos, sin, positions, eps, bool(interleaved))
    return _rotary_forward(_rows(q), _rows(k), q_weight, k_weight, cos, sin, positions, eps, bool(interleaved))


def _dense(t):
    """the elements lie in one consecutive block of memory, in whatever order of the dimensions"""
    if t.is_contiguous():
        return True
    at = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != at:
            return False
        at *= size
    return True


def clip_gradients(grads, max_norm, out=None, eps=1e-6):
    """Scales a list of gradients by ``min(1, max_norm / (norm + eps))`` and returns ``norm``, the 2-norm of all of them together, as a
    float32 scalar on their device (no synchronisation): the arithmetic of ``torch.nn.utils.clip_grad_norm_`` in two passes over the
    values, whatever their number.

    In place, or into ``out``: a list of tensors of the same shapes and strides, each float32, bfloat16 or float16 (half-precision
    gradients into the float32 gradients of master weights).  ``max_norm = math.inf``: only the norm, nothing is written.  Squares are summed
    in float64, in a fixed order.  A norm that is not finite scales as its arithmetic says (NaN everywhere, or zeros and NaN).

    Every tensor is dense (its elements fill one block of memory).  What is written must not overlap with anything else in the call; the
    same memory twice in one list is refused.
    """
    grads = list(grads)
    max_norm, eps = float(max_norm), float(eps)
    if not max_norm >= 0 or not eps >= 0 or math.isinf(eps):
        raise ValueError(f"max_norm {max_norm}, eps {eps}: not negative")
    if not grads:
        raise ValueError("no gradients")
    device = grads[0].device
    into = grads if out is None else list(out)
    if len(into) != len(grads):
        raise ValueError(f"{len(grads)} gradients, {len(into)} tensors to write")
    for g in (grads if into is grads else grads + into):
        if not g.is_cuda or g.device != device:
            raise RuntimeError("every gradient must be a CUDA tensor on one device")
        if g.dtype not in _TYPES or g.layout is not torch.strided:
            raise ValueError(f"a gradient is {g.dtype}, {g.layout}: dense float32, bfloat16 or float16")
        if not _dense(g):
            raise ValueError(f"a gradient of shape {tuple(g.shape)} and strides {g.stride()} does not fill one block of memory")
    n = len(grads)
    read = [g.data_ptr() for g in grads]
    numel = [g.numel() for g in grads]
    write = read
    if into is not grads:
        for g, o in zip(grads, into):
            if o.shape != g.shape or (o.stride() != g.stride() and not (o.is_contiguous() and g.is_contiguous())):
                raise ValueError(f"out {tuple(o.shape)} {o.stride()} for a gradient {tuple(g.shape)} {g.stride()}")
        write = [o.data_ptr() for o in into]
    if not math.isinf(max_norm):
        _refuse_overlap(read, write, numel, grads, into)
    lib = load_library()
    norm = torch.empty((), device=device, dtype=torch.float32)
    kinds = (ctypes.c_int * n)(*[_TYPES[g.dtype] for g in grads])
    out_kinds = kinds if into is grads else (ctypes.c_int * n)(*[_TYPES[o.dtype] for o in into])
    with torch.cuda.device(device):
        workspace = torch.empty(lib.danra_clip_gradients_workspace(n) // 8, device=device, dtype=torch.float64)
        _check(lib, lib.danra_clip_gradients((ctypes.c_void_p * n)(*read), (ctypes.c_void_p * n)(*write), (ctypes.c_size_t * n)(*numel),
                                             kinds, out_kinds, n, max_norm, eps, _ptr(norm), _ptr(workspace), _stream()),
               "danra_clip_gradients")
    if not math.isinf(max_norm):
        for o in into:
            torch.autograd.graph.increment_version(o)
    return norm


def _refuse_overlap(read, write, numel, grads, into):
    """what one tensor's part of the call writes may be read or written by no other part"""
    spans = []
    for r, w, n, g, o in zip(read, write, numel, grads, into):
        if n:
            spans.append((w, w + n * o.element_size(), True))
            if r != w or g.dtype != o.dtype:
                spans.append((r, r + n * g.element_size(), False))
    spans.sort()
    end = written_end = 0    # of all spans so far, and of the written ones
    for begin, stop, written in spans:
        if begin < written_end or (written and begin < end):
            raise ValueError("a gradient that is written overlaps with another tensor of the call")
        end = max(end, stop)
        if written:
            written_end = max(written_end, stop)
