"""Token operators of the native library: attention with capped scores, a distance bias and masks; the norms of queries and keys with the
position rotation; clipping of a list of gradients.

They stand beside the attention core and the token LayerNorm of ``hip_engine`` for attention blocks that the reference's networks
do not have: sequences packed from several documents, a bidirectional prefix, one new token over a cache, half-precision tensors.
``training.GraphedTrainStep`` and ``training.eager_train_step`` clip through ``clip_gradients``.

All of them take CUDA tensors in float32, bfloat16 or float16, run on the current stream of the tensors' device, allocate nothing
outside torch's allocator, never synchronise, and may be captured into a graph.  There is no fallback: a call that the library does
not take raises.  Derivatives are those of reverse mode, once: forward-mode tangents and second derivatives are refused.
"""
import ctypes
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .hip_engine import QkNormRotary, TokenAttention, _check, load_library

__all__ = ["token_attention", "qk_norm_rotary", "rotary_tables", "clip_gradients"]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_LARGEST = torch.finfo(torch.float32).max


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


def _no_tangents(*lists):
    """Forward-mode derivatives stay behind in tensors whose memory alone is read: no result may come without them.  (The level is asked for
    first: there may be hundreds of tensors.)"""
    if getattr(forward_ad, "_current_level", 0) >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for ts in lists for t in ts):
        raise NotImplementedError("the token operators have no forward-mode derivatives")


def _rows(t):
    """`t` where the kernels can read it as it lies - consecutive channels, every row on 16 bytes, tokens apart and a few of them within
    32-bit offsets (a tile of 64 rows spans 32 tokens of two heads, and 64 tokens of one head fit at any step that is taken) -, else a
    contiguous copy"""
    size = t.element_size()
    per = 16 // size
    (n0, n1, n2, n3), (s0, s1, s2, s3) = t.shape, t.stride()
    if (s3 == 1 and t.data_ptr() % 16 == 0 and (s0 % per == 0 or n0 <= 1) and (n1 <= 1 or (s1 % per == 0 and n3 <= s1 < 1 << 22))
            and (n2 <= 1 or (s2 % per == 0 and (33 * s1 + n2 * s2) * size < (1 << 31) - 1024))):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _at(t):
    return None if t is None else t.data_ptr()


_Strides = ctypes.c_int64 * 12


def _call(lib, name, device, *args):
    """The entry with `args` and the current stream of `device`, which is made the current device where it is not.  (These calls take as
    long as the shortest kernels: the stream is asked for without a Stream object around it, and no context is entered without need.)"""
    fn, stream = getattr(lib, name), torch._C._cuda_getCurrentRawStream    # (a torch without a GPU has no such name, but no call either)
    if device.index == torch.cuda.current_device():
        rc = fn(*args, stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream(device.index))
    if rc == -1:    # DANRA_EINVAL: what only the library can tell
        raise ValueError(f"{name}: {lib.danra_last_error().decode()}")
    if rc:
        _check(lib, rc, name)


def _describe(q, k, v, beside, scale, softcap, causal, dout=None):
    slopes, prefix, kv_lens, q_docs, k_docs = beside
    B, Lq, H, D = q.shape
    return TokenAttention(_TYPES[q.dtype], B, Lq, k.shape[1], H, k.shape[2], D, causal, scale, softcap, _at(slopes), _at(prefix),
                          _at(kv_lens), _at(q_docs), _at(k_docs),
                          _Strides(*q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *(() if dout is None else dout.stride()[:3])))


def _workspace(size, device):
    return torch.empty(size, device=device, dtype=torch.uint8) if size else None


def _attention_forward(q, k, v, beside, scale, softcap, causal, keep):
    """out of tensors that _rows returned; with `keep` (out, rest, stats) for the backward pass"""
    lib = load_library()
    B, Lq, H, D = q.shape
    device = q.device
    out = torch.empty((B, Lq, H, D), device=device, dtype=q.dtype)
    rest = stats = None
    if keep:
        stats = torch.empty((B, H, Lq, 2), device=device, dtype=torch.float32)
        if q.dtype != torch.float32:
            rest = torch.empty((B, Lq, H, D), device=device, dtype=q.dtype)
    d = ctypes.byref(_describe(q, k, v, beside, scale, softcap, causal))
    workspace = _workspace(lib.danra_token_attention_fwd_workspace(d), device)
    _call(lib, "danra_token_attention_fwd", device, d, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _at(rest),
          _at(stats), _at(workspace))
    return (out, rest, stats) if keep else out


class _TokenAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, prefix, kv_lens, q_docs, k_docs, scale, softcap, causal):
        q, k, v = _rows(q), _rows(k), _rows(v)
        beside = (slopes, prefix, kv_lens, q_docs, k_docs)
        out, rest, stats = _attention_forward(q, k, v, beside, scale, softcap, causal, True)
        ctx.save_for_backward(q, k, v, out, rest, stats, *beside)
        ctx.call = (scale, softcap, causal)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        lib = load_library()
        q, k, v, out, rest, stats, *beside = ctx.saved_tensors
        dout = _rows(dout)
        need_q, need_k, need_v = ctx.needs_input_grad[:3]
        device, dtype = q.device, q.dtype
        dq = torch.empty(q.shape, device=device, dtype=dtype) if need_q else None
        dk, dv = (torch.empty(k.shape, device=device, dtype=dtype) for _ in range(2)) if need_k or need_v else (None, None)
        d = ctypes.byref(_describe(q, k, v, beside, *ctx.call, dout=dout))
        workspace = _workspace(lib.danra_token_attention_bwd_workspace(d), device)
        _call(lib, "danra_token_attention_bwd", device, d, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _at(rest), dout.data_ptr(),
              stats.data_ptr(), _at(dq), _at(dk), _at(dv), _at(workspace))
        return (dq, dk if need_k else None, dv if need_v else None) + (None,) * 8


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
    past ``n_b`` may hold anything.  A non-finite value in a key that some query may see can reach every query of its head; a query with an
    infinite score, or with none but scores of -infinity, gives NaN.

    D is a multiple of 8, at most 128.  Tensors are read in place where channels are consecutive and rows start on 16 bytes (parts of a
    fused projection's output do), else copied first.  Scores, softmax and sums are float32; for their products the probabilities are
    rounded to the tensors' type, the score gradients to two parts of it (value and remainder).  Results are the same bits for the same inputs.
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
    softcap = min(max(softcap, 1e-30), 1e30) if softcap else 0.0    # (in float32; what lies outside acts like these)
    beside = (_beside(slopes, "slopes", q, torch.float32, (H,)), _beside(prefix, "prefix", q, torch.int32, (B,)),
              _beside(kv_lens, "kv_lens", q, torch.int32, (B,)), _beside(q_docs, "q_docs", q, torch.int32, (B, Lq)),
              _beside(k_docs, "k_docs", q, torch.int32, (B, Lk)))
    _no_tangents((q, k, v, slopes))
    causal = int(bool(causal))
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _TokenAttention.apply(q, k, v, *beside, scale, softcap, causal)
    return _attention_forward(_rows(q), _rows(k), _rows(v), beside, scale, softcap, causal, False)


def rotary_tables(length, rotated, base=10000.0, device=None):
    """(cos, sin) of position * base^(-2 p / rotated) for positions 0 .. length - 1 and pairs p, [length, rotated / 2] float32.
    The angles are formed in float64: far positions keep their place in the circle."""
    if rotated < 2 or rotated % 2:
        raise ValueError(f"rotated {rotated}: even and positive")
    rate = float(base) ** (-torch.arange(0, rotated, 2, dtype=torch.float64, device=device) / rotated)
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * rate
    return angle.cos().float(), angle.sin().float()


def _describe_rotary(q, k, weight, cos, sin, positions, eps, interleaved, dq=None, dk=None):
    B, L, H, D = q.shape
    kind = _TYPES[q.dtype]
    return QkNormRotary(kind, kind if weight is None else _TYPES[weight.dtype], B, L, H, k.shape[2], D, 2 * cos.shape[1], cos.shape[0],
                        interleaved, eps, cos.data_ptr(), sin.data_ptr(), _at(positions),
                        _Strides(*q.stride()[:3], *k.stride()[:3], *(() if dq is None else (*dq.stride()[:3], *dk.stride()[:3]))))


def _rotary_forward(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved):
    lib = load_library()
    device = q.device
    q_out = torch.empty(q.shape, device=device, dtype=q.dtype)
    k_out = torch.empty(k.shape, device=device, dtype=q.dtype)
    d = _describe_rotary(q, k, q_weight if q_weight is not None else k_weight, cos, sin, positions, eps, interleaved)
    _call(lib, "danra_qk_norm_rotary_fwd", device, ctypes.byref(d), q.data_ptr(), k.data_ptr(), _at(q_weight), _at(k_weight),
          q_out.data_ptr(), k_out.data_ptr())
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
        dq_out, dk_out = _rows(dq_out), _rows(dk_out)
        device, dtype = q.device, q.dtype
        d = ctypes.byref(_describe_rotary(q, k, q_weight if q_weight is not None else k_weight, cos, sin, positions, *ctx.call, dq_out, dk_out))
        dq = torch.empty(q.shape, device=device, dtype=dtype)
        dk = torch.empty(k.shape, device=device, dtype=dtype)
        dqw = torch.empty_like(q_weight) if q_weight is not None and ctx.needs_input_grad[2] else None
        dkw = torch.empty_like(k_weight) if k_weight is not None and ctx.needs_input_grad[3] else None
        workspace = None
        if dqw is not None or dkw is not None:
            workspace = _workspace(lib.danra_qk_norm_rotary_bwd_workspace(d), device)
        _call(lib, "danra_qk_norm_rotary_bwd", device, d, q.data_ptr(), k.data_ptr(), _at(q_weight), _at(k_weight), dq_out.data_ptr(),
              dk_out.data_ptr(), dq.data_ptr(), dk.data_ptr(), _at(dqw), _at(dkw), _at(workspace))
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
    _no_tangents((q, k, q_weight, k_weight, cos, sin))
    interleaved = int(bool(interleaved))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _QkNormRotary.apply(q, k, q_weight, k_weight, cos, sin, positions, eps, interleaved)
    return _rotary_forward(_rows(q), _rows(k), q_weight, k_weight, cos, sin, positions, eps, interleaved)


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


class NotClipped(ValueError, RuntimeError):
    """raised by ``clip_gradients`` for tensors that the library does not take, before anything is done"""


def clip_gradients(grads, max_norm, out=None, eps=1e-6):
    """Scales a list of gradients by ``min(1, max_norm / (norm + eps))`` and returns ``norm``, the 2-norm of all of them together, as a
    float32 scalar on their device (no synchronisation): the arithmetic of ``torch.nn.utils.clip_grad_norm_`` in two passes over the
    values, whatever their number.

    In place, or into ``out``: a list of tensors of as many elements, contiguous like the gradients or with the same strides, each
    float32, bfloat16 or float16 (half-precision gradients into the float32 gradients of master weights).  ``max_norm = math.inf``: only
    the norm, nothing is written, to ``out`` neither; a finite one counts as at most float32's largest number.  Squares are summed in
    float64, in a fixed order.  A norm that is not finite scales as its arithmetic says (NaN everywhere, or zeros and NaN).

    Every tensor is dense (its elements fill one block of memory).  What is written must not overlap with anything else in the call; the
    same memory twice in one list is refused.
    """
    grads = list(grads)
    max_norm, eps = float(max_norm), float(eps)
    if not max_norm >= 0 or not eps >= 0 or math.isinf(eps):
        raise ValueError(f"max_norm {max_norm}, eps {eps}: not negative")
    # (the entry takes float32, where a larger number would be infinity: no limit)
    eps, max_norm = min(eps, _LARGEST), max_norm if math.isinf(max_norm) else min(max_norm, _LARGEST)
    if not grads:
        raise ValueError("no gradients")
    into = grads if out is None else list(out)
    if len(into) != len(grads):
        raise ValueError(f"{len(grads)} gradients, {len(into)} tensors to write")
    device = grads[0].device
    n = len(grads)
    read, numel, kinds, plain = _facts(grads, device.index)
    write, out_kinds = read, kinds
    if out is not None:
        write, out_numel, out_kinds, out_plain = _facts(into, device.index)
        if numel != out_numel or not (plain and out_plain):
            for g, o in zip(grads, into):
                if o.numel() != g.numel() or (o.stride() != g.stride() and not (o.is_contiguous() and g.is_contiguous())):
                    raise ValueError(f"out {tuple(o.shape)} {o.stride()} for a gradient {tuple(g.shape)} {g.stride()}")
    _no_tangents(grads, into)
    lib = load_library()
    norm = torch.empty((), device=device, dtype=torch.float32)
    workspace = _workspace(lib.danra_clip_gradients_workspace(n), device)
    pointers, integers = ctypes.c_void_p * n, ctypes.c_int * n
    kinds = integers(*kinds)
    read = pointers(*read)
    _call(lib, "danra_clip_gradients", device, read, read if out is None else pointers(*write), (ctypes.c_size_t * n)(*numel), kinds,
          kinds if out is None else integers(*out_kinds), n, max_norm, eps, norm.data_ptr(), workspace.data_ptr())
    if not math.isinf(max_norm):
        torch.autograd.graph.increment_version(into)
    return norm


def _facts(tensors, index):
    """addresses, numbers of elements, types of dense tensors on device `index`, and whether all are contiguous (each asked of all tensors
    in turn: there may be hundreds, and the kernels take as long as a few dozen such loops)"""
    if any(t.get_device() != index for t in tensors) or index is None:
        raise NotClipped("every gradient must be a CUDA tensor on one device")
    kinds = [_TYPES.get(t.dtype, -1) for t in tensors]
    if -1 in kinds or {t.layout for t in tensors} != {torch.strided}:
        raise NotClipped("a gradient is not a dense float32, bfloat16 or float16 tensor")
    plain = all([t.is_contiguous() for t in tensors])
    if not plain:
        for t in tensors:
            if not _dense(t):
                raise NotClipped(f"a gradient of shape {tuple(t.shape)} and strides {t.stride()} does not fill one block of memory")
    return [t.data_ptr() for t in tensors], [t.numel() for t in tensors], kinds, plain
