"""The token operators where their definitions have corners: infinite scores, caps and limits of any size, calls that have to be refused."""
import math

import pytest
import torch

from tests.test_gpu_token_ops import TYPES, attention_inputs, check_attention, gen, ops
from tests.token_util import assert_within, attention_reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("documents", ["", "mixed", "one"])
@pytest.mark.parametrize("rows,keys", [(70, 70), (1, 3000), (900, 900)])
@pytest.mark.parametrize("value", [math.inf, -math.inf])
def test_attention_infinite_scores_are_not_numbers(dtype, documents, rows, keys, value):
    """A query whose seen scores are all infinite, or partly: its softmax is no number, in the result and in every gradient that it takes part
    in.  One that sees no key is zero, infinite or not.  (Rows by keys, split and not, and by rows.)"""
    token_attention = ops().token_attention
    H, Hk, D = 16 if rows == 900 else 2, 2, 32
    q, k, v, dout = attention_inputs(50, dtype, 1, rows, keys, H, Hk, D)
    k[0, :, 0, 5] = k[0, :, 0, 5].abs() + 0.25     # the first key head: every score has the sign of the query's channel 5
    r, G = rows // 2, H // Hk
    q[0, r, 0, 5] = value                          # all scores +inf, or all -inf
    q[0, r, G, 5] = value                          # the second key head: scores of both signs
    kw = {}
    if documents:
        ids_q = torch.full((1, rows), 3, device="cuda", dtype=torch.int32)
        ids_k = torch.full((1, keys), 3, device="cuda", dtype=torch.int32)
        if documents == "mixed":
            ids_k[0] = torch.arange(keys, device="cuda", dtype=torch.int32) % 3 + 2
        if rows > 1:
            q[0, 1] = value
            ids_q[0, 1], ids_q[0, 0] = 7, 7        # of a document without keys, one of the two infinite
        kw.update(q_docs=ids_q, k_docs=ids_k)
        seen = ids_k[0] == 3
    else:
        seen = torch.ones(keys, device="cuda", dtype=torch.bool)
    xs = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = token_attention(*xs, **kw)
    dq, dk, dv = torch.autograd.grad(out, xs, dout)
    none = torch.zeros(1, rows, H, dtype=torch.bool, device="cuda")
    none[0, r, 0] = none[0, r, G] = True
    for name, t in (("out", out), ("dq", dq), ("out without a graph", token_attention(q, k, v, **kw))):
        assert torch.equal(torch.isnan(t), none[..., None].expand_as(t)), name
        if documents and rows > 1:
            assert not t[0, :2].any(), name
    for name, t in (("dk", dk), ("dv", dv)):
        assert torch.isnan(t[0][seen]).all(), name


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [255.0, 257.0, 1e4, 1e5, 1e6, 1e12, 3e38, 1e39])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_caps_of_any_size(dtype, cap, D):
    """A cap far above the scores bends nothing: the result is as exact as without one.

    From 1e4 on the bound is that of the same scores uncapped, whose exponent may be off by 2 (D + 8) 2^-24 of sum |q k|: the scaling, the
    tangent and its factor add at most ten roundings of the score, 10 / 72 of that, and the derivative 1 - tanh^2 sixteen of a score
    gradient that is granted Lk + 16 = 216 of them, so a quarter more covers both."""
    q, k, v, dout = attention_inputs(51, dtype, 1, 200, 200, 2, 2, D)
    for kw in (dict(), dict(causal=True, slopes=torch.tensor([0.1, 0.0], device="cuda"))):
        if cap < 1e4:
            check_attention(q, k, v, dout, softcap=cap, **kw)
            continue
        xs = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = ops().token_attention(*xs, softcap=cap, **kw)
        got = [out, *torch.autograd.grad(out, xs, dout)]
        want, _ = attention_reference(q, k, v, dout, softcap=cap, **kw)
        _, bound = attention_reference(q, k, v, dout, **kw)
        for a, b, c, n in zip(got, want, bound, ("out", "dq", "dk", "dv")):
            assert_within(a, b, 1.25 * c, n)
        one = ops().token_attention(q[:, -1:], k, v, softcap=cap, **kw)     # the form by keys, without a backward pass
        assert_within(one, want[0][:, -1:], 1.25 * bound[0][:, -1:], "last token")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cap", [1e-50, 1e-38, 1e-20])
def test_attention_caps_near_zero(dtype, cap):
    """every score is the cap's size, nothing beside the bias: the gradients of q and k vanish"""
    q, k, v, dout = attention_inputs(52, dtype, 1, 100, 100, 2, 2, 32)
    got = check_attention(q, k, v, dout, softcap=cap, slopes=torch.tensor([0.5, 20.0], device="cuda"))
    assert not got[1].any() and not got[2].any()


@pytest.mark.parametrize("limit", [3.4e38, 3.5e38, 1e39, 1e300])
def test_clip_limits_past_float32(limit):
    """finite, so what is asked for is written: the gradients as they are"""
    grads = [torch.randn(n, device="cuda", generator=gen(n)) for n in (5, 5000)]
    out = [torch.full_like(g, 7.0) for g in grads]
    norm = ops().clip_gradients(grads, limit, out=out)
    assert all(torch.equal(a, b) for a, b in zip(grads, out))
    assert abs(float(norm) / math.sqrt(sum(float(g.double().square().sum()) for g in grads)) - 1) <= 2.0 ** -23
    before = [g.clone() for g in grads]
    ops().clip_gradients(grads, limit)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    assert float(ops().clip_gradients(grads, 1.0, eps=limit, out=out)) == float(norm) and all(float(o.abs().max()) < 1e-37 for o in out)


def test_tangents_are_refused():
    """forward-mode derivatives: none of the operators has one, so that a result without its tangent would be a wrong one"""
    from torch.autograd import forward_ad
    t = ops()
    q, k, v, _ = attention_inputs(53, torch.float32, 1, 8, 8, 2, 2, 16)
    cos, sin = t.rotary_tables(8, 16, device="cuda")
    w, slopes = torch.ones(16, device="cuda"), torch.ones(2, device="cuda")
    calls = [(t.token_attention, (q, k, v)), (lambda s: t.token_attention(q, k, v, slopes=s), (slopes,)), (lambda *a: t.qk_norm_rotary(*a)[0], (q, k, w, w, cos, sin)),
             (lambda *a: t.clip_gradients(a, 1e9), (q, k)), (lambda *a: t.clip_gradients((v, slopes), 1e9, out=a), (v.clone(), slopes.clone()))]
    with forward_ad.dual_level():
        for call, args in calls:
            call(*args)
            for n in range(len(args)):
                dual = [forward_ad.make_dual(a, torch.ones_like(a)) if i == n else a for i, a in enumerate(args)]
                with pytest.raises(RuntimeError, match="forward"):
                    call(*dual)
    for call, args in calls:
        call(*args)


def test_clip_grad_norm_of_every_parameter_that_torch_takes():
    """gradients that the library does not take go through torch's own function, whatever the first one is"""
    from diffusionmodelscustom_amd.training import clip_grad_norm_

    def parameters(*kinds):
        made = []
        for n, (dtype, device) in enumerate(kinds):
            p = torch.nn.Parameter(torch.zeros(7, 3, dtype=dtype, device=device))
            p.grad = torch.randn(7, 3, dtype=torch.float64, generator=torch.Generator().manual_seed(n)).to(device, dtype)
            made.append(p)
        return made
    gpu, cpu = torch.device("cuda"), torch.device("cpu")
    for kinds in ([(torch.float64, gpu)] * 2, [(torch.float32, gpu), (torch.float64, gpu)], [(torch.float32, gpu), (torch.float32, cpu)],
                  [(torch.float32, cpu), (torch.bfloat16, gpu)], [(torch.float32, gpu), (torch.bfloat16, gpu)]):
        got, want = parameters(*kinds), parameters(*kinds)
        a, b = clip_grad_norm_(got, 0.5), torch.nn.utils.clip_grad_norm_(want, 0.5)
        assert abs(float(a) / float(b) - 1) < 1e-2
        for p, w in zip(got, want):
            # one rounding of the gradient's type each, and torch's norm in the types' own (bfloat16: 2^-8)
            assert float((p.grad - w.grad).abs().max()) <= (2.0 ** -6 if p.dtype == torch.bfloat16 or torch.bfloat16 in [k[0] for k in kinds] else 1e-6) * float(w.grad.abs().max())
    sparse = torch.nn.Parameter(torch.zeros(4, 2, device="cuda"))
    sparse.grad = torch.sparse_coo_tensor([[1]], torch.ones(1, 2), (4, 2)).to("cuda")
    try:
        want = torch.nn.utils.clip_grad_norm_([sparse], 0.5)
    except (RuntimeError, NotImplementedError) as e:
        with pytest.raises(type(e)):
            clip_grad_norm_([sparse], 0.5)
    else:
        sparse.grad = torch.sparse_coo_tensor([[1]], torch.ones(1, 2), (4, 2)).to("cuda")
        assert abs(float(clip_grad_norm_([sparse], 0.5)) - float(want)) < 1e-5


def documents(rows, lengths, tail):
    """[1, rows] ids of documents one after the other, as long as given in turn, the last `tail` places of none"""
    ids = torch.cat([torch.full((n,), i, dtype=torch.int32) for i, n in enumerate(lengths)])[:rows - tail]
    return torch.cat([ids, torch.full((rows - len(ids),), -1, dtype=torch.int32)])[None].cuda()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_packed_documents_in_split_rows(dtype, causal):
    """A row of packed documents so long that the backward pass splits the rows of its keys and that lists of tiles take more than one look:
    more than 64 tiles of rows and of keys, long documents, short ones, padding."""
    import ctypes
    from diffusionmodelscustom_amd import hip_engine
    B, L, H, Hk, D = 1, 2200, 4, 1, 128
    q, k, v, dout = attention_inputs(54, dtype, B, L, L, H, Hk, D)
    ids = documents(L, (900, 5, 130, 1, 700, 64, 264), 150)
    d = ops()._describe(q, k, v, (None, None, None, ids, ids), D ** -0.5, 0.0, int(causal), dout)
    # (two or more partial results of dk and dv in float32)
    assert hip_engine.load_library().danra_token_attention_bwd_workspace(ctypes.byref(d)) > 2 * B * L * Hk * 2 * D * 4
    check_attention(q, k, v, dout, causal=causal, softcap=30.0 if causal else 0.0, q_docs=ids, k_docs=ids)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_documents_over_many_tiles_of_keys(dtype):
    """a forward pass by rows with more than 64 tiles of keys; documents in another order there, so that those of a row lie far apart"""
    q, k, v, _ = attention_inputs(55, dtype, 1, 2600, 4500, 4, 1, 64)
    ids_q = documents(2600, (800, 3, 1200, 500), 97)
    ids_k = documents(4500, (40, 1500, 2, 958), 0)
    ids_k[0, 2500:4400] = documents(1900, (1000, 300, 600), 0)[0]
    check_attention(q, k, v, q_docs=ids_q, k_docs=ids_k, softcap=30.0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("rows,keys", [(1, 20000), (4, 5000), (64, 3000)])
def test_attention_split_keys_joined_in_every_type(dtype, rows, keys):
    q, k, v, dout = attention_inputs(56, dtype, 2, rows, keys, 4, 2, 128)
    lens = torch.tensor([keys, 37], device="cuda", dtype=torch.int32)
    check_attention(q, k, v, kv_lens=lens, softcap=50.0, slopes=torch.tensor([0.5, 0.01, 0.0, 0.1], device="cuda"))
    check_attention(q, k, v, dout, kv_lens=lens, causal=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mean", [0.0, 1.0])
def test_attention_gradients_are_as_exact_as_one_rounding(dtype, mean):
    """The gradients of q and k of two-byte tensors are off by little more than the rounding of the exact ones is (e, in the 2-norm).

    With scores of a spread of 1 over 400 keys a row's probabilities spread over 1 / sum p^2 = 400 / e of them, more than 100.  Rounding P
    shifts delta = rowsum(dout . out) by e |dS|, which reaches dq through sum p k, a tenth of a key: together sqrt(1 + 1 / 100) e.  Rounding dS in
    one part would add another e, sqrt(2) e in all.  Values around `mean` with a spread s = 1 / 16 leave a difference dP - delta s times
    as large as its parts: a delta of the rounded result alone would be e / s = 16 e off.  1.2 e lies between."""
    q, k, v, dout = attention_inputs(57, dtype, 2, 400, 400, 4, 2, 64, spread=1.0)
    if mean:
        v = (mean + v.float() / 16).to(dtype)
    xs = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = ops().token_attention(*xs)
    got = torch.autograd.grad(out, xs, dout)
    want = attention_reference(q, k, v, dout)[0]
    for g, w, name in ((got[0], want[1], "dq"), (got[1], want[2], "dk")):
        one = float((w.to(dtype).double() - w).norm())
        assert float((g.double().cpu() - w).norm()) <= 1.2 * one, name


@pytest.mark.parametrize("dtype", TYPES)
def test_rotary_gains_of_many_tokens_are_rounded_once(dtype):
    """dw = sum g n over 32768 tokens of 4 heads, all terms positive.  Each term's own roundings are of either sign and shrink with the
    root of their number (362) beside the sum; what is left is the rounding of the result, 2^-24 at most, and a quarter for the rest.
    (A float32 sum of the 64 last partial sums alone would add 2^-24 sqrt(64) / 3 in the mean.)"""
    t = ops()
    g = gen(60)
    B, L, H, D = 2, 16384, 4, 32
    q, k = (torch.randn(B, L, H, D, device="cuda", generator=g).to(dtype) for _ in range(2))
    w = [torch.ones(D, device="cuda").requires_grad_(True) for _ in range(2)]
    cos, sin = torch.ones(L, D // 2, device="cuda"), torch.zeros(L, D // 2, device="cuda")
    out = t.qk_norm_rotary(q, k, *w, cos, sin)
    got = torch.autograd.grad(out, w, (q, k))
    for x, dw in ((q, got[0]), (k, got[1])):
        x = x.double()
        want = (x * x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt()).sum((0, 1, 2))
        assert float(((dw.double() - want) / want).abs().max()) <= 1.25 * 2.0 ** -24


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_scales_far_above_the_cap(dtype):
    """scale / cap past float32's range: scores are -cap, 0 and cap, and a product of 0 stays 0"""
    q, k, v, dout = attention_inputs(58, dtype, 1, 40, 40, 2, 2, 16)
    q[0, 7] = 0
    k[0, 9] = 0
    for cap, scale in ((1e-20, 1e25), (3.0, 8e37)):
        check_attention(q, k, v, softcap=cap, scale=scale)


def test_clip_in_inference_mode():
    with torch.inference_mode():
        g = [torch.full((5,), 2.0, device="cuda"), torch.full((4,), 2.0, device="cuda")]
        assert float(ops().clip_gradients(g, 3.0)) == 6.0
        assert all(float((x - 1).abs().max()) < 1e-6 for x in g)
        out = [torch.empty(5, device="cuda"), torch.empty(4, device="cuda")]
        assert abs(float(ops().clip_gradients(g, 1.0, out=out)) - 3.0) < 1e-6
    h = [torch.full((5,), 2.0, device="cuda")]
    with torch.inference_mode():
        ops().clip_gradients(h, 1.0)
    assert abs(float(h[0].norm()) - 1) < 1e-5
