"""The token operators against their definitions in float64, each element within a bound derived from its roundings (token_util)."""
import math

import pytest
import torch

from tests.token_util import assert_within, attention_reference, rotary_reference

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def ops():
    from diffusionmodelscustom_amd import token_ops
    return token_ops


def normal(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * scale).to(dtype)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def attention_inputs(seed, dtype, B, Lq, Lk, H, Hk, D, spread=3.0):
    g = gen(seed)
    return (normal(g, B, Lq, H, D, dtype=dtype, scale=spread), normal(g, B, Lk, Hk, D, dtype=dtype), normal(g, B, Lk, Hk, D, dtype=dtype),
            normal(g, B, Lq, H, D, dtype=dtype))


def check_attention(q, k, v, dout=None, **kw):
    token_attention = ops().token_attention
    if dout is None:
        got = [token_attention(q, k, v, **kw)]
    else:
        q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
        out = token_attention(q, k, v, **kw)
        got = [out, *torch.autograd.grad(out, (q, k, v), dout)]
    want, bound = attention_reference(q, k, v, dout, **kw)
    worst = [assert_within(a, b, c, n) for a, b, c, n in zip(got, want, bound, ("out", "dq", "dk", "dv"))]
    print("share of the bound:", ["%.2f" % w for w in worst], flush=True)
    return got


# (B, Lq, Lk, H, Hk, D): one token to several tiles, odd lengths, shared heads, every width of the tiles
SHAPES = [(1, 1, 1, 1, 1, 8), (2, 1, 65, 4, 2, 16), (1, 33, 33, 3, 1, 24), (2, 129, 129, 4, 4, 32), (1, 70, 70, 6, 2, 40), (1, 257, 257, 2, 2, 64),
          (2, 31, 100, 4, 1, 72), (1, 130, 130, 2, 1, 96), (1, 200, 200, 5, 1, 128), (3, 5, 300, 8, 2, 128), (1, 300, 7, 2, 2, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("masks", ["plain", "capped causal", "all"])
def test_attention_matches_float64(shape, dtype, masks):
    B, Lq, Lk, H, Hk, D = shape
    q, k, v, dout = attention_inputs(Lq * 7 + Lk, dtype, B, Lq, Lk, H, Hk, D)
    g = gen(1)
    kw = {}
    if masks != "plain":
        kw.update(softcap=20.0, causal=True)
    if masks == "all":
        kw.update(slopes=torch.rand(H, device="cuda", generator=g), prefix=torch.randint(0, Lk + 1, (B,), device="cuda", generator=g, dtype=torch.int32),
                  kv_lens=torch.randint(0, Lk + 1, (B,), device="cuda", generator=g, dtype=torch.int32),
                  q_docs=torch.randint(-1, 3, (B, Lq), device="cuda", generator=g, dtype=torch.int32).sort(dim=1).values.contiguous(),
                  k_docs=torch.randint(-1, 3, (B, Lk), device="cuda", generator=g, dtype=torch.int32).sort(dim=1).values.contiguous())
    check_attention(q, k, v, dout, **kw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-3])
def test_attention_scales_of_any_sign(dtype, scale):
    for D, L in ((64, 90), (128, 140)):
        q, k, v, dout = attention_inputs(21, dtype, 1, L, L, 4, 2, D)
        check_attention(q, k, v, dout, scale=scale, causal=True)
        check_attention(q, k, v, dout, scale=scale, softcap=6.0, slopes=torch.tensor([0.0, 0.3, 1.0, 0.01], device="cuda"))
        check_attention(q[:, -1:], k, v, scale=scale, slopes=torch.full((4,), 0.05, device="cuda"))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [1, 40, 700])
def test_attention_documents_in_any_order(dtype, rows):
    """ids that alternate, so that no tile is of one document; the last ones of no document"""
    q, k, v, dout = attention_inputs(3, dtype, 2, rows, rows, 4, 2, 64)
    ids = (torch.arange(rows, device="cuda", dtype=torch.int32) * 5 % 7 - 1)[None].repeat(2, 1)
    check_attention(q, k, v, dout, q_docs=ids, k_docs=ids, causal=True, softcap=30.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Lq", [1, 300])
def test_attention_masked_places_hold_anything(dtype, Lq):
    """NaN and infinity in keys past the length and in padding, in queries that see nothing, and in their gradients"""
    B, Lk, H, Hk, D = 4, 400, 4, 2, 64
    q, k, v, dout = attention_inputs(5, dtype, B, Lq, Lk, H, Hk, D)
    lens = torch.tensor([0, 1, 333, 400], device="cuda", dtype=torch.int32)
    for b, n in enumerate(lens.tolist()):
        k[b, n:] = math.nan
        v[b, n:] = math.inf
    q[0], dout[0] = math.nan, math.inf
    for causal in (False, True):
        if causal and Lq > 1:   # sequence 1: every query but the last stands in front of its only key
            q[1, :-1], dout[1, :-1] = math.inf, math.nan
        got = check_attention(q, k, v, dout, kv_lens=lens, causal=causal)
        assert not got[0][0].any() and not got[1][0].any() and not got[2][0].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_padding_documents_hold_anything(dtype):
    q, k, v, dout = attention_inputs(6, dtype, 2, 150, 150, 2, 1, 32)
    ids = torch.zeros(2, 150, device="cuda", dtype=torch.int32)
    ids[0, 100:], ids[1, :40] = -1, -1
    for t, value in ((q, math.nan), (k, math.inf), (v, math.nan), (dout, math.nan)):
        t[ids < 0] = value
    got = check_attention(q, k, v, dout, q_docs=ids, k_docs=ids, softcap=10.0)
    assert all(not g[ids < 0].any() for g in got)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_large_and_tiny_values(dtype):
    """scores of +-80 and gradients far from 1 (in half precision: near its smallest and largest numbers)"""
    q, k, v, dout = attention_inputs(7, dtype, 1, 200, 200, 2, 2, 64, spread=20.0)
    small = 2.0 ** -14 if dtype == torch.float16 else 2.0 ** -60
    check_attention(q, k, v, dout * small, causal=True)
    check_attention(q, k, v * 2.0 ** -8, dout * 2.0 ** 8, softcap=50.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_not_finite_inputs_reach_the_result(dtype):
    q, k, v, _ = attention_inputs(8, dtype, 1, 40, 40, 2, 2, 32)
    q[0, 3, 1, 5] = math.nan
    out = ops().token_attention(q, k, v)
    nan = torch.isnan(out)
    assert nan[0, 3, 1].all() and int(nan.sum()) == 32
    q, k, v, _ = attention_inputs(8, dtype, 1, 40, 40, 2, 2, 32)
    k[0, 39, 0, 0] = math.nan
    assert torch.isnan(ops().token_attention(q, k, v)[0, :, 0]).all() and not torch.isnan(ops().token_attention(q, k, v)[0, :, 1]).any()


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_reads_parts_of_a_projection_in_place(dtype):
    B, L, H, Hk, D = 2, 150, 4, 2, 64
    g = gen(9)
    qkv = normal(g, B, L, H + 2 * Hk, D, dtype=dtype)
    dout = normal(g, B, H, L, D, dtype=dtype).transpose(1, 2)          # another order of dimensions
    q, k, v = qkv.split((H, Hk, Hk), dim=2)
    check_attention(q, k, v, dout, causal=True)
    # heads in front of tokens; a broadcast key; channels apart; a start off 16 bytes
    check_attention(q.transpose(1, 2).contiguous().transpose(1, 2), k[:1].expand(B, -1, -1, -1), v, dout, softcap=5.0)
    wide = normal(g, B, L, H, 2 * D, dtype=dtype)
    flat = normal(g, B * L * Hk * D + 1, dtype=dtype)
    check_attention(wide[..., ::2], flat[1:].view(B, L, Hk, D), v, dout)


def test_attention_gradients_of_shared_tensors():
    """one tensor as query, key and value; a broadcast key's gradient is the sum"""
    token_attention = ops().token_attention
    x = normal(gen(10), 2, 60, 2, 32).requires_grad_(True)
    y = token_attention(x, x, x, causal=True)
    (got,) = torch.autograd.grad(y.square().sum(), x)
    want, bound = attention_reference(x, x, x, 2 * y.detach(), causal=True)
    assert_within(got, sum(want[1:]), 2 * sum(bound[1:]), "dx")
    k1 = normal(gen(11), 1, 60, 2, 32).requires_grad_(True)
    (got,) = torch.autograd.grad(token_attention(x, k1.expand(2, -1, -1, -1), x).sum(), k1)
    want, bound = attention_reference(x, k1.expand(2, -1, -1, -1), x, torch.ones_like(y))
    assert_within(got, want[2].sum(0, keepdim=True), 2 * bound[2].sum(0, keepdim=True), "dk")


def test_attention_gradient_against_differences():
    """directional differences of the loss in float32, central, step h: the third-order remainder h^2 and the loss's rounding over h"""
    token_attention = ops().token_attention
    q, k, v, dout = (t.double() for t in attention_inputs(12, torch.float32, 1, 37, 37, 4, 2, 16, spread=1.0))
    kw = dict(softcap=4.0, causal=True, slopes=torch.full((4,), 0.1, device="cuda"))
    f32 = [t.float().requires_grad_(True) for t in (q, k, v)]
    out = token_attention(*f32, **kw)
    grads = torch.autograd.grad(out, f32, dout.float())

    def loss(*xs):
        return float((token_attention(*(x.float() for x in xs), **kw).double() * dout).sum())
    h = 2.0 ** -6
    for n, grad in enumerate(grads):
        d = torch.randn(grad.shape, device="cuda", generator=gen(n), dtype=torch.float64)
        d /= d.norm()
        xs = [[t + (s * h * d if i == n else 0) for i, t in enumerate((q, k, v))] for s in (1, -1)]
        slope = (loss(*xs[0]) - loss(*xs[1])) / (2 * h)
        # rounding: 2368 outputs of size about 1 with errors of a few 2^-22, over h; remainder: |f'''| h^2 / 6 with |f'''| of a few |dout|
        assert abs(slope - float((grad.double() * d).sum())) < 2368 ** 0.5 * 8 * 2.0 ** -22 / h + 20 * h * h, n


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_same_bits_again_and_on_another_stream(dtype):
    q, k, v, dout = attention_inputs(13, dtype, 2, 333, 333, 4, 2, 64)
    ids = (torch.arange(333, device="cuda", dtype=torch.int32) // 50)[None].repeat(2, 1)

    def step():
        qs = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = ops().token_attention(*qs, softcap=30.0, q_docs=ids, k_docs=ids)
        return [out.detach(), *torch.autograd.grad(out, qs, dout)]
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))


def test_attention_empty_sizes():
    token_attention = ops().token_attention
    for B, Lq, Lk in ((0, 5, 5), (2, 0, 5), (2, 5, 0), (1, 0, 0)):
        q, k, v = (torch.randn(B, n, 2, 16, device="cuda").requires_grad_(True) for n in (Lq, Lk, Lk))
        out = token_attention(q, k, v, causal=True)
        assert out.shape == q.shape and not out.any()
        for g in torch.autograd.grad(out, (q, k, v), torch.ones_like(out)):
            assert not g.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_long_cache_past_32_bits(dtype):
    """a cache of more than 2^32 bytes; the last sequence's keys lie past 2^31 elements' worth of bytes"""
    B, Lk, Hk, D = (9, 131072, 8, 128) if dtype == torch.bfloat16 else (9, 65536, 8, 128)
    cache = torch.zeros(2, B, Lk, Hk, D, device="cuda", dtype=dtype)
    g = gen(14)
    cache[:, -1, -700:] = normal(g, 2, 700, Hk, D, dtype=dtype)
    q = normal(g, B, 1, 16, D, dtype=dtype)
    out = ops().token_attention(q, cache[0], cache[1])
    # the zero keys have score 0 and value 0: they only add their count to the sum
    qd, kd, vd = q[-1, 0].double().cpu(), cache[0, -1, -700:].double().cpu(), cache[1, -1, -700:].double().cpu()
    s = torch.einsum("hd,khd->hk", qd, kd.repeat_interleave(2, 1)) * D ** -0.5
    e = s.exp()
    want = torch.einsum("hk,khd->hd", e, vd.repeat_interleave(2, 1)) / (e.sum(-1, keepdim=True) + Lk - 700)
    size = torch.einsum("hk,khd->hd", e, vd.abs().repeat_interleave(2, 1)) / (e.sum(-1, keepdim=True) + Lk - 700)
    u = torch.finfo(dtype).eps / 2
    # roundings of P and of the result; float32 sums of Lk terms, in runs of at most 256 / 4 per wave, joined: 2^-24 times 4096 covers them
    assert_within(out[-1, 0], want, u * want.abs() + (u + 4096 * 2.0 ** -24) * size, "out")
    assert not out[:-1].any()


@pytest.mark.parametrize("rows,keys", [(1, 20000), (4, 5000), (64, 3000), (2000, 2000)])
def test_attention_every_form_of_the_forward_pass(rows, keys):
    """keys split over many workgroups, over the waves of one, and shared by them; keys that some splits do not see"""
    q, k, v, _ = attention_inputs(15, torch.bfloat16, 2, rows, keys, 4, 2, 128)
    lens = torch.tensor([keys, 37], device="cuda", dtype=torch.int32)
    check_attention(q, k, v, kv_lens=lens, softcap=50.0, slopes=torch.tensor([0.5, 0.01, 0.0, 0.1], device="cuda"))
    check_attention(q, k, v, kv_lens=lens, causal=True)


def test_attention_in_a_captured_step():
    """forward and backward of norm, rotation and attention in one graph, replayed between eager steps"""
    t = ops()
    B, L, H, Hk, D = 2, 130, 4, 2, 32
    g = gen(16)
    static = normal(g, B, L, H + 2 * Hk, D, dtype=torch.bfloat16)
    dout = normal(g, B, L, H, D, dtype=torch.bfloat16)
    weights = [(1 + normal(g, D, scale=0.1)).requires_grad_(True) for _ in range(2)]
    cos, sin = t.rotary_tables(L, D, device="cuda")
    ids = (torch.arange(L, device="cuda", dtype=torch.int32) // 40)[None].repeat(B, 1)

    def step():
        x = static.detach().requires_grad_(True)
        q, k, v = x.split((H, Hk, Hk), dim=2)
        q, k = t.qk_norm_rotary(q, k, *weights, cos, sin)
        out = t.token_attention(q, k, v, causal=True, softcap=20.0, q_docs=ids, k_docs=ids)
        return [out.detach(), *torch.autograd.grad(out, (x, *weights), dout)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other):
        held2 = step()
    for n in range(4):
        static.copy_(normal(gen(20 + n), *static.shape, dtype=torch.bfloat16))
        eager = step()
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, held)), n
        assert all(torch.equal(a, b) for a, b in zip(eager, held2)), n


def test_attention_refusals():
    token_attention = ops().token_attention
    q, k, v, _ = attention_inputs(17, torch.bfloat16, 2, 8, 8, 4, 2, 32)
    ids = torch.zeros(2, 8, device="cuda", dtype=torch.int32)
    with pytest.raises(RuntimeError):
        token_attention(q.cpu(), k.cpu(), v.cpu())
    with pytest.raises(RuntimeError):
        token_attention(q, k, v, kv_lens=torch.zeros(2, dtype=torch.int32))
    for bad in (dict(prefix=torch.zeros(2, device="cuda", dtype=torch.int32)), dict(q_docs=ids), dict(k_docs=ids), dict(softcap=-1.0),
                dict(softcap=math.inf), dict(scale=math.nan), dict(kv_lens=torch.zeros(2, device="cuda", dtype=torch.int64)),
                dict(slopes=torch.zeros(3, device="cuda")), dict(slopes=torch.zeros(4, device="cuda").requires_grad_(True)),
                dict(q_docs=ids[:, :4], k_docs=ids), dict(causal=True, prefix=torch.zeros(3, device="cuda", dtype=torch.int32))):
        with pytest.raises(ValueError):
            token_attention(q, k, v, **bad)
    for a, b, c in ((q.double(), k.double(), v.double()), (q, k.float(), v), (q, k, v[:, :4]), (q, k[:1], v[:1]), (q[:, :, :3], k, v), (q[..., :20], k[..., :20], v[..., :20]),
                    (q[0], k[0], v[0])):
        with pytest.raises(ValueError):
            token_attention(a, b, c)


# ---------------------------------------------------------------------------------------------------------------- rotary
ROTARY = [(1, 1, 1, 1, 8, 8), (2, 5, 3, 1, 16, 12), (1, 67, 4, 2, 24, 24), (3, 33, 2, 2, 32, 16), (2, 20, 4, 1, 40, 20), (1, 130, 6, 2, 64, 64), (2, 9, 5, 5, 80, 40),
          (1, 300, 8, 2, 128, 128), (1, 40, 4, 4, 128, 2), (2, 17, 2, 1, 96, 94)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", ROTARY)
def test_rotary_matches_float64(shape, interleaved, dtype):
    B, L, H, Hk, D, R = shape
    g = gen(D + L)
    t = ops()
    qkv = normal(g, B, L, H + 2 * Hk, D, dtype=dtype, scale=3.0)
    q, k = (x.detach().requires_grad_(True) for x in (qkv[:, :, :H], qkv[:, :, H:H + Hk]))
    wtype = torch.float32 if D % 32 == 0 else dtype
    qw, kw = ((1 + normal(g, D, scale=0.3)).to(wtype).requires_grad_(True) for _ in range(2))
    cos, sin = t.rotary_tables(512, R, device="cuda")
    positions = torch.randint(0, 512, (B, L), device="cuda", generator=g) if L % 2 else None
    dq, dk = normal(g, B, L, H, D, dtype=dtype), normal(g, B, Hk, L, D, dtype=dtype).transpose(1, 2)
    out = t.qk_norm_rotary(q, k, qw, kw, cos, sin, positions=positions, eps=1e-5, interleaved=interleaved)
    got = [*out, *torch.autograd.grad(out, (q, k, qw, kw), (dq, dk))]
    want, bound = rotary_reference(q, k, qw, kw, cos, sin, positions, 1e-5, interleaved, dq, dk)
    for a, b, c, n in zip(got, want, bound, ("q", "k", "dq", "dk", "dqw", "dkw")):
        assert_within(a, b, c, n)
    with torch.no_grad():
        again = t.qk_norm_rotary(q, k, qw, kw, cos, sin, positions=positions, eps=1e-5, interleaved=interleaved)
    assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_rotary_many_tokens_without_gains_and_with_one():
    t = ops()
    g = gen(30)
    q, k = (normal(g, 4, 2100, h, 16, dtype=torch.bfloat16).requires_grad_(True) for h in (4, 4))
    cos, sin = t.rotary_tables(2100, 12, device="cuda")
    dq, dk = normal(g, 4, 2100, 4, 16, dtype=torch.bfloat16), normal(g, 4, 2100, 4, 16, dtype=torch.bfloat16)
    kw = (1 + normal(g, 16, scale=0.3)).requires_grad_(True)
    out = t.qk_norm_rotary(q, k, None, kw, cos, sin)
    got = [*out, *torch.autograd.grad(out, (q, k, kw), (dq, dk))]
    want, bound = rotary_reference(q, k, None, kw, cos, sin, dq=dq, dk=dk)
    for a, n in zip(got, (0, 1, 2, 3, 5)):
        assert_within(a, want[n], bound[n], n)
    out = t.qk_norm_rotary(q, k, None, None, cos, sin)
    assert_within(torch.autograd.grad(out, q, (dq, dk))[0] if False else torch.autograd.grad(out, (q, k), (dq, dk))[0], want[2], bound[2], "dq")


def test_rotary_zero_rows_and_positions_outside_the_tables():
    t = ops()
    q = torch.zeros(1, 4, 2, 16, device="cuda").requires_grad_(True)
    k = torch.ones(1, 4, 1, 16, device="cuda").requires_grad_(True)
    cos, sin = t.rotary_tables(8, 8, device="cuda")
    at = torch.tensor([[0, -1, 8, 7]], device="cuda")
    qo, ko = t.qk_norm_rotary(q, k, None, None, cos, sin, positions=at)
    want, bound = rotary_reference(q, k, None, None, cos, sin, at)
    assert_within(qo, want[0], bound[0], "q")
    assert_within(ko, want[1], bound[1], "k")
    assert torch.isnan(ko[0, 1:3, 0, :8]).all() and not torch.isnan(ko[0, 1:3, 0, 8:]).any()
    (dq,) = torch.autograd.grad(qo[0, 0].sum() + ko[0, 0].sum(), q)
    assert torch.isfinite(dq[0, 0]).all()


def test_rotary_empty_and_refusals():
    t = ops()
    g = gen(31)
    q, k = normal(g, 2, 8, 4, 32), normal(g, 2, 8, 2, 32)
    cos, sin = t.rotary_tables(8, 32, device="cuda")
    w = torch.ones(32, device="cuda").requires_grad_(True)
    for B, L in ((0, 8), (2, 0)):
        out = t.qk_norm_rotary(q[:B, :L].requires_grad_(True), k[:B, :L], w, None, cos, sin)
        assert out[0].shape == (B, L, 4, 32)
        assert not torch.autograd.grad(out[0].sum() + out[1].sum(), w)[0].any()
    with pytest.raises(RuntimeError):
        t.qk_norm_rotary(q.cpu(), k.cpu(), None, None, cos, sin)
    with pytest.raises(RuntimeError):
        t.qk_norm_rotary(q, k, torch.ones(32), None, cos, sin)
    for args, kw in (((q, k[:, :4], None, None, cos, sin), {}), ((q, k, torch.ones(16, device="cuda"), None, cos, sin), {}),
                     ((q, k, w.half(), None, cos, sin), {}), ((q, k.half(), None, None, cos, sin), {}), ((q, k, None, None, cos[:4], sin[:4]), {}),
                     ((q, k, None, None, cos.double(), sin.double()), {}), ((q, k, None, None, cos, sin[:, :8]), {}),
                     ((q, k, None, None, cos, sin), dict(eps=-1.0)), ((q, k, None, None, cos, sin), dict(positions=torch.zeros(2, 4, device="cuda", dtype=torch.int64))),
                     ((q, k, None, None, torch.ones(8, 17, device="cuda"), torch.ones(8, 17, device="cuda")), {})):
        with pytest.raises(ValueError):
            t.qk_norm_rotary(*args, **kw)


# ------------------------------------------------------------------------------------------------------------------ clip
def clip_reference(grads, max_norm, eps=1e-6):
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    f = min(1.0, max_norm / (norm + eps))
    return norm, [g.double() * f for g in grads], f


def check_clip(grads, max_norm, out=None):
    norm, want, f = clip_reference(grads, max_norm)
    before = [g.clone() for g in grads]
    got = ops().clip_gradients(grads, max_norm, out=out)
    # float64 sums: the norm's only rounding that counts is that to float32; a result has the factor's, the product's and its own
    assert abs(float(got) - norm) <= 2 * 2.0 ** -24 * norm
    for w, o, b in zip(want, grads if out is None else out, before):
        u = torch.finfo(o.dtype).eps / 2
        # (half of the smallest steps: 2^-24 in float16, 2^-149 in float32, 2^-133 in bfloat16)
        least = {torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134}[o.dtype]
        assert_within(o, w.cpu(), ((u + 3 * 2.0 ** -24) * w.abs() + least).cpu(), "clipped")
        if f == 1.0 and o.dtype == b.dtype:
            assert torch.equal(o, b)
    return got


SIZES = [(1,), (4096,), (4097,), (3, 5, 7), (64, 64, 3, 3), (123457,), (0,), (2,)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("limit", [0.0, 0.37, 1e9])
def test_clip_in_place_and_out_of_place(dtype, limit):
    g = gen(40)
    grads = [normal(g, *s, dtype=dtype) for s in SIZES]
    flat = torch.full((sum(x.numel() for x in grads) + 8,), 7.0, device="cuda")
    out, at = [], 3   # a buffer whose parts do not start on 16 bytes
    for x in grads:
        out.append(flat[at:at + x.numel()].view(x.shape))
        at += x.numel()
    before = [x.clone() for x in grads]
    check_clip(grads, limit, out=out)
    assert all(torch.equal(a, b) for a, b in zip(grads, before)) and (flat[:3] == 7).all() and (flat[at:] == 7).all()
    check_clip(grads, limit)


def test_clip_mixed_types_strides_and_many_tensors():
    g = gen(41)
    grads = [normal(g, 1 + n % 37, 5, dtype=TYPES[n % 3]) for n in range(500)]
    check_clip(grads, 1.0)
    image = normal(g, 4, 6, 8, 8).contiguous(memory_format=torch.channels_last)
    turned = normal(g, 30, 20).t()
    check_clip([image, turned, normal(g, 9)[3:7]], 0.5)


def test_clip_large_values_and_not_finite_norms():
    t = ops()
    check_clip([torch.full((5000,), 1e30, device="cuda"), torch.full((7,), 1e-30, device="cuda")], 1.0)
    check_clip([torch.zeros(10, device="cuda")], 1.0)
    x = [torch.ones(5000, device="cuda"), torch.ones(3, device="cuda")]
    x[0][4999] = math.nan
    assert math.isnan(float(t.clip_gradients(x, 1.0))) and all(torch.isnan(a).all() for a in x)
    x = [torch.ones(5000, device="cuda")]
    x[0][0] = math.inf
    assert math.isinf(float(t.clip_gradients(x, 1.0))) and torch.isnan(x[0][0]) and not x[0][1:].any()
    x = [torch.ones(16, device="cuda")]
    assert float(t.clip_gradients(x, math.inf)) == 4.0 and (x[0] == 1).all()
    assert float(t.clip_gradients([torch.ones(0, device="cuda")], 1.0)) == 0.0


def test_clip_more_than_2_to_the_32_elements():
    x = torch.full(((1 << 32) + 4099,), 2.0, device="cuda", dtype=torch.bfloat16)
    norm = ops().clip_gradients([x], 1.0)
    want = 2.0 * math.sqrt(x.numel())
    assert abs(float(norm) - want) <= 2 * 2.0 ** -24 * want
    value = torch.tensor(2.0 / want).bfloat16()
    assert abs(float(x[0]) / float(value) - 1) <= 2.0 ** -7 and bool((x == x[0]).all())


def test_clip_refusals():
    t = ops()
    a, b = torch.ones(8, device="cuda"), torch.ones(8, device="cuda")
    flat = torch.ones(32, device="cuda")
    with pytest.raises(RuntimeError):
        t.clip_gradients([torch.ones(3)], 1.0)
    for grads, limit, kw in (([], 1.0, {}), ([a], -1.0, {}), ([a], math.nan, {}), ([a, a], 1.0, {}), ([flat[:8], flat[4:12]], 1.0, {}), ([a], 1.0, dict(out=[b, b])),
                             ([a, b], 1.0, dict(out=[b, a])), ([a, b], 1.0, dict(out=[flat[:8], flat[7:15]])), ([a.double()], 1.0, {}),
                             ([torch.ones(4, 4, device="cuda")[:, :2]], 1.0, {}), ([torch.ones(1, device="cuda").expand(8)], 1.0, {}), ([a], 1.0, dict(out=[b[:4]])),
                             ([flat[:8], flat[8:16]], 1.0, dict(out=[flat[4:12], flat[20:28]])), ([a], 1.0, dict(out=[a.half().view(8).view(torch.bfloat16).float()[:4]]))):
        with pytest.raises(ValueError):
            t.clip_gradients(grads, limit, **kw)
    assert float(t.clip_gradients([a, a], math.inf)) == 4.0   # (nothing is written)


def test_clip_captured_and_replayed():
    g = gen(42)
    src = [normal(g, *s) for s in SIZES]
    grads = [x.clone() for x in src]
    t = ops()
    t.clip_gradients(grads, 0.5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = t.clip_gradients(grads, 0.5)
    for n in range(3):
        for x, s in zip(grads, src):
            x.copy_(s * (n + 1) * 0.001 if n == 1 else s * (n + 1))
        eager = [x.clone() for x in grads]
        want = t.clip_gradients(eager, 0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(a, b) for a, b in zip(grads, eager))


# -------------------------------------------------------------------------------------------------- as they are used together
class TokenBlock(torch.nn.Module):
    """x + out_proj(attention(norm and rotation of q and k)), with shared key heads, over packed documents"""

    def __init__(self, width, heads, kv_heads):
        super().__init__()
        self.heads, self.kv_heads, self.dim = heads, kv_heads, width // heads
        self.qkv = torch.nn.Linear(width, (heads + 2 * kv_heads) * self.dim)
        self.out = torch.nn.Linear(width, width)
        self.q_gain, self.k_gain = (torch.nn.Parameter(torch.ones(self.dim)) for _ in range(2))

    def forward(self, x, cos, sin, ids):
        from diffusionmodelscustom_amd.hip_engine import token_linear
        t = ops()
        B, L, C = x.shape
        qkv = token_linear(x, self.qkv.weight, self.qkv.bias).view(B, L, -1, self.dim)
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=2)
        q, k = t.qk_norm_rotary(q, k, self.q_gain, self.k_gain, cos, sin)
        y = t.token_attention(q, k, v, softcap=20.0, causal=True, q_docs=ids, k_docs=ids)
        return x + token_linear(y.view(B, L, C), self.out.weight, self.out.bias)

    def plain(self, x, cos, sin, ids):
        """the same in elementary operations, in the type of x"""
        B, L, C = x.shape
        q, k, v = torch.nn.functional.linear(x, self.qkv.weight, self.qkv.bias).view(B, L, -1, self.dim).split((self.heads, self.kv_heads, self.kv_heads), dim=2)

        def turned(t, gain):
            t = t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt() * gain
            a, b = t.chunk(2, -1)
            c, s = cos.to(x.dtype)[:L, None], sin.to(x.dtype)[:L, None]
            return torch.cat((a * c - b * s, b * c + a * s), -1)
        q, k = turned(q, self.q_gain), turned(k, self.k_gain)
        k, v = (t.repeat_interleave(self.heads // self.kv_heads, 2) for t in (k, v))
        s = 20.0 * torch.tanh(torch.matmul(q.transpose(1, 2), k.permute(0, 2, 3, 1).contiguous()) * self.dim ** -0.5 / 20.0)
        seen = (ids[:, :, None] == ids[:, None]) & (ids >= 0)[:, :, None] & torch.ones(L, L, device=x.device, dtype=torch.bool).tril()
        alive = seen.any(-1)[:, None, :, None]
        p = s.masked_fill(~seen[:, None] & alive, -math.inf).softmax(-1).masked_fill(~alive, 0.0)
        y = torch.matmul(p, v.transpose(1, 2).contiguous()).transpose(1, 2).reshape(B, L, C)
        return x + torch.nn.functional.linear(y, self.out.weight, self.out.bias)


def test_a_training_step_of_a_token_block():
    """projections, norm and rotation, attention, loss, backward, clipping, against the same in float64.

    Bound: the longest sums are those of the weight gradients (260 rows) and of the projections (128 and 256 terms); six products follow
    one another in a gradient, each off by at most 260 * 2^-24 = 1.6e-5 of the sum of its absolute values, which a norm of the result
    under-estimates by a few times: 6 * 1.6e-5 * 5 = 5e-4."""
    from diffusionmodelscustom_amd.training import clip_grad_norm_
    torch.manual_seed(3)
    block = TokenBlock(128, 4, 2).cuda()
    exact = TokenBlock(128, 4, 2).cuda().double()
    exact.load_state_dict({k: v.double() for k, v in block.state_dict().items()})
    cos, sin = ops().rotary_tables(130, 32, device="cuda")
    x, target = torch.randn(2, 130, 128, device="cuda"), torch.randn(2, 130, 128, device="cuda")
    ids = torch.tensor([0] * 40 + [1] * 75 + [-1] * 15, device="cuda", dtype=torch.int32)[None].repeat(2, 1)
    loss = (block(x, cos, sin, ids) - target).square().mean()
    loss.backward()
    norm = clip_grad_norm_(block.parameters(), 0.05)
    want = (exact.plain(x.double(), cos, sin, ids) - target.double()).square().mean()
    want.backward()
    want_norm = torch.nn.utils.clip_grad_norm_(exact.parameters(), 0.05)
    assert float(want_norm) > 0.05
    assert abs(float(loss) - float(want)) < 5e-4 * float(want) and abs(float(norm) - float(want_norm)) < 5e-4 * float(want_norm)
    for (n, p), w in zip(block.named_parameters(), exact.parameters()):
        off = float((p.grad.double() - w.grad).norm() / w.grad.norm())
        assert off < 5e-4, (n, off)


def test_the_training_step_clips():
    """GraphedTrainStep and eager_train_step with max_grad_norm: plain SGD moves the parameters by lr * max_grad_norm"""
    import copy
    from diffusionmodelscustom_amd import DiffusionUtils
    from diffusionmodelscustom_amd.training import GraphedTrainStep, clip_grad_norm_, eager_train_step
    from tests.model_util import build_model
    torch.manual_seed(6)
    base = build_model()
    base.train()
    B = 4
    batch = dict(images=torch.randn(B, 1, 64, 64, device="cuda"), seasons=torch.randint(0, 4, (B,), device="cuda"), cond_images=torch.randn(B, 1, 64, 64, device="cuda"),
                 lsm=torch.rand(B, 1, 64, 64, device="cuda"), topo=torch.randn(B, 1, 64, 64, device="cuda"), t=torch.randint(1, 1000, (B,), device="cuda"),
                 noise=torch.randn(B, 1, 64, 64, device="cuda"))
    du = DiffusionUtils(1000, 1e-4, 0.02, device="cuda")
    lossfunc, limit, lr = torch.nn.MSELoss(), 0.01, 0.5
    norms = []
    for form in ("unclipped", "eager", "graphed"):
        model = copy.deepcopy(base).cuda()
        before = [p.detach().clone() for p in model.parameters()]
        opt = torch.optim.SGD(model.parameters(), lr=lr)
        if form == "graphed":
            step = GraphedTrainStep(model, opt, du, lossfunc, batch, external_draws=True, max_grad_norm=limit)
            for n in range(3):
                if n:
                    with torch.no_grad():
                        for p, b in zip(model.parameters(), before):
                            p.copy_(b)
                step(**batch)
                norms.append(float(step.grad_norm))
        else:
            eager_train_step(model, opt, du, lossfunc, **batch, max_grad_norm=limit if form == "eager" else None)
        moved = math.sqrt(sum(float((p.detach().double() - b.double()).square().sum()) for p, b in zip(model.parameters(), before)))
        if form == "unclipped":
            size = moved / lr
            assert size > 10 * limit
        else:
            # a parameter of size up to about 1 rounds by 2^-25, its change (0.005 over 17 million of them) is of 1e-6: a few per cent of it,
            # of random sign, so that the norm over all is off by the square of that
            assert abs(moved / (lr * limit) - 1) < 1e-2, (form, moved)
    # atomics in torch's own kernels of the step order sums differently: 1e-4 (see test_graphed_train_step_equals_the_eager_loop_body)
    assert all(abs(n / size - 1) < 1e-2 for n in norms), (norms, size)
    model.zero_grad()
    assert float(clip_grad_norm_(model.parameters(), 1.0)) == 0.0
