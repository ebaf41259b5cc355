"""Float64 evaluations of the token operators and, beside each value, how far a kernel of a given type may be from it.

Rounding to a type is off by at most half a step: u = eps / 2 relative (2^-8 bfloat16, 2^-11 float16, 2^-24 float32).  The bounds below add up,
element by element, what the kernels round (results, probabilities, score gradients: u each) and what float32 arithmetic may
lose before that (w = 2^-24 per operation, over the length of the sums), each times the absolute values that it applies to.
"""
import math

import torch

W = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attention_reference(q, k, v, dout=None, scale=None, softcap=0.0, slopes=None, causal=False, prefix=None, kv_lens=None, q_docs=None,
                        k_docs=None):
    """(values, bounds): lists [out] or [out, dq, dk, dv] of float64 tensors on the CPU."""
    dtype = q.dtype
    u = half_step(dtype)
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    B, Lq, H, D = q.shape
    Lk, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    n = torch.full((B,), Lk) if kv_lens is None else kv_lens.cpu().long().clamp(0, Lk)
    i, j = torch.arange(Lq), torch.arange(Lk)
    pos = i[None] + (n - Lq)[:, None]
    seen = (j[None, None] < n[:, None, None]).repeat(1, Lq, 1)
    usable = j[None] < n[:, None]
    if causal:
        past = j[None, None] <= pos[:, :, None]
        if prefix is not None:
            past |= j[None, None] < prefix.cpu().long()[:, None, None]
        seen &= past
    if q_docs is not None:
        a, b = q_docs.cpu(), k_docs.cpu()
        seen &= (a[:, :, None] == b[:, None]) & (a >= 0)[:, :, None]
        usable &= b >= 0
    alive = seen.any(-1)
    # what the operator does not read counts as zero
    q = torch.where(alive[:, :, None, None], q, 0.0).permute(0, 2, 1, 3)
    k = torch.where(usable[:, :, None, None], k, 0.0).permute(0, 2, 1, 3).repeat_interleave(G, 1)
    v = torch.where(usable[:, :, None, None], v, 0.0).permute(0, 2, 1, 3).repeat_interleave(G, 1)
    s = scale * (q @ k.transpose(2, 3))
    s_abs = abs(scale) * (q.abs() @ k.abs().transpose(2, 3))
    es = (D + 4) * W * s_abs                                    # the product's error
    bent = torch.zeros_like(s)
    if softcap:
        bent = torch.tanh(s / softcap)
        s = softcap * bent
        # tanh: a few roundings of values up to 1, times cap (the two-byte types' form 1 - 2 / (1 + e^2y) loses up to 4 W of it more)
        es = es + softcap * 8 * W
    es = es + 4 * W * s.abs()
    if slopes is not None:
        far = slopes.detach().double().cpu().view(1, H, 1, 1) * (pos[:, :, None] - j).abs()[:, None]
        s = s - far
        es = es + 4 * W * (far + s.abs())
    shut = ~seen[:, None]
    s = s.masked_fill(shut, -math.inf)
    top = s.amax(-1, keepdim=True) if Lk else s.new_zeros(B, H, Lq, 1)
    top = torch.where(top == -math.inf, 0.0, top)
    p = (s - top).exp()
    # exponent: the score's error, the maximum's and the difference's rounding; a factor 2 because numerator and denominator both have it
    es = torch.where(shut, 0.0, es)
    ep = 2 * (es.amax(-1, keepdim=True) if Lk else 0.0) + 8 * W * torch.where(shut, 0.0, (s - top).abs()).clamp(max=150) + (Lk + 16) * W
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p @ v
    tiny = 2.0 ** -30 if dtype == torch.float16 else 2.0 ** -120  # below the smallest step of a scaled half-precision P
    out_b = u * out.abs() + ((u + ep + Lk * W) * p + tiny) @ v.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)

    def tokens(t):
        return t.permute(0, 2, 1, 3)

    def fold(t):
        return tokens(t.view(B, Hk, G, *t.shape[2:]).sum(2))
    if dout is None:
        return [tokens(out)], [tokens(out_b)]
    do = torch.where(alive[:, :, None, None], dout.detach().double().cpu(), 0.0).permute(0, 2, 1, 3)
    dp = do @ v.transpose(2, 3)
    dp_b = (D + 2) * W * (do.abs() @ v.abs().transpose(2, 3))
    delta = (do * out).sum(-1, keepdim=True)
    delta_b = (do.abs() * (out_b + (D + 2) * W * out.abs())).sum(-1, keepdim=True)   # from the rounded result
    slope = 1 - bent * bent
    slope_b = 16 * W + 2 * es / max(softcap, 1e-30) if softcap else torch.zeros_like(s)
    ds = p * (dp - delta) * slope
    # each factor's error times the others; the subtraction's rounding
    gap = (dp - delta).abs()
    ds_b = p * (ep * gap * slope + (dp_b + delta_b + 2 * W * (dp.abs() + delta.abs())) * slope + gap * slope_b) + u * ds.abs()
    narrow = 2.0 ** -33 if dtype == torch.float16 else 0.0
    rows_b, cols_b = narrow * ds.abs().amax(-1, keepdim=True), narrow * ds.abs().amax(-2, keepdim=True)
    # numbers under float32's smallest normal one, 2^-126, may count as zero: each score gradient, and each term of a sum
    ds_b = torch.where(shut, 0.0, ds_b + 2.0 ** -126)
    least = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126 * (Lk + Lq * G + 1)
    dq = scale * (ds @ k)
    dq_b = u * dq.abs() + abs(scale) * ((ds_b + rows_b + Lk * W * ds.abs()) @ k.abs()) + least
    dk = scale * (ds.transpose(2, 3) @ q)
    dk_b = abs(scale) * ((ds_b + cols_b + (Lq * G) * W * ds.abs()).transpose(2, 3) @ q.abs())
    dv = p.transpose(2, 3) @ do
    dv_b = ((u + ep + (Lq * G) * W) * p + (2.0 ** -36 if dtype == torch.float16 else 0.0)).transpose(2, 3) @ do.abs()
    dk, dv = fold(dk), fold(dv)
    return ([tokens(out), tokens(dq), dk, dv],
            [tokens(out_b), tokens(dq_b), fold(dk_b) + u * dk.abs() + least, fold(dv_b) + u * dv.abs() + least])


def rotary_reference(q, k, qw, kw, cos, sin, positions=None, eps=1e-6, interleaved=False, dq=None, dk=None):
    """(values, bounds): [q, k] or [q, k, dq, dk, dqw, dkw]"""
    outs, grads = [], []
    for x, w, dy in ((q, qw, dq), (k, kw, dk)):
        dtype = x.dtype
        u = half_step(dtype)
        x, B, L, D = x.detach().double().cpu(), x.shape[0], x.shape[1], x.shape[3]
        wd = torch.ones(D, dtype=torch.float64) if w is None else w.detach().double().cpu()
        at = torch.arange(L)[None].expand(B, L) if positions is None else positions.cpu()
        inside = (at >= 0) & (at < cos.shape[0])
        c, s = (torch.where(inside[..., None], t.double().cpu()[at.clamp(0, cos.shape[0] - 1)], math.nan)[:, :, None] for t in (cos, sin))
        R = 2 * c.shape[-1]

        def turn(t, s, absolute=False):
            a, b = (t[..., 0:R:2], t[..., 1:R:2]) if interleaved else (t[..., :R // 2], t[..., R // 2:R])
            if absolute:
                one, two = a.abs() * c.abs() + b.abs() * s.abs(), b.abs() * c.abs() + a.abs() * s.abs()
            else:
                one, two = a * c - b * s, b * c + a * s
            turned = torch.stack((one, two), -1).flatten(-2) if interleaved else torch.cat((one, two), -1)
            return torch.cat((turned, t[..., R:].abs() if absolute else t[..., R:]), -1)
        rate = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
        n = x * rate
        y = turn(n * wd, s)
        y_abs = turn(n * wd, s, True)
        # the mean's sum (D W / 2 through the root), the root, the division, two products, the rotation's three roundings
        # (half a step of a float16 below 2^-14 is 2^-25, whatever the value)
        least = 2.0 ** -25 if dtype == torch.float16 else 0.0
        outs.append((y, u * y.abs() + (D / 2 + 10) * W * y_abs + least))
        if dy is None:
            continue
        dy = dy.detach().double().cpu()
        g, g_abs = turn(dy, -s), turn(dy, s, True)
        gw, gw_abs = g * wd, g_abs * wd.abs()
        pull = (gw * n).mean(-1, keepdim=True)
        pull_abs = (gw_abs * n.abs()).mean(-1, keepdim=True)
        dx = rate * (gw - n * pull)
        dx_b = u * dx.abs() + (2 * D + 24) * W * rate * (gw_abs + n.abs() * pull_abs) + least
        uw = u if w is None or w.dtype == dtype else W
        dw = (g * n).sum((0, 1, 2))
        terms = B * L * x.shape[2]
        dw_b = uw * dw.abs() + (D / 2 + 16 + min(terms, 4096)) * W * (g_abs * n.abs()).sum((0, 1, 2))
        grads.append((dx, dx_b, dw, dw_b))
    if dq is None:
        return [o[0] for o in outs], [o[1] for o in outs]
    return ([outs[0][0], outs[1][0], grads[0][0], grads[1][0], grads[0][2], grads[1][2]],
            [outs[0][1], outs[1][1], grads[0][1], grads[1][1], grads[0][3], grads[1][3]])


def assert_within(got, want, bound, what):
    """every element within its bound; NaN exactly where NaN is wanted"""
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places"
    over = torch.where(nan, 0.0, (got - want).abs() / (bound + 1e-300))
    over = torch.where(~nan & (got == want), 0.0, over)
    worst = float(over.max()) if over.numel() else 0.0
    at = int(over.argmax()) if over.numel() else 0
    assert worst <= 1.0, (f"{what}: {worst:.3g} times its bound at {at}: {float(got.flatten()[at])!r} for {float(want.flatten()[at])!r}, "
                          f"bound {float(bound.flatten()[at])!r}")
    return worst
