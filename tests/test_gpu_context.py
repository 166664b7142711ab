"""Long-context decoding operators on the GPU against plain forms in 64 bits: rotary positions over
several axes, sliding-window attention with visible first tokens (forward, gradients, decoding step), the
4-bit paged cache, verification of drafted tokens, and a run of them together.

Tolerances are worst-case bounds computed with each reference: U is half a step of the stored type (bf16
2^-8, fp32 2^-24), counted once for every value that is rounded to that type (the output, the
probabilities and score gradients that enter a product, the saved output), F = 2^-24 times the length of
each 32-bit sum, and 2^-20 for the hardware's exp2 / log2 / sin / cos."""
import math

import numpy as np
import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a GPU")]

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
F = 2.0 ** -24


def _rand(*shape, seed=0, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _close(got, ref, tol, what=""):
    assert got.shape == ref.shape, what
    assert torch.isfinite(got).all(), what
    over = (got.double() - ref).abs() - tol
    assert float(over.max()) <= 0, f"{what}: {float(over.max()):.3g} over the bound at {int(over.argmax())}"


# ------------------------------------------------------------------------------------ rotary ---
def _rope_ref(x, pos, freq, axis, interleaved, sign=1.0):
    """(turned x, bound of the error besides the output's rounding) in 64 bits."""
    P = freq.shape[0]
    x = x.double()
    pos = pos if pos.dim() == 3 else pos.unsqueeze(1).expand(-1, x.shape[0], -1)
    a = (pos[axis.long()].double() * freq.view(-1, 1, 1)).permute(1, 2, 0).unsqueeze(2)
    i = torch.arange(P, device="cuda")
    e1, e2 = (2 * i, 2 * i + 1) if interleaved else (i, i + P)
    y, slack = x.clone(), torch.zeros_like(x)
    x1, x2, c, s = x[..., e1], x[..., e2], a.cos(), sign * a.sin()
    y[..., e1], y[..., e2] = x1 * c - x2 * s, x1 * s + x2 * c
    slack[..., e1] = slack[..., e2] = (x1.abs() + x2.abs()) * 2.0 ** -20
    return y, slack


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,N,H,Hk,hd,pairs,interleaved", [
    (1, 1, 1, 1, 64, 32, False), (3, 17, 12, 12, 64, 32, False), (2, 130, 8, 2, 128, 64, True),
    (2, 9, 3, 1, 80, 20, False), (1, 33, 4, 4, 96, 24, True), (5, 7, 2, 1, 30, 11, False), (1, 2100, 2, 2, 32, 16, False)])
def test_axis_rope(dtype, B, N, H, Hk, hd, pairs, interleaved):
    from capk import context
    dt = DT[dtype]
    q, k = _rand(B, N, H, hd, seed=1, dtype=dt), _rand(B, N, Hk, hd, seed=2, dtype=dt)
    axis = torch.arange(pairs, device="cuda") % 3
    freq = torch.tensor([10000.0 ** (-i / pairs) for i in range(pairs)], dtype=torch.float64, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    pos = torch.randint(-1000, 300000, (3, B, N), generator=g, device="cuda", dtype=torch.int32)
    got = context.axis_rope(q, k, pos, freq, axis, interleaved=interleaved)
    for x, y in zip((q, k), got):
        ref, slack = _rope_ref(x, pos, freq, axis, interleaved)
        _close(y, ref, U[dt] * ref.abs() + slack, "forward")
    # the gradient turns back
    q.requires_grad_(), k.requires_grad_()
    y = context.axis_rope(q, k, pos, freq, axis, interleaved=interleaved)
    w = [_rand(*t.shape, seed=4 + i, dtype=dt) for i, t in enumerate(y)]
    for x, d, u in zip((q, k), torch.autograd.grad(y, (q, k), w), w):
        ref, slack = _rope_ref(u, pos, freq, axis, interleaved, -1.0)
        _close(d, ref, U[dt] * ref.abs() + slack, "gradient")


def test_axis_rope_views_shared_positions_in_place_and_one_side():
    from capk import context, ops
    B, N, H, hd = 2, 21, 4, 64
    freq, axis = context.axis_frequencies((8, 12, 12))
    pos = torch.stack([torch.arange(N), torch.arange(N) // 5, torch.arange(N) % 5]).int().cuda()
    qkv = _rand(B, N, 3, H, hd, seed=5)
    q, k = qkv[:, :, 0], qkv[:, :, 1]
    ref = [_rope_ref(x, pos, freq, axis, False) for x in (q, k)]
    got = context.axis_rope(q, k, pos, freq, axis)
    v0 = qkv[:, :, 2].clone()
    ops.axis_rope(q, k, pos, freq, axis, out_q=q, out_k=k)  # in place, inside the fused buffer
    for y, z, (r, slack) in zip(got, (q, k), ref):
        _close(y, r, F * r.abs() + slack)
        assert torch.equal(y, z)
    assert torch.equal(qkv[:, :, 2], v0)
    t = _rand(B, H, N, hd, seed=6).transpose(1, 2)  # [B, N, H, hd] with heads outside
    y, none = context.axis_rope(t, None, pos, freq, axis)
    r, slack = _rope_ref(t, pos, freq, axis, False)
    _close(y, r, F * r.abs() + slack)
    assert none is None
    odd = _rand(B * N * H * hd + 1, seed=7)[1:].view(B, N, H, hd)  # 4-B aligned only
    y, _ = context.axis_rope(odd, None, pos, freq, axis)
    r, slack = _rope_ref(odd, pos, freq, axis, False)
    _close(y, r, F * r.abs() + slack)
    a = _rand(B, N, H, hd, seed=8).requires_grad_()
    b = _rand(B, N, H, hd, seed=9).requires_grad_()
    context.axis_rope(a, b, pos, freq, axis)[1].sum().backward()  # only k is used
    assert a.grad is None or not a.grad.any()
    r, slack = _rope_ref(torch.ones_like(b), pos, freq, axis, False, -1.0)
    _close(b.grad, r, F * r.abs() + slack)
    assert context.axis_rope(a[:0], b[:0], pos, freq, axis)[0].shape == (0, N, H, hd)


# --------------------------------------------------------------------------------- attention ---
def _see(B, Nq, Nk, window, sinks, key_pad, kv_len):
    last = torch.full((B,), Nk, device="cuda") if kv_len is None else kv_len.clamp(0, Nk).long()
    p = (last - Nq).view(B, 1, 1) + torch.arange(Nq, device="cuda").view(1, Nq, 1)
    j = torch.arange(Nk, device="cuda").view(1, 1, Nk)
    see = (j <= p) & (j < last.view(B, 1, 1))
    if window:
        see &= (j < sinks) | (p - j < window)
    return see if key_pad is None else see & ~key_pad.view(B, 1, Nk)


def _attention_ref(q, k, v, see, do=None, scale=None, u=0.0, up=None):
    """{name: (value, bound)} in 64 bits; u: rounding of outputs, up: of the probabilities."""
    up = u if up is None else up
    B, Nq, H, hd = q.shape
    G = H // k.shape[2]
    scale = hd ** -0.5 if scale is None else scale
    heads = lambda x: x.double().permute(0, 2, 1, 3).repeat_interleave(H // x.shape[2], 1)  # noqa: E731
    back = lambda x: x.permute(0, 2, 1, 3)  # noqa: E731
    q, k, v, see = heads(q), heads(k), heads(v), see.unsqueeze(1)
    hide = ~see
    k, v = (x.nan_to_num(0, 0, 0) if not torch.isfinite(x).all() else x for x in (k, v))
    s = (q @ k.transpose(-1, -2) * scale).masked_fill(hide, -math.inf)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(s - m)
    z = p.sum(-1, keepdim=True)
    lse = (m + z.log()).squeeze(-1)
    p = p / torch.where(z == 0, 1.0, z)
    o = p @ v
    # a probability's relative error: its score's (an hd-term sum) twice, the sum over keys, exp2 and log2
    big = float(((q.abs() @ k.abs().transpose(-1, -2)) * scale * see).max())
    ep = (2 * big * (hd + 4) + big + k.shape[2]) * F + 2.0 ** -20
    A = p @ v.abs()
    out = {"o": (back(o), back((up + 2 * ep) * A + u * o.abs())), "lse": (lse, lse.abs() * 2 * F + ep)}
    if do is None:
        return out
    do = heads(do)
    share = lambda x: back(x.view(B, H // G, G, *x.shape[2:]).sum(2))  # noqa: E731
    dp, delta = do @ v.transpose(-1, -2), (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta) * scale
    # delta from the saved output (its own bound), 32-bit sums over hd
    d_delta = (do.abs() * ((up + 2 * ep) * A + u * o.abs())).sum(-1, keepdim=True) + hd * F * (do * o).abs().sum(-1, keepdim=True)
    d_dp = hd * F * (do.abs() @ v.abs().transpose(-1, -2))
    d_ds = up * ds.abs() + p * scale * (d_delta + d_dp + 2 * ep * (dp.abs() + delta.abs()))
    n = Nq * F * G
    dv, dq, dk = p.transpose(-1, -2) @ do, ds @ k, ds.transpose(-1, -2) @ q
    t_dv = (up + 2 * ep + n) * (p.transpose(-1, -2) @ do.abs())
    t_dq = d_ds @ k.abs() + k.shape[2] * F * (ds.abs() @ k.abs())
    t_dk = d_ds.transpose(-1, -2) @ q.abs() + n * (ds.abs().transpose(-1, -2) @ q.abs())
    for name, x, t in (("dq", back(dq), back(t_dq)), ("dk", share(dk), share(t_dk)), ("dv", share(dv), share(t_dv))):
        out[name] = (x, t + u * x.abs() + 1e-30)
    return out


def _slide_case(dtype, B, Nq, Nk, H, Hk, hd, window, sinks, pad=None, kv_len=None, grad=True, seed=0, scale=None):
    from capk import context, ops
    dt = DT[dtype]
    q, k, v = (_rand(B, n, h, hd, seed=seed + i, dtype=dt) for i, (n, h) in enumerate(((Nq, H), (Nk, Hk), (Nk, Hk))))
    do = _rand(B, Nq, H, hd, seed=seed + 3, dtype=dt) if grad else None
    key_pad = None if pad is None else (torch.arange(Nk, device="cuda") >= torch.tensor(pad, device="cuda").view(B, 1))
    kv_len = None if kv_len is None else torch.tensor(kv_len, dtype=torch.int32, device="cuda")
    ref = _attention_ref(q, k, v, _see(B, Nq, Nk, window, sinks, key_pad, kv_len), do, scale, U[dt])
    o, lse = ops.sliding_attention_fwd(q, k, v, window, sinks, hd ** -0.5 if scale is None else scale, key_pad, kv_len)
    _close(o, *ref["o"], "o")
    inf = torch.isinf(ref["lse"][0])
    assert torch.equal(inf, lse == -math.inf)
    _close(lse.masked_fill(inf, 0), ref["lse"][0].masked_fill(inf, 0), ref["lse"][1].nan_to_num(0, 0).masked_fill(inf, 0), "lse")
    assert not o.permute(0, 2, 1, 3)[inf].any()
    if not grad:
        return
    q, k, v = (x.requires_grad_() for x in (q, k, v))
    kw = dict(window=window, sinks=sinks, scale=scale, key_pad=key_pad, kv_len=kv_len)
    got = torch.autograd.grad(context.sliding_attention(q, k, v, **kw), (q, k, v), do)
    for name, x in zip(("dq", "dk", "dv"), got):
        _close(x, *ref[name], name)
    again = torch.autograd.grad(context.sliding_attention(q, k, v, **kw), (q, k, v), do)
    assert all(torch.equal(a, b) for a, b in zip(got, again))  # deterministic


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,N,H,Hk,hd,window,sinks", [
    (1, 1, 1, 1, 64, 1, 0), (2, 2, 2, 1, 32, 1, 1), (1, 63, 2, 2, 64, 5, 0), (2, 64, 4, 2, 128, 64, 4),
    (1, 65, 3, 1, 96, 200, 0), (1, 129, 2, 1, 80, 16, 3), (1, 200, 2, 2, 8, 0, 0), (2, 333, 4, 1, 64, 50, 130),
    (1, 700, 2, 1, 64, 30, 4), (1, 1300, 2, 1, 128, 100, 131), (1, 900, 1, 1, 64, 900, 900), (1, 1500, 2, 2, 32, 1, 0)])
def test_sliding_attention_sizes(dtype, B, N, H, Hk, hd, window, sinks):
    _slide_case(dtype, B, N, N, H, Hk, hd, window, sinks)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,Nq,Nk,window,sinks,pad,kv_len", [
    (3, 100, 100, 20, 0, (100, 37, 1), None),        # right-padded; late rows see nothing
    (2, 100, 100, 20, 5, (0, 60), None),             # one sequence entirely hidden
    (3, 70, 300, 64, 7, None, (300, 70, 129)),       # chunks against caches of different lengths
    (3, 70, 300, 0, 0, None, (0, 30, 71)),           # fewer keys than queries, none at all
    (2, 40, 1500, 200, 140, (1500, 900), (1400, 1500)),
    (1, 300, 77, 16, 2, None, None),                 # more queries than keys
])
def test_sliding_attention_masks_and_lengths(dtype, B, Nq, Nk, window, sinks, pad, kv_len):
    _slide_case(dtype, B, Nq, Nk, 4, 2, 64, window, sinks, pad, kv_len, seed=11)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,Nq,Nk,H,Hk,hd,window,sinks,pad,kv_len", [
    (1, 1, 1, 1, 1, 64, 1, 0, None, None), (2, 1, 100, 12, 12, 64, 0, 0, None, (100, 1)),
    (3, 1, 1000, 8, 1, 128, 100, 4, None, (1000, 513, 0)), (2, 7, 600, 6, 2, 96, 33, 50, (600, 400), (599, 600)),
    (1, 16, 5000, 8, 1, 128, 0, 0, None, None), (2, 5, 3000, 32, 2, 80, 1024, 197, None, (3, 3000)),
    (1, 16, 40, 6, 1, 32, 3, 0, None, (10,)), (40, 1, 300, 16, 16, 64, 64, 4, None, tuple(range(7, 287, 7)))])
def test_sliding_attention_step(dtype, B, Nq, Nk, H, Hk, hd, window, sinks, pad, kv_len):
    """Few queries: the kernel that splits the keys (gradients run the others)."""
    _slide_case(dtype, B, Nq, Nk, H, Hk, hd, window, sinks, pad, kv_len, seed=21, grad=Nk <= 1000)


def test_sliding_attention_step_matches_prefill_rows():
    """Decoding token by token gives the rows of the whole pass."""
    from capk import context
    B, N, H, Hk, hd, kw = 2, 150, 4, 2, 64, dict(window=40, sinks=3)
    q, k, v = _rand(B, N, H, hd, seed=31), _rand(B, N, Hk, hd, seed=32), _rand(B, N, Hk, hd, seed=33)
    whole = context.sliding_attention(q, k, v, **kw)
    for t in (0, 1, 39, 40, 42, 43, 149):
        n = torch.full((B,), t + 1, dtype=torch.int32, device="cuda")
        one = context.sliding_attention(q[:, t:t + 1], k, v, kv_len=n, **kw)
        ref = _attention_ref(q[:, t:t + 1], k, v, _see(B, 1, N, 40, 3, None, n), u=F)["o"]
        _close(one, *ref)
        _close(whole[:, t:t + 1], *ref)


@pytest.mark.parametrize("Nq", [1, 100])
def test_sliding_attention_hidden_values_are_not_used(Nq):
    """NaN and infinities behind kv_len, under key_pad and before the window change nothing."""
    from capk import context
    B, Nk, H, hd = 2, 400, 2, 64
    q, k, v = (_rand(B, n, H, hd, seed=41 + i, dtype=torch.bfloat16) for i, n in enumerate((Nq, Nk, Nk)))
    n = torch.tensor([300, 350], dtype=torch.int32, device="cuda")
    pad = torch.zeros(B, Nk, dtype=torch.bool, device="cuda")
    pad[:, 290:295] = True
    kw = dict(window=50, sinks=4, key_pad=pad, kv_len=n)
    clean = context.sliding_attention(q, k, v, **kw)
    k2, v2 = k.clone(), v.clone()
    for b in range(B):
        first = int(n[b]) - Nq - 50 + 1
        for x, bad in ((k2, math.nan), (v2, math.inf), (v2, math.nan)):
            x[b, int(n[b]):] = bad
            x[b, 290:295] = bad
            x[b, 4:max(4, first)] = bad
    assert torch.equal(clean, context.sliding_attention(q, k2, v2, **kw))
    k3, v3 = (x.clone().requires_grad_() for x in (k2, v2))
    q3 = q.clone().requires_grad_()
    grads = torch.autograd.grad(context.sliding_attention(q3, k3, v3, **kw).sum(), (q3, k3, v3))
    assert all(torch.isfinite(g).all() for g in grads)


def test_sliding_attention_views_and_orders():
    """Heads outside tokens, fused q/k/v rows, a batch-expanded cache, an unaligned slice and an expanded gradient."""
    from capk import context
    B, N, H, hd = 2, 90, 4, 64
    kw = dict(window=25, sinks=2)
    qkv = _rand(B, N, 3, H, hd, seed=51, dtype=torch.bfloat16)
    q, k, v = qkv.unbind(2)
    ref = _attention_ref(q, k, v, _see(B, N, N, 25, 2, None, None), u=2.0 ** -8)["o"]
    _close(context.sliding_attention(q, k, v, **kw), *ref)
    t = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    _close(context.sliding_attention(*t, **kw), *ref)
    one = [x[:1].expand(B, N, H, hd) for x in (k, v)]
    ref1 = _attention_ref(q, *one, _see(B, N, N, 25, 2, None, None), u=2.0 ** -8)["o"]
    _close(context.sliding_attention(q, *one, **kw), *ref1)
    odd = torch.empty(B, N, H, hd + 4, dtype=torch.bfloat16, device="cuda")[..., 4:]
    odd.copy_(q)
    _close(context.sliding_attention(odd, k, v, **kw), *ref)
    x = [y.detach().clone().requires_grad_() for y in (q, k, v)]
    context.sliding_attention(*x, **kw).sum().backward()  # a gradient of stride 0
    y = [z.detach().clone().requires_grad_() for z in (q, k, v)]
    context.sliding_attention(*y, **kw).backward(torch.ones_like(q))
    assert all(torch.equal(a.grad, b.grad) for a, b in zip(x, y))
    e = context.sliding_attention(q[:, :0], k, v, **kw)
    assert e.shape == (B, 0, H, hd)
    assert not context.sliding_attention(q, k[:, :0], v[:, :0], **kw).any()


def test_sliding_attention_gradient_against_differences():
    from capk import context
    B, N, H, Hk, hd, window, sinks = 1, 70, 2, 1, 32, 20, 3
    x = [_rand(B, N, h, hd, seed=61 + i) for i, h in enumerate((H, Hk, Hk))]
    w = _rand(B, N, H, hd, seed=64).double()
    see = _see(B, N, N, window, sinks, None, None)
    loss = lambda y: float((_attention_ref(*y, see)["o"][0] * w).sum())  # noqa: E731
    leaf = [y.clone().requires_grad_() for y in x]
    grads = torch.autograd.grad(context.sliding_attention(*leaf, window=window, sinks=sinks), leaf, w.float())
    for i, g in enumerate(grads):
        d = _rand(*x[i].shape, seed=65 + i).double()
        h = 1e-4
        ends = [loss([y.double() + (s * h * d if j == i else 0) for j, y in enumerate(x)]) for s in (1, -1)]
        num, ana = (ends[0] - ends[1]) / (2 * h), float((g.double() * d).sum())
        # second-order term h^2 f''' (f''' of this loss is below 1e4 of its gradient's size), 32-bit gradients
        assert abs(num - ana) <= 1e-4 * float((g.double() * d).abs().sum()), (i, num, ana)


def test_sliding_attention_offsets_past_32_bits():
    """A cache of more than 2^31 elements: the sinks at its start and the window at its end."""
    from capk import context
    N, hd, Nq = 17_000_000, 128, 3
    k, v = (torch.zeros(1, N, 1, hd, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    tail = 200
    for x, s in ((k, 71), (v, 72)):
        x[:, :8] = _rand(1, 8, 1, hd, seed=s, dtype=torch.bfloat16)
        x[:, -tail:] = _rand(1, tail, 1, hd, seed=s + 2, dtype=torch.bfloat16)
    for nq in (Nq, 40):
        q = _rand(1, nq, 2, hd, seed=75, dtype=torch.bfloat16)
        got = context.sliding_attention(q, k, v, window=100, sinks=8)
        ks, vs = (torch.cat([x[:, :8], x[:, -tail:]], 1) for x in (k, v))
        _close(got, *_attention_ref(q, ks, vs, _see(1, nq, 8 + tail, 100, 8, None, None), u=2.0 ** -8)["o"])
    del k, v
    torch.cuda.empty_cache()


# ----------------------------------------------------------------------------- 4-bit cache ---
LEVELS = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])


def _kv4_ref(x):
    """What 32-element blocks of x [..., hd] stand for after rounding, element by element in 64 bits."""
    x = x.double().cpu().numpy()
    b = x.reshape(-1, 32)
    out = np.empty_like(b)
    for i, r in enumerate(b):
        if not np.isfinite(r).all():
            out[i] = np.nan
            continue
        amax = np.abs(r).max()
        e = 0
        if amax > 0:
            e = max(-126, math.frexp(amax)[1] - 5)
            while amax > 6 * 2.0 ** e:
                e += 1
        y = np.abs(r) / 2.0 ** e
        d = np.abs(y[:, None] - LEVELS)
        best = d.min(1)
        near = d == best[:, None]
        pick = [next((c for c in np.flatnonzero(n) if c % 2 == 0), np.flatnonzero(n)[0]) for n in near]  # ties: even
        out[i] = np.sign(r) * LEVELS[pick] * 2.0 ** e
    return torch.from_numpy(out.reshape(x.shape)).cuda()


def _table(B, per, pages, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[:B * per].view(B, per).int().cuda()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,n,Hk,hd,page,start", [
    (1, 1, 1, 32, 16, (0,)), (2, 37, 2, 64, 16, (0, 15)), (3, 20, 1, 96, 48, (5, 47, 100)), (2, 70, 3, 128, 64, (63, 1))])
def test_kv4_append_and_read(dtype, B, n, Hk, hd, page, start):
    from capk import context
    dt = DT[dtype]
    k, v = (_rand(B, n, Hk, hd, seed=81 + i, dtype=dt, scale=s) for i, s in enumerate((1.0, 37.0)))
    # all the levels and the ties between them, at several powers of two; a block of zeros; tiny values
    edge = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, -6] * 2, device="cuda")
    for i, s in enumerate((1.0, 2.0 ** -9, 2.0 ** 20, 0.0, 2.0 ** -130)):
        k.view(-1, 32)[i % (k.numel() // 32)] = (edge * s).to(dt)
    cache = context.KV4Cache.empty(B * 12 + 2, Hk, hd, page)
    table = _table(B, 12, B * 12 + 2)
    start = torch.tensor(start, dtype=torch.int32, device="cuda")
    before = cache.codes.clone()
    cache.append(k, v, table, start)
    gk, gv = cache.read(table, start, n, torch.float32)
    assert torch.equal(gk.double(), _kv4_ref(k)) and torch.equal(gv.double(), _kv4_ref(v))
    # nothing beside the written tokens moved
    t = start.long().view(-1, 1) + torch.arange(n, device="cuda")
    at = table.long().gather(1, t // page), t % page
    after = cache.codes.clone()
    for i in (0, 1):
        after[:, i].permute(0, 2, 1, 3)[at] = before[:, i].permute(0, 2, 1, 3)[at]
    assert torch.equal(after, before)


def test_kv4_bad_pages_counts_and_non_finite():
    """Tokens without a page are dropped and read as zeros; count leaves the padded rows alone; a block with an
    infinity or a NaN stands for NaN."""
    from capk import context
    B, n, Hk, hd, page = 3, 40, 1, 64, 16
    k, v = (_rand(B, n, Hk, hd, seed=91 + i) for i in (0, 1))
    k[1, 3, 0, 5], v[1, 4, 0, 40] = math.inf, math.nan
    cache = context.KV4Cache.empty(9, Hk, hd, page)
    table = torch.tensor([[0, -1, 2], [3, 4, 9], [6, 7, 8]], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, 0, 30], dtype=torch.int32, device="cuda")  # the last runs past its table
    count = torch.tensor([40, 40, 12], dtype=torch.int32, device="cuda")
    cache.append(k, v, table, start, count)
    gk, gv = cache.read(table, torch.zeros_like(start), 48, torch.float32)
    rk, rv = (_kv4_ref(x) for x in (k, v))
    for got, ref in ((gk, rk), (gv, rv)):
        got = got.double()
        assert not got[0, 16:32].any() and torch.equal(got[0, :16], ref[0, :16]) and torch.equal(got[0, 32:40], ref[0, 32:])
        assert torch.allclose(got[1, :32], ref[1, :32], rtol=0, atol=0, equal_nan=True) and not got[1, 32:].any()
        assert not got[2, :30].any() and torch.equal(got[2, 30:42], ref[2, :12]) and not got[2, 42:].any()
    assert torch.isnan(gk[1, 3, 0, :32]).all() and torch.isfinite(gk[1, 3, 0, 32:]).all()
    assert torch.isnan(gv[1, 4, 0, 32:]).all()
    # keys without a page are hidden
    q = _rand(B, 1, 2, hd, seed=94)
    kv_len = torch.tensor([40, 2, 42], dtype=torch.int32, device="cuda")
    got = cache.attend(q, table, kv_len)
    see = _see(B, 1, 48, 0, 0, None, kv_len)
    see[0, :, 16:32] = False
    _close(got, *_attention_ref(q, gk, gv, see, u=F)["o"])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,Nq,H,Hk,hd,page,cols,kv_len,window,sinks", [
    (1, 1, 1, 1, 32, 16, 1, (1,), 0, 0), (2, 1, 12, 12, 64, 64, 4, (256, 3), 0, 0), (3, 5, 8, 2, 128, 16, 40, (640, 5, 0), 0, 0),
    (2, 8, 32, 2, 96, 48, 30, (1400, 700), 100, 5), (1, 2, 8, 1, 128, 128, 100, (12800,), 0, 0),
    (2, 1, 16, 4, 64, 32, 70, (2240, 2000), 500, 40), (1, 64, 4, 1, 128, 16, 20, (300,), 0, 0), (1, 3, 4, 4, 64, 16, 3, (2,), 0, 0),
    (70, 1, 4, 2, 64, 32, 5, tuple(range(1, 141, 2)), 40, 2)])
def test_kv4_attention(dtype, B, Nq, H, Hk, hd, page, cols, kv_len, window, sinks):
    from capk import context
    dt = DT[dtype]
    n = cols * page
    cache = context.KV4Cache.empty(B * cols + 5, Hk, hd, page)
    table = _table(B, cols, B * cols + 5, seed=1)
    k, v = (_rand(B, n, Hk, hd, seed=101 + i, scale=2.0) for i in (0, 1))
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    cache.append(k, v, table, zero)
    k, v = cache.read(table, zero, n, torch.float32)
    q = _rand(B, Nq, H, hd, seed=103, dtype=dt)
    kv_len = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
    got = cache.attend(q, table, kv_len, window=window, sinks=sinks)
    _close(got, *_attention_ref(q, k, v, _see(B, Nq, n, window, sinks, None, kv_len), u=U[dt])["o"])


def test_kv4_stale_slots_and_shared_pages():
    """NaN in slots behind the length is never used, and two sequences may read the same pages."""
    from capk import context
    cache = context.KV4Cache.empty(4, 1, 64, 16)
    cache.scales.fill_(255)
    table = torch.tensor([[0, 1], [0, 2]], dtype=torch.int32, device="cuda")
    k = _rand(1, 20, 1, 64, seed=111)
    cache.append(k, k, table[:1], torch.zeros(1, dtype=torch.int32, device="cuda"))
    cache.append(k[:, 16:18], k[:, 16:18], table[1:], torch.full((1,), 16, dtype=torch.int32, device="cuda"))
    q = _rand(1, 1, 2, 64, seed=112).expand(2, 1, 2, 64)
    kv_len = torch.tensor([18, 18], dtype=torch.int32, device="cuda")
    got = cache.attend(q, table, kv_len)
    assert torch.isfinite(got).all() and torch.equal(got[0], got[1])


def test_kv4_offsets_past_32_bits():
    """Pages past 2^31 bytes of codes."""
    from capk import context
    page, Hk, hd = 128, 8, 128
    pages = (1 << 31) // (2 * Hk * page * hd // 2) + 40
    cache = context.KV4Cache(torch.zeros(pages, 2, Hk, page, hd // 2, dtype=torch.uint8, device="cuda"),
                             torch.full((pages, 2, Hk, page, hd // 32), 127, dtype=torch.uint8, device="cuda"))
    table = torch.arange(pages - 1, pages - 4, -1, dtype=torch.int32, device="cuda").view(1, 3)
    k, v = (_rand(1, 300, Hk, hd, seed=121 + i) for i in (0, 1))
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache.append(k, v, table, zero)
    gk, gv = cache.read(table, zero, 300, torch.float32)
    assert torch.equal(gk.double(), _kv4_ref(k)) and torch.equal(gv.double(), _kv4_ref(v))
    q = _rand(1, 2, 16, hd, seed=123)
    n = torch.tensor([300], dtype=torch.int32, device="cuda")
    _close(cache.attend(q, table, n), *_attention_ref(q, gk, gv, _see(1, 2, 300, 0, 0, None, n), u=F)["o"])


# ----------------------------------------------------------------------------- verification ---
def _verify_ref(target, ids, u, draft, draft_len, t):
    """Sequence by sequence in 64 bits on the host."""
    B, K1, V = target.shape
    soft = lambda x: (lambda e: e / e.sum())(np.exp(x - x.max()))  # noqa: E731
    target = target.double().cpu().numpy() / t
    draft = None if draft is None else draft.double().cpu().numpy() / t
    ids, u = ids.cpu().numpy(), u.double().cpu().numpy()
    acc, tok = np.zeros(B, np.int32), np.full((B, K1), -1, np.int64)
    for b in range(B):
        n, length = 0, K1 - 1 if draft_len is None else min(max(int(draft_len[b]), 0), K1 - 1)
        rest = None
        while n < length:
            p = soft(target[b, n])
            x = ids[b, n]
            q = soft(draft[b, n]) if draft is not None else np.eye(1, V, x if 0 <= x < V else V)[0]
            if not (0 <= x < V and u[b, n] * q[x] < p[x]):
                rest = np.maximum(p - q, 0)
                break
            tok[b, n] = x
            n += 1
        if rest is None or not rest.sum() > 0:
            rest = soft(target[b, n])
        c = np.cumsum(rest)
        tok[b, n] = np.argmax(c > u[b, K1 - 1] * c[-1])
        acc[b] = n
    return acc, tok


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,K,V,one_hot,ragged,t", [
    (1, 1, 2, False, False, 1.0), (1, 0, 100, False, False, 1.0), (5, 4, 1000, False, True, 0.7), (3, 7, 4096, True, False, 1.0),
    (2, 3, 4097, False, False, 1.5), (9, 5, 50257, False, True, 1.0), (4, 2, 50257, True, True, 0.9), (40, 1, 7, False, False, 1.0)])
def test_verify_drafts(dtype, B, K, V, one_hot, ragged, t):
    from capk import context
    dt = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(131)
    target = (3 * _rand(B, K + 1, V, seed=132)).to(dt)
    draft = (target[:, :K].float() + _rand(B, K, V, seed=133)).to(dt) if K else None
    ids = torch.randint(0, V, (B, K), generator=g, device="cuda")
    if K:
        best = draft.float().argmax(-1)
        ids = torch.where(torch.rand(B, K, generator=g, device="cuda") < 0.8, best, ids)
    u = torch.rand(B, K + 1, generator=g, device="cuda")
    draft_len = torch.randint(-1, K + 2, (B,), generator=g, device="cuda") if ragged else None
    draft = None if one_hot else draft
    n, tok = context.verify_drafts(target, ids, u, draft, draft_len=draft_len, temperature=t)
    rn, rt = _verify_ref(target, ids, u, draft, draft_len, t)
    assert n.cpu().numpy().tolist() == rn.tolist()
    assert tok.cpu().numpy().tolist() == rt.tolist()


def test_verify_drafts_edges():
    """Padded vocabulary columns, hidden tokens (-inf), ids outside the vocabulary, equal distributions, u at its ends."""
    from capk import context
    B, K, V, ld = 6, 2, 300, 320
    target, draft = _rand(B, K + 1, ld, seed=141), _rand(B, K, ld, seed=142)
    target[..., V:] = draft[..., V:] = 1e30  # never read
    target[:, :, 7] = -math.inf
    draft[1], ids = target[1, :K], torch.randint(0, V, (B, K), device="cuda", generator=torch.Generator("cuda").manual_seed(143))
    ids[0, 0], ids[2, 1], ids[3, 0], ids[4, 0] = 7, V, -1, 5
    u = torch.rand(B, K + 1, device="cuda", generator=torch.Generator("cuda").manual_seed(144))
    u[4], u[5] = 0.0, 1 - 2.0 ** -24
    n, tok = context.verify_drafts(target, ids, u, draft, vocab_size=V)
    rn, rt = _verify_ref(target[..., :V], ids, u, draft[..., :V], None, 1.0)
    assert n.cpu().numpy().tolist() == rn.tolist() and tok.cpu().numpy().tolist() == rt.tolist()
    assert (tok != 7).all()
    # a refusal that leaves no residual (the same rows, an impossible token) draws from the target
    draft[0] = target[0, :K]
    n, tok = context.verify_drafts(target, ids, u, draft, vocab_size=V)
    assert int(n[0]) == 0 and 0 <= int(tok[0, 0]) < V
    # rows of NaN or of nothing but -inf still give a token of the vocabulary
    for bad in (math.nan, -math.inf):
        target[3] = bad
        n, tok = context.verify_drafts(target, ids, u, draft, vocab_size=V)
        assert int(n[3]) == 0 and 0 <= int(tok[3, 0]) < V and (tok[3, 1:] == -1).all()
    # strides: every second row of a larger buffer
    big = _rand(B, 2 * (K + 1), V, seed=145)
    a = context.verify_drafts(big[:, ::2], ids, u, None)
    b = context.verify_drafts(big[:, ::2].contiguous(), ids, u, None)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert context.verify_drafts(target[:0], ids[:0], u[:0], draft[:0], vocab_size=V)[1].shape == (0, K + 1)


# --------------------------------------------------------------------------------- together ---
def _decode_step(state, x, ids, pos, start, u):
    """Rotate, append to the 4-bit cache, attend over it, project to logits and verify: one speculative step."""
    from capk import context
    B, n = x.shape[:2]
    q, k, v = (torch.matmul(x.float(), w).to(x.dtype).view(B, n, -1, 64) for w in state["w"])
    q, k = context.axis_rope(q, k, pos, state["freq"], state["axis"])
    state["cache"].append(k, v, state["table"], start)
    o = state["cache"].attend(q, state["table"], start + n, window=48, sinks=5)
    logits = torch.matmul(o.reshape(B, n, -1).float(), state["head"]).to(x.dtype)
    return o, logits, context.verify_drafts(logits, ids, u)


def _state(B):
    from capk import context
    freq, axis = context.axis_frequencies((8, 12, 12))
    return {"w": [_rand(128, d, seed=151 + d, scale=0.1) for d in (256, 128, 128)], "head": _rand(256, 500, seed=155, scale=0.2),
            "freq": freq, "axis": axis, "cache": context.KV4Cache.empty(20, 2, 64, 16), "table": _table(B, 8, 20, seed=2)}


@pytest.mark.parametrize("dtype", DT)
def test_together(dtype):
    """A prompt in one pass and two speculative steps, against the same computation in 64 bits on what the cache holds."""
    from capk import context
    B, n0, K, dt = 2, 60, 3, DT[dtype]
    s = _state(B)
    x = _rand(B, n0, 128, seed=161, dtype=dt)
    pos = torch.arange(n0, device="cuda", dtype=torch.int32).expand(3, n0).contiguous()
    q, k, v = (torch.matmul(x.float(), w).to(dt).view(B, n0, -1, 64) for w in s["w"])
    q, k = context.axis_rope(q, k, pos, s["freq"], s["axis"])
    o = context.sliding_attention(q, k, v, window=48, sinks=5)
    _close(o, *_attention_ref(q, k, v, _see(B, n0, n0, 48, 5, None, None), u=U[dt])["o"])
    start = torch.zeros(B, dtype=torch.int32, device="cuda")
    s["cache"].append(k, v, s["table"], start)
    start = start + n0
    for step in range(2):
        x = _rand(B, K + 1, 128, seed=162 + step, dtype=dt)
        ids = torch.randint(0, 500, (B, K), device="cuda")
        u = torch.rand(B, K + 1, device="cuda")
        pos = (start.view(1, B, 1) + torch.arange(K + 1, device="cuda", dtype=torch.int32)).expand(3, B, K + 1).contiguous()
        o, logits, (n, tok) = _decode_step(s, x, ids, pos, start, u)
        q = torch.matmul(x.float(), s["w"][0]).to(dt).view(B, K + 1, -1, 64)
        q, _ = context.axis_rope(q, None, pos, s["freq"], s["axis"])
        ck, cv = s["cache"].read(s["table"], torch.zeros_like(start), 128, torch.float32)
        _close(o, *_attention_ref(q, ck, cv, _see(B, K + 1, 128, 48, 5, None, start + K + 1), u=U[dt])["o"])
        rn, rt = _verify_ref(logits, ids, u, None, None, 1.0)
        assert n.cpu().numpy().tolist() == rn.tolist() and tok.cpu().numpy().tolist() == rt.tolist()
        start = start + n + 1


def test_together_captured_and_replayed():
    """The speculative step in a HIP graph: every replay equals the eager call on the same inputs."""
    B, K = 2, 3
    s = _state(B)
    start = torch.tensor([40, 17], dtype=torch.int32, device="cuda")
    x = _rand(B, K + 1, 128, seed=171, dtype=torch.bfloat16)
    ids = torch.randint(0, 500, (B, K), device="cuda")
    u = torch.rand(B, K + 1, device="cuda")
    pos = torch.zeros(3, B, K + 1, dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _decode_step(s, x, ids, pos, start, u)  # (work on another stream than the default one)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, logits, (n, tok) = _decode_step(s, x, ids, pos, start, u)
    for r in range(4):
        x.copy_(_rand(B, K + 1, 128, seed=172 + r, dtype=torch.bfloat16))
        u.copy_(torch.rand(B, K + 1, device="cuda"))
        pos.copy_(torch.full_like(pos, 40 + r))
        start.copy_(torch.tensor([40 + 3 * r, 17 + r], dtype=torch.int32))
        graph.replay()
        got = [t.clone() for t in (o, logits, n, tok)]
        eo, el, (en, et) = _decode_step(s, x, ids, pos, start, u)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (eo, el, en, et))), r


def test_training_pass_captured_and_replayed():
    """Forward and gradients of rotary positions and sliding attention in a graph (fresh leaves, no eager graph alive)."""
    from capk import ops, context
    B, N, H, Hk, hd = 2, 200, 4, 2, 64
    freq, axis = context.axis_frequencies((8, 12, 12))
    pos = torch.arange(N, device="cuda", dtype=torch.int32).expand(3, N).contiguous()
    q, k, v, do = (_rand(B, N, h, hd, seed=181 + i, dtype=torch.bfloat16) for i, h in enumerate((H, Hk, Hk, H)))

    def step():
        rq, rk = ops.axis_rope(q, k, pos, freq, axis)
        o, lse = ops.sliding_attention_fwd(rq, rk, v, 30, 140, hd ** -0.5)
        dq, dk, dv = ops.sliding_attention_bwd(rq, rk, v, o, do, lse, 30, 140, hd ** -0.5)
        return (o, dv) + ops.axis_rope(dq, dk, pos, freq, axis, inverse=True)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for r in range(3):
        for i, t in enumerate((q, k, v, do)):
            t.copy_(_rand(*t.shape, seed=190 + 4 * r + i, dtype=torch.bfloat16))
        graph.replay()
        got = [t.clone() for t in out]
        ref = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, ref)), r


# --------------------------------------------------------------------------------- refusals ---
def test_refusals():
    from capk import context, ops
    from capk._lib import CapkError
    q, k = _rand(2, 5, 4, 64), _rand(2, 5, 2, 64)
    freq, axis = context.axis_frequencies((8, 12, 12))
    pos = torch.zeros(3, 2, 5, dtype=torch.int32, device="cuda")
    for call in (lambda: context.axis_rope(q.half(), k.half(), pos, freq, axis),
                 lambda: context.axis_rope(q, k.bfloat16(), pos, freq, axis),
                 lambda: context.axis_rope(q.cpu(), k, pos, freq, axis),
                 lambda: context.axis_rope(q, k[:1], pos, freq, axis),
                 lambda: context.axis_rope(q, k, pos[:, :, :4], freq, axis),
                 lambda: context.axis_rope(q, k, pos.float(), freq, axis),
                 lambda: context.axis_rope(q, k, pos, freq.float(), axis),
                 lambda: context.axis_rope(q, k, pos, freq, axis[:-1]),
                 lambda: context.axis_rope(q[..., :32], k[..., :32], pos, freq, axis),  # more pairs than the head has
                 lambda: context.sliding_attention(q, k, k, window=-1),
                 lambda: context.sliding_attention(q, k, k, window=1, sinks=-2),
                 lambda: context.sliding_attention(q[:, :, :3], k, k, window=1),
                 lambda: context.sliding_attention(q, k, k[:, :4], window=1),
                 lambda: context.sliding_attention(q[..., :60], k[..., :60], k[..., :60], window=1),
                 lambda: context.sliding_attention(q, k, k, kv_len=torch.ones(3, dtype=torch.int32, device="cuda")),
                 lambda: context.sliding_attention(q, k, k, key_pad=torch.zeros(2, 5, device="cuda")),
                 lambda: ops.sliding_attention_fwd(q[..., 1:], k[..., 1:], k[..., 1:], 1, 0, 1.0),
                 lambda: context.KV4Cache.empty(4, 1, 48), lambda: context.KV4Cache.empty(4, 1, 64, page=20)):
        with pytest.raises((CapkError, ValueError)):
            call()
    c = context.KV4Cache.empty(4, 2, 64, 16)
    t, z = torch.zeros(2, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    u, ids = torch.rand(2, 3, device="cuda"), torch.zeros(2, 2, dtype=torch.int64, device="cuda")
    logits = _rand(2, 3, 50)
    for call in (lambda: c.append(k[..., :32], k[..., :32], t, z), lambda: c.append(k, k, t[:1], z),
                 lambda: c.append(k, k, t.float(), z), lambda: c.append(k, k, t, z[:1]),
                 lambda: c.append(q, q, t, z), lambda: c.read(t, z, 4, torch.float16), lambda: c.read(t, z, -1),
                 lambda: c.attend(_rand(2, 65, 4, 64), t, z), lambda: c.attend(q[:, :, :3], t, z),
                 lambda: c.attend(q, t, None), lambda: c.attend(q, t, z, window=-3),
                 lambda: context.KV4Cache(c.codes[..., :16], c.scales).attend(q, t, z),
                 lambda: context.verify_drafts(logits, ids, u, temperature=0.0),
                 lambda: context.verify_drafts(logits, ids, u, vocab_size=51),
                 lambda: context.verify_drafts(logits, ids[:, :1], u), lambda: context.verify_drafts(logits, ids, u[:, :2]),
                 lambda: context.verify_drafts(logits, ids, u.double()), lambda: context.verify_drafts(logits, ids, u, logits),
                 lambda: context.verify_drafts(logits, ids.float(), u)):
        with pytest.raises((CapkError, ValueError)):
            call()


# --------------------------------------------------------------------------- rarely used calls ---
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd", [64, 96])
def test_kv4_attention_over_non_finite_blocks(dtype, hd):
    """A visible block that stands for NaN makes its heads' queries NaN (all elements for a key, the block's for
    a value), and nothing else."""
    from capk import context
    B, n, Hk = 2, 90, 3
    cache, table = context.KV4Cache.empty(12, Hk, hd, 16), _table(B, 6, 12, seed=3)
    k, v = (_rand(B, n, Hk, hd, seed=201 + i) for i in (0, 1))
    k[0, 70, 0, 40], v[0, 71, 1, 33] = math.nan, math.inf
    k[1, 3], v[1, 4] = math.nan, math.nan  # (hidden by the window)
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    cache.append(k, v, table, zero)
    q = _rand(B, 1, 2 * Hk, hd, seed=203, dtype=DT[dtype])
    o = cache.attend(q, table, zero + n, window=40, sinks=2)[:, 0]
    assert torch.isnan(o[0, :2]).all() and torch.isfinite(o[1]).all() and torch.isfinite(o[0, 4:]).all()
    assert torch.isnan(o[0, 2:4, 32:64]).all() and torch.isfinite(o[0, 2:4, :32]).all() and torch.isfinite(o[0, 2:4, 64:]).all()


@pytest.mark.parametrize("size", [1.0, 2.0 ** 60])
@pytest.mark.parametrize("t", [1e-3, 2.0 ** -40, 1e-30, 1e12])
def test_verify_drafts_temperatures(t, size):
    """Temperatures down to an arg max and up to a flat row, at logits of any size (in steps of 2^-6 of them, so that
    no two probabilities but equal ones are near each other)."""
    from capk import context
    B, K, V = 4, 3, 1000
    target, draft = ((torch.round(_rand(B, n, V, seed=211 + n) * 64) / 64 * size) for n in (K + 1, K))
    ids = target[:, :K].argmax(-1)
    ids[1, 1] = 5
    u = torch.rand(B, K + 1, device="cuda", generator=torch.Generator("cuda").manual_seed(212))
    for d in (draft, None):
        n, tok = context.verify_drafts(target, ids, u, d, temperature=t)
        rn, rt = _verify_ref(target, ids, u, d, None, t)
        assert n.cpu().numpy().tolist() == rn.tolist() and tok.cpu().numpy().tolist() == rt.tolist()


def test_sliding_attention_layouts_that_are_copied():
    """Tokens 2^22 elements apart, an integer key_pad of any non-zero values, and no keys at all."""
    from capk import context
    wide = torch.zeros(20, (1 << 22) // 64, 64, dtype=torch.bfloat16, device="cuda")
    wide[:, :4] = _rand(20, 4, 64, seed=221, dtype=torch.bfloat16)
    q = wide[:, :4].unsqueeze(0)
    assert q.stride(1) == 1 << 22
    pad = torch.zeros(1, 20, dtype=torch.int64, device="cuda")
    pad[0, 3] = 256
    o = context.sliding_attention(q, q, q, window=7, sinks=1, key_pad=pad)
    assert torch.equal(o, context.sliding_attention(*[q.contiguous()] * 3, window=7, sinks=1, key_pad=pad != 0))
    q = torch.full((2, 3, 4, 64), math.inf, device="cuda", requires_grad=True)
    o = context.sliding_attention(q, q[:, :0], q[:, :0])
    o.sum().backward()
    assert o.shape == q.shape and not o.any() and not q.grad.any()


def test_sliding_attention_unseeing_rows_with_any_gradient():
    """Rows before their sequence's first key: whatever their q and do hold, they give zeros and change nothing."""
    from capk import ops
    B, N, H, hd = 1, 700, 2, 64
    q, k, v, do = (_rand(B, N, H, hd, seed=231 + i, dtype=torch.bfloat16) for i in range(4))
    kv_len = torch.tensor([600], dtype=torch.int32, device="cuda")  # rows 0..99 stand before position 0
    args = (0, 0, hd ** -0.5, None, kv_len)
    o, lse = ops.sliding_attention_fwd(q, k, v, *args)
    ref = ops.sliding_attention_bwd(q, k, v, o, do, lse, *args)
    q[:, :100], do[:, :100] = math.nan, math.nan
    o2, lse2 = ops.sliding_attention_fwd(q, k, v, *args)
    got = ops.sliding_attention_bwd(q, k, v, o2, do, lse2, *args)
    assert torch.equal(o, o2) and torch.equal(lse, lse2) and not o[:, :100].any() and not got[0][:, :100].any()
    assert all(torch.equal(a, b) for a, b in zip(ref, got))


def test_one_tensor_for_all_operands():
    """q, k and v the same leaf: its gradient is the sum of the three."""
    from capk import context
    x = _rand(2, 150, 2, 32, seed=241).requires_grad_()
    do = _rand(2, 150, 2, 32, seed=242)
    context.sliding_attention(x, x, x, window=20, sinks=3).backward(do)
    leaves = [x.detach().clone().requires_grad_() for _ in range(3)]
    context.sliding_attention(*leaves, window=20, sinks=3).backward(do)
    three = [t.grad for t in leaves]
    # two additions in either order: a step of 2^-24 each, of sums no larger than the magnitudes'
    bound = 4 * F * sum(g.double().abs() for g in three)
    _close(x.grad, sum(g.double() for g in three), bound)


def test_calls_on_two_streams_and_graphs_that_take_turns():
    """Steps with split keys at once on two streams, and two captured graphs replayed in turn, each with workspaces of
    its own: every result equals the call alone."""
    from capk import context
    n, Hk, hd = 4000, 2, 128
    sets, alone = [], []
    for i in range(2):
        cache, table = context.KV4Cache.empty(64, Hk, hd, 64), torch.randperm(64, device="cuda").int().view(1, 64)
        k, v = (_rand(1, n, Hk, hd, seed=251 + 3 * i + j) for j in (0, 1))
        cache.append(k, v, table, torch.zeros(1, dtype=torch.int32, device="cuda"))
        q = _rand(1, 4, 8, hd, seed=253 + 3 * i, dtype=torch.bfloat16)
        sets.append((q, k.bfloat16(), v.bfloat16(), cache, table, torch.tensor([n], dtype=torch.int32, device="cuda")))

    def call(s):
        q, k, v, cache, table, length = s
        return cache.attend(q, table, length), context.sliding_attention(q, k, v, window=3000, sinks=4)

    alone = [[t.clone() for t in call(s)] for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for r in range(6):
        with torch.cuda.stream(streams[r % 2]):
            got.append(call(sets[r % 2]))
    torch.cuda.synchronize()
    for r, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, alone[r % 2])), r
    graphs, outs = [], []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call(s))
    for r in range(6):
        graphs[r % 2].replay()
        call(sets[(r + 1) % 2])
    torch.cuda.synchronize()
    for o, a in zip(outs, alone):
        assert all(torch.equal(x, y) for x, y in zip(o, a))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,N,H,Hk,hd,window,sinks", [
    (22, 400, 4, 4, 32, 40, 5), (33, 300, 8, 4, 64, 30, 140), (65, 257, 2, 2, 96, 0, 0), (1, 1400, 4, 1, 128, 70, 9),
    (1, 1400, 4, 1, 64, 0, 0), (2, 1000, 6, 1, 32, 5, 300)])
def test_sliding_attention_large_and_small_grids(dtype, B, N, H, Hk, hd, window, sinks):
    """Enough key tiles for every compute unit, and so few that their queries are cut into chunks."""
    _slide_case(dtype, B, N, N, H, Hk, hd, window, sinks)


@pytest.mark.parametrize("B,window,sinks", [(30, 60, 3), (30, 0, 0), (4, 60, 150)])
def test_sliding_attention_grids_of_ragged_sequences(B, window, sinks):
    pad, kv_len = (tuple((1 + k * i) % 301 for i in range(B)) for k in (37, 113))
    _slide_case("bf16", B, 200, 300, 8, 4, 64, window, sinks, pad, None, seed=5)
    _slide_case("bf16", B, 200, 300, 8, 4, 64, window, sinks, None, kv_len, seed=6)


def test_axis_rope_gradient_of_one_output():
    """Only q', only k', neither, and expanded gradients."""
    from capk import context
    freq, axis = context.axis_frequencies((8, 12, 12))
    pos = torch.randint(0, 5000, (3, 2, 9), device="cuda")
    q, k = (_rand(2, 9, h, 64, seed=261 + h).requires_grad_() for h in (4, 2))
    gq, gk = _rand(2, 9, 1, 64, seed=265).expand(2, 9, 4, 64), _rand(2, 9, 2, 64, seed=266)
    both = torch.autograd.grad(context.axis_rope(q, k, pos, freq, axis), (q, k), (gq, gk))
    dq, = torch.autograd.grad(context.axis_rope(q, k, pos, freq, axis)[0], q, gq)
    dk, none = torch.autograd.grad(context.axis_rope(q, k, pos, freq, axis)[1], (k, q), gk, allow_unused=True)
    alone, = torch.autograd.grad(context.axis_rope(q, None, pos, freq, axis)[0], q, gq)
    assert torch.equal(both[0], dq) and torch.equal(both[1], dk) and none is None and torch.equal(alone, dq)
    back, _ = _rope_ref(gq, pos, freq, axis, False, -1.0)
    _close(dq, back, gq.double().abs().amax(-1, keepdim=True).expand_as(back) * 2.0 ** -19 + 2.0 ** -24 * back.abs())


def test_fewer_query_heads_than_key_heads_are_refused():
    """In the forward, in the backward (whose workspace is asked for before its entry checks the sizes) and over the
    4-bit cache."""
    from capk import context, ops
    from capk._lib import CapkError
    q, lse = _rand(1, 20, 1, 64, seed=271), torch.zeros(1, 1, 20, device="cuda")
    for Hk in (2, 3):
        k = _rand(1, 20, Hk, 64, seed=272)
        cache, table = context.KV4Cache.empty(2, Hk, 64, 16), torch.zeros(1, 2, dtype=torch.int32, device="cuda")
        for call in (lambda: ops.sliding_attention_bwd(q, k, k, q, q, lse, 8, 2, 1.0), lambda: ops.sliding_attention_fwd(q, k, k, 8, 2, 1.0),
                     lambda: context.sliding_attention(q, k, k, window=8, sinks=2), lambda: cache.attend(q, table, table[:, 0] + 20)):
            with pytest.raises((CapkError, ValueError)):
                call()


@pytest.mark.parametrize("dtype", DT)
def test_kv4_empty_batches(dtype):
    """No sequences, or no tokens: append, read and attend leave the pages alone and give empty results."""
    from capk import context
    cache, dt = context.KV4Cache.empty(3, 2, 64, 16), DT[dtype]
    before = cache.codes.clone()
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    x, table = _rand(0, 5, 2, 64, dtype=dt), torch.zeros(0, 2, dtype=torch.int32, device="cuda")
    cache.append(x, x, table, none, none)
    k, v = cache.read(table, none, 5, dt)
    assert k.shape == v.shape == (0, 5, 2, 64) and k.dtype == dt
    assert cache.attend(_rand(0, 1, 4, 64, dtype=dt), table, none).shape == (0, 1, 4, 64)
    x, table, zero = _rand(1, 0, 2, 64, dtype=dt), torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    cache.append(x, x, table, zero)
    assert cache.read(table, zero, 0, dt)[0].shape == (1, 0, 2, 64) and torch.equal(cache.codes, before)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,Nq,Nk", [(2, 3, 0), (2, 0, 5), (0, 3, 5), (2, 0, 0)])
def test_sliding_attention_of_nothing(dtype, B, Nq, Nk):
    """No queries, keys or sequences: zeros, gradients of zeros for each operand that asks for one, and the refusals of
    any other call."""
    from capk import context
    from capk._lib import CapkError
    dt = DT[dtype]
    q0, k0, v0 = (_rand(B, n, h, 64, seed=281, dtype=dt) for n, h in ((Nq, 4), (Nk, 2), (Nk, 2)))
    assert not context.sliding_attention(q0, k0, v0, window=3).any()
    for need in ((True, True, True), (False, True, True), (True, False, False), (False, False, True)):
        x = [t.detach().clone().requires_grad_(r) for t, r in zip((q0, k0, v0), need)]
        o = context.sliding_attention(*x, window=3, sinks=1)
        assert o.shape == q0.shape and o.dtype == dt and not o.any()
        o.sum().backward()
        for t, r in zip(x, need):
            assert (t.grad is not None and t.grad.shape == t.shape and not t.grad.any()) if r else t.grad is None
    for call in (lambda: context.sliding_attention(q0.half(), k0.half(), v0.half()), lambda: context.sliding_attention(q0[:, :, :3], k0, v0),
                 lambda: context.sliding_attention(q0, k0[..., :32], v0[..., :32]), lambda: context.sliding_attention(q0, k0, v0, window=-1),
                 lambda: context.sliding_attention(q0, k0, v0, sinks=-1), lambda: context.sliding_attention(q0.cpu(), k0.cpu(), v0.cpu()),
                 lambda: context.sliding_attention(q0, k0, v0, key_pad=torch.zeros(B, Nk + 1, dtype=torch.bool, device="cuda"))):
        with pytest.raises((CapkError, ValueError)):
            call()


# ------------------------------------------------------------------- 32 bits through three parts ---
# fp32 products run as six products of bf16 parts, x = h + m + l.  The bounds below are those of 32-bit arithmetic
# alone (a value of two parts is off by up to 2^-17, 128 F); every test also shows on the CPU that operands of two
# parts would break its bound.  E counts a product x y: three dropped part products (2^-26 in all, F / 4 at most)
# and six additions of at most 2 F each, rounded up.
E = 16 * F


def _full(*shape, seed, scale=1.0):
    """Values in +-[scale, 2 scale) with all 24 bits in use."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(1 << 23, 1 << 24, shape, generator=g).float() * 2.0 ** -23
    return x * scale * (torch.randint(0, 2, shape, generator=g) * 2 - 1)


def _two_parts(x):
    h = x.bfloat16().float()
    return h.double() + (x - h).bfloat16().double()


def _tight(got, ref, tol, planted=None, what=""):
    """`got` within `tol` of `ref`, and the value of two-part operands not."""
    if planted is not None:
        assert float(((planted - ref).abs() - 1.5 * tol).max()) > 0, f"{what}: the bound would not see two parts"
    _close(got.cpu(), ref, tol, what)


def _columns(hd, at, x):
    """[..., hd] with x in one column and zeros beside it."""
    y = torch.zeros(*x.shape, hd)
    y[..., at] = x
    return y


FP32_FORMS = [(1, 12, 2, 64), (1, 300, 2, 32), (1, 300, 2, 64), (1, 300, 1, 80), (1, 300, 2, 128), (32, 300, 4, 32), (32, 300, 4, 64),
              (32, 300, 4, 96), (32, 300, 4, 128)]  # few queries; small grids (two groups, cut queries); large grids


@pytest.mark.parametrize("B,N,H,hd", FP32_FORMS)
def test_fp32_scores_keep_32_bits(B, N, H, hd):
    """One visible key: lse = scale q k.  Off by a product (E), the rounded factor, product with it, ln 2 and result
    (6 F), and log2 (2^-20)."""
    from capk import ops
    q, k = _full(B, N, H, seed=1, scale=16.0), _full(B, N, H, seed=2, scale=8.0)
    v = torch.zeros(B, N, H, hd).cuda()
    lse = ops.sliding_attention_fwd(_columns(hd, 3, q).cuda(), _columns(hd, 3, k).cuda(), v, 1, 0, 0.75)[1]
    ref = 0.75 * q.double() * k.double()
    planted = 0.75 * _two_parts(q) * _two_parts(k)
    t = lambda x: x.permute(0, 2, 1)  # noqa: E731
    _tight(lse, t(ref), t((E + 6 * F) * ref.abs() + 2.0 ** -20), t(planted), "lse")


@pytest.mark.parametrize("B,N,H,hd", FP32_FORMS)
def test_fp32_values_and_gradients_keep_32_bits(B, N, H, hd):
    """Scores of zero and one visible key: P = 1, o = v and dv = do, off by the sums of their three parts (4 F)."""
    from capk import context
    q = torch.zeros(B, N, H, hd).cuda().requires_grad_()
    k, v = (_full(B, N, H, hd, seed=s).cuda().requires_grad_() for s in (3, 4))
    do = _full(B, N, H, hd, seed=5)
    o = context.sliding_attention(q, k, v, window=1)
    dv, = torch.autograd.grad(o, v, do.cuda())
    for got, x, name in ((o, v.detach().cpu(), "o"), (dv, do, "dv")):
        _tight(got.detach(), x.double(), 4 * F * x.double().abs(), _two_parts(x) if N > 16 or name == "dv" else None, name)


@pytest.mark.parametrize("B,N,H,hd", FP32_FORMS)
def test_fp32_probabilities_keep_32_bits(B, N, H, hd):
    """Two visible keys, scores in [-1/2, 1/2): P = exp2(c s - m).  Exponents are off by at most 4 F (the factor, its
    product, the maximum's, their difference), so a P by 3 F and exp2's 2 F, relative.  o with v = 1 at every other
    key is one P over the sum of two: 10 F, the sum of its parts 4 F, of the row F, quotient and product 2 F.  dv with
    do = 1 at every other row is one P recomputed from lse, each rounding at most 2 F where values reach 1.8: c s and its
    difference from lse 4 F; in lse the row's sum, off by 6 F, or 9 F of its log2, log2 itself 2 F, the maximum and
    three roundings 5 F; back to base 2 3 F; 23 F in all, times ln 2 16 F, exp2 2 F, parts 4 F."""
    from capk import context
    k = _full(B, N, H, seed=6, scale=0.25)
    even = (torch.arange(N) % 2 == 0).float()
    q = _columns(hd, 1, torch.ones(B, N, H)).cuda()
    v = even.view(1, N, 1, 1).expand(B, N, H, hd).contiguous().cuda().requires_grad_()
    o = context.sliding_attention(q, _columns(hd, 1, k).cuda(), v, window=2, scale=1.0)
    do = even.view(1, N, 1, 1).expand(B, N, H, hd).contiguous().cuda()
    dv, = torch.autograd.grad(o, v, do)
    s = k.double()
    prev = torch.cat([torch.full_like(s[:, :1], -math.inf), s[:, :-1]], 1)
    top = torch.maximum(s, prev)
    p1, p0 = (s - top).exp(), (prev - top).exp()  # own key, the one before
    z = p1 + p0
    e = even.view(1, N, 1).double()
    ref = (p1 * e + p0 * (1 - e)) / z
    ref[:, 0] = 1
    planted = (_two_parts(p1.float()) * e + _two_parts(p0.float()) * (1 - e)) / z
    planted[:, 0] = 1
    wide = lambda x: x.unsqueeze(-1).expand(B, N, H, hd)  # noqa: E731
    _tight(o.detach(), wide(ref), wide(17 * F * ref), wide(planted) if N > 16 else None, "o")
    own, before = p1 / z, torch.cat([(p0 / z)[:, 1:], torch.zeros_like(s[:, :1])], 1)  # P of key j in rows j and j + 1
    rows = torch.cat([even[1:], torch.zeros(1)]).view(1, N, 1).double()
    ref = own * e + before * rows
    planted = _two_parts(own.float()) * e + _two_parts(before.float()) * rows
    _tight(dv, wide(ref), wide(24 * F * ref), wide(planted), "dv")


@pytest.mark.parametrize("B,N,H,hd", FP32_FORMS)
def test_fp32_score_gradients_keep_32_bits(B, N, H, hd):
    """Two visible keys of score zero (q and k in different columns), P = 1/2; v, q and k are zero at every odd token,
    so a row has one do v = x, dS = +-x / 4, and dq, dk have one term each, scale dS k and scale dS q.  Off by: x (E), P
    (exponent 3 F, times ln 2 2 F, exp2 2 F), D = P x (6 F), x - D = x / 2 (7 F), P again and the product (5 F), the
    last product (E) and the scale (F): 2 E + 13 F."""
    from capk import context
    even = (torch.arange(N) % 2 == 0).float().view(1, N, 1)
    qx, kx, vx = (_full(B, N, H, seed=7 + i) * even for i in range(3))
    dx = _full(B, N, H, seed=10)
    dx[:, 0] = 0
    q, k, v = (_columns(hd, c, x).cuda().requires_grad_() for c, x in ((1, qx), (2, kx), (5, vx)))
    do = _columns(hd, 5, dx).cuda()
    scale = 0.75
    dq, dk, _ = torch.autograd.grad(context.sliding_attention(q, k, v, window=2, scale=scale), (q, k, v), do)

    def grads(q, k, v, d, cut):
        shift = lambda x: torch.cat([torch.zeros_like(x[:, :1]), x[:, :-1]], 1)  # noqa: E731
        own, prev = d * v, d * shift(v)                      # do v^T of a row's two keys, one of them zero
        ds1, ds0 = cut((own - prev) / 4), cut((prev - own) / 4)
        dk0 = torch.cat([(ds0 * q)[:, 1:], torch.zeros_like(q[:, :1])], 1)  # of the row behind, at key j
        return scale * (ds1 * k + ds0 * shift(k)), scale * (ds1 * q + dk0)

    ref = grads(*(x.double() for x in (qx, kx, vx, dx)), lambda x: x)
    planted = grads(*(_two_parts(x) for x in (qx, kx, vx, dx)), lambda x: _two_parts(x.float()))
    for got, r, p, c, name in ((dq, ref[0], planted[0], 2, "dq"), (dk, ref[1], planted[1], 1, "dk")):
        _tight(got[..., c], r, (2 * E + 13 * F) * r.abs(), p if B * N * H > 100 else None, name)  # (of 12 dk all may lie within)


def test_fp32_queries_over_the_4_bit_cache_keep_32_bits():
    """One visible key: lse = scale q k (three part products, 6 F of sums, and 6 F as above); two, with v = 1 and 0:
    o = P_0 / (P_0 + P_1) as above with 3 F more for each score."""
    from capk import context, ops
    B, H, hd = 300, 4, 64
    cache, table = context.KV4Cache.empty(B, 2, hd, 16), torch.arange(B, dtype=torch.int32).view(B, 1).cuda()
    lev = torch.tensor([0.5, 1, 1.5, 2, 3, 4, 6])
    kx = lev[torch.randint(0, 7, (B, 2, 2), generator=torch.Generator().manual_seed(11))] * 0.125
    vx = torch.tensor([1.0, 0.0]).view(1, 2, 1, 1).expand(B, 2, 2, hd)
    cache.append(_columns(hd, 9, kx).cuda(), vx.contiguous().cuda(), table, torch.zeros(B, dtype=torch.int32, device="cuda"))
    kx = kx.repeat_interleave(2, 2)  # [B, 2 keys, H]
    for n, size in ((1, 64.0), (2, 2.0 ** -2)):
        q = _full(B, 1, H, seed=12, scale=size)
        lse = torch.empty(B, H, 1, device="cuda")
        o = ops.kv4_attention(_columns(hd, 9, q).cuda(), cache.codes, cache.scales, table, torch.full((B,), n, device="cuda"), 0, 0,
                              1.0, lse=lse)
        s, cut = (x * kx.double() for x in (q.double(), _two_parts(q)))  # [B, 2, H]
        if n == 1:
            _tight(lse[..., 0], s[:, 0], 12 * F * s[:, 0].abs() + 2.0 ** -20, cut[:, 0], "lse")
        else:
            p = torch.softmax(s, 1)
            e = (s - s.amax(1, keepdim=True)).exp()
            planted = (_two_parts(e.float()) / e.sum(1, keepdim=True))[:, 0]
            # (exponents up to 0.75 log2 e: 2 F and 3 F of the score each; both weighted by the other's share)
            tol = (4 + 2 * 8) * F * p[:, 0] * p[:, 1] + 7 * F * p[:, 0]
            wide = lambda x: x.unsqueeze(-1).expand(B, H, hd)  # noqa: E731
            _tight(o[:, 0], wide(p[:, 0]), wide(tol), wide(planted), "o")


# ------------------------------------------------------------------- what a call may not touch, outputs ---
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("hd,page", [(32, 16), (64, 48), (96, 16), (128, 32)])
def test_kv4_append_leaves_all_other_codes_and_scales(dtype, hd, page):
    """Pages of random bytes: only the written slots change, of codes and of scales, whatever a block holds (zeros, NaN
    and infinities too)."""
    from capk import context
    B, n, Hk, cols = 3, 21, 3, 4
    g = torch.Generator(device="cuda").manual_seed(301)
    pages = B * cols + 3
    codes, scales = (torch.randint(0, 256, (pages, 2, Hk, page, hd // d), generator=g, device="cuda", dtype=torch.uint8) for d in (2, 32))
    cache, table = context.KV4Cache(codes.clone(), scales.clone()), _table(B, cols, pages, seed=4)
    table[1, 1] = -1
    k, v = (_rand(B, n, Hk, hd, seed=302 + i, dtype=DT[dtype]) for i in (0, 1))
    k[0, 2], v[0, 3, 0], k[2, 5, 1, 7], v[2, 6, 2, 0] = 0, 0, math.nan, math.inf
    start = torch.tensor([0, page - 5, 2 * page + 1], dtype=torch.int32, device="cuda")
    count = torch.tensor([n, n, n - 4], dtype=torch.int32, device="cuda")
    cache.append(k, v, table, start, count)
    written = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for b in range(B):
        for t in range(int(start[b]), int(start[b]) + int(count[b])):
            pg = int(table[b, t // page])
            if pg >= 0:
                written[pg, t % page] = True
    for now, before in ((cache.codes, codes), (cache.scales, scales)):
        beside = ~written.view(pages, 1, 1, page, 1).expand_as(now)
        assert torch.equal(now[beside], before[beside])
    # the written slots hold what the same append into cleared pages holds
    clean = context.KV4Cache.empty(pages, Hk, hd, page)
    clean.append(k, v, table, start, count)
    for now, other in ((cache.codes, clean.codes), (cache.scales, clean.scales)):
        at = written.view(pages, 1, 1, page, 1).expand_as(now)
        assert torch.equal(now[at], other[at])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,Nq,H,Hk,hd,cols,kv_len", [
    (70, 3, 8, 8, 64, 4, (0, 1, 2, 3, 50) + tuple(range(5, 64)) + (0, 64, 64, 63, 33, 32)),  # a workgroup for each: not split
    (3, 2, 8, 2, 128, 60, (0, 960, 500))])                                                    # split and joined
def test_kv4_attention_lse(dtype, B, Nq, H, Hk, hd, cols, kv_len):
    """lse of the 4-bit cache, -inf where a query sees nothing."""
    from capk import _lib, context, ops
    dt, page = DT[dtype], 16
    cache, table = context.KV4Cache.empty(B * cols + 1, Hk, hd, page), _table(B, cols, B * cols + 1, seed=5)
    k, v = (_rand(B, cols * page, Hk, hd, seed=311 + i) for i in (0, 1))
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    cache.append(k, v, table, zero)
    k, v = cache.read(table, zero, cols * page, torch.float32)
    kv_len = torch.tensor(kv_len, dtype=torch.int32, device="cuda")
    q, lse = _rand(B, Nq, H, hd, seed=313, dtype=dt), torch.full((B, H, Nq), 7.0, device="cuda")
    split = _lib.load().capk_kv4_attention_workspace(1, B, H, Hk, Nq, hd, 0, 0, page, cols) > 0
    assert split == (B == 3)
    o = ops.kv4_attention(q, cache.codes, cache.scales, table, kv_len, 0, 0, hd ** -0.5, lse=lse)
    ref = _attention_ref(q, k, v, _see(B, Nq, cols * page, 0, 0, None, kv_len), u=U[dt])
    _close(o, *ref["o"], "o")
    none = torch.isinf(ref["lse"][0])
    assert bool(none[0].all()) and torch.equal(none, lse == -math.inf)
    _close(lse.masked_fill(none, 0), ref["lse"][0].masked_fill(none, 0), ref["lse"][1].nan_to_num(0, 0).masked_fill(none, 0), "lse")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("Nq,Nk", [(1, 2000), (5, 40), (150, 150)])
def test_sliding_attention_into_a_strided_output(dtype, Nq, Nk):
    """out= inside a larger buffer, heads outside tokens: the result's bits, and nothing beside them; with and without
    lse, and refusals of another shape, type or alignment."""
    from capk import ops
    from capk._lib import CapkError
    B, H, hd, dt = 2, 4, 64, DT[dtype]
    q, k, v = (_rand(B, n, H, hd, seed=321 + i, dtype=dt) for i, n in enumerate((Nq, Nk, Nk)))
    rule = (30, 2, hd ** -0.5)
    ref, lse = ops.sliding_attention_fwd(q, k, v, *rule)
    big = torch.full((B, H, Nq + 3, hd + 8), 3.0, dtype=dt, device="cuda")
    out = big[:, :, 1:Nq + 1, :hd].transpose(1, 2)
    for want in (True, False):
        out.zero_()
        got, got_lse = ops.sliding_attention_fwd(q, k, v, *rule, out=out, want_lse=want)
        assert got is out and torch.equal(out, ref) and (torch.equal(got_lse, lse) if want else got_lse is None)
        assert (big[:, :, 0] == 3).all() and (big[:, :, Nq + 1:] == 3).all() and (big[..., hd:] == 3).all()
    for bad in (ref[:, :, :2], ref.double(), ref.cpu(), torch.zeros(B, Nq, H, hd + 1, dtype=dt, device="cuda")[..., 1:]):
        with pytest.raises((CapkError, ValueError)):
            ops.sliding_attention_fwd(q, k, v, *rule, out=bad)


# ------------------------------------------------------------------- a chunk of queries over a long cache ---
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("B,Nq,Nk,H,Hk,hd,window,sinks,pad,kv_len,split", [
    (1, 16, 4100, 4, 2, 64, 0, 0, None, None, True), (1, 17, 4100, 4, 2, 64, 0, 0, None, None, True),
    (1, 17, 300, 4, 2, 64, 0, 0, None, None, False), (1, 64, 2500, 8, 1, 128, 0, 0, None, (2311,), True),
    (1, 129, 3000, 3, 1, 80, 2000, 5, (2900,), None, True), (2, 100, 3001, 2, 2, 32, 2200, 300, None, (3001, 60), True),
    (2, 100, 3001, 2, 1, 96, 0, 0, (3000, 5), (2999, 3001), True), (1, 512, 2100, 2, 1, 64, 0, 0, None, None, True),
    (1, 513, 2100, 2, 1, 64, 0, 0, None, None, False), (1, 40, 4000, 4, 2, 64, 100, 3, None, None, False),
    (70, 20, 2100, 6, 6, 32, 0, 0, None, tuple(range(0, 2100, 30)), False)])
def test_sliding_attention_chunks_over_a_long_cache(dtype, B, Nq, Nk, H, Hk, hd, window, sinks, pad, kv_len, split):
    """Both sides of the rule that sends a chunk of queries to the kernel that splits the keys."""
    from capk import _lib
    ws = _lib.load().capk_sliding_attention_fwd_workspace(dtype == "bf16", B, H, Hk, Nq, Nk, hd, window, sinks)
    assert (ws > 0) == split, ws
    _slide_case(dtype, B, Nq, Nk, H, Hk, hd, window, sinks, pad, kv_len, grad=Nq <= 129 and B < 70, seed=331)


def test_windows_and_sinks_past_32_bits():
    """A window or a number of sinks of any size means what it says: past all keys, none are hidden."""
    import sys

    from capk import context
    from capk._lib import CapkError
    q, k = _rand(1, 40, 2, 64, seed=341), _rand(1, 40, 2, 64, seed=342)
    cache, table = context.KV4Cache.empty(4, 2, 64, 16), torch.arange(4, device="cuda").view(1, 4)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    cache.append(k, k, table, zero)
    n = zero + 40
    for nq in (40, 3):
        x = q[:, :nq]
        whole = context.sliding_attention(x, k, k)
        few = context.sliding_attention(x, k, k, window=5)
        for big in (1 << 31, (1 << 32) + 5, (1 << 32) - 1, sys.maxsize):
            assert torch.equal(context.sliding_attention(x, k, k, window=big), whole), big
            assert torch.equal(context.sliding_attention(x, k, k, window=5, sinks=big), whole), big
            assert torch.equal(cache.attend(x, table, n, window=big), cache.attend(x, table, n)), big
            assert torch.equal(cache.attend(x, table, n, window=5, sinks=big), cache.attend(x, table, n)), big
            for kw in (dict(window=-big), dict(sinks=-big)):
                with pytest.raises((CapkError, ValueError)):
                    context.sliding_attention(x, k, k, **kw)
                with pytest.raises((CapkError, ValueError)):
                    cache.attend(x, table, n, **kw)
        assert not torch.equal(few, whole)


@pytest.mark.parametrize("V", [50, 9000])
@pytest.mark.parametrize("dtype", DT)
def test_verify_drafts_rows_with_an_infinity(dtype, V):
    """A target row with +inf has no mass: its draft is refused and token 0 drawn.  A draft row with one accepts nothing,
    and the next token is drawn from the target."""
    from capk import context
    B, K, dt = 3, 2, DT[dtype]
    target, draft = _rand(B, K + 1, V, seed=351, dtype=dt), _rand(B, K, V, seed=352, dtype=dt)
    ids = target[:, :K].float().argmax(-1)
    u = torch.full((B, K + 1), 0.5, device="cuda")
    u[:, :K] = 0
    ref = context.verify_drafts(target, ids, u, draft)
    target[0, 0, V - 3], draft[1, 0, 7] = math.inf, math.inf
    n, tok = context.verify_drafts(target, ids, u, draft)
    assert n.tolist() == [0, 0, K] and tok[0].tolist() == [0, -1, -1] and torch.equal(tok[2], ref[1][2])
    c = torch.softmax(target[1, 0].double(), -1).cumsum(-1)
    assert tok[1].tolist() == [int((c > 0.5 * c[-1]).long().argmax()), -1, -1]


@pytest.mark.parametrize("dtype", DT)
def test_sliding_attention_chunks_and_what_is_hidden(dtype):
    """A chunk that splits its keys: NaN behind kv_len, under key_pad, between the sinks and every window, and in the
    rows before position 0 changes nothing; the replays of a captured call equal the eager ones."""
    from capk import _lib, ops
    B, Nq, Nk, H, hd, dt = 2, 100, 6000, 2, 64, DT[dtype]
    assert _lib.load().capk_sliding_attention_fwd_workspace(dtype == "bf16", B, H, H, Nq, Nk, hd, 2500, 40) > 0
    q, k, v = (_rand(B, n, H, hd, seed=361 + i, dtype=dt) for i, n in enumerate((Nq, Nk, Nk)))
    n = torch.tensor([5500, 60], dtype=torch.int32, device="cuda")
    pad = torch.zeros(B, Nk, dtype=torch.bool, device="cuda")
    pad[:, 5100:5110] = True
    args = (2500, 40, hd ** -0.5, pad, n)
    clean = ops.sliding_attention_fwd(q, k, v, *args)
    for x in (k, v):
        for b in range(B):
            x[b, int(n[b]):] = math.nan
        x[0, 5100:5110], x[0, 40:5500 - Nq - 2500 + 1] = math.nan, math.inf
    q[1, :Nq - 60] = math.nan
    got = ops.sliding_attention_fwd(q, k, v, *args)
    assert all(torch.equal(a, b) for a, b in zip(got, clean)) and not got[0][1, :Nq - 60].any()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = ops.sliding_attention_fwd(q, k, v, *args)
    for r in range(3):
        q.copy_(_rand(B, Nq, H, hd, seed=371 + r, dtype=dt))
        n.copy_(torch.tensor([5000 + r, 200], dtype=torch.int32))
        k.copy_(_rand(B, Nk, H, hd, seed=381 + r, dtype=dt))
        v.copy_(_rand(B, Nk, H, hd, seed=391 + r, dtype=dt))
        graph.replay()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, ops.sliding_attention_fwd(q, k, v, *args))), r
