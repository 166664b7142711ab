"""Refusals of the long-context entry points that need no GPU: the C entries check their arguments before
any launch, the Python ones their tensors' devices."""
import pytest
import torch

OK, EINVAL = 0, -1
P = 1 << 20  # an aligned address that no refused call may touch


def _lib():
    from capk import _lib
    return _lib.load()


def _rope(L, dtype=0, B=1, N=4, hd=64, pairs=32, axes=3, pos=P, Hq=2, q=P, Hk=1, k=P):
    return L.capk_axis_rope(dtype, B, N, hd, pairs, 0, 0, axes, pos, N, 0, P, P, Hq, q, 0, hd, hd, P, 0, hd, hd, Hk, k, 0,
                            hd, hd, P, 0, hd, hd, None)


def test_axis_rope_refusals():
    L = _lib()
    for kw in (dict(dtype=2), dict(B=-1), dict(N=-1), dict(hd=0), dict(pairs=0), dict(pairs=33), dict(axes=0), dict(Hq=0),
               dict(Hk=-1), dict(pos=None), dict(q=None), dict(k=None), dict(hd=2048)):
        assert _rope(L, **kw) == EINVAL, kw
        assert b"capk_axis_rope" in L.capk_last_error()
    assert _rope(L, B=0) == OK and _rope(L, N=0) == OK  # nothing to do


def _fwd(L, dtype=1, B=1, H=4, Hk=2, Nq=40, Nk=50, hd=64, window=8, sinks=2, q=P, rs=256, o=P, ws=None, wsb=0):
    return L.capk_sliding_attention_fwd(dtype, B, H, Hk, Nq, Nk, hd, 1.0, window, sinks, q, 0, rs, 64, P, 0, 128, 64, P, 0,
                                        128, 64, None, None, o, 0, 256, 64, None, ws, wsb, None)


def test_sliding_attention_refusals():
    L = _lib()
    for kw in (dict(dtype=3), dict(B=0), dict(H=3), dict(Hk=0), dict(Nq=0), dict(Nk=0), dict(hd=60), dict(hd=136), dict(window=-1),
               dict(sinks=-1), dict(q=None), dict(q=P + 2), dict(rs=257), dict(o=None), dict(Nk=1 << 29), dict(B=70000)):
        assert _fwd(L, **kw) == EINVAL, kw
    need = L.capk_sliding_attention_fwd_workspace(1, 1, 4, 2, 1, 100000, 64, 0, 0)
    assert need > 0
    assert _fwd(L, Nq=1, Nk=100000, window=0, sinks=0) == EINVAL  # a step without its workspace
    assert _fwd(L, Nq=1, Nk=100000, window=0, sinks=0, ws=P, wsb=need - 1) == EINVAL
    assert L.capk_sliding_attention_fwd_workspace(1, 1, 4, 2, 1000, 100000, 64, 0, 0) == 0
    # the backward's workspace covers the far queries of the keys that stay visible, and on small grids the chunks
    # of the near ones
    small = L.capk_sliding_attention_bwd_workspace(8, 8, 8, 5000, 5000, 64, 100, 0)
    assert small == 64 * 5000 * 4
    assert L.capk_sliding_attention_bwd_workspace(8, 8, 8, 5000, 5000, 64, 100, 4) > small
    assert L.capk_sliding_attention_bwd_workspace(1, 4, 2, 5000, 5000, 64, 100, 0) > 4 * 5000 * 4


def test_kv4_and_verify_refusals():
    L = _lib()

    def append(dtype=1, B=1, n=4, Hk=2, hd=64, k=P, codes=P, pages=8, page=16, table=P, ld=4, cols=4, start=P):
        return L.capk_kv4_append(dtype, B, n, Hk, hd, k, 0, 128, 64, P, 0, 128, 64, codes, P, pages, page, table, ld, cols,
                                 start, None, None)

    for kw in (dict(dtype=5), dict(hd=48), dict(hd=160), dict(page=8), dict(page=24), dict(page=8192), dict(pages=0), dict(codes=None),
               dict(codes=P + 4), dict(table=None), dict(cols=0), dict(ld=3), dict(k=None), dict(k=P + 8), dict(start=None), dict(Hk=0),
               dict(n=-1), dict(page=4096, ld=1 << 20, cols=1 << 20)):
        assert append(**kw) == EINVAL, kw
    assert append(n=0) == OK and append(B=0) == OK

    def attend(Nq=1, H=4, Hk=2, window=0, sinks=0, kv_len=P, ws=P, wsb=1 << 40, cols=64):
        return L.capk_kv4_attention(1, 1, H, Hk, Nq, 64, 1.0, window, sinks, P, 0, 256, 64, P, P, 8, 64, P, cols, cols, kv_len, P,
                                    0, 256, 64, None, ws, wsb, None)

    for kw in (dict(Nq=0), dict(Nq=65), dict(H=3), dict(window=-1), dict(sinks=-1), dict(kv_len=None), dict(wsb=0), dict(ws=None),
               dict(ws=P + 4)):
        assert attend(**kw) == EINVAL, kw

    def verify(B=2, K=3, V=1000, temperature=1.0, target=P, ids=P, ws=P, wsb=1 << 40):
        return L.capk_verify_drafts(0, B, K, V, target, 0, 0, None, 0, 0, ids, 0, P, 0, None, temperature, P, P, K + 1, ws, wsb, None)

    for kw in (dict(B=-1), dict(K=-1), dict(V=0), dict(K=2000), dict(B=60000), dict(temperature=0.0), dict(temperature=-1.0),
               dict(temperature=float("nan")), dict(temperature=float("inf")), dict(target=None), dict(ids=None), dict(ws=None),
               dict(wsb=8), dict(ws=P + 4)):
        assert verify(**kw) == EINVAL, kw
    assert verify(B=0) == OK


def test_python_entry_points_need_a_gpu():
    from capk import context
    from capk._lib import CapkError
    q = torch.zeros(1, 2, 2, 64)
    freq, axis = context.axis_frequencies((8, 12, 12), device="cpu")
    assert freq.shape == (32,) and axis.tolist() == [0] * 8 + [1] * 12 + [2] * 12 and float(freq[8]) == 1.0
    cache = context.KV4Cache.empty(2, 2, 64, 16, device="cpu")
    table, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (lambda: context.axis_rope(q, q, torch.zeros(3, 2, dtype=torch.int32), freq, axis),
                 lambda: context.sliding_attention(q, q, q, window=1),
                 lambda: cache.append(q, q, table, n), lambda: cache.read(table, n, 1), lambda: cache.attend(q, table, n),
                 lambda: context.verify_drafts(torch.zeros(1, 2, 9), torch.zeros(1, 1, dtype=torch.int64), torch.zeros(1, 2))):
        with pytest.raises(CapkError):
            call()
    for bad in ((), (0, 0), (4, -1)):
        with pytest.raises(ValueError):
            context.axis_frequencies(bad, device="cpu")
    for bad in (dict(pages=0, heads=1, head_dim=64), dict(pages=1, heads=0, head_dim=64), dict(pages=1, heads=1, head_dim=40),
                dict(pages=1, heads=1, head_dim=64, page=17)):
        with pytest.raises(ValueError):
            context.KV4Cache.empty(device="cpu", **bad)


def test_scale_stride_and_size_limits():
    L = _lib()

    def fwd(scale=1.0, rs=128, Nq=40, Nk=50, B=1, H=2):
        return L.capk_sliding_attention_fwd(1, B, H, 2, Nq, Nk, 64, scale, 8, 2, P, 0, 128, 64, P, 0, rs, 64, P, 0, 128, 64, None,
                                            None, P, 0, 128, 64, None, None, 0, None)

    for bad in (0.0, -1.0, float("inf"), float("nan")):
        assert fwd(scale=bad) == EINVAL
        assert L.capk_kv4_attention(1, 1, 4, 2, 1, 64, bad, 0, 0, P, 0, 256, 64, P, P, 8, 64, P, 4, 4, P, P, 0, 256, 64, None, P,
                                    1 << 30, None) == EINVAL
    assert fwd(rs=1 << 22) == EINVAL and fwd(rs=-128) == EINVAL
    assert fwd(B=65535, H=65534, Nq=1 << 20) == EINVAL  # more workgroups than a launch has
    for kw in (dict(hd=514), dict(Hq=1000, Hk=25), dict(B=1 << 20, N=1 << 20)):
        assert _rope(L, **kw) == EINVAL, kw
    assert L.capk_verify_drafts(0, 1, 1, 9, P, 0, 0, None, 0, 0, P, 0, P, 0, None, 1e-310, P, P, 2, P, 1 << 20, None) == EINVAL


def test_backward_workspace_stays_small():
    """Partial sums of the far queries, for few and many keys that stay visible."""
    L = _lib()
    for N, Hk, G, hd in ((16384, 4, 1, 128), (16384, 1, 8, 128), (65536, 2, 4, 64), (4096, 8, 2, 128)):
        for window in (1, 128, 2000):
            for sinks in (1, 4, 200, 2048, N // 2, N):
                for B in (1, 4):
                    size = L.capk_sliding_attention_bwd_workspace(B, Hk * G, Hk, N, N, hd, window, sinks)
                    assert size <= B * Hk * G * N * 4 + (1 << 29), (N, Hk, G, hd, window, sinks, B)


def test_workspace_queries_of_refused_sizes():
    """A size that the entry refuses has a workspace of 0 bytes: the query neither divides by a group of no heads nor
    overflows."""
    L = _lib()
    for B, H, Hk, Nq, Nk, hd in ((1, 1, 2, 20, 20, 64), (1, 3, 2, 20, 20, 64), (1, 0, 1, 20, 20, 64), (1, 1, 0, 20, 20, 64),
                                 (0, 1, 1, 20, 20, 64), (1, 1 << 28, 1, 16, 20, 64), (1, 1, 1, 2, (1 << 31) - 1, 64), (1, 1, 1, 20, 20, 0)):
        assert L.capk_sliding_attention_bwd_workspace(B, H, Hk, Nq, Nk, hd, 8, 2) == 0, (B, H, Hk, Nq, Nk, hd)
        assert L.capk_sliding_attention_fwd_workspace(1, B, H, Hk, min(Nq, 16), Nk, hd, 8, 2) == 0, (B, H, Hk, Nq, Nk, hd)
    for kw in (dict(H=1), dict(H=3), dict(H=1 << 27, Hk=1), dict(Nq=0), dict(Nq=65), dict(page=4096, cols=1 << 20), dict(cols=0), dict(B=0)):
        a = dict(dict(B=1, H=2, Hk=2, Nq=64, page=64, cols=1000), **kw)
        assert L.capk_kv4_attention_workspace(1, a["B"], a["H"], a["Hk"], a["Nq"], 64, 0, 0, a["page"], a["cols"]) == 0, kw
    assert L.capk_kv4_attention_workspace(1, 1, 2, 2, 64, 64, 0, 0, 64, 1000) > 0
    # (the same overflow in the entry itself)
    assert L.capk_kv4_attention(1, 1, 1 << 30, 1, 64, 64, 1.0, 0, 0, P, 0, 256, 64, P, P, 8, 64, P, 4, 4, P, P, 0, 256, 64, None, P,
                                1 << 30, None) == EINVAL


def test_kv4_empty_batches():
    """A batch of no sequences, whose tensors have no memory, is nothing to do."""
    L = _lib()
    assert L.capk_kv4_append(1, 0, 4, 2, 64, None, 0, 128, 64, None, 0, 128, 64, P, P, 8, 16, None, 4, 4, None, None, None) == OK
    assert L.capk_kv4_read(1, 0, 4, 2, 64, P, P, 8, 16, None, 4, 4, None, None, 0, 128, 64, None, 0, 128, 64, None) == OK
    assert L.capk_kv4_attention(1, 0, 4, 2, 1, 64, 1.0, 0, 0, None, 0, 256, 64, P, P, 8, 64, None, 4, 4, None, None, 0, 256, 64,
                                None, None, 0, None) == OK
    # with sequences the table is needed
    assert L.capk_kv4_append(1, 1, 4, 2, 64, P, 0, 128, 64, P, 0, 128, 64, P, P, 8, 16, None, 4, 4, P, None, None) == EINVAL
    assert L.capk_kv4_attention(1, 1, 4, 2, 1, 64, 1.0, 0, 0, P, 0, 256, 64, P, P, 8, 64, None, 4, 4, P, P, 0, 256, 64, None, P,
                                1 << 30, None) == EINVAL


def test_derivatives_are_not_dropped():
    """Forward-mode tangents, and a gradient through attention over the 4-bit cache, are refused in words (ahead of
    the refusal of a tensor that is not on a GPU)."""
    import torch.autograd.forward_ad as fw

    from capk import context
    from capk._lib import CapkError
    x = torch.ones(1, 2, 2, 64)
    pos, (freq, axis) = torch.zeros(3, 2, dtype=torch.int32), context.axis_frequencies((8, 12, 12), device="cpu")
    cache, table = context.KV4Cache.empty(2, 2, 64, 16, device="cpu"), torch.zeros(1, 2, dtype=torch.int32)
    n = torch.ones(1, dtype=torch.int32)
    with fw.dual_level():
        d = fw.make_dual(x, x)
        for call in (lambda: context.axis_rope(d, x, pos, freq, axis), lambda: context.axis_rope(x, d, pos, freq, axis),
                     lambda: context.axis_rope(d, None, pos, freq, axis), lambda: context.sliding_attention(d, x, x, window=1),
                     lambda: context.sliding_attention(x, d, x, window=1), lambda: context.sliding_attention(x, x, d, window=1),
                     lambda: context.sliding_attention(x, x[:, :0], d[:, :0]), lambda: cache.attend(d, table, n)):
            with pytest.raises(CapkError, match="forward-mode"):
                call()
        with pytest.raises(CapkError, match="GPU|device"):  # (no tangent: the usual refusal)
            context.axis_rope(x, x, pos, freq, axis)
    g = x.clone().requires_grad_()
    with pytest.raises(CapkError, match="no gradient"):
        cache.attend(g, table, n)
    for q in (g.detach(), g):
        with torch.no_grad(), pytest.raises(CapkError, match="GPU|device"):
            cache.attend(q, table, n)


def test_kv4_pages_that_no_call_takes():
    from capk import context
    for page in (4112, 8192):
        with pytest.raises(ValueError):
            context.KV4Cache.empty(1, 1, 64, page, device="cpu")
    assert context.KV4Cache.empty(1, 1, 64, 4096, device="cpu").codes.shape == (1, 2, 1, 4096, 32)
