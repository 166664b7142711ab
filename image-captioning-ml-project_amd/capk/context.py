"""Operators of long-context decoding on libcapk kernels, differentiable where training needs them.

    freq, axis = axis_frequencies((8, 12, 12))              # pairs for time, height, width
    q, k = axis_rope(q, k, pos, freq, axis)                 # [B, N, heads, hd], pos [3, B, N]
    o = sliding_attention(q, k, v, window=1024, sinks=4)    # training, prefill, a decoding step
    cache = KV4Cache.empty(pages, heads, head_dim)          # 4.25 bits per element, paged
    cache.append(k, v, table, start)
    o = cache.attend(q, table, kv_len, window=1024, sinks=4)
    accepted, tokens = verify_drafts(target, ids, u, draft)

axis_rope and sliding_attention have backward passes (once) and no forward-mode derivatives; what the cache holds
and what the verification returns has none: KV4Cache.attend refuses queries that require a gradient, append stores
its tensors' values alone.  The tensor-level wrappers, which know nothing of gradients, are capk.ops.axis_rope, sliding_attention_fwd / _bwd, kv4_* and verify_drafts;
layouts and rules are those of include/capk.h.
"""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import ops
from ._lib import CapkError
from .ops import verify_drafts  # noqa: F401


def axis_frequencies(sections, theta=10000.0, device="cuda"):
    """(freq fp64 [pairs], axis uint8 [pairs]): sections[a] pairs follow axis a, each axis on its own ladder
    theta^(-i / sections[a]).  Any other assignment of frequencies and axes to pairs works as well."""
    if not sections or any(int(n) < 0 for n in sections) or not sum(sections):
        raise ValueError(f"axis_frequencies: sections {sections!r}")
    freq = [theta ** (-i / n) for n in sections for i in range(n)]
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    return (torch.tensor(freq, dtype=torch.float64, device=device), torch.tensor(axis, dtype=torch.uint8, device=device))


def _rows(t):
    """`t` itself where its rows start 16-B aligned with unit element stride, and its tokens less than 2^22
    elements apart, else a contiguous copy."""
    if t is None or t.dim() != 4:
        return t
    n, s, d = 16 // t.element_size(), t.stride(), t.shape
    if (t.data_ptr() % 16 == 0 and (s[3] == 1 or d[3] == 1) and (s[0] % n == 0 or d[0] == 1)
            and ((s[1] % n == 0 and s[1] < 1 << 22) or d[1] == 1) and (s[2] % n == 0 or d[2] == 1)):
        return t
    return t.contiguous()


def _unit(t):
    return t if t is None or t.dim() != 4 or t.stride(3) == 1 else t.contiguous()


def _differentiable(what, *ts):
    """Whether a call on `ts` needs a graph.  A forward-mode dual tensor requires no gradient and would lose its
    tangent without a word, so it is refused."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise CapkError(f"{what} has no forward-mode derivatives")
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


# (The backward passes run in the engine's thread, on a cold core: what can be checked, converted and looked up is,
# in the forward.)
class _AxisRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos, freq, axis, interleaved):
        ctx.set_materialize_grads(False)
        q, k = _unit(q), _unit(k)
        sizes, *table = ops._axis_rope_args(q, k, pos, freq, axis)
        out_q, out_k = q.new_empty(q.shape), None if k is None else k.new_empty(k.shape)
        ops._axis_rope_run(sizes, *table, q, k, out_q, out_k, int(interleaved), 0)
        ctx.save_for_backward(*table)
        ctx.rule = (sizes, int(interleaved))
        return out_q, out_k

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        sizes, interleaved = ctx.rule
        if gq is None and gk is None:
            return None, None, None, None, None, None
        g = [_unit(x) for x in (gq, gk)]
        d = [None if x is None else x.new_empty(x.shape) for x in g]
        first = 0 if gq is not None else 1
        second = 1 if first == 0 else 0
        ops._axis_rope_run(sizes, *ctx.saved_tensors, g[first], g[second], d[first], d[second], interleaved, 1)
        return d[0], d[1], None, None, None, None


def axis_rope(q, k, pos, freq, axis, *, interleaved=False):
    """(q', k') turned by their positions (ops.axis_rope); k may be None.  Differentiable in q and k."""
    if _differentiable("axis_rope", q, k):
        return _AxisRope.apply(q, k, pos, freq, axis, interleaved)
    return ops.axis_rope(_unit(q), _unit(k), pos, freq, axis, interleaved=interleaved)


class _SlidingAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, scale, key_pad, kv_len):
        q, k, v = _rows(q), _rows(k), _rows(v)
        args = ops._sliding_args("sliding_attention", q, k, v, window, sinks, key_pad, kv_len)
        o, lse = ops._sliding_fwd_run(*args, q, scale, q.new_empty(q.shape), True)
        code, dims, rule, _, key_pad, kv_len = args
        ctx.save_for_backward(q, k, v, o, lse, key_pad, kv_len)
        ctx.rule = ((code, *dims), rule, scale)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, key_pad, kv_len = ctx.saved_tensors
        dq, dk, dv = ops._sliding_bwd_run(*ctx.rule, q, k, v, o, _rows(do), lse, key_pad, kv_len)
        return dq, dk, dv, None, None, None, None, None


class _NoAttention(torch.autograd.Function):
    """No queries or no keys: zeros, and zeros as the gradients of all three operands."""

    @staticmethod
    def forward(ctx, q, k, v):
        ctx.shapes = (q.shape, k.shape, v.shape)
        return q.new_zeros(q.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        return tuple(do.new_zeros(s) if need else None for s, need in zip(ctx.shapes, ctx.needs_input_grad))


def sliding_attention(q, k, v, *, window=0, sinks=0, scale=None, key_pad=None, kv_len=None):
    """o [B, Nq, H, hd]: the queries are the last Nq positions of kv_len[b] (default Nk) keys; position p sees
    j <= p with j < sinks or p - j < window (0: no window), less key_pad[b, j].  k / v [B, Nk, Hk, hd] with
    H % Hk == 0; scale defaults to hd ** -0.5.  Differentiable in q, k and v."""
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    track = _differentiable("sliding_attention", q, k, v)
    if q.dim() == 4 and k.dim() == 4 and not (q.numel() and k.numel()):  # nothing to attend, or to
        ops._sliding_args("sliding_attention", q, k, v, window, sinks, key_pad, kv_len)
        if window < 0 or sinks < 0:
            raise ValueError(f"sliding_attention: window {window} and sinks {sinks} must not be negative")
        return _NoAttention.apply(q, k, v) if track else q.new_zeros(q.shape)
    if track:
        return _SlidingAttention.apply(q, k, v, window, sinks, scale, key_pad, kv_len)
    return ops.sliding_attention_fwd(_rows(q), _rows(k), _rows(v), window, sinks, scale, key_pad, kv_len,
                                     want_lse=False)[0]


class KV4Cache:
    """Pages of keys and values in 4 bits: codes [pages, 2, heads, page, hd/2] and scales [pages, 2, heads, page,
    hd/32] (uint8).  The caller keeps the page tables (int [B, pages of a sequence]) and lengths, as one table
    serves every layer's cache; a page may stand in several tables (shared prefixes, beams) as long as
    no call appends to the same slot twice."""

    def __init__(self, codes, scales):
        self.codes, self.scales = codes, scales

    @classmethod
    def empty(cls, pages, heads, head_dim, page=64, device="cuda"):
        if head_dim % 32 or not 32 <= head_dim <= 128 or page % 16 or not 16 <= page <= 4096 or pages < 1 or heads < 1:
            raise ValueError(f"KV4Cache: {pages} pages of {page} tokens, {heads} heads x {head_dim}: need head_dim "
                             "32, 64, 96 or 128 and pages of a multiple of 16 tokens, up to 4096")
        return cls(torch.zeros(pages, 2, heads, page, head_dim // 2, dtype=torch.uint8, device=device),
                   torch.full((pages, 2, heads, page, head_dim // 32), 127, dtype=torch.uint8, device=device))

    def append(self, k, v, table, start, count=None):
        """The values of k, v [B, n, heads, hd] become tokens start[b] + i (i < count[b]); tokens without a page are
        dropped."""
        ops.kv4_append(_rows(k), _rows(v), self.codes, self.scales, table, start, count)

    def read(self, table, start, n, dtype=torch.bfloat16):
        """(k, v) [B, n, heads, hd] of tokens start[b] + i: the values the cache stands for."""
        return ops.kv4_read(self.codes, self.scales, table, start, n, dtype)

    def attend(self, q, table, kv_len, *, window=0, sinks=0, scale=None):
        """o [B, Nq, H, hd] of the last Nq <= 64 tokens of kv_len[b], visible as in sliding_attention.  For decoding:
        a q that requires a gradient is refused (detach it, or call under torch.no_grad())."""
        if _differentiable("KV4Cache.attend", q):
            raise CapkError("KV4Cache.attend has no gradient: detach q, or call it under torch.no_grad()")
        scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
        return ops.kv4_attention(_rows(q), self.codes, self.scales, table, kv_len, window, sinks, scale)
