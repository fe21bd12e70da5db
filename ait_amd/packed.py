"""Transformer operators on packed token sequences, with gradients: sequences of any lengths lie one behind another in
[rows, ...] tensors, `cu_seqlens` [n_seq + 1] int32 holds where each begins.

    packed_attention(q, k, v, cu_q, cu_k)                 any lengths, grouped heads, causal or not, caches for new tokens
    relative_buckets / RelativePositionBias               a learned bias of its scores by buckets of the relative position
    gated_norm(x, f, post_weight=..., pre_weight=...)     the norms behind and before a block, its gate and residual scale

The general-length counterparts of the 64-token blocks in ait_amd/system.py (ScaledDotProductAttention,
lib/model/system/Modules.py:16-29; the sinusoid table of PositionalEncoding, lib/model/system/Models.py:26-50; the residual and
LayerNorm behind a sub-layer, lib/model/system/SubLayers.py:98-100).  float32 or
bfloat16 tensors on a GPU; there is no CPU path.  The kernels run on the current stream of the tensors' device, take their
scratch from torch's allocator per call and may be captured into a graph.
"""
import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _lib, ops


def _recorded(op, *tensors):
    """whether a gradient of the call is wanted.  A dual tensor of forward mode, whose tangent the kernels would drop, is refused"""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise _lib.AitHipError(op + ": there is no forward-mode derivative")
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _once(backward):
    """once_differentiable, whose guard of a second derivative is entered only where one is recorded (autograd's worker thread
    pays about 8 us for it, of some 160 us that a small training step takes on the host)"""
    guarded = torch.autograd.function.once_differentiable(backward)
    return lambda ctx, *grads: guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, cu_q, cu_k, k_len, max_q, max_k, causal, scale, bucket_of):
        p, keep = ops.packed_attn_desc(q, k, v, cu_q, cu_k, k_len, max_q, max_k, causal, scale, table, bucket_of)
        o, lse, rest = ops.packed_attn_fwd(p, q, k, v, for_backward=True)
        ctx.save_for_backward(q, k, v, o, lse, rest, *keep)
        ctx.p = p
        return o

    @staticmethod
    @_once
    def backward(ctx, d_o):
        q, k, v, o, lse, rest, *keep = ctx.saved_tensors
        p, n = ctx.p, ctx.needs_input_grad
        ops.packed_attn_point(p, *keep)
        dq, dk, dv, dt = ops.packed_attn_bwd(p, q, k, v, o, rest, d_o, lse, want_table=n[3])
        return dq if n[0] else None, dk if n[1] else None, dv if n[2] else None, dt, None, None, None, None, \
            None, None, None, None


def packed_attention(q, k, v, cu_q, cu_k=None, *, k_len=None, max_q=None, max_k=None, causal=False, scale=None, bias=None):
    """softmax(scale q k^T + bias) v of every sequence and head -> [total_q, heads, d].

    q [total_q, heads, d], k / v [total_k, kv_heads, d] (float32 or bfloat16; head h reads key head h // (heads // kv_heads); any
    strides, views of a fused projection are read in place where their rows are whole 16-byte vectors and copied where not; d a
    multiple of 8 up to 128).  cu_q, cu_k: int32 starts [n_seq + 1], the first 0, not descending; cu_k None: the keys are packed
    like the queries.  k_len int32 [n_seq]: the sequence's keys are the first k_len of its rows -- a cache whose rows behind them
    may hold anything.  causal: the last query is level with the last key and a query sees no later key.  scale: a number, d ** -0.5.
    bias: (table [n_buckets, heads], bucket_of), or a RelativePositionBias.  max_q / max_k: the longest lengths where the host
    knows them; they guide how the work is cut up (a few new tokens against long caches are spread over the key axis; bfloat16
    inference rounds its probabilities to bfloat16 only where max_q * heads / kv_heads is over 128).

    A query that sees no key gives zeros; so do rows behind the last sequence, and neither takes part in a gradient.  Gradients
    of q, k, v and the table, in reverse mode, not differentiable again.  In a captured graph the backward belongs to a forward
    captured with it, while no eager graph of the same leaves is alive (autograd would wait for their streams inside the capture,
    which ends the process: capture first, or with detached leaves)."""
    table = bucket_of = None
    if bias is not None:
        if isinstance(bias, RelativePositionBias):
            bias = bias.weight, bias.bucket_of
        if not (isinstance(bias, (tuple, list)) and len(bias) == 2 and all(torch.is_tensor(t) for t in bias)):
            raise _lib.AitHipError("packed_attention: `bias` must be (table, bucket_of) or a RelativePositionBias")
        table, bucket_of = bias
    if cu_k is None:
        cu_k = cu_q
    if torch.is_tensor(scale) and scale.requires_grad and torch.is_grad_enabled():
        raise _lib.AitHipError("packed_attention: `scale` is a number and gets no gradient (multiply q by a learned one)")
    if all(torch.is_tensor(t) for t in (q, k, v)) and _recorded("packed_attention", q, k, v, table):
        return _PackedAttention.apply(q, k, v, table, cu_q, cu_k, k_len, max_q, max_k, causal, scale, bucket_of)
    p, _keep = ops.packed_attn_desc(q, k, v, cu_q, cu_k, k_len, max_q, max_k, causal, scale, table, bucket_of)
    return ops.packed_attn_fwd(p, q, k, v)[0]


def relative_buckets(n_buckets, max_distance, two_sided, device=None):
    """int32 [2 * max_distance + 1]: the bucket of every relative position key - query from -max_distance to max_distance (those
    further away share the outermost ones').  The bucketing of Raffel et al., "Exploring the Limits of Transfer Learning with a
    Unified Text-to-Text Transformer" (2020), section 2.1: of the n buckets of a side the first n // 2 hold one distance each,
    the others steps of equal ratio up to max_distance.  two_sided: half the buckets for keys behind the query, half for those
    ahead; else all keys ahead share bucket 0.  Borders are found in whole numbers: step t begins at the least distance a with
    (a / e) ** N >= (max_distance / e) ** t, e the exact buckets and N the others."""
    side = n_buckets // 2 if two_sided else n_buckets
    e = side // 2
    if n_buckets <= 0 or (two_sided and n_buckets % 2) or e < 1 or max_distance <= e:
        raise ValueError("relative_buckets: %d buckets%s do not reach from exact steps to a distance of %d"
                         % (n_buckets, " on two sides" if two_sided else "", max_distance))
    if n_buckets > _lib.MAX_BUCKETS or max_distance > _lib.MAX_BIAS_DISTANCE:
        raise ValueError("relative_buckets: at most %d buckets and a distance of %d" % (_lib.MAX_BUCKETS, _lib.MAX_BIAS_DISTANCE))
    N, of = side - e, []
    t = 0
    for a in range(max_distance + 1):
        while t < N - 1 and a >= e and a ** N * e ** (t + 1) >= max_distance ** (t + 1) * e ** N:
            t += 1
        of.append(a if a < e else e + t)
    of[max_distance] = side - 1
    ahead = [side + of[a] for a in range(1, max_distance + 1)] if two_sided else [0] * max_distance
    return torch.tensor(of[::-1] + ahead, dtype=torch.int32, device=device)


class RelativePositionBias(nn.Module):
    """A learned bias per head and bucket of the relative position, for packed_attention(bias=...); as the sinusoid table of
    PositionalEncoding it is shared by all sequences.  weight [n_buckets, n_head]."""

    def __init__(self, n_head, n_buckets=32, max_distance=128, two_sided=True):
        super().__init__()
        self.weight = nn.Parameter(torch.zeros(n_buckets, n_head))
        self.register_buffer("bucket_of", relative_buckets(n_buckets, max_distance, two_sided), persistent=False)


def _f32(t):
    return None if t is None else t.float()


class _GatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, gate, w_post, b_post, w_pre, b_pre, scale, cu_seqlens, layer, eps):
        p, keep = ops.gated_norm_desc(x, f, _f32(w_post), _f32(w_pre), _f32(b_post), _f32(b_pre), gate, _f32(scale), layer, eps, cu_seqlens)
        y, h, stats = ops.gated_norm_fwd(p, x, f, want_stats=True)
        ctx.save_for_backward(stats, *keep)
        ctx.p, ctx.types = p, [None if t is None else t.dtype for t in (w_post, b_post, w_pre, b_pre, scale)]
        return y, h

    @staticmethod
    @_once
    def backward(ctx, dy, dh):
        stats, *keep = ctx.saved_tensors
        p = ctx.p
        ops.gated_norm_point(p, *keep)
        dx, df, dg, *par = ops.gated_norm_bwd(p, keep[0], keep[1], keep[2], stats, dy, dh)
        grads = [dx, df, dg] + [None if t is None else t.to(dt) for t, dt in zip(par, ctx.types)]
        return tuple(g if n else None for g, n in zip(grads, ctx.needs_input_grad)) + (None, None, None)


def gated_norm(x, f, *, post_weight, pre_weight, post_bias=None, pre_bias=None, gate=None, scale=None, kind="rms", eps=1e-6, cu_seqlens=None):
    """The norm behind a block and the one before the next, with what is between them, in one pass over the rows -> (y, h):

        m = norm(f) * post_weight (+ post_bias);   y = x + scale * gate * m;   h = norm(y) * pre_weight (+ pre_bias)

    x [..., width] the residual stream, f the block's output: both float32, both bfloat16, or a float32 stream with a bfloat16
    branch; y is of x's type, h of f's.  kind: "rms" (by the root of the mean square) or "layer" (about the mean).  gate: None,
    one of f's shape and type, or with cu_seqlens (int32 [n_seq + 1], the first 0, not descending) one row per sequence of the
    packed rows of a two-dimensional x; rows behind the last sequence then give zeros.  scale: None or [width], the learned
    factor of the branch.  Parameters are float32 or bfloat16 [width]; sums, statistics and the row between the two norms are
    f32.  width up to 8192; up to 67 million rows of 512, fewer of wider ones (their waves' lanes stay below 2^32)."""
    if kind not in ("rms", "layer"):
        raise ValueError("gated_norm: kind must be 'rms' or 'layer'")
    if not (torch.is_tensor(x) and torch.is_tensor(f) and x.dim() >= 1 and x.shape == f.shape):
        raise _lib.AitHipError("gated_norm: x and f must be tensors of one shape")
    if gate is not None and not torch.is_tensor(gate):
        raise _lib.AitHipError("gated_norm: the gate must be a tensor")
    if cu_seqlens is not None and x.dim() != 2:
        raise _lib.AitHipError("gated_norm: with cu_seqlens x must be [rows, width]")
    for n, t in (("post_weight", post_weight), ("pre_weight", pre_weight), ("post_bias", post_bias), ("pre_bias", pre_bias), ("scale", scale)):
        if t is not None and not (torch.is_tensor(t) and t.dtype in _lib.DTYPES):
            raise _lib.AitHipError("gated_norm: `%s` must be a float32 or bfloat16 tensor" % n)
    shape = x.shape
    if x.dim() != 2:
        if gate is not None and gate.shape != shape:
            raise _lib.AitHipError("gated_norm: a gate without cu_seqlens has x's shape")
        x, f, gate = (None if t is None else t[None] if len(shape) == 1 else t.flatten(0, -2) for t in (x, f, gate))
    if _recorded("gated_norm", x, f, gate, post_weight, post_bias, pre_weight, pre_bias, scale):
        y, h = _GatedNorm.apply(x, f, gate, post_weight, post_bias, pre_weight, pre_bias, scale, cu_seqlens, kind == "layer", eps)
    else:
        p, keep = ops.gated_norm_desc(x, f, _f32(post_weight), _f32(pre_weight), _f32(post_bias), _f32(pre_bias), gate, _f32(scale),
                                      kind == "layer", eps, cu_seqlens)
        y, h, _ = ops.gated_norm_fwd(p, x, f)
    return (y, h) if len(shape) == 2 else (y.view(shape), h.view(shape))
