"""QKNormRotation and RelativeAttention: attention over the tokens of an image or a sequence (the
rows of an equirectangular image, which close on themselves; its pixels in scan order; a decoder's
tokens over a cache).  No counterpart in the reference; the work is done by the HIP kernels behind
`_C.qk_norm_rotate_*` and `_C.relative_attention_*`."""
import torch
import torch.nn as nn

from .. import _C


class FirstDerivative(torch.autograd.Function):
    """A gradient that depends on what it was computed from in a way that is not differentiated
    again: on the inputs too, since the output's gradient need not be a variable (that of a plain
    sum is not)."""

    @staticmethod
    def forward(ctx, gradient, *computed_from):
        return gradient

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("second derivatives through the attention layers are not supported")


def first_derivatives(gradients, *computed_from):
    if not torch.is_grad_enabled():  # no graph of the backward pass is recorded
        return tuple(gradients)
    return tuple(None if g is None else FirstDerivative.apply(g, *computed_from) for g in gradients)


class QKNormRotationFunction(torch.autograd.Function):

    @staticmethod
    def forward(ctx, query, key, query_weight, key_weight, cos, sin, positions, eps, adjacent):
        ctx.save_for_backward(query, key, query_weight, key_weight, cos, sin, positions)
        ctx.eps, ctx.adjacent = eps, adjacent
        return tuple(_C.qk_norm_rotate_forward(query, key, query_weight, key_weight, cos, sin,
                                               positions, eps, adjacent))

    @staticmethod
    def backward(ctx, grad_query, grad_key):
        grads = _C.qk_norm_rotate_backward(grad_query, grad_key, *ctx.saved_tensors, ctx.eps,
                                           ctx.adjacent, needs=tuple(ctx.needs_input_grad[:4]))
        return first_derivatives(grads, grad_query, grad_key, *ctx.saved_tensors[:4]) + (None,) * 5


class QKNormRotation(nn.Module):
    """Every head of every token of queries and keys divided by its root mean square, times a weight
    per value, and its first values turned in pairs by the angles of the token's place.  Parameters
    of another type than the data are cast to it, as under mixed precision."""

    def __init__(self, head_dim, eps=1e-6, adjacent=False):
        super().__init__()
        self.eps, self.adjacent = eps, adjacent
        self.query_weight = nn.Parameter(torch.ones(head_dim))
        self.key_weight = nn.Parameter(torch.ones(head_dim))

    def forward(self, query, key, cos, sin, positions=None):
        """query [B, L, Hq, D], key [B, L, Hk, D]; cos, sin float32 [places, F] (see
        util.rotation_table); positions int64 [B, L], or the index along L -> (query, key)."""
        return QKNormRotationFunction.apply(query, key, self.query_weight.to(query.dtype),
                                            self.key_weight.to(query.dtype), cos, sin, positions,
                                            self.eps, self.adjacent)


class RelativeAttentionFunction(torch.autograd.Function):

    @staticmethod
    def forward(ctx, query, key, value, table, buckets, zero, scale, causal, query_start,
                key_lengths, recording):
        ctx.args = dict(bucket_zero=zero, scale=scale, causal=causal)
        training = recording and any(ctx.needs_input_grad[:4])
        out, saved = _C.relative_attention_forward(
            query, key, value, table, buckets, query_start=query_start, key_lengths=key_lengths,
            for_backward=training, **ctx.args)
        if training:
            ctx.save_for_backward(query, key, value, table, buckets, query_start, key_lengths, out,
                                  *saved)
        return out

    @staticmethod
    def backward(ctx, grad_output):
        query, key, value, table, buckets, start, lengths, out, *saved = ctx.saved_tensors
        needs = tuple(ctx.needs_input_grad[:4])
        grads = _C.relative_attention_backward(
            grad_output, query, key, value, out, saved, table, buckets, query_start=start,
            key_lengths=lengths, needs=needs, **ctx.args)
        return first_derivatives(grads, grad_output, query, key, value, table) + (None,) * 7


class RelativeAttention(nn.Module):
    """Softmax attention whose scores get a learned bias by the relative position of key and query:
    `table` [heads, buckets], the bucket of a difference coming from `buckets` and `zero` (see
    util.distance_buckets).  With `buckets` None there is no bias.  A table of another type than the
    data is cast to it, as under mixed precision."""

    def __init__(self, num_heads, buckets=None, zero=0, num_buckets=None, causal=False, scale=None):
        super().__init__()
        self.zero, self.causal, self.scale = zero, causal, scale
        if buckets is None:
            self.register_buffer('buckets', None)
            self.register_parameter('table', None)
        else:
            assert buckets.dtype == torch.int32 and buckets.dim() == 1, \
                'Buckets must be a vector of int32'
            count = int(buckets.max()) + 1 if num_buckets is None else num_buckets
            self.register_buffer('buckets', buckets)
            self.table = nn.Parameter(torch.zeros(num_heads, count))

    def forward(self, query, key, value, query_start=None, key_lengths=None):
        """query [B, Lq, H, D], key and value [B, Lk, Hk, D], Hk a divisor of H; query_start int32
        [B]: the position of each first query (0 by default); key_lengths int32 [B]: keys in use
        -> [B, Lq, H, D]."""
        table = None if self.table is None else self.table.to(query.dtype)
        return RelativeAttentionFunction.apply(query, key, value, table, self.buckets, self.zero,
                                               self.scale, self.causal, query_start, key_lengths,
                                               torch.is_grad_enabled())
