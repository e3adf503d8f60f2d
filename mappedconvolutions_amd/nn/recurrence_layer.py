"""GatedRecurrence and GroupNormActivation: a linear-time mixer of tokens (the rows of an equirectangular
image, its pixels in scan order, a decoder's tokens from a kept state) and a norm with an activation for
tokens whose channels lie last.  No counterpart in the reference; the work is done by the HIP kernels
behind `_C.gated_recurrence_*` and `_C.group_norm_*`."""
import torch
import torch.nn as nn

from .. import _C
from .relative_attention_layer import first_derivatives


class GatedRecurrenceFunction(torch.autograd.Function):

    @staticmethod
    def forward(ctx, value, forget, gate, initial, lengths, reverse, recording):
        ctx.set_materialize_grads(False)
        ctx.reverse = reverse
        training = recording and any(ctx.needs_input_grad[:4])
        out, final, saved = _C.gated_recurrence_forward(value, forget, gate, initial, lengths, reverse,
                                                        for_backward=training)
        if training:
            ctx.save_for_backward(value, forget, gate, initial, lengths, saved)
        return out, final

    @staticmethod
    def backward(ctx, grad_output, grad_final):
        value, forget, gate, initial, lengths, saved = ctx.saved_tensors
        given = [t for t in (grad_output, grad_final) if t is not None]
        if grad_output is None:
            grad_output = torch.zeros_like(value)
        grads = _C.gated_recurrence_backward(grad_output, value, forget, gate, saved, grad_final, lengths,
                                             ctx.reverse, needs=tuple(ctx.needs_input_grad[:4]))
        return first_derivatives(grads, *given, value, forget, gate, initial) + (None,) * 3


class GatedRecurrence(nn.Module):
    """h_t = a_t h_{t-1} + (1 - a_t) value_t with a_t = sigmoid(forget_t), every channel for itself, and
    out_t = h_t gate_t sigmoid(gate_t) (h_t without a gate); with `reverse` from the last token to the
    first.  It has no parameters: value, forget and gate are usually parts of one projection, whose bias
    sets how long the channels remember (a forget gate of x keeps a state for about e^x tokens)."""

    def __init__(self, reverse=False):
        super().__init__()
        self.reverse = reverse

    def forward(self, value, forget, gate=None, initial=None, lengths=None):
        """value, forget, gate [B, L, C]; initial float32 [B, C]: the state to begin with (zeros by
        default); lengths int32 [B]: tokens in use -> (out [B, L, C], the last state float32 [B, C])."""
        return GatedRecurrenceFunction.apply(value, forget, gate, initial, lengths, self.reverse,
                                             torch.is_grad_enabled())

    @torch.no_grad()
    def step(self, state, value, forget, gate=None):
        """The next tokens, value, forget, gate [B, L, C], from `state` float32 [B, C], which is changed in
        place (no gradients) -> [B, L, C]."""
        assert not self.reverse, 'Tokens that come one by one have no last one to begin with'
        return _C.gated_recurrence_forward(value, forget, gate, state, final=state)[0]


class GroupNormActivationFunction(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, activation, recording):
        ctx.groups, ctx.activation = groups, activation
        training = recording and any(ctx.needs_input_grad[:3])
        y, saved = _C.group_norm_forward(x, groups, weight, bias, eps, activation, for_backward=training)
        if training:
            ctx.save_for_backward(x, weight, bias, saved)
        return y

    @staticmethod
    def backward(ctx, grad_output):
        x, weight, bias, saved = ctx.saved_tensors
        grads = _C.group_norm_backward(grad_output, x, saved, ctx.groups, weight, bias, ctx.activation,
                                       needs=tuple(ctx.needs_input_grad[:3]))
        return first_derivatives(grads, grad_output, x, weight, bias) + (None,) * 4


class GroupNormActivation(nn.Module):
    """Every group of neighbouring channels of a sample normed over all its tokens, times a weight per
    channel plus a bias, and an activation (None, 'silu' or 'gelu').  Parameters of another type than the
    data are cast to it, as under mixed precision: a weight's rounding (2^-8 of it in bfloat16) is no larger
    than that of the values it is multiplied by, and the gradients' sums, taken in 32 bits, are rounded once."""

    def __init__(self, num_groups, num_channels, eps=1e-5, activation=None, affine=True):
        super().__init__()
        assert num_channels % num_groups == 0, 'Number of channels must be divisible by the groups'
        assert activation in _C.ACTIVATIONS, 'Activation must be None, \'silu\' or \'gelu\''
        self.num_groups, self.num_channels, self.eps = num_groups, num_channels, eps
        self.activation = activation
        if affine:
            self.weight = nn.Parameter(torch.ones(num_channels))
            self.bias = nn.Parameter(torch.zeros(num_channels))
        else:
            self.register_parameter('weight', None)
            self.register_parameter('bias', None)

    def forward(self, x):
        """x [B, ..., C] -> the same shape (an image that has its channels last in memory goes as
        x.permute(0, 2, 3, 1))."""
        assert x.dim() >= 2 and x.shape[-1] == self.num_channels, \
            'Input must end in %d channels' % self.num_channels
        weight = None if self.weight is None else self.weight.to(x.dtype)
        bias = None if self.bias is None else self.bias.to(x.dtype)
        tokens = x.flatten(1, -2) if x.dim() > 2 else x[:, None]
        return GroupNormActivationFunction.apply(tokens, weight, bias, self.num_groups, self.eps,
                                                 self.activation, torch.is_grad_enabled()).view(x.shape)
