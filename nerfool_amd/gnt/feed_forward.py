"""The feed-forward half of a transformer layer as operators of its own, at any width and in float32, bfloat16 or float16: the
root-mean-square norm with the residual's addition, and the gated feed-forward block.  GNT's own layers (LayerNorm and a ReLU block of
width 64, gnt/transformer_network.py:38-50, :121-202) run inside the whole-network kernels of `GNT`; these stand beside them for networks with
other layers.

    y, h = rms_norm(x, weight, residual=r)                      # h = x + r, y = weight * h / sqrt(mean(h^2) + eps)
    out = gated_feed_forward(y, w_gate, w_up, w_down)           # (act(y Wg^T) * (y Wu^T)) Wd^T

Both have a backward pass, and no second one: backward() and grad() with create_graph raise.  On 8 bits, for inference:

    q, scale, h = rms_norm_8bit(x, weight, residual=r)
    out = gated_feed_forward_8bit((q, scale), quantize_8bit(w_gate), quantize_8bit(w_up), quantize_8bit(w_down), dtype=torch.bfloat16)

An 8-bit tensor is a pair: the values, float8_e4m3fn [..., n], and the scales, float8_e8m0fnu [..., ceil(n / 32)] -- 32 consecutive values of the
last axis share a power of two, the least 2^e with max|block| <= 448 * 2^e.  A block that holds an infinity or a NaN is NaN as a whole.

In float16 and bfloat16 the product in the middle, and its gradients, are rounded to that type (in float16: infinite beyond 65504, the gradients
held times a power of two that keeps those of a small dy from the subnormal values); sums are float32.  relu's gradient takes the side of zero on which the
exact sum x Wg^T lies: one that a float32 sum cannot tell from zero is summed again in double.  Where weights need
gradients, or dim is above 64, the forward keeps x Wg^T and x Wu^T in float32 for the backward pass; for constant weights at dim <= 64 nothing is kept (rows and hidden
permitting: `ops.gated_ff_bwd_recomputes`).

Any number of leading axes; a call's tensors are of one type and on one device; tensors that are not contiguous are copied.  Work is enqueued on the
current stream; results do not depend on scheduling (no atomics).  A row's result may depend on how many rows the call has, as the order of its sums does, and on 8 bits with a
bfloat16 result a little more: see `gated_feed_forward_8bit`.  In float32 with more than 64 rows (or, in a gradient, any number) an infinity in an operand of a product gives NaN
where the exact sum would be infinite: operands are split into parts, and the parts that are zero, or of the other sign, meet the infinity.  (Up to 64 rows the forward multiplies
float32 values as they are.)"""
import torch
import torch.nn as nn
from torch.autograd import forward_ad

from .. import ops


def _last_axis(t, name):
    if t.dim() < 1 or not t.shape[-1]:
        raise ValueError('%s must have a last axis of at least one value (got the shape %s)' % (name, tuple(t.shape)))
    return t


def _rows(t, name):
    _last_axis(t, name)
    return t if t.dim() == 2 else t.reshape(-1, t.shape[-1])          # (a view is a node of its own in the backward pass)


def _as(t, shape):
    return t if t.dim() == len(shape) else t.reshape(shape)


def _differentiated(*tensors):
    """whether the call is part of a gradient: decided here, as a Function's needs_input_grad says the same under no_grad, where nothing is to be kept.  (Forward mode goes through
    the Function too, which refuses it.)"""
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _first_only():
    if torch.is_grad_enabled():          # create_graph: the gradients would enter the new graph as constants
        raise RuntimeError('rms_norm and gated_feed_forward have no second derivative: call backward() or grad() without create_graph')


class _RMSNorm(torch.autograd.Function):
    # takes x and the residual in their own shapes: their gradient is one tensor, and a view between it and a leaf would hide from the leaf's accumulation that the other
    # leaf has it too (both .grad would be one memory, and the next pass would add to it twice)
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        h, y, rstd = ops.rms_norm_fwd(x, weight, residual, eps, want_rstd=True)
        ctx.set_materialize_grads(False)
        # from h as rounded to 16 bits both gradients would carry that rounding beside their own -- dx many times over where dy lies along xhat, which it subtracts -- so x and
        # the residual are kept and added again; in float32 h as stored is their sum, and half the reading
        if h is None or x.dtype != torch.float32:
            ctx.save_for_backward(x, residual, weight, rstd)
        else:
            ctx.save_for_backward(h, None, weight, rstd)
        return y if h is None else (y, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        _first_only()
        need_x, need_w, need_r, _ = ctx.needs_input_grad
        h, residual, weight, rstd = ctx.saved_tensors
        if dy is None:          # only the sum was used
            return (dh if need_x else None, torch.zeros_like(weight) if need_w else None, dh if need_r else None, None)
        dx, dw = ops.rms_norm_bwd_saved(dy, dh, h, residual, weight, rstd, need_w)
        return dx if need_x else None, dw, dx if need_r else None, None


def rms_norm(x, weight=None, residual=None, eps=1e-6):
    """x, residual [..., dim], weight [dim] -> y, or (y, h) with a residual: h = x + residual in the inputs' type, y from the sum before that rounding"""
    _last_axis(x, 'x')
    if _differentiated(x, weight, residual):
        return _RMSNorm.apply(x, weight, residual, float(eps))
    h, y, _ = ops.rms_norm_fwd(x, weight, residual, eps)
    return y if residual is None else (y, h)


def _no_gradient(what, tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError('%s has no backward pass: call it under torch.no_grad(), or on tensors that do not require a gradient' % what)


def rms_norm_8bit(x, weight=None, residual=None, eps=1e-6):
    """rms_norm with y in 8 bits -> (q, scale), or (q, scale, h) with a residual; no backward pass"""
    _no_gradient('rms_norm_8bit', (x, weight, residual))
    if residual is not None and residual.shape != x.shape:
        raise ValueError('residual has the shape %s, x %s' % (tuple(residual.shape), tuple(x.shape)))
    h, (q, scale), _ = ops.rms_norm_fwd(_rows(x, 'x'), weight, None if residual is None else _rows(residual, 'residual'), float(eps), quantize=True)
    q, scale = q.reshape(x.shape), scale.reshape(*x.shape[:-1], scale.shape[-1])
    return (q, scale) if residual is None else (q, scale, h.reshape(x.shape))


def quantize_8bit(x):
    """x [..., n] -> (q, scale); no backward pass"""
    _no_gradient('quantize_8bit', (x,))
    q, scale = ops.quantize_8bit(_rows(x, 'x'))
    return q.reshape(x.shape), scale.reshape(*x.shape[:-1], scale.shape[-1])


class _GatedFeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, activation):
        need = any(ctx.needs_input_grad[:4])
        save = need and (any(ctx.needs_input_grad[1:4]) or w_gate.dim() != 2 or not ops.gated_ff_bwd_recomputes(*x.shape, w_gate.shape[0]))
        out, g, u = ops.gated_ff_fwd(x, w_gate, w_up, w_down, activation, save=save)
        ctx.activation = activation
        if need:
            ctx.save_for_backward(x, w_gate, w_up, w_down, g, u)
        return out

    @staticmethod
    def backward(ctx, dy):
        _first_only()
        x, w_gate, w_up, w_down, g, u = ctx.saved_tensors
        return (*ops.gated_ff_bwd(x, w_gate, w_up, w_down, dy, g, u, ctx.activation, ctx.needs_input_grad[:4]), None)


def gated_feed_forward(x, w_gate, w_up, w_down, activation='silu'):
    """x [..., dim], w_gate, w_up [hidden, dim], w_down [dim, hidden] -> [..., dim]; activation: 'silu', 'gelu' (the error function), 'relu'.
    Constant weights (requires_grad False, as everywhere in an attack) cost no gradient of their own."""
    ops.ff_activation(activation)
    rows = _rows(x, 'x')
    if _differentiated(x, w_gate, w_up, w_down):
        return _as(_GatedFeedForward.apply(rows, w_gate, w_up, w_down, activation), x.shape)
    return _as(ops.gated_ff_fwd(rows, w_gate, w_up, w_down, activation)[0], x.shape)


def gated_feed_forward_8bit(x, w_gate, w_up, w_down, activation='silu', dtype=torch.bfloat16):
    """`gated_feed_forward` on 8-bit pairs (q, scale), dim and hidden multiples of 32: x [..., dim] -> [..., dim] in dtype.  The product in the
    middle is brought to 8 bits by the same rule from its float32 values.  No backward pass.

    float32 and float16 results, and all results of up to 64 rows, are of exact products in float32 sums.  With more rows a bfloat16 result is of the matrix instruction's own 8-bit
    products, which drops what lies below 2^-12 of the largest of 16, at twice the rate (0.0020 from the exact sums where rounding alone is 0.0017): dtype=torch.float32 and
    .to(torch.bfloat16) has the exact ones."""
    _no_gradient('gated_feed_forward_8bit', (*x, *w_gate, *w_up, *w_down))
    (q, scale), lead = x, x[0].shape[:-1]
    if scale.shape[:-1] != lead:
        raise ValueError("x: the scales' leading axes %s are not the values' %s" % (tuple(scale.shape[:-1]), tuple(lead)))
    out = ops.gated_ff_fwd_8bit((_rows(q, 'x'), _rows(scale, "x's scales")), w_gate, w_up, w_down, activation, dtype)
    return out.reshape(*lead, out.shape[-1])


class RMSNorm(nn.Module):
    """`rms_norm` with its weight; called with a residual it returns (y, h)"""

    def __init__(self, dim, eps=1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(dim))
        self.eps = eps

    def forward(self, x, residual=None):
        return rms_norm(x, self.weight, residual, self.eps)


class GatedFeedForward(nn.Module):
    """`gated_feed_forward` with its weights, `[out, in]` as nn.Linear keeps them and under nn.Linear's names"""

    def __init__(self, dim, hid, activation='silu'):
        super().__init__()
        ops.ff_activation(activation)
        self.activation = activation
        self.gate = nn.Linear(dim, hid, bias=False)
        self.up = nn.Linear(dim, hid, bias=False)
        self.down = nn.Linear(hid, dim, bias=False)

    def forward(self, x):
        return gated_feed_forward(x, self.gate.weight, self.up.weight, self.down.weight, self.activation)
