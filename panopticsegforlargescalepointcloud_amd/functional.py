"""Differentiable row operators on [rows, channels] features: thin autograd nodes over ops.* (csrc/pp_groupnorm.hip, pp_linear.hip)."""
import torch
from torch.autograd import forward_ad

from . import ops


def _refuse_tangents(name, *tensors):
    """the operators have no forward-mode derivative: a tangent is refused, not dropped (the level is -1 outside forward_ad.dual_level)"""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("%s has no forward-mode derivative" % name)


class _GroupNormActFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, offsets, num_groups, weight, bias, eps, act, slope, order):
        with ops.device_of(x):
            y, stat = ops._group_norm_fwd(x, offsets, num_groups, weight, bias, eps, act, slope, order)
        ctx.save_for_backward(x, offsets, weight, bias, stat, order)
        ctx.cfg = (num_groups, act, slope)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, offsets, weight, bias, stat, order = ctx.saved_tensors
        num_groups, act, slope = ctx.cfg
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0] or need[3] or need[4]:
            at = stat.data_ptr()
            with ops.device_of(x):
                dx, dw, db = ops._group_norm_bwd(x, dy, offsets, num_groups, weight, bias, at, at + 2 * stat.numel(), act, slope, order,
                                                 need[0], need[3], need[4])
        return dx, None, None, dw, db, None, None, None, None


def group_norm_act(x, offsets, num_groups, weight=None, bias=None, eps=1e-5, activation="none", slope=0.2, order=None):
    """y = act(group_norm(x)): statistics over the rows of each batch element and the channels of each group, differentiable in x,
    weight and bias.  x [n, c] (float32, bfloat16 or float16), weight / bias float32 [c] or None.  Batch element s owns the
    positions offsets[s] .. offsets[s+1] of the row sequence (int64 [batch + 1] on the device, ascending); position p is row
    order[p] (int64 [n], each row once) or, without an order, row p.  Rows of no batch element (padding) come out as zeros and
    get zero gradients.  activation: none, relu, leaky_relu (with `slope`), silu or gelu (exact).  num_groups = c: instance norm.
    Beside FastBatchNorm1d: the result for a row does not depend on the other batch elements, in training and in inference."""
    act = ops.activation_id(activation)
    _refuse_tangents("group_norm_act", x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _GroupNormActFn.apply(x, offsets, num_groups, weight, bias, eps, act, slope, order)
    return ops.group_norm_fwd(x, offsets, num_groups, weight, bias, eps, act, slope, order)[0]


class _LinearActFn(torch.autograd.Function):
    """keeps x, weight and bias only: the backward recomputes the pre-activation (csrc/pp_linear.hip)"""

    @staticmethod
    def forward(ctx, x, weight, bias, act, slope, residual):
        ctx.save_for_backward(x, weight, bias)
        ctx.cfg = (act, slope)
        return ops.linear_act_fwd(x, weight, bias, act, slope, residual)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, bias = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dw = db = None
        if need[0] or need[1] or need[2]:
            dx, dw, db = ops.linear_act_bwd(x, dy, weight, bias, *ctx.cfg, want_input=need[0], want_weight=need[1], want_bias=need[2])
        return dx, dw, db, None, None, dy if need[5] else None


def linear_act(x, weight, bias=None, activation="none", slope=0.2, residual=None):
    """y = act(x W^T + bias) + residual as one launch, differentiable in all four operands.  x [..., cin], weight [cout, cin] (the
    layout of torch.nn.Linear), bias [cout] or None, residual [..., cout] or None, all of one type (float32, bfloat16, float16), which is
    the result's.  Under torch.autocast operands of different types are brought to its type; operands of one type stay as they are
    (fp32 features go on to sparse convolutions, which take nothing else).
    activation: none, relu, leaky_relu (with `slope`), silu or gelu (exact); it acts before the residual is added, as in ResBlock."""
    act = ops.activation_id(activation)
    _refuse_tangents("linear_act", x, weight, bias, residual)
    if torch.is_autocast_enabled("cuda") and any(t is not None and t.dtype != x.dtype for t in (weight, bias, residual)):
        dtype = torch.get_autocast_dtype("cuda")
        x, weight, bias, residual = (t if t is None or t.dtype == torch.float64 else t.to(dtype) for t in (x, weight, bias, residual))
    if x.dim() != 2:
        if x.dim() == 0 or (residual is not None and residual.shape != (*x.shape[:-1], weight.shape[0])):
            raise ValueError("linear_act: input %s, weight %s and residual %s do not fit" % (
                tuple(x.shape), tuple(weight.shape), None if residual is None else tuple(residual.shape)))
        rows = x.reshape(x.shape[:-1].numel(), x.shape[-1])
        more = None if residual is None else residual.reshape(rows.shape[0], weight.shape[0])
        return _linear_act(rows, weight, bias, act, slope, more).view(*x.shape[:-1], weight.shape[0])
    return _linear_act(x, weight, bias, act, slope, residual)


def _linear_act(x, weight, bias, act, slope, residual):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
        return _LinearActFn.apply(x, weight, bias, act, slope, residual)
    return ops.linear_act_fwd(x, weight, bias, act, slope, residual)
