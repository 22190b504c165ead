"""bfloat-emulated RMSNorm (reference: mx/layernorm.py:98-200, fused kernel for bfloat16 CUDA tensors) and
LayerNorm (mx/layernorm.py:17-96, 203-210).  fused_layer_norm / FusedLayerNorm have no counterpart there: a layer norm that
emulates no vector format, computed in fp32 in one pass each way and rounded once."""
import torch
from torch.autograd.function import once_differentiable

from . import _backend
from ._autograd import call
from ._backend import MxqError
from .norm_utils import norm_backward_ln, norm_forward
from .specs import apply_mx_specs, get_backwards_mx_specs, mx_assert_test
from .vector_ops import (fused_bf16_ok, vec_add, vec_mul, vec_quantize, vec_recip, vec_reduce_mean, vec_reduce_sum,
                         vec_sqrt, vec_sub)


class RMSNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, mx_specs=None, name=None):
        sp = mx_specs
        if fused_bf16_ok(sp, x, weight, bias) and x.shape[-1] == weight.numel() == bias.numel():
            if any(ctx.needs_input_grad[:3]):
                out, x_norm, rms_inv = _backend.rmsnorm_bf16(x.contiguous(), weight.contiguous(), bias.contiguous(),
                                                             eps, want_saved=True)
            else:                                             # inference: nothing is kept for backward
                out = _backend.rmsnorm_bf16(x.contiguous(), weight.contiguous(), bias.contiguous(), eps)
                ctx.mx_specs = get_backwards_mx_specs(sp)
                return out
            bf_w = weight
        else:
            x = vec_quantize(x, mx_specs=sp)
            ms = vec_reduce_mean(vec_mul(x, x, mx_specs=sp), -1, keepdim=True, mx_specs=sp)
            rms_inv = vec_recip(vec_sqrt(vec_add(ms, eps, mx_specs=sp), mx_specs=sp), mx_specs=sp)
            x_norm = vec_mul(x, rms_inv, mx_specs=sp)
            bf_w = vec_quantize(weight, mx_specs=sp)
            bf_b = vec_quantize(bias, mx_specs=sp)
            out = vec_add(vec_mul(bf_w, x_norm, mx_specs=sp), bf_b, mx_specs=sp)
        ctx.save_for_backward(x_norm, rms_inv, bf_w if sp["quantize_backprop"] else weight)
        ctx.mx_specs = get_backwards_mx_specs(sp)
        return out

    @staticmethod
    def backward(ctx, grad_output):
        sp = ctx.mx_specs
        x_norm, rms_inv, weight = ctx.saved_tensors
        lead = list(range(grad_output.dim() - 1))
        g = vec_quantize(grad_output, mx_specs=sp)
        grad_bias = vec_reduce_sum(g, lead, mx_specs=sp)
        grad_weight = vec_reduce_sum(vec_mul(g, x_norm, mx_specs=sp), lead, mx_specs=sp)
        dx1 = vec_mul(vec_mul(g, weight, mx_specs=sp), rms_inv, mx_specs=sp)
        m = vec_reduce_mean(vec_mul(dx1, x_norm, mx_specs=sp), -1, keepdim=True, mx_specs=sp)
        grad_input = vec_sub(dx1, vec_mul(x_norm, m, mx_specs=sp))       # last step unrounded, as in the reference
        return (grad_input, grad_weight, grad_bias, None, None, None)


class RMSNorm(torch.nn.LayerNorm):
    def __init__(self, hidden_size, eps=1e-12, mx_specs=None, name=None):
        mx_assert_test(mx_specs)
        self.name = name
        self.mx_specs = apply_mx_specs(mx_specs)
        super().__init__(normalized_shape=hidden_size, eps=eps)

    def apply_mx_specs(self, mx_specs):
        self.mx_none = mx_specs is None
        self.mx_specs = apply_mx_specs(mx_specs)

    def append_name(self, postfix):
        self.name += postfix

    def forward(self, x):
        return call(RMSNormFunction, x, self.weight, self.bias, self.eps, self.mx_specs, self.name)


torch_layer_norm = torch.nn.functional.layer_norm


class LayerNormFunction(torch.autograd.Function):
    """Normalisation over the last dimension, eps inside the square root; keeps the normalised input and
    (variance + eps) for the gradient."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, mx_specs=None, name=None):
        sp = mx_specs
        bf_w = vec_quantize(weight, mx_specs=sp)
        r = norm_forward(vec_quantize(x, mx_specs=sp), -1, bf_w, vec_quantize(bias, mx_specs=sp), eps, sp)
        ctx.save_for_backward(r.x_norm, r.x_vare, bf_w if sp["quantize_backprop"] else weight)
        ctx.mx_specs = get_backwards_mx_specs(sp)
        return r.output

    @staticmethod
    def backward(ctx, grad_output):
        sp = ctx.mx_specs
        x_norm, x_vare, weight = ctx.saved_tensors
        lead = list(range(grad_output.ndim - 1))
        g = vec_quantize(grad_output, mx_specs=sp)
        grad_bias = vec_reduce_sum(g, lead, mx_specs=sp)
        grad_weight = vec_reduce_sum(vec_mul(g, x_norm, mx_specs=sp), lead, mx_specs=sp)
        return (norm_backward_ln(g, -1, weight, x_norm, x_vare, sp), grad_weight, grad_bias, None, None, None)


class LayerNorm(torch.nn.LayerNorm):
    def __init__(self, hidden_size, eps=1e-12, mx_specs=None, name=None):
        mx_assert_test(mx_specs)
        self.mx_none = mx_specs is None
        self.name = name
        self.mx_specs = apply_mx_specs(mx_specs)
        super().__init__(normalized_shape=hidden_size, eps=eps)

    def apply_mx_specs(self, mx_specs):
        self.mx_none = mx_specs is None
        self.mx_specs = apply_mx_specs(mx_specs)

    def append_name(self, postfix):
        self.name += postfix

    def forward(self, x):
        if self.mx_none:
            return super().forward(x)
        return LayerNormFunction.apply(x, self.weight, self.bias, self.eps, self.mx_specs, self.name)


def layer_norm(input, normalized_shape, weight, bias, eps=1e-12, mx_specs=None, name=None):
    mx_assert_test(mx_specs)
    if mx_specs is None:
        return torch_layer_norm(input, normalized_shape, weight, bias, eps)
    assert normalized_shape == weight.shape
    return LayerNormFunction.apply(input, weight, bias, eps, apply_mx_specs(mx_specs), name)


class FusedLayerNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2 = _backend.rows_of(x)
        y, mean, rstd = _backend.layer_norm_fwd(x2, weight, bias, eps, True)
        ctx.save_for_backward(x2, weight, mean, rstd)
        ctx.sums_dtype = x.dtype if weight is None and bias is None else (bias if weight is None else weight).dtype
        return y if x.dim() == 2 else y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, weight, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad[:3]
        dx, dw, db = _backend.layer_norm_bwd(_backend.rows_of(dy), x2, weight, mean, rstd, ctx.sums_dtype, need)
        return dx.view(dy.shape) if need[0] and dy.dim() != 2 else dx, dw, db, None


_FLOATS = (torch.float32, torch.float16, torch.bfloat16)


def fused_layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension, in fp32 and rounded once to x's dtype; no
    vector format is emulated (layer_norm does that).  weight and bias: [cols], both of x's dtype or both float32; either may be
    None.  Gradients: dx of x's dtype; dw and db summed over the rows in fp32, in a fixed order."""
    if not isinstance(x, torch.Tensor) or x.dtype not in _FLOATS:
        raise MxqError("x must be a float32, float16 or bfloat16 tensor")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise MxqError("x needs at least one value along its last dimension")
    if not eps >= 0:
        raise MxqError("eps must not be negative")
    grad = x.requires_grad
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            if t.shape != x.shape[-1:] or t.dtype not in (x.dtype, torch.float32) or t.device != x.device or not t.is_contiguous():
                raise MxqError("%s must be a contiguous tensor of %d values of x's dtype or float32 on x's device" %
                               (name, x.shape[-1]))
            grad = grad or t.requires_grad
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise MxqError("weight and bias must have one dtype")
    if x.is_cuda:
        if grad and torch.is_grad_enabled():
            return FusedLayerNormFunction.apply(x, weight, bias, float(eps))
        if x.dim() == 2:
            return _backend.layer_norm_fwd(_backend.rows_of(x), weight, bias, float(eps), False)[0]
        with torch.no_grad():
            return _backend.layer_norm_fwd(_backend.rows_of(x), weight, bias, float(eps), False)[0].view(x.shape)
    v = x.float()
    d = v - v.mean(-1, keepdim=True)
    y = d / ((d * d).mean(-1, keepdim=True) + eps).sqrt()
    y = y if weight is None else y * weight.float()
    return (y if bias is None else y + bias.float()).to(x.dtype)


class FusedLayerNorm(torch.nn.LayerNorm):
    """Layer normalisation over the last dimension on fused_layer_norm."""

    def __init__(self, hidden_size, eps=1e-5, elementwise_affine=True, bias=True, device=None, dtype=None):
        super().__init__(hidden_size, eps=eps, elementwise_affine=elementwise_affine, bias=bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise MxqError("FusedLayerNorm normalises the last dimension only")

    def forward(self, x):
        return fused_layer_norm(x, self.weight, self.bias, self.eps)
