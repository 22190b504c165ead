"""8-bit products with one fp32 scale per 128 values: quantizer, matrix product, linear layer with its gradients.

Coarser than MX (blocks of 32, power-of-two scales): the scheme in which many 8-bit checkpoints are kept.  A block with
maximum magnitude a has the scale s = max(a, 2^-100) * (1 / top) and the codes RNE(v * (1 / s)), top the largest value of
the format (448 for fp8_e4m3, 57344 for fp8_e5m2); 1 / top, s, 1 / s and the product are fp32.  Activations and gradients
have 1 x 128 blocks along the axis that a product sums over, weights 128 x 128 blocks, which serve both directions.

    linear, forward   y  = q(x) q(w)^T + b        blocks along in_features
    gradients         dx = q(dy) q(w)             blocks along out_features
                      dw = q(dy^T) q(x^T)^T       blocks along the tokens
                      db = sum over tokens of dy  (not quantized)

CUDA tensors run the sm_100a kernels; CPU tensors the same definition as torch operations.  Sums are fp32 and every result
is rounded once.  A value that is infinite or NaN makes every result NaN that sums over its block.  The framework has no counterpart
of this in the reference."""
import torch
from torch.autograd.function import once_differentiable

from . import _backend
from ._backend import MxqError

FORMATS = ("fp8_e4m3", "fp8_e5m2")                       # index = the library's format id
_DTYPES = (torch.float8_e4m3fn, torch.float8_e5m2)
_TOP = (448.0, 57344.0)
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
BLOCK = 128


def _fmt(name):
    if name not in FORMATS:
        raise MxqError("element format of an 8-bit block operand must be one of %s, not %r" % (FORMATS, name))
    return FORMATS.index(name)


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


class BlockFP8:
    """An 8-bit operand [rows, K] of a product that sums over K.

    codes   float8_e4m3fn or float8_e5m2 [rows, K], unit stride along K, rows a multiple of 16 bytes apart and 16-byte
            aligned (any K: allocate rows of ceil(K / 16) * 16 bytes and pass the slice [:, :K])
    scales  float32, contiguous: [ceil(K / 128), rows], or [ceil(K / 128), ceil(rows / 128)] for 128 x 128 blocks
    Nothing is copied: the operand holds these tensors."""

    __slots__ = ("codes", "scales", "tile", "fmt", "transposed")

    def __init__(self, codes, scales, transposed=None):
        if codes.dtype not in _DTYPES or codes.dim() != 2:
            raise MxqError("codes must be a 2-D float8_e4m3fn or float8_e5m2 tensor")
        rows, K = codes.shape
        if K == 0:
            raise MxqError("an operand needs at least one value along K")
        if codes.stride(1) != 1 and K > 1 or rows > 1 and (codes.stride(0) % 16 or codes.stride(0) < K) or \
                codes.data_ptr() % 16:
            raise MxqError("codes need unit stride along K, rows a multiple of 16 bytes apart, 16-byte alignment")
        if scales.dtype != torch.float32 or not scales.is_contiguous() or scales.device != codes.device:
            raise MxqError("scales must be a contiguous float32 tensor on the codes' device")
        if scales.dim() != 2 or scales.shape[0] != _blocks(K) or scales.shape[1] not in (rows, _blocks(rows)):
            raise MxqError("scales of a [%d, %d] operand must be [%d, %d] or [%d, %d], not %s" %
                           (rows, K, _blocks(K), rows, _blocks(K), _blocks(rows), list(scales.shape)))
        if transposed is not None and tuple(transposed.codes.shape) != (K, rows):
            raise MxqError("the transposed operand has the wrong shape")
        self._set(codes, scales, scales.shape[1] != rows, _DTYPES.index(codes.dtype), transposed)

    def _set(self, codes, scales, tile, fmt, transposed=None):
        self.codes, self.scales, self.tile, self.fmt, self.transposed = codes, scales, tile, fmt, transposed
        return self

    @property
    def shape(self):
        return self.codes.shape

    @property
    def elem_format(self):
        return FORMATS[self.fmt]

    def dequantize(self, dtype=torch.float32):
        """The values that codes and scales stand for, [rows, K]."""
        rows, K = self.codes.shape
        s = self.scales.t()
        if self.tile:
            s = s.repeat_interleave(BLOCK, 0)[:rows]
        return (self.codes.float() * s.repeat_interleave(BLOCK, 1)[:, :K]).to(dtype)


def _operand(parts, tile, fmt, transposed=None):
    """BlockFP8 of tensors that the quantizer has just laid out."""
    return BlockFP8.__new__(BlockFP8)._set(parts[0], parts[1], tile and parts[1].shape[1] != parts[0].shape[0], fmt, transposed)


def _host_quantize(x, fmt, tile):
    """The definition as torch operations, codes in rows of a multiple of 16 bytes."""
    rows, K = x.shape
    per, rp, kb = (BLOCK, _blocks(rows) * BLOCK, _blocks(K)) if tile else (1, rows, _blocks(K))
    v = torch.nn.functional.pad(x.float(), (0, kb * BLOCK - K, 0, rp - rows)).view(rp // per, per, kb, BLOCK)
    inv_top = torch.tensor(1.0 / _TOP[fmt], dtype=torch.float32, device=x.device)
    s = v.abs().amax((1, 3)).clamp(min=2.0 ** -100) * inv_top
    r = s.reciprocal()[:, None, :, None]
    q = (v * r).clamp(-_TOP[fmt], _TOP[fmt]).reshape(rp, kb * BLOCK)[:rows]
    pitch = (K + 15) // 16 * 16
    return q[:, :pitch].to(_DTYPES[fmt]).contiguous()[:, :K], s.t().contiguous()


def _quantize(x, fmt, tile, rows, cols, colsum=False):
    """x [rows, K] -> (operand or None, transposed operand or None, column sums [n, K] in fp32 or None)"""
    if x.is_cuda:
        x = _backend.rows_of(x)
        if x.shape[0] == 0:                              # nothing to launch: sums over no rows are zero
            sums = torch.zeros((1, x.shape[1]), dtype=torch.float32, device=x.device) if colsum else None
            a, b, _ = _backend.fp8_quantize(x, fmt, tile, rows, cols)
        else:
            a, b, sums = _backend.fp8_quantize(x, fmt, tile, rows, cols, colsum)
    else:
        a = _host_quantize(x, fmt, tile) if rows else None
        b = _host_quantize(x.t(), fmt, tile) if cols else None
        sums = x.float().sum(0, keepdim=True) if colsum else None
    return (_operand(a, tile, fmt) if rows else None), (_operand(b, tile, fmt) if cols else None), sums


def _check_float(t, name):
    if not isinstance(t, torch.Tensor) or t.dtype not in _FLOATS:
        raise MxqError("%s must be a float32, float16 or bfloat16 tensor" % name)


def quantize_fp8_block(x, elem_format="fp8_e4m3", axes=-1, tile=False):
    """8-bit operand(s) of x, whose leading dimensions are taken as one (its rows).

    axes=-1: the operand [rows, K], blocks along the last dimension; axes=-2: the operand [K, rows] of x transposed, blocks
    along the rows; axes=(-1, -2): both, x read once.  tile: one scale per 128 x 128 block instead of one per 128 values."""
    fmt = _fmt(elem_format)
    _check_float(x, "x")
    want = (axes,) if isinstance(axes, int) else tuple(axes)
    if want not in ((-1,), (-2,), (-1, -2), (-2, -1)):
        raise MxqError("axes must be -1, -2 or both, not %r" % (axes,))
    if x.dim() == 0 or x.shape[-1] == 0:
        raise MxqError("x needs at least one value along its last dimension")
    if x.requires_grad:
        x = x.detach()
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if -2 in want and x.shape[0] == 0:
        raise MxqError("blocks along the rows need at least one row")
    a, b, _ = _quantize(x, fmt, bool(tile), -1 in want, -2 in want)
    got = {-1: a, -2: b}
    return got[want[0]] if len(want) == 1 else tuple(got[w] for w in want)


def _check_bias(bias, n, device):
    if bias is not None and (bias.dtype not in _FLOATS or bias.shape != (n,) or bias.device != device or bias.stride(0) != 1 and n > 1):
        raise MxqError("bias must be a contiguous float tensor of %d values on the operands' device" % n)


def _matmul(a, b, bias, out_dtype):
    if a.codes.is_cuda:
        return _backend.fp8_gemm(a, b, bias, out_dtype)
    y = a.dequantize() @ b.dequantize().t()
    return (y if bias is None else y + bias.float()).to(out_dtype)


def fp8_block_matmul(a, b, bias=None, out_dtype=torch.bfloat16):
    """a b^T (+ bias): a [M, K] and b [N, K] are BlockFP8 operands (of either format and either kind of block), the
    result is [M, N] of out_dtype.  The product of two blocks' scales has to be representable in float32."""
    if not isinstance(a, BlockFP8) or not isinstance(b, BlockFP8):
        raise MxqError("fp8_block_matmul takes BlockFP8 operands")
    if a.codes.shape[1] != b.codes.shape[1]:
        raise MxqError("operands [%d, %d] and [%d, %d] sum over different lengths" % (*a.codes.shape, *b.codes.shape))
    if a.codes.device != b.codes.device:
        raise MxqError("operands are on different devices")
    if out_dtype not in _FLOATS:
        raise MxqError("out_dtype must be float32, float16 or bfloat16")
    _check_bias(bias, b.codes.shape[0], a.codes.device)
    return _matmul(a, b, bias.detach() if bias is not None else None, out_dtype)


def _forward(x2, w, bias, fmt):
    """x2 [tokens, K] times a packed weight, no gradient."""
    if x2.is_cuda:
        return _backend.fp8_linear_fwd(_backend.rows_of(x2), fmt, w, bias)
    return _matmul(_quantize(x2, fmt, False, True, False)[0], w, bias, x2.dtype)


class PackedLinearFunction(torch.autograd.Function):
    """The layer with a weight that was packed before: gradients of x and bias."""

    @staticmethod
    def forward(ctx, x, bias, w, fmt, grad_fmt):
        wt = w.transposed
        if ctx.needs_input_grad[0]:
            if wt is None:
                raise MxqError("the gradient of x needs a packed weight that carries its transposed operand")
            ctx.save_for_backward(wt.codes, wt.scales)
            ctx.wt_kind = (wt.tile, wt.fmt)
        ctx.args = (grad_fmt, x.shape, x.dtype, None if bias is None else bias.dtype)
        return _forward(x.reshape(-1, x.shape[-1]), w, bias, fmt).view(*x.shape[:-1], w.codes.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_x, need_b = ctx.needs_input_grad[:2]
        grad_fmt, x_shape, x_dtype, b_dtype = ctx.args
        q, _, sums = _quantize(dy.reshape(-1, dy.shape[-1]), grad_fmt, False, True, False, need_b)
        dx = db = None
        if need_x:
            wt = BlockFP8.__new__(BlockFP8)._set(*ctx.saved_tensors, *ctx.wt_kind)
            dx = _matmul(q, wt, None, x_dtype).view(x_shape)
        if need_b:
            db = _backend.sum_partials(sums, b_dtype) if dy.is_cuda else sums[0].to(b_dtype)
        return dx, db, None, None, None


class Fp8BlockLinearFunction(torch.autograd.Function):
    """The layer with its weight quantized in the call, which keeps the transposed operands for the gradients."""

    @staticmethod
    def forward(ctx, x, weight, bias, fmt, grad_fmt):
        x2 = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x
        n = weight.shape[0]
        ctx.args = (fmt, grad_fmt, ctx.needs_input_grad[:2], x.shape, tuple(weight.shape),
                    (x.dtype, weight.dtype, None if bias is None else bias.dtype))
        if x.is_cuda and x2.shape[0] > 0:
            y, saved = _backend.fp8_linear_fwd_train(_backend.rows_of(x2), _backend.rows_of(weight), bias, fmt,
                                                     *ctx.needs_input_grad[:2])
            ctx.save_for_backward(saved)
        else:
            ctx.save_for_backward(x2, weight)
            w, _, _ = _quantize(weight, fmt, True, True, False)
            y = _matmul(_quantize(x2, fmt, False, True, False)[0], w, bias, x.dtype)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], n)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        fmt, grad_fmt, saved_for, x_shape, w_shape, dtypes = ctx.args
        need = ctx.needs_input_grad[:3]
        dy2 = dy.reshape(-1, dy.shape[-1]) if dy.dim() != 2 else dy
        if len(ctx.saved_tensors) == 1:
            dx, dw, db = _backend.fp8_linear_bwd(_backend.rows_of(dy2), ctx.saved_tensors[0], saved_for, grad_fmt, fmt, w_shape,
                                                 dtypes, need)
            return dx.view(x_shape) if need[0] and len(x_shape) != 2 else dx, dw, db, None, None
        x2, weight = ctx.saved_tensors
        if dy2.shape[0] == 0:                                # no tokens
            dx, dw, db = (dy.new_zeros(s, dtype=t) if n else None
                          for s, t, n in zip((x_shape, w_shape, w_shape[:1]), dtypes, need))
            return dx, dw, db, None, None
        dx = dw = db = None
        if need[0]:
            dx = _matmul(_quantize(dy2, grad_fmt, False, True, False)[0], _quantize(weight, fmt, True, False, True)[1], None,
                         dtypes[0]).view(x_shape)
        if need[1]:
            dw = _matmul(_quantize(dy2, grad_fmt, False, False, True)[1], _quantize(x2, fmt, False, False, True)[1], None, dtypes[1])
        if need[2]:
            db = dy2.float().sum(0).to(dtypes[2])
        return dx, dw, db, None, None


def fp8_block_linear(x, weight, bias=None, elem_format="fp8_e4m3", grad_elem_format="fp8_e4m3"):
    """x w^T (+ bias) in 8 bits with a scale per block; x [..., in_features], result [..., out_features] of x's dtype.

    weight: a [out_features, in_features] tensor, quantized in the call (128 x 128 blocks, elem_format) and differentiable;
    or a BlockFP8 that was packed once, which gets no gradient (x gets one if it was packed with its transposed operand).
    x is quantized in the call (1 x 128 blocks, elem_format), and in the backward pass so is the incoming gradient
    (grad_elem_format), along out_features for dx and along the tokens for dw."""
    fmt, grad_fmt = _fmt(elem_format), _fmt(grad_elem_format)
    _check_float(x, "x")
    packed = isinstance(weight, BlockFP8)
    if packed:
        (n, k), dev = weight.codes.shape, weight.codes.device
    else:
        _check_float(weight, "weight")
        if weight.dim() != 2:
            raise MxqError("weight must be 2-D")
        (n, k), dev = weight.shape, weight.device
    if x.dim() == 0 or x.shape[-1] != k or k == 0 or n == 0:
        raise MxqError("x %s does not fit a weight [%d, %d]" % (list(x.shape), n, k))
    if x.device != dev:
        raise MxqError("x and weight are on different devices")
    if bias is not None:
        _check_bias(bias, n, dev)
    grad = torch.is_grad_enabled() and (x.requires_grad or not packed and weight.requires_grad or
                                        bias is not None and bias.requires_grad)
    if grad:
        return PackedLinearFunction.apply(x, bias, weight, fmt, grad_fmt) if packed else \
            Fp8BlockLinearFunction.apply(x, weight, bias, fmt, grad_fmt)
    with torch.no_grad():
        w = weight if packed else _quantize(weight, fmt, True, True, False)[0]
        if x.dim() == 2:
            return _forward(x, w, bias, fmt)
        return _forward(x.reshape(-1, k), w, bias, fmt).view(*x.shape[:-1], n)


class Fp8BlockLinear(torch.nn.Linear):
    """Linear layer on fp8_block_linear.  prequantize_weights() packs the weight once for inference, as
    Linear.prequantize_weights does: the forward pass then reads the packed copy until the next call of it, whatever
    happens to the parameter, and refuses to run in training mode."""

    def __init__(self, in_features, out_features, bias=True, elem_format="fp8_e4m3", grad_elem_format="fp8_e4m3", device=None,
                 dtype=None):
        _fmt(elem_format), _fmt(grad_elem_format)
        self.elem_format, self.grad_elem_format = elem_format, grad_elem_format
        self.packed = None
        super().__init__(in_features, out_features, bias, device=device, dtype=dtype)

    def prequantize_weights(self):
        self.packed = quantize_fp8_block(self.weight, self.elem_format, tile=True)

    def forward(self, inputs):
        w = self.weight
        if self.packed is not None:
            assert self.training is False, "Cannot use prequantized weights when training!"
            w = self.packed
        return fp8_block_linear(inputs, w, self.bias, self.elem_format, self.grad_elem_format)
