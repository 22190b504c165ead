"""The 8-bit block operators without a GPU: the definition on CPU tensors, gradients, refusals."""
import pytest
import torch

import fp8_reference as ref
import microxcaling_b200 as mx
from microxcaling_b200._backend import MxqError


def values(rows, cols, seed, dtype=torch.float32):
    return torch.randn(rows, cols, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("shape", [(1, 1), (3, 130), (129, 257), (200, 16)])
@pytest.mark.parametrize("tile", [False, True])
def test_quantize(shape, tile):
    for fmt in ("fp8_e4m3", "fp8_e5m2"):
        x = values(*shape, 0, torch.bfloat16)
        a, b = mx.quantize_fp8_block(x, fmt, axes=(-1, -2), tile=tile)
        for q, v in ((a, x), (b, x.t())):
            codes, scales, value = ref.quantize(v, fmt, tile)
            assert torch.equal(q.codes.double(), codes) and torch.equal(q.scales, scales)
            # the stated value is codes times scale, rounded to fp32
            assert bool(((q.dequantize().double() - value).abs() <= value.abs() * 2.0 ** -24).all())


def test_linear_and_gradients():
    x, w, b, dy = (values(*s, i) for i, s in enumerate([(37, 200), (150, 200), (1, 150), (37, 150)]))
    b = b[0]
    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    layer_out = mx.fp8_block_linear(*leaves)
    dx, dw, db = torch.autograd.grad(layer_out, leaves, dy)
    xv, wv = ref.quantize(x, "fp8_e4m3")[2], ref.quantize(w, "fp8_e4m3", True)[2]
    for got, (want, _) in ((layer_out, ref.product_bound(xv, wv, torch.float32, b)),
                           (dx, ref.product_bound(ref.quantize(dy, "fp8_e4m3")[2], wv.t(), torch.float32)),
                           (dw, ref.product_bound(ref.quantize(dy.t(), "fp8_e4m3")[2], ref.quantize(x.t(), "fp8_e4m3")[2], torch.float32))):
        # fp32 sums of at most 200 terms on the CPU, whatever their order, after operands rounded to fp32
        assert torch.allclose(got.double(), want, rtol=0, atol=float(202 * 2.0 ** -24 * want.abs().max() * 200))
    assert torch.allclose(db, dy.sum(0), rtol=0, atol=1e-4)


def test_gradient_is_that_of_the_unquantized_product_up_to_the_codes_rounding():
    """dx against a difference quotient of the exact product: the codes' rounding, 2^-4 of each value at most, bounds the gap."""
    x, w, dy = values(8, 128, 3).double(), values(16, 128, 4).double(), values(8, 16, 5).double()
    leaf = x.float().requires_grad_()
    dx, = torch.autograd.grad(mx.fp8_block_linear(leaf, w.float()), leaf, dy.float())
    h, at = 1e-3, (2, 17)
    xp, xm = x.clone(), x.clone()
    xp[at] += h
    xm[at] -= h
    diff = (((xp - xm) @ w.t()) * dy).sum() / (2 * h)
    room = ((1 + 2.0 ** -4) ** 2 - 1) * (dy.abs() @ w.abs())[at] + 2.0 ** -9 * float(w.abs().max()) * float(dy.abs().max()) * 16
    assert abs(float(dx[at]) - float(diff)) <= float(room)


def test_module_and_packed_weight():
    layer = mx.Fp8BlockLinear(130, 20)
    x = values(5, 130, 6)
    want = layer(x).detach()
    layer.prequantize_weights()
    with pytest.raises(AssertionError, match="training"):
        layer(x)
    layer.eval()
    assert torch.equal(layer(x).detach(), want)
    layer.weight.data.mul_(2)
    assert torch.equal(layer(x).detach(), want)           # the packed copy, until it is made again
    layer.prequantize_weights()
    assert not torch.equal(layer(x).detach(), want)


def test_double_backward_is_refused():
    x = values(4, 16, 7).requires_grad_()
    w = values(8, 16, 8).requires_grad_()
    g, = torch.autograd.grad(mx.fp8_block_linear(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals():
    x, w = values(4, 32, 9), values(8, 32, 10)
    q = mx.quantize_fp8_block(w, tile=True)
    bad = [
        (lambda: mx.quantize_fp8_block(x, "fp6_e3m2"), "element format"),
        (lambda: mx.quantize_fp8_block(x.double()), "float32"),
        (lambda: mx.quantize_fp8_block(x.int()), "float32"),
        (lambda: mx.quantize_fp8_block(x, axes=0), "axes"),
        (lambda: mx.quantize_fp8_block(x, axes=(-1, -1)), "axes"),
        (lambda: mx.quantize_fp8_block(torch.empty(4, 0)), "at least one value"),
        (lambda: mx.quantize_fp8_block(torch.empty(0, 4), axes=-2), "at least one row"),
        (lambda: mx.BlockFP8(w, q.scales), "codes must be"),
        (lambda: mx.BlockFP8(q.codes, q.scales.double()), "scales must be"),
        (lambda: mx.BlockFP8(q.codes, q.scales[:, :0]), "scales of a"),
        (lambda: mx.BlockFP8(q.codes[:, 1:], q.scales), "alignment"),
        (lambda: mx.BlockFP8(torch.zeros(8, 20, dtype=torch.uint8).view(torch.float8_e4m3fn), q.scales), "16 bytes apart"),
        (lambda: mx.BlockFP8(q.codes.t(), q.scales), "unit stride"),
        (lambda: mx.BlockFP8(q.codes[:, :0], q.scales), "at least one value"),
        (lambda: mx.BlockFP8(q.codes, q.scales, q), "transposed"),
        (lambda: mx.fp8_block_matmul(q, w), "BlockFP8"),
        (lambda: mx.fp8_block_matmul(q, mx.quantize_fp8_block(values(3, 31, 1))), "different lengths"),
        (lambda: mx.fp8_block_matmul(q, q, out_dtype=torch.float64), "out_dtype"),
        (lambda: mx.fp8_block_matmul(q, q, torch.zeros(7)), "bias"),
        (lambda: mx.fp8_block_linear(x, w, torch.zeros(4)), "bias"),
        (lambda: mx.fp8_block_linear(x, w[:, :31]), "does not fit"),
        (lambda: mx.fp8_block_linear(x, w[0]), "2-D"),
        (lambda: mx.fp8_block_linear(x, w.double()), "weight must be"),
        (lambda: mx.fp8_block_linear(x, w, elem_format="int8"), "element format"),
        (lambda: mx.fp8_block_linear(x.clone().requires_grad_(), q), "transposed operand"),
        (lambda: mx.Fp8BlockLinear(4, 4, elem_format="int8"), "element format"),
    ]
    for call, words in bad:
        with pytest.raises(MxqError, match=words):
            call()


def test_c_entries_refuse_before_they_launch():
    from microxcaling_b200 import _backend
    L = _backend.lib()
    p = 1 << 20                                            # never dereferenced: every call below is refused
    BAD, ALIGN = -1, -4
    assert L.mxq_fp8_quantize(p, 0, 4, 32, 31, 0, 0, p, 32, p, None, 0, None, None, None) == BAD        # rows overlap
    assert L.mxq_fp8_quantize(p, 0, 4, 32, 32, 2, 0, p, 32, p, None, 0, None, None, None) == BAD        # format
    assert L.mxq_fp8_quantize(p, 0, 4, 32, 32, 0, 0, None, 32, p, None, 0, None, None, None) == BAD     # nothing to write
    assert L.mxq_fp8_quantize(p, 0, 4, 32, 32, 0, 0, p, 40, p, None, 0, None, None, None) == ALIGN
    assert L.mxq_fp8_quantize(p, 0, 4, 32, 32, 0, 0, None, 0, None, p, 2, p, None, None) == ALIGN       # pitch below rows
    assert L.mxq_fp8_quantize(p, 0, 0, 32, 32, 0, 0, p, 32, p, None, 0, None, None, None) == 0
    assert L.mxq_fp8_gemm(p, 32, p, 0, 0, p, 32, p, 0, 0, p, 2, None, 0, 4, 8, 0, None) == BAD          # K = 0
    assert L.mxq_fp8_gemm(p, 16, p, 0, 0, p, 32, p, 0, 0, p, 2, None, 0, 4, 8, 32, None) == BAD         # pitch below K
    assert L.mxq_fp8_gemm(p + 8, 32, p, 0, 0, p, 32, p, 0, 0, p, 2, None, 0, 4, 8, 32, None) == ALIGN
    assert L.mxq_fp8_gemm(p, 32, p, 0, 0, p, 32, p, 0, 0, p, 5, None, 0, 4, 8, 32, None) == BAD         # output type
    assert L.mxq_fp8_gemm(p, 32, p, 0, 0, p, 32, p, 0, 0, p, 2, None, 0, 0, 8, 32, None) == 0
    assert L.mxq_fp8_linear_fwd(p, 0, 32, 0, p, 32, p, 1, 0, p, 0, None, 0, 4, 8, 32, p, 100, None) == BAD   # workspace too small
    assert L.mxq_fp8_linear_fwd(p, 0, 32, 0, p, 32, p, 1, 0, p, 0, None, 0, 4, 8, 32, p + 16, 1 << 20, None) == ALIGN
    assert L.mxq_sum_partials(p, -1, 4, p, 0, None) == BAD
    big = 1 << 30
    assert L.mxq_fp8_linear_fwd_train(p, 0, 32, p, 0, 32, 0, None, 0, p, 0, 1, 1, p, 10, p, big, 4, 8, 32, None) == BAD    # saved too small
    assert L.mxq_fp8_linear_fwd_train(p, 0, 32, p, 0, 32, 0, None, 0, p, 0, 0, 1, None, 0, p, big, 4, 8, 32, None) == BAD
    assert L.mxq_fp8_linear_fwd_train(p, 0, 32, p, 0, 32, 0, None, 0, p, 0, 1, 1, p + 16, big, p, big, 4, 8, 32, None) == ALIGN
    assert L.mxq_fp8_linear_bwd(p, 0, 8, 0, 0, p, big, 0, 1, p, 0, p, 0, None, 0, p, big, 4, 8, 32, None) == BAD           # dx, nothing saved
    assert L.mxq_fp8_linear_bwd(p, 0, 8, 0, 0, p, big, 1, 1, p, 0, p, 0, None, 0, p, 10, 4, 8, 32, None) == BAD
