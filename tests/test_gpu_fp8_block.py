"""The 8-bit block operators on the GPU: codes and scales bit for bit against the definition, products within the rounding
they are allowed (fp8_reference.product_bound), gradients against the formula's."""
import pytest
import torch

import fp8_reference as ref

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def mx():
    import microxcaling_b200 as mx
    yield mx
    from microxcaling_b200 import _backend
    assert _backend.device_status() == 0


def values(rows, cols, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * scale
    x[:, ::7] *= 30
    return x.to(dtype)


def same_operand(q, x, fmt, tile):
    codes, scales, _ = ref.quantize(x, fmt, tile)
    assert torch.equal(q.scales.cpu(), scales)
    assert torch.equal(q.codes.cpu().double(), codes)


SHAPES = [(1, 1), (1, 4096), (3, 16), (7, 129), (128, 128), (129, 127), (200, 333), (257, 1000), (1030, 640)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("fmt", ["fp8_e4m3", "fp8_e5m2"])
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize(mx, shape, fmt, dtype):
    x = values(*shape, dtype, 1)
    for tile in (False, True):
        a, b = mx.quantize_fp8_block(x.cuda(), fmt, axes=(-1, -2), tile=tile)
        same_operand(a, x, fmt, tile)
        same_operand(b, x.t(), fmt, tile)
        same_operand(mx.quantize_fp8_block(x.cuda(), fmt, tile=tile), x, fmt, tile)
        same_operand(mx.quantize_fp8_block(x.cuda(), fmt, axes=-2, tile=tile), x.t(), fmt, tile)


def test_quantize_every_bf16_value(mx):
    """Every finite bf16 pattern, in blocks whose maxima run over the exponents."""
    bits = torch.arange(0, 1 << 16, dtype=torch.int32).to(torch.int16).view(BF16)
    bits = torch.where(torch.isfinite(bits.float()), bits.float(), torch.zeros(())).to(BF16)
    order = torch.randperm(1 << 16, generator=torch.Generator().manual_seed(0))
    for x in (bits.view(512, 128), bits[order].view(512, 128)):
        same_operand(mx.quantize_fp8_block(x.cuda()), x, "fp8_e4m3", False)
        same_operand(mx.quantize_fp8_block(x.cuda(), "fp8_e5m2"), x, "fp8_e5m2", False)


def test_quantize_special_values(mx):
    x = values(130, 300, F32, 2)
    x[0] = 0
    x[1, :128] = 1e-38
    x[2, 5], x[3, 200], x[4, 299] = float("inf"), float("nan"), float("-inf")
    for tile in (False, True):
        a, b = mx.quantize_fp8_block(x.cuda(), axes=(-1, -2), tile=tile)
        for q, v in ((a, x), (b, x.t())):
            codes, scales, _ = ref.quantize(v, "fp8_e4m3", tile)
            assert torch.equal(q.scales.cpu().isnan(), scales.isnan())
            assert torch.equal(q.scales.cpu().nan_to_num(7), scales.nan_to_num(7))
            assert torch.equal(q.codes.cpu().float().isnan(), codes.isnan())
            assert torch.equal(q.codes.cpu().double().nan_to_num(7), codes.nan_to_num(7))


def test_quantize_strides_and_leading_dimensions(mx):
    x = values(64, 1024, BF16, 3)
    for view in (x[:, 3:600], x[::2, 8:520], x.t()[5:300], x[:, :512].reshape(4, 16, 512)):
        flat = view.reshape(-1, view.shape[-1])
        dev = x.cuda()
        dview = {(64, 597): dev[:, 3:600], (32, 512): dev[::2, 8:520], (295, 64): dev.t()[5:300],
                 (4, 16, 512): dev[:, :512].reshape(4, 16, 512)}[tuple(view.shape)]
        a, b = mx.quantize_fp8_block(dview, axes=(-1, -2))
        same_operand(a, flat, "fp8_e4m3", False)
        same_operand(b, flat.t(), "fp8_e4m3", False)


PRODUCTS = [(1, 1, 1), (1, 4096, 4096), (3, 130, 100), (16, 128, 128), (17, 300, 512), (33, 1, 2000), (64, 256, 1024), (65, 129, 4097),
            (128, 128, 256), (200, 1000, 1511), (300, 520, 640), (777, 1032, 1160), (1024, 1024, 2048),
            (2050, 2304, 1100), (1500, 2311, 384), (9500, 200, 130), (300, 5000, 1)]   # enough 256 x 256 tiles for CTA pairs


@pytest.mark.parametrize("shape", PRODUCTS)
def test_matmul(mx, shape):
    M, N, K = shape
    a, b = values(M, K, BF16, 4), values(N, K, BF16, 5, 0.02)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(6))
    for i, (a_tile, b_tile, fa, fb, out, with_bias) in enumerate([
            (False, True, "fp8_e4m3", "fp8_e4m3", BF16, False), (False, False, "fp8_e5m2", "fp8_e4m3", F32, True),
            (True, False, "fp8_e4m3", "fp8_e5m2", F16, True), (True, True, "fp8_e5m2", "fp8_e5m2", F32, False)]):
        qa, qb = mx.quantize_fp8_block(a.cuda(), fa, tile=a_tile), mx.quantize_fp8_block(b.cuda(), fb, tile=b_tile)
        bb = bias.to(out) if with_bias else None
        y = mx.fp8_block_matmul(qa, qb, None if bb is None else bb.cuda(), out)
        want, room = ref.product_bound(ref.quantize(a, fa, a_tile)[2], ref.quantize(b, fb, b_tile)[2], out, bb)
        off = (y.cpu().double() - want).abs()
        assert y.dtype == out and bool((off <= room).all()), (i, float((off / room).max()))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [(1, 64, 128), (5, 100, 37), (130, 257, 300), (384, 512, 640), (1024, 1024, 1152)])
def test_linear_and_gradients(mx, shape, dtype):
    t, k, n = shape
    x, w = values(t, k, dtype, 7), values(n, k, dtype, 8, 0.01)
    b, dy = values(1, n, dtype, 9)[0], values(t, n, dtype, 10, 1e-2)
    xd, wd, bd = (v.cuda().requires_grad_() for v in (x, w, b))
    y = mx.fp8_block_linear(xd, wd, bd, grad_elem_format="fp8_e5m2")
    dx, dw, db = torch.autograd.grad(y, (xd, wd, bd), dy.cuda())
    xv, wv = ref.quantize(x, "fp8_e4m3")[2], ref.quantize(w, "fp8_e4m3", True)[2]
    dyv, dytv = ref.quantize(dy, "fp8_e5m2")[2], ref.quantize(dy.t(), "fp8_e5m2")[2]
    xtv = ref.quantize(x.t(), "fp8_e4m3")[2]
    for got, (want, room) in ((y, ref.product_bound(xv, wv, dtype, b)), (dx, ref.product_bound(dyv, wv.t(), dtype)),
                              (dw, ref.product_bound(dytv, xtv, dtype))):
        assert got.dtype == dtype and bool(((got.cpu().double() - want).abs() <= room).all())
    want = dy.double().sum(0)
    room = (t + 1) * 2.0 ** -24 * dy.double().abs().sum(0) + want.abs() * torch.finfo(dtype).eps / 2
    assert bool(((db.cpu().double() - want).abs() <= room).all())
    # one gradient at a time is the same gradient
    for i, leaf in enumerate((xd, wd, bd)):
        only = [v.detach().requires_grad_(v is leaf) for v in (xd, wd, bd)]
        g, = torch.autograd.grad(mx.fp8_block_linear(*only, grad_elem_format="fp8_e5m2"), only[i], dy.cuda())
        assert torch.equal(g, (dx, dw, db)[i])


def test_linear_packed_weight(mx):
    x, w, b = values(40, 512, BF16, 11).cuda(), values(300, 512, BF16, 12, 0.02).cuda(), values(1, 300, BF16, 13)[0].cuda()
    full = mx.fp8_block_linear(x, w, b)
    q, qt = mx.quantize_fp8_block(w, axes=(-1, -2), tile=True)
    assert torch.equal(full, mx.fp8_block_linear(x, q, b))
    xl = x.clone().requires_grad_()
    dy = values(40, 300, BF16, 14).cuda()
    g, = torch.autograd.grad(mx.fp8_block_linear(xl, mx.BlockFP8(q.codes, q.scales, qt), b), xl, dy)
    wl = w.clone()
    xr = x.clone().requires_grad_()
    r, = torch.autograd.grad(mx.fp8_block_linear(xr, wl, b), xr, dy)
    assert torch.equal(g, r)
    with pytest.raises(RuntimeError, match="transposed"):
        mx.fp8_block_linear(xl, q, b)
    layer = mx.Fp8BlockLinear(512, 300, device="cuda", dtype=BF16).eval()
    want = layer(x)
    layer.prequantize_weights()
    assert torch.equal(layer(x), want)


def test_linear_no_tokens(mx):
    x = torch.empty(0, 64, device="cuda", dtype=BF16, requires_grad=True)
    w = torch.randn(32, 64, device="cuda", dtype=BF16, requires_grad=True)
    b = torch.randn(32, device="cuda", dtype=BF16, requires_grad=True)
    y = mx.fp8_block_linear(x, w, b)
    assert y.shape == (0, 32)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(0, 32, device="cuda", dtype=BF16))
    assert dx.shape == (0, 64) and not dw.any() and not db.any()
    assert mx.fp8_block_linear(x.detach(), mx.quantize_fp8_block(w, tile=True)).shape == (0, 32)


def test_nan_reaches_every_result_over_its_block(mx):
    x, w = values(20, 256, BF16, 15), values(30, 256, BF16, 16)
    x[3, 7] = float("inf")
    y = mx.fp8_block_linear(x.cuda(), w.cuda()).cpu()
    assert bool(y[3].isnan().all()) and not bool(y[:3].isnan().any()) and not bool(y[4:].isnan().any())


def test_repeats_exactly_on_other_streams_and_in_graphs(mx):
    x, w, b = values(48, 2048, BF16, 17).cuda(), values(512, 2048, BF16, 18, 0.02).cuda(), values(1, 512, BF16, 19)[0].cuda()
    q = mx.quantize_fp8_block(w, tile=True)
    want = mx.fp8_block_linear(x, q, b)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = mx.fp8_block_linear(x, q, b)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = mx.fp8_block_linear(x, q, b)
    x2 = values(48, 2048, BF16, 20).cuda()
    x.copy_(x2)
    for _ in range(3):
        g.replay()
    assert torch.equal(y, mx.fp8_block_linear(x2, q, b))


def test_linear_mixed_types_one_dimension_and_views(mx):
    x, w, b = values(6, 260, BF16, 21), values(260, 90, F32, 22, 0.05), values(1, 90, F32, 23)[0]
    xd, wd, bd = x.cuda().requires_grad_(), w.cuda().t().requires_grad_(), b.cuda().requires_grad_()      # a transposed view as weight
    dy = values(6, 90, BF16, 24)
    y = mx.fp8_block_linear(xd, wd, bd)
    got = (y, *torch.autograd.grad(y, (xd, wd, bd), dy.cuda()))
    xv, wv = ref.quantize(x, "fp8_e4m3")[2], ref.quantize(w.t(), "fp8_e4m3", True)[2]
    dyv, dytv, xtv = (ref.quantize(v, "fp8_e4m3")[2] for v in (dy, dy.t(), x.t()))
    for t, (want, room), dt in ((got[0], ref.product_bound(xv, wv, BF16, b), BF16), (got[1], ref.product_bound(dyv, wv.t(), BF16), BF16),
                                (got[2], ref.product_bound(dytv, xtv, F32), F32)):
        assert t.dtype == dt and bool(((t.detach().cpu().double() - want).abs() <= room).all())
    assert got[3].dtype == F32
    one = mx.fp8_block_linear(xd.detach()[3], wd.detach(), bd.detach())
    assert one.shape == (90,) and torch.equal(one, y.detach()[3])
    leaf = xd.detach()[3].clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(mx.fp8_block_linear(leaf, wd.detach(), bd.detach()), leaf, dy.cuda()[3])[0], got[1][3])


def test_prefix_of_a_larger_buffer_is_left_alone_behind_its_end(mx):
    """The product writes [M, N] and nothing behind it; the operands' padding is not read as values."""
    from microxcaling_b200 import _backend
    for M, N, K in ((3, 130, 100), (300, 1000, 130), (2050, 2311, 200)):
        a, b = (mx.quantize_fp8_block(values(r, K, BF16, r).cuda(), tile=t) for r, t in ((M, False), (N, True)))
        want = mx.fp8_block_matmul(a, b)
        dirty = []
        for o in (a, b):                                       # other bytes in the padding between rows
            pitch = o.codes.stride(0) if o.codes.shape[0] > 1 else (K + 15) // 16 * 16
            buf = torch.full((o.codes.shape[0], pitch), 0x7f, dtype=torch.uint8, device="cuda")
            buf[:, :K] = o.codes.view(torch.uint8) if o.codes.is_contiguous() else o.codes.contiguous().view(torch.uint8)
            dirty.append(mx.BlockFP8(buf.view(torch.float8_e4m3fn)[:, :K], o.scales))
        out = torch.full((M * N + 64,), 7.0, dtype=BF16, device="cuda")
        L = _backend.lib()
        p = [(o.codes.data_ptr(), _backend._pitch(o.codes), o.scales.data_ptr(), int(o.tile), 0) for o in dirty]
        _backend.check(L.mxq_fp8_gemm(*p[0], *p[1], out.data_ptr(), 2, None, 0, M, N, K, _backend._stream(out)))
        assert torch.equal(out[:M * N].view(M, N), want) and bool((out[M * N:] == 7).all())
