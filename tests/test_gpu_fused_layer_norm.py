"""fused_layer_norm on the GPU against 64 bits, within bounds derived in norm_reference."""
import pytest
import torch

import norm_reference as ref

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def inputs(rows, cols, dtype, wdtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g) * 2 + 0.7).to(dtype)
    w, b = (1 + 0.3 * torch.randn(cols, generator=g)).to(wdtype), torch.randn(cols, generator=g).to(wdtype)
    return x, w, b, torch.randn(rows, cols, generator=g).to(dtype)


@pytest.fixture(scope="module")
def mx():
    import microxcaling_b200 as mx
    return mx


# around every border of the row shapes, whole vectors and odd lengths, and past what registers and shared memory hold
COLS = [1, 2, 7, 8, 64, 250, 256, 260, 512, 513, 1000, 1024, 1032, 2048, 2049, 4096, 4104, 8192, 8200, 16384, 20001, 25600, 25608]


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtypes", [(BF16, BF16), (BF16, F32), (F16, F16), (F32, F32)])
def test_forward_and_gradients(mx, cols, dtypes):
    for rows in (1, 5, 333 if cols <= 8200 else 170):
        x, w, b, dy = inputs(rows, cols, *dtypes, seed=rows)
        leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
        y = mx.fused_layer_norm(*leaves, eps=1e-5)
        got = (y, *torch.autograd.grad(y, leaves, dy.cuda()))
        for t, pair, like in zip(got, ref.layer_norm(x, w, b, 1e-5, dy), (x, x, w, b)):
            assert t.dtype == like.dtype and t.shape == like.shape
            ref.check(t, pair)


@pytest.mark.parametrize("cols", [16, 264, 520, 1024, 1032, 2048, 2056, 4096, 4104, 8192, 9008])
@pytest.mark.parametrize("dtypes", [(BF16, BF16), (F16, F32), (F32, F32)])
def test_many_rows(mx, cols, dtypes):
    """More rows than four on an SM: other shapes of the forward kernel, and every ring of the gradient's wraps around."""
    x, w, b, dy = inputs(1300 if cols <= 4104 else 700, cols, *dtypes, seed=cols)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = mx.fused_layer_norm(*leaves)
    for t, pair in zip((y, *torch.autograd.grad(y, leaves, dy.cuda())), ref.layer_norm(x, w, b, 1e-5, dy)):
        ref.check(t, pair)


@pytest.mark.parametrize("cols", [24, 129, 4096, 9000])
def test_parts_and_missing_weights(mx, cols):
    x, w, b, dy = inputs(40, cols, BF16, F32)
    full = [t.cuda().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(mx.fused_layer_norm(*full), full, dy.cuda())
    for i in range(3):
        only = [t.detach().requires_grad_(j == i) for j, t in enumerate(full)]
        assert torch.equal(torch.autograd.grad(mx.fused_layer_norm(*only), only[i], dy.cuda())[0], grads[i])
    for ww, bb in ((w, None), (None, b), (None, None)):
        leaves = [None if t is None else t.cuda().requires_grad_() for t in (x, ww, bb)]
        y = mx.fused_layer_norm(*leaves)
        want = ref.layer_norm(x, ww, bb, 1e-5, dy)
        ref.check(y, want[0])
        have = [t for t in leaves if t is not None]
        got = torch.autograd.grad(y, have, dy.cuda())
        pairs = [want[1]] + ([want[2]] if ww is not None else []) + ([want[3]] if bb is not None else [])
        if bb is not None and ww is None:
            pairs[-1] = (want[3][0], want[3][1])
        for t, pair in zip(got, pairs):
            ref.check(t, pair)


def test_strides_offsets_and_leading_dimensions(mx):
    x, w, b, dy = inputs(64, 1040, BF16, BF16)
    xd, wd, bd = x.cuda(), w.cuda(), b.cuda()
    for view, dview in ((x[:, 3:700], xd[:, 3:700]), (x[::2, 8:1032], xd[::2, 8:1032]), (x.t()[:300], xd.t()[:300]),
                        (x.view(4, 16, 1040), xd.view(4, 16, 1040)), (x[:, :1].expand(64, 16), xd[:, :1].expand(64, 16))):
        n = view.shape[-1]
        flat = view.reshape(-1, n)
        y = mx.fused_layer_norm(dview, wd[:n].contiguous(), bd[:n].contiguous())
        assert y.shape == view.shape
        ref.check(y.reshape(-1, n), ref.layer_norm(flat, w[:n], b[:n], 1e-5)[0])
    # weights that start off a 16-byte border, a gradient that is expanded
    leaf = xd[:, :1024].clone().requires_grad_()
    off = wd[1:1025]
    g, = torch.autograd.grad(mx.fused_layer_norm(leaf, off, bd[1:1025]).sum(), leaf)
    ref.check(g, ref.layer_norm(x[:, :1024], w[1:1025], b[1:1025], 1e-5, torch.ones(64, 1024, dtype=BF16))[1])


def test_constant_rows_nan_and_no_rows(mx):
    x = torch.full((3, 512), 7.0, device="cuda", dtype=BF16)
    assert not mx.fused_layer_norm(x).any()
    x[1, 5] = float("nan")
    y = mx.fused_layer_norm(x)
    assert y[1].isnan().all() and not y[0].any() and not y[2].any()
    e = torch.empty(0, 64, device="cuda", dtype=BF16, requires_grad=True)
    w = torch.ones(64, device="cuda", dtype=BF16, requires_grad=True)
    y = mx.fused_layer_norm(e, w)
    ge, gw = torch.autograd.grad(y, (e, w), y.detach())
    assert y.shape == (0, 64) and ge.shape == (0, 64) and not gw.any()


def test_same_bits_on_another_stream_and_in_a_graph(mx):
    x, w, b, dy = (t.cuda() for t in inputs(777, 2048, BF16, BF16))

    def step():
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = mx.fused_layer_norm(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(p, q) for p, q in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    x.copy_(x.flip(0))
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(step(), held))
