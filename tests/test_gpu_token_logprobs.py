"""token_logprobs on the GPU against 64 bits.

Room, with u = 2^-24 and t = x - max: the hardware's 2^v is off by 2^-22 relative, its argument by 2 roundings of |t| log2(e),
so a term of z is off by r(t) = 2^-22 + 3 u (1 + |t|) relative; the sum adds one u per addition of a thread's chain (vocab / 256 for
short rows, vocab / 1024 for long ones) and 12 across threads.  A log probability adds the roundings of x_t - max, log z and
their difference."""
import pytest
import torch

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


@pytest.fixture(scope="module")
def mx():
    import microxcaling_b200 as mx
    return mx


def logits(rows, vocab, dtype, seed=0, barred=0.1):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * 3
    x[torch.rand(rows, vocab, generator=g) < barred] = -float("inf")
    t = torch.randint(0, vocab, (rows,), generator=g)
    x[torch.arange(rows), t] = torch.randn(rows, generator=g) + 2
    return x.to(dtype), t


def reference(x, t, temperature=1.0):
    """lp, H, p, and the rooms of log z, lp and H, in 64 bits."""
    v = x.double() * (1.0 / temperature)
    d = v - v.amax(1, keepdim=True)
    lp = v.log_softmax(1)
    p = lp.exp()
    lp0 = torch.where(p > 0, lp, torch.zeros_like(lp))
    d0 = torch.where(p > 0, d, torch.zeros_like(d)).abs()
    scaling = 2 * U * torch.where(p > 0, v, torch.zeros_like(v)).abs()                 # temperature and its reciprocal in fp32
    r = 2.0 ** -22 + 3 * U * (1 + d0) + scaling + (x.shape[1] / 256 + 14) * U
    e_z = (p * r).sum(1) + U
    H = -(p * lp0).sum(1)
    at = t.clamp(0, x.shape[1] - 1)[:, None]
    log_z = -d.gather(1, lp.argmax(1, keepdim=True))[:, 0] - lp.amax(1)
    e_lp = e_z + 3 * U * (log_z.abs() + d0.gather(1, at)[:, 0] + lp0.gather(1, at)[:, 0].abs()) + scaling.gather(1, at)[:, 0]
    e_H = e_z + (p * d0 * (r + 4 * U)).sum(1) + (p * d0).sum(1) * e_z + 4 * U * (log_z.abs() + H.abs())
    return lp, H, p, e_z + 3 * U * log_z.abs(), e_lp, e_H, r, scaling


VOCABS = [1, 2, 7, 8, 64, 255, 1000, 2048, 8192, 8193, 32000, 50257]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_values_and_gradient(mx, vocab, dtype, temperature):
    x, t = logits(9, vocab, dtype, seed=vocab)
    top = min(vocab, 20)
    leaf = x.cuda().requires_grad_()
    r = mx.token_logprobs(leaf, t.cuda(), top=top, entropy=True, temperature=temperature)
    lp, H, p, e_lz, e_lp, e_H, rel, scaling = reference(x, t, temperature)
    want = lp[torch.arange(9), t]
    assert bool(((r.logprobs.detach().cpu().double() - want).abs() <= e_lp).all())
    assert bool(((r.entropy.detach().cpu().double() - H).abs() <= e_H).all())
    order = x.sort(dim=1, descending=True, stable=True)[1][:, :top]
    assert torch.equal(r.top_tokens.cpu(), order)
    tl, wl = r.top_logprobs.cpu().double(), lp.gather(1, order)
    assert torch.equal(tl.isinf(), wl.isinf())
    room = e_lz[:, None] + 6 * U * (wl.abs() + 40)
    assert bool(((tl - wl).abs().nan_to_num(0) <= room).all())
    # gradient: p is off by its exponent's error (log z, the roundings of log p) and that of 2^v
    g_lp, g_h = torch.randn(9, generator=torch.Generator().manual_seed(1)), torch.randn(9, generator=torch.Generator().manual_seed(2))
    dx, = torch.autograd.grad([r.logprobs, r.entropy], leaf, [g_lp.cuda(), g_h.cuda()])
    lp0 = torch.where(p > 0, lp, torch.zeros_like(lp))
    a, b = g_lp.double()[:, None], g_h.double()[:, None]
    one = torch.zeros_like(p)
    one[torch.arange(9), t] = 1
    inv = 1 / temperature
    want = inv * (a * (one - p) - b * p * (lp0 + H[:, None]))
    size = p * (a.abs() + b.abs() * (lp0.abs() + H.abs()[:, None])) * inv
    r_p = 2.0 ** -22 + 4 * U * (1 + lp0.abs()) + 2 * e_lz[:, None] + scaling + 6 * U
    room = size * (r_p + 8 * U) + inv * p * b.abs() * (r_p * 2 + e_H[:, None]) + 4 * U * want.abs() + \
        (one * a.abs() * inv) * 4 * U + want.abs() * torch.finfo(dtype).eps / 2 + \
        torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps + 2.0 ** -126
    assert dx.dtype == dtype
    assert bool(((dx.cpu().double() - want).abs() <= room).all()), float(((dx.cpu().double() - want).abs() / room).max())
    # each output alone
    leaf2 = x.cuda().requires_grad_()
    one_r = mx.token_logprobs(leaf2, t.cuda(), temperature=temperature)
    assert torch.equal(one_r.logprobs, r.logprobs) and one_r.entropy is None and one_r.top_tokens is None
    g1, = torch.autograd.grad(one_r.logprobs, leaf2, g_lp.cuda())
    want1 = inv * a * (one - p)
    room1 = inv * p * a.abs() * (r_p + 8 * U) + (one * a.abs() * inv) * 4 * U + \
        want1.abs() * (torch.finfo(dtype).eps / 2 + 4 * U) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps + 2.0 ** -126
    assert bool(((g1.cpu().double() - want1).abs() <= room1).all())
    e = mx.token_logprobs(x.cuda(), entropy=True, temperature=temperature)
    assert e.logprobs is None and torch.equal(e.entropy, r.entropy)


@pytest.mark.parametrize("vocab", [8200, 32003])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_rows(mx, vocab, dtype):
    """More rows than SMs: another number of threads a row; rows that start off every 16-byte border."""
    x, t = logits(200, vocab, dtype, seed=7)
    leaf = x.cuda().requires_grad_()
    r = mx.token_logprobs(leaf, t.cuda(), top=32, entropy=True)
    lp, H, p, e_lz, e_lp, e_H, *_ = reference(x, t)
    assert bool(((r.logprobs.detach().cpu().double() - lp[torch.arange(200), t]).abs() <= e_lp).all())
    assert bool(((r.entropy.detach().cpu().double() - H).abs() <= e_H).all())
    assert torch.equal(r.top_tokens.cpu(), x.sort(dim=1, descending=True, stable=True)[1][:, :32])
    g, = torch.autograd.grad(r.logprobs.sum(), leaf)
    want = -p
    want[torch.arange(200), t] += 1
    # 2^-18: log p is at most 40 in magnitude, its exponent and log z are off by a few 2^-22 of that
    room = p * 2.0 ** -18 + want.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -22) + 2.0 ** -40
    assert bool(((g.cpu().double() - want).abs() <= room).all())


def test_gradient_against_differences(mx):
    """d lp / d x_j by central differences of the 64-bit function."""
    x, t = logits(3, 50, F32, seed=5, barred=0)
    leaf = x.cuda().requires_grad_()
    r = mx.token_logprobs(leaf, t.cuda(), entropy=True)
    dx, = torch.autograd.grad((r.logprobs.sum() + 0.5 * r.entropy.sum()), leaf)

    def f(v):
        lp = v.log_softmax(1)
        return lp[torch.arange(3), t].sum() + 0.5 * -(lp.exp() * lp).sum()

    h = 1e-5
    for at in ((0, 0), (1, 17), (2, 49), (0, int(t[0]))):
        hi, lo = x.double(), x.double()
        hi[at] += h
        lo[at] -= h
        # the difference is off by h^2 / 6 times a third derivative (below 10 here) and 2^-53 / h of a sum below 100
        assert abs(float(dx[at]) - float((f(hi) - f(lo)) / (2 * h))) <= 10 * h * h + 100 * 2.0 ** -52 / h + 1e-6


def test_rows_without_a_finite_logit_and_special_values(mx):
    inf = float("inf")
    for dtype in (BF16, F16, F32):
        low = torch.finfo(dtype).min
        for vocab in (100, 9000, 9001):
            x = torch.randn(7, vocab, generator=torch.Generator().manual_seed(3)).to(dtype)
            x[0] = -inf
            x[1] = low                                   # a uniform row of the type's lowest value
            x[2, 1:] = -inf                              # one token left
            x[3, :-1] = low
            x[4, 7] = inf
            x[5, 9] = float("nan")
            t = torch.tensor([3, 3, 0, vocab - 1, 7, 9, 4])
            leaf = x.cuda().requires_grad_()
            r = mx.token_logprobs(leaf, t.cuda(), top=5, entropy=True)
            lp, h = r.logprobs.tolist(), r.entropy.tolist()
            assert lp[0] == -inf and h[0] == 0 and r.top_tokens[0].tolist() == [0, 1, 2, 3, 4]
            assert r.top_logprobs[0].tolist() == [-inf] * 5
            n = torch.log(torch.tensor(float(vocab), dtype=torch.float64)).item()
            assert abs(lp[1] + n) <= 2.0 ** -20 * n and abs(h[1] - n) <= 2.0 ** -20 * n
            assert r.top_tokens[1].tolist() == [0, 1, 2, 3, 4]
            assert lp[2] == 0 and h[2] == 0 and r.top_tokens[2].tolist() == [0, 1, 2, 3, 4]
            assert r.top_logprobs[2].tolist() == [0] + [-inf] * 4
            assert lp[3] == 0 and h[3] == 0 and r.top_tokens[3].tolist() == [vocab - 1, 0, 1, 2, 3]
            assert all(v != v for v in (lp[4], lp[5], h[4], h[5]))
            assert r.top_tokens[4][0] == 7 and r.top_tokens[5][0] == 9
            dx, = torch.autograd.grad((r.logprobs.sum() + r.entropy.sum()), leaf)
            assert not dx[0].any() and not dx[2].any() and not dx[3].any() and dx[4].isnan().all() and dx[5].isnan().all()
            assert dx[6].isfinite().all()


def test_ties_go_to_the_lowest_index(mx):
    x = torch.zeros(4, 20000)
    x[1, ::3] = 1
    x[2] = torch.randint(0, 4, (20000,), generator=torch.Generator().manual_seed(4))
    x[3, 5:] = -0.0
    for dtype in (BF16, F32):
        for top in (1, 20, 32):
            r = mx.token_logprobs(x.to(dtype).cuda(), top=top)
            assert torch.equal(r.top_tokens.cpu(), x.sort(dim=1, descending=True, stable=True)[1][:, :top])


def test_ignored_and_invalid_tokens(mx):
    x, t = logits(6, 300, BF16)
    t[1], t[2], t[3], t[4] = -100, 300, -1, 2 ** 40
    leaf = x.cuda().requires_grad_()
    r = mx.token_logprobs(leaf, t.cuda())
    lp = r.logprobs.tolist()
    assert lp[1] == 0 and all(lp[i] != lp[i] for i in (2, 3, 4))
    dx, = torch.autograd.grad(r.logprobs.sum(), leaf)
    assert not dx[1].any() and dx[2:5].isnan().all() and dx[0].isfinite().all() and dx[5].isfinite().all()
    r = mx.token_logprobs(leaf, t.cuda(), ignore_index=-1)
    assert r.logprobs[3] == 0 and r.logprobs[1].isnan()


def test_strides_and_leading_dimensions(mx):
    x, _ = logits(24, 3000, BF16, seed=8)
    xd = x.cuda()
    for view, dview in ((x[:, 1:2000], xd[:, 1:2000]), (x[::3, 8:2008], xd[::3, 8:2008]), (x.t()[:40], xd.t()[:40]),
                        (x.view(2, 3, 4, 3000), xd.view(2, 3, 4, 3000)), (x[0], xd[0])):
        lead, n = view.shape[:-1], view.shape[-1]
        t = torch.randint(0, n, lead, generator=torch.Generator().manual_seed(9))
        r = mx.token_logprobs(dview, t.cuda(), top=3)
        flat = view.reshape(-1, n)
        lp, _, _, _, e_lp, *_ = reference(flat, t.reshape(-1))
        want = lp[torch.arange(len(flat)), t.reshape(-1)]
        got = r.logprobs.cpu().double()
        assert got.shape == lead and r.top_tokens.shape == (*lead, 3)
        same = (got.reshape(-1) - want).abs() <= e_lp
        assert bool((same | (got.reshape(-1) == want)).all())
        assert torch.equal(r.top_tokens.cpu().reshape(-1, 3), flat.sort(dim=1, descending=True, stable=True)[1][:, :3])


def test_no_rows_streams_and_graphs(mx):
    e = torch.empty(0, 50, device="cuda", requires_grad=True)
    r = mx.token_logprobs(e, torch.empty(0, dtype=torch.int64, device="cuda"), top=3, entropy=True)
    assert r.logprobs.shape == (0,) and r.top_tokens.shape == (0, 3)
    assert torch.autograd.grad(r.logprobs.sum(), e)[0].shape == (0, 50)
    x, t = (v.cuda() for v in logits(64, 32000, BF16, seed=11))

    def step():
        leaf = x.detach().requires_grad_()
        r = mx.token_logprobs(leaf, t, top=20, entropy=True)
        return [r.logprobs.detach(), r.entropy.detach(), r.top_logprobs, r.top_tokens,
                torch.autograd.grad(r.logprobs.sum() + r.entropy.sum(), leaf)[0]]

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    x.copy_(x.flip(0))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(step(), held))
