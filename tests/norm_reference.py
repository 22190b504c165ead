"""Layer normalisation in 64 bits with bounds on what fp32 arithmetic may change, for the tests.

u = 2^-24 is the largest relative rounding error of an fp32 operation.  A sum over n terms held by 32 to 1024 threads
is a chain of at most max(16, n / 1024) additions in a thread and 10 in the tree across threads, so with D that depth plus a few
operations around it a sum is off by at most D u times the sum of magnitudes."""
import torch

U = 2.0 ** -24


def half_step(y, dtype):
    return y.abs() * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def layer_norm(x, w, b, eps, dy=None):
    """[(value in 64 bits, room)] of y, and with dy of dx, dw, db; x, w, b, dy on the CPU."""
    dt, wt = x.dtype, None if w is None else w.dtype
    x = x.double()
    rows, n = x.shape
    D = max(16, n / 1024) + 16
    one = torch.ones(n, dtype=torch.float64)
    w64, b64 = (one if w is None else w.double()), (one * 0 if b is None else b.double())
    mean = x.mean(1, keepdim=True)
    c = x - mean
    var = (c * c).mean(1, keepdim=True)
    rstd = (var + eps) ** -0.5
    e_mean = D * U * x.abs().mean(1, keepdim=True)
    # the variance: its own sum, the centred values' rounding and the mean's error (which enters squared, and times a sum of c
    # that vanishes); half of that, the root and the division reach rstd
    r_rstd = (D + 4) * U + e_mean ** 2 / (var + eps) + 2 * U * (x.abs().amax(1, keepdim=True) + e_mean) * (var + eps) ** -0.5 + 4 * U
    xh = c * rstd
    e_xh = rstd * (e_mean + 2 * U * x.abs()) + xh.abs() * (r_rstd + 2 * U)
    y = xh * w64 + b64
    out = [(y, e_xh * w64.abs() + 2 * U * (y.abs() + (xh * w64).abs()) + half_step(y, dt))]
    if dy is None:
        return out
    dy = dy.double()
    g = dy * w64
    mg, mgx = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    e_mg = D * U * g.abs().mean(1, keepdim=True)
    e_mgx = D * U * (g * xh).abs().mean(1, keepdim=True) + (g.abs() * e_xh).mean(1, keepdim=True)
    dx = rstd * (g - mg - xh * mgx)
    e = rstd * (e_mg + e_xh * mgx.abs() + xh.abs() * e_mgx + 4 * U * (g.abs() + mg.abs() + (xh * mgx).abs())) * (1 + r_rstd) + \
        dx.abs() * (r_rstd + 2 * U)
    out.append((dx, e + half_step(dx, dt)))
    dw, db = (dy * xh).sum(0), dy.sum(0)
    e_dw = (rows + 4) * U * (dy * xh).abs().sum(0) + (dy.abs() * e_xh).sum(0)
    out.append((dw, e_dw + half_step(dw, wt or dt)))
    out.append((db, (rows + 4) * U * dy.abs().sum(0) + half_step(db, wt or dt)))
    return out


def check(got, pair):
    want, room = pair
    off = (got.detach().cpu().double() - want).abs()
    assert bool((off <= room).all()), float((off / room).max())
