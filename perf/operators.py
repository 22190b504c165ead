"""Cases that measure the operators around a language model's projections: the 8-bit block quantization, the
products on its operands (serving and training), layer normalisation and token log probabilities.

`run` computes a case in its plain form, elementary torch operations in 32 bits; with `own` set it makes the calls a
user makes of microxcaling_b200.  `exact` computes the same outputs in 64 bits from the definitions.

Definitions.  A block of 128 values with maximum magnitude a has the scale s = max(a, 2^-100) * (1 / top), its inverse
r = 1 / s, and the codes RNE(v * r), where top is the largest finite value of the 8-bit format (448 for e4m3, 57344 for
e5m2) and RNE rounds to the format's grid, ties to even.  1 / top, s (which is stored), r and v * r are 32-bit numbers,
each rounded to nearest: values of 8 significant bits over a maximum of 8 significant bits are often ties of the grid, and
which way such a tie falls is part of the definition.  Blocks are 1 x 128 along the contraction axis, or 128 x 128 tiles for weights; a last block may be
shorter.  Scales are stored [K block, row]."""
import math

import torch

own = False

LEAST = 2.0 ** -100
TOP = {"fp8_e4m3": 448.0, "fp8_e5m2": 57344.0}
F8 = {"fp8_e4m3": torch.float8_e4m3fn, "fp8_e5m2": torch.float8_e5m2}
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token's activations before a projection: latency is all there is
        dict(name="quantize_token", op="quantize", rows=1, cols=4096, dtype="bf16", fmt="fp8_e4m3", mode="row"),
        # a training layer's activations: along the features for the product, along the tokens for the weight's gradient
        dict(name="quantize_both", op="quantize", rows=8192, cols=4096, dtype="bf16", fmt="fp8_e4m3", mode="both"),
        # one token through a feed-forward block's gate projection, weights kept in 8 bits
        dict(name="linear_token", op="serve", tokens=1, k=8192, n=28672, dtype="bf16", fmt="fp8_e4m3", bias=False),
        # the same projection of a long prompt batch
        dict(name="linear_prompt", op="serve", tokens=16384, k=8192, n=28672, dtype="bf16", fmt="fp8_e4m3", bias=False),
        # a training step of a square projection
        dict(name="linear_train", op="train", tokens=8192, k=4096, n=4096, dtype="bf16", fmt="fp8_e4m3", grad_fmt="fp8_e4m3", bias=True),
        # a training step of a small projection with no round size, in fp32, gradients in e5m2
        dict(name="linear_train_odd", op="train", tokens=1037, k=1000, n=1511, dtype="fp32", fmt="fp8_e4m3", grad_fmt="fp8_e5m2", bias=True),
        # a few generated tokens through a norm, no gradient
        dict(name="norm_tokens", op="norm", rows=4, cols=8192, dtype="bf16", wdtype="bf16", grad=False),
        # a training step of a block's norm, 4 x 4096 tokens
        dict(name="norm_train", op="norm", rows=16384, cols=8192, dtype="bf16", wdtype="bf16", grad=True),
        # a small model's norm, odd sizes, in fp32
        dict(name="norm_train_odd", op="norm", rows=4099, cols=1001, dtype="fp32", wdtype="fp32", grad=True),
        # generated tokens of a small batch: chosen tokens' log probabilities, entropy and the 20 best alternatives
        dict(name="logprob_tokens", op="logprob", rows=8, vocab=32000, dtype="bf16", top=20, entropy=True, grad=False),
        # scoring and a policy-gradient step over a batch of sequences, large vocabulary
        dict(name="logprob_train", op="logprob", rows=4096, vocab=131072, dtype="bf16", top=0, entropy=True, grad=True),
        # evaluation of a text in fp32 with an odd vocabulary, five alternatives
        dict(name="logprob_odd", op="logprob", rows=333, vocab=50257, dtype="fp32", top=5, entropy=True, grad=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def _odd(rng, n, to):
    """n, half of the time rounded to a multiple of `to`."""
    return max(to, n // to * to) if rng.random() < 0.5 else n


def draw(rng):
    op = rng.choice(["quantize", "serve", "train", "norm", "logprob"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    fmt = rng.choice(["fp8_e4m3", "fp8_e4m3", "fp8_e5m2"])
    if op == "quantize":
        cols = _odd(rng, _log(rng, 16, 16384), 64)
        rows = _odd(rng, _log(rng, 1, min(16384, (1 << 26) // cols)), 8)
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, fmt=fmt, mode=rng.choice(["row", "both", "tile"]))
    if op == "serve":
        k, n = _odd(rng, _log(rng, 64, 16384), 128), _odd(rng, _log(rng, 64, 8192), 128)
        return dict(op=op, tokens=_odd(rng, _log(rng, 1, 4096), 8), k=k, n=n, dtype=dtype, fmt=fmt, bias=rng.random() < 0.5)
    if op == "train":
        k, n = _odd(rng, _log(rng, 16, 8192), 128), _odd(rng, _log(rng, 16, 8192), 128)
        return dict(op=op, tokens=_odd(rng, _log(rng, 1, 8192), 64), k=k, n=n, dtype=dtype, fmt="fp8_e4m3",
                    grad_fmt=rng.choice(["fp8_e4m3", "fp8_e5m2"]), bias=rng.random() < 0.5)
    if op == "norm":
        cols = _odd(rng, _log(rng, 8, 32768), 64)
        rows = _odd(rng, _log(rng, 1, min(32768, (1 << 27) // cols)), 8)
        return dict(op=op, rows=rows, cols=cols, dtype=dtype, wdtype=rng.choice([dtype, "fp32"]), grad=rng.random() < 0.7)
    vocab = _odd(rng, _log(rng, 64, 200000), 64)
    rows = _log(rng, 1, min(8192, (1 << 28) // vocab))
    return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, top=min(rng.choice([0, 1, 5, 20]), vocab), entropy=rng.random() < 0.5,
                grad=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------------- inputs
def _activations(g, rows, cols, dtype):
    """Normal values, a few channels of them far larger, as the activations of language models are."""
    x = torch.randn(rows, cols, generator=g, device="cuda")
    loud = torch.rand(cols, generator=g, device="cuda") < 0.01
    return torch.where(loud, x * 16, x).to(dtype)


def _weight(g, n, k, dtype):
    return ((torch.rand(n, k, generator=g, device="cuda") * 2 - 1) * math.sqrt(3.0 / k)).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    dt = DTYPE[case["dtype"]]
    op = case["op"]
    if op == "quantize":
        s["x"] = _activations(g, case["rows"], case["cols"], dt)
    elif op == "serve":
        t, k, n = case["tokens"], case["k"], case["n"]
        s["x"] = _activations(g, t, k, dt)
        # the weight as a checkpoint in 8 bits holds it: codes with rows padded to 16 bytes, one scale a tile
        codes, s["w_scales"] = _quantize_plain(_weight(g, n, k, torch.float32), case["fmt"], "tile")
        pitch = -(-k // 16) * 16
        held = torch.zeros(n, pitch, dtype=torch.uint8, device="cuda")
        held[:, :k] = codes.view(torch.uint8)
        s["w_codes"] = held.view(F8[case["fmt"]])[:, :k]
        s["bias"] = torch.randn(n, generator=g, device="cuda").to(dt) if case["bias"] else None
    elif op == "train":
        t, k, n = case["tokens"], case["k"], case["n"]
        s["x"] = _activations(g, t, k, dt).requires_grad_()
        s["w"] = _weight(g, n, k, dt).requires_grad_()
        s["bias"] = torch.randn(n, generator=g, device="cuda").to(dt).requires_grad_() if case["bias"] else None
        s["dy"] = (torch.randn(t, n, generator=g, device="cuda") * 1e-3).to(dt)
    elif op == "norm":
        s["x"] = (_activations(g, case["rows"], case["cols"], torch.float32) + 0.5).to(dt).requires_grad_(case["grad"])
        wt = DTYPE[case["wdtype"]]
        s["w"] = (1 + 0.1 * torch.randn(case["cols"], generator=g, device="cuda")).to(wt).requires_grad_(case["grad"])
        s["b"] = (0.1 * torch.randn(case["cols"], generator=g, device="cuda")).to(wt).requires_grad_(case["grad"])
        s["dy"] = torch.randn(case["rows"], case["cols"], generator=g, device="cuda").to(dt) if case["grad"] else None
    else:
        rows, vocab = case["rows"], case["vocab"]
        x = torch.empty(rows, vocab, dtype=dt, device="cuda")
        for i in range(0, rows, 512):                          # in parts: the fp32 values of the largest case need not exist at once
            part = 2.5 * torch.randn(min(512, rows - i), vocab, generator=g, device="cuda")
            part[torch.rand(part.shape, generator=g, device="cuda") < 0.02] = -math.inf      # tokens that a grammar bars
            x[i:i + 512] = part
        s["tokens"] = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
        x[torch.arange(rows, device="cuda"), s["tokens"]] = (6 + torch.randn(rows, generator=g, device="cuda")).to(dt)
        s["x"] = x.requires_grad_(case["grad"])
        s["g_lp"] = torch.randn(rows, generator=g, device="cuda") / rows if case["grad"] else None
        s["g_h"] = torch.randn(rows, generator=g, device="cuda") * 0.01 / rows if case["grad"] and case["entropy"] else None
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _quantize_plain(x, fmt, mode):
    """(codes, scales [K block, row or 128-row tile]) of x [rows, K], blocks along K."""
    x = x.float()
    rows, k = x.shape
    kb = -(-k // 128)
    rp = -(-rows // 128) * 128 if mode == "tile" else rows
    full = torch.nn.functional.pad(x, (0, kb * 128 - k, 0, rp - rows))
    per = 128 if mode == "tile" else 1
    blocks = full.view(rp // per, per, kb, 128)
    s = blocks.abs().amax(dim=(1, 3)).clamp(min=LEAST) * torch.tensor(1.0 / TOP[fmt], dtype=torch.float32, device=x.device)
    r = torch.ones_like(s) / s
    q = (blocks * r[:, None, :, None]).clamp(-TOP[fmt], TOP[fmt]).view(rp, kb * 128)[:rows, :k]
    return q.to(F8[fmt]), s.t().contiguous()


def _tile_values(codes, scales):
    n, k = codes.shape
    return codes.float() * scales.t().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]


def _row_values(x, fmt):
    codes, s = _quantize_plain(x, fmt, "row")
    return codes.float() * s.t().repeat_interleave(128, 1)[:, :x.shape[1]]


def _plain(s):
    op, dt = s["op"], DTYPE[s["dtype"]]
    x = s["x"].detach()
    if op == "quantize":
        codes, scales = _quantize_plain(x, s["fmt"], "tile" if s["mode"] == "tile" else "row")
        if s["mode"] == "row":
            return [codes, scales]
        if s["mode"] == "tile":
            return [codes, scales, codes.view(torch.uint8).t().contiguous().view(codes.dtype), scales.t().contiguous()]
        tcodes, tscales = _quantize_plain(x.t(), s["fmt"], "row")
        return [codes, scales, tcodes, tscales]
    if op == "serve":
        y = _row_values(x, s["fmt"]) @ _tile_values(s["w_codes"], s["w_scales"]).t()
        return [(y if s["bias"] is None else y + s["bias"].float()).to(dt)]
    if op == "train":
        w, dy = s["w"].detach(), s["dy"]
        wq = _tile_values(*_quantize_plain(w, s["fmt"], "tile"))
        y = _row_values(x, s["fmt"]) @ wq.t()
        if s["bias"] is not None:
            y = y + s["bias"].detach().float()
        dx = _row_values(dy, s["grad_fmt"]) @ wq
        dw = _row_values(dy.t(), s["grad_fmt"]) @ _row_values(x.t(), s["fmt"]).t()
        out = [y.to(dt), dx.to(dt), dw.to(dt)]
        return out + ([dy.float().sum(0).to(dt)] if s["bias"] is not None else [])
    if op == "norm":
        w, b = s["w"].detach(), s["b"].detach()
        xf = x.float()
        d = xf - xf.mean(1, keepdim=True)
        rstd = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + 1e-5)
        xhat = d * rstd
        y = (xhat * w.float() + b.float()).to(dt)
        if not s["grad"]:
            return [y]
        dy = s["dy"].float()
        g = dy * w.float()
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        return [y, dx.to(dt), (dy * xhat).sum(0).to(w.dtype), dy.sum(0).to(b.dtype)]
    xf = x.float()
    m = xf.amax(1, keepdim=True)
    e = torch.exp(xf - m)
    z = e.sum(1, keepdim=True)
    lse = m + torch.log(z)
    out = [(xf.gather(1, s["tokens"][:, None]) - lse).squeeze(1)]
    p = e / z
    lp = xf - lse
    plp = torch.where(e > 0, p * lp, torch.zeros_like(p)) if s["entropy"] else None
    h = -plp.sum(1) if s["entropy"] else None
    if s["entropy"]:
        out.append(h)
    if s["top"]:
        v, i = torch.sort(x, dim=1, descending=True, stable=True)
        out += [v[:, :s["top"]].float() - lse, i[:, :s["top"]]]
    if s["grad"]:
        d = -p * s["g_lp"][:, None]
        if s["entropy"]:
            d = d - s["g_h"][:, None] * (plp + p * h[:, None])
        d.scatter_add_(1, s["tokens"][:, None], s["g_lp"][:, None])
        out.append(d.to(dt))
    return out


# ---------------------------------------------------------------------------------------------------- the framework's calls
def _own(s):
    import microxcaling_b200 as mx
    op = s["op"]
    if op == "quantize":
        if s["mode"] == "row":
            q = mx.quantize_fp8_block(s["x"], s["fmt"])
            return [q.codes, q.scales]
        a, b = mx.quantize_fp8_block(s["x"], s["fmt"], axes=(-1, -2), tile=s["mode"] == "tile")
        return [a.codes, a.scales, b.codes, b.scales]
    if op == "serve":
        w = mx.BlockFP8(s["w_codes"], s["w_scales"])
        return [mx.fp8_block_linear(s["x"], w, s["bias"], elem_format=s["fmt"])]
    if op == "train":
        y = mx.fp8_block_linear(s["x"], s["w"], s["bias"], elem_format=s["fmt"], grad_elem_format=s["grad_fmt"])
        leaves = [s["x"], s["w"]] + ([s["bias"]] if s["bias"] is not None else [])
        return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]
    if op == "norm":
        y = mx.fused_layer_norm(s["x"], s["w"], s["b"], eps=1e-5)
        return [y.detach(), *torch.autograd.grad(y, [s["x"], s["w"], s["b"]], s["dy"])] if s["grad"] else [y]
    r = mx.token_logprobs(s["x"], s["tokens"], top=s["top"], entropy=s["entropy"])
    out = [r.logprobs.detach()] + ([r.entropy.detach()] if s["entropy"] else [])
    if s["top"]:
        out += [r.top_logprobs, r.top_tokens]
    if s["grad"]:
        outs, gs = ([r.logprobs, r.entropy], [s["g_lp"], s["g_h"]]) if s["entropy"] else ([r.logprobs], [s["g_lp"]])
        out += torch.autograd.grad(outs, [s["x"]], gs)
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


# ---------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    op, b = case["op"], SIZE[case["dtype"]]
    if op == "quantize":
        n, rb, cb = case["rows"] * case["cols"], -(-case["rows"] // 128), -(-case["cols"] // 128)
        out = n + 4 * case["rows"] * cb
        if case["mode"] == "both":
            out += n + 4 * case["cols"] * rb
        elif case["mode"] == "tile":
            out = 2 * (n + 4 * rb * cb)
        return {"bytes": n * b + out, "flops": 3 * n}
    if op in ("serve", "train"):
        t, k, n = case["tokens"], case["k"], case["n"]
        if op == "serve":
            return {"bytes": t * k * b + n * k + 4 * -(-n // 128) * -(-k // 128) + t * n * b + (n * b if case["bias"] else 0), "flops": 2 * t * k * n}
        return {"bytes": 2 * b * (t * k + n * k + t * n) + (2 * n * b if case["bias"] else 0), "flops": 6 * t * k * n}
    if op == "norm":
        n, wb = case["rows"] * case["cols"], SIZE[case["wdtype"]]
        # the backward pass needs the statistics of the whole row: x and dy are read once, y and dx written once
        return {"bytes": n * b * (4 if case["grad"] else 2) + case["cols"] * wb * (4 if case["grad"] else 2), "flops": n * (20 if case["grad"] else 8)}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * b * (2 if case["grad"] else 1) + case["rows"] * (24 + 12 * case["top"]), "flops": n * (10 if case["grad"] else 5)}


# ---------------------------------------------------------------------------------------------------- 64 bits
def _grid64(v, fmt):
    """v rounded to the format's grid in 64 bits, ties to even, magnitudes above the largest value set to it."""
    bits, low = (3, -6) if fmt == "fp8_e4m3" else (2, -14)
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), torch.clamp(e - 1, min=low) - bits)
    return torch.clamp(torch.round(v / step) * step, -TOP[fmt], TOP[fmt])


def _quantize64(x, fmt, per=1):
    """(codes, scale of each value, scales [K block, row group]) of x [rows, K] in 64 bits, but for the numbers that
    the definition rounds to 32; `per` rows share a scale."""
    rows, k = x.shape
    x = x.double()
    rp, kb = -(-rows // per), -(-k // 128)
    a = torch.zeros(rp * per, kb * 128, dtype=torch.float64, device=x.device)
    a[:rows, :k] = x.abs()
    a = a.reshape(rp, per, kb, 128).amax(3).amax(1)
    inv_top = torch.tensor(1 / TOP[fmt], dtype=torch.float64, device=x.device).float().double()
    s = (torch.maximum(a, torch.full_like(a, LEAST)) * inv_top).float().double()
    r = (1 / s).float().double()
    row, block = torch.arange(rows, device=x.device) // per, torch.arange(k, device=x.device) // 128
    return _grid64((x * r[row][:, block]).float().double(), fmt), s[row][:, block], s.T


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    with torch.no_grad():
        x = s["x"].detach()
        if op == "quantize":
            per = 128 if case["mode"] == "tile" else 1
            q, _, sc = _quantize64(x, case["fmt"], per)
            if case["mode"] == "row":
                return [q, sc]
            qt, _, sct = _quantize64(x.T, case["fmt"], per)
            return [q, sc, qt, sct]
        if op in ("serve", "train"):
            q, each, _ = _quantize64(x, case["fmt"])
            xv = q * each
            del q, each
            if op == "serve":
                n, k = s["w_codes"].shape
                sw = s["w_scales"].double().T[torch.arange(n, device="cuda") // 128][:, torch.arange(k, device="cuda") // 128]
                y = torch.matmul(xv, (s["w_codes"].double() * sw).T)
                return [y if s["bias"] is None else y.add_(s["bias"].double())]
            q, each, _ = _quantize64(s["w"].detach(), case["fmt"], 128)
            wv = q * each
            y = torch.matmul(xv, wv.T)
            if s["bias"] is not None:
                y += s["bias"].detach().double()
            q, each, _ = _quantize64(s["dy"], case["grad_fmt"])
            dx = torch.matmul(q * each, wv)
            q, each, _ = _quantize64(s["dy"].T, case["grad_fmt"])
            qx, ex, _ = _quantize64(x.T, case["fmt"])
            dw = torch.matmul(q * each, (qx * ex).T)
            return [y, dx, dw] + ([s["dy"].double().sum(0)] if s["bias"] is not None else [])
        if op == "norm":
            x, w, b = x.double(), s["w"].detach().double(), s["b"].detach().double()
            n = x.shape[1]
            mu = x.sum(1, keepdim=True) / n
            var = ((x - mu) ** 2).sum(1, keepdim=True) / n
            inv = (var + 1e-5) ** -0.5
            xh = (x - mu) * inv
            y = w * xh + b
            if not case["grad"]:
                return [y]
            dy = s["dy"].double()
            t = dy * w
            dx = (n * t - t.sum(1, keepdim=True) - xh * (t * xh).sum(1, keepdim=True)) * (inv / n)
            return [y, dx, (dy * xh).sum(0), dy.sum(0)]
        lp = torch.log_softmax(x.double(), 1)
        rows = torch.arange(x.shape[0], device="cuda")
        out = [lp[rows, s["tokens"]]]
        p = lp.exp()
        if case["entropy"]:
            lp0 = torch.where(p > 0, lp, 0.0)
            h = -(p * lp0).sum(1)
            out.append(h)
        if case["top"]:
            # larger values first, the lowest index first among equals
            i = torch.argsort(-x.double(), dim=1, stable=True)[:, :case["top"]]
            out += [lp.gather(1, i), i]
        if case["grad"]:
            d = -s["g_lp"].double()[:, None] * p
            if case["entropy"]:
                d -= s["g_h"].double()[:, None] * p * (lp0 + h[:, None])
            d[rows, s["tokens"]] += s["g_lp"].double()
            out.append(d)
        return out
