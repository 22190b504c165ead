"""The operators together, as the head of a language model runs them: layer norm, 8-bit projection to the vocabulary, log
probabilities; a training step eagerly and captured, then scoring with the packed weight."""
import pytest
import torch

import fp8_reference as ref
import norm_reference

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def mx():
    import microxcaling_b200 as mx
    return mx


def head(mx, width, vocab):
    g = torch.Generator().manual_seed(0)
    norm = mx.FusedLayerNorm(width, device="cuda", dtype=BF16)
    proj = mx.Fp8BlockLinear(width, vocab, device="cuda", dtype=BF16)
    with torch.no_grad():
        norm.weight.copy_(1 + 0.1 * torch.randn(width, generator=g))
        norm.bias.copy_(0.1 * torch.randn(width, generator=g))
        proj.weight.copy_(torch.randn(vocab, width, generator=g) * (2 / width ** 0.5))
        proj.bias.copy_(0.1 * torch.randn(vocab, generator=g))
    return norm, proj


def step(mx, norm, proj, x, tokens):
    leaves = [x, norm.weight, norm.bias, proj.weight, proj.bias]
    r = mx.token_logprobs(proj(norm(x)), tokens, entropy=True)
    loss = -(r.logprobs.sum() + 0.01 * r.entropy.sum())
    return [r.logprobs.detach(), r.entropy.detach(), *torch.autograd.grad(loss, leaves)]


@pytest.mark.parametrize("shape", [(2, 50, 192, 1000), (1, 3, 1024, 4100)])
def test_training_step(mx, shape):
    b, t, width, vocab = shape
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(b, t, width, generator=g) + 0.2).to(BF16)
    tokens = torch.randint(0, vocab, (b, t), generator=g)
    tokens[0, 1] = -100                                        # a padded place
    norm, proj = head(mx, width, vocab)
    xd, td = x.cuda().requires_grad_(), tokens.cuda()
    # stage by stage: every stage against 64 bits on the values that the stage before it gave
    h = norm(xd)
    logits = proj(h)
    r = mx.token_logprobs(logits, td, entropy=True)
    norm_reference.check(h.reshape(-1, width), norm_reference.layer_norm(x.reshape(-1, width), norm.weight.detach().cpu(),
                                                                         norm.bias.detach().cpu(), 1e-5)[0])
    hv = ref.quantize(h.detach().reshape(-1, width), "fp8_e4m3")[2]
    wv = ref.quantize(proj.weight, "fp8_e4m3", True)[2]
    norm_reference.check(logits.reshape(-1, vocab), ref.product_bound(hv, wv, BF16, proj.bias.detach().cpu()))
    lp = logits.detach().cpu().double().log_softmax(-1)
    want = lp.gather(-1, tokens.clamp(0)[..., None])[..., 0].masked_fill(tokens < 0, 0.0)
    # fp32 sums over the vocabulary (test_gpu_token_logprobs derives 2^-19 as ample for logits below 32 in magnitude)
    assert float((r.logprobs.detach().cpu().double() - want).abs().max()) <= 2.0 ** -19 * 32
    # the gradient at the logits goes back through the same operands
    got = step(mx, norm, proj, xd, td)
    assert torch.equal(got[0], r.logprobs) and torch.equal(got[1], r.entropy)
    leaf = logits.detach().requires_grad_()
    rr = mx.token_logprobs(leaf, td, entropy=True)
    dl, = torch.autograd.grad(-(rr.logprobs.sum() + 0.01 * rr.entropy.sum()), leaf)
    hl = h.detach().requires_grad_()
    dh, dw, db = torch.autograd.grad(proj(hl), (hl, proj.weight, proj.bias), dl)
    dx, dnw, dnb = torch.autograd.grad(norm(xd), (xd, norm.weight, norm.bias), dh)
    for a, e in zip(got[2:], (dx, dnw, dnb, dw, db)):
        assert torch.equal(a, e)
    # captured and replayed on other values; torch cannot capture a backward pass while an eager graph of its leaves lives
    del h, logits, r, rr, leaf, dl, hl, dh
    graph = torch.cuda.CUDAGraph()
    xs = xd.detach().clone().requires_grad_()
    with torch.cuda.graph(graph):
        held = step(mx, norm, proj, xs, td)
    with torch.no_grad():
        xs.copy_(xd.flip(1))
    graph.replay()
    assert all(torch.equal(a, e) for a, e in zip(step(mx, norm, proj, xd.detach().flip(1).requires_grad_(), td), held))


def test_scoring_with_a_packed_head_on_two_streams(mx):
    norm, proj = head(mx, 512, 3000)
    norm.eval(), proj.eval()
    xs = [torch.randn(n, 512, generator=torch.Generator().manual_seed(n)).to(BF16).cuda() for n in (1, 37)]
    with torch.no_grad():
        want = [mx.token_logprobs(proj(norm(x)), top=5) for x in xs]
        proj.prequantize_weights()
        streams = [torch.cuda.Stream() for _ in xs]
        got = []
        for x, s in zip(xs, streams):                          # both at work at once
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                for _ in range(3):
                    r = mx.token_logprobs(proj(norm(x)), top=5)
                got.append(r)
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
    for a, e in zip(got, want):
        assert torch.equal(a.top_tokens, e.top_tokens) and torch.equal(a.top_logprobs, e.top_logprobs)
    from microxcaling_b200 import _backend
    torch.cuda.synchronize()
    assert _backend.device_status() == 0
