"""fused_layer_norm and token_logprobs without a GPU: CPU tensors, refusals, the C entries' checks."""
import pytest
import torch

import microxcaling_b200 as mx
import norm_reference as ref
from microxcaling_b200._backend import MxqError


def rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_norm(dtype):
    x, w, b, dy = rand(11, 130, dtype=dtype), rand(130, seed=1, dtype=dtype), rand(130, seed=2, dtype=dtype), rand(11, 130, seed=3, dtype=dtype)
    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    y = mx.fused_layer_norm(*leaves)
    for got, (want, room) in zip((y, *torch.autograd.grad(y, leaves, dy)), ref.layer_norm(x, w, b, 1e-5, dy)):
        # torch's CPU sums may be plain chains over the 130 values: eight times the depth of the kernels'
        assert bool(((got.double() - want).abs() <= 8 * room).all())
    layer = mx.FusedLayerNorm(130)
    assert layer(x.float()).shape == (11, 130) and layer.eps == 1e-5


def test_layer_norm_refusals():
    x, w = rand(4, 32), rand(32)
    for call, words in [(lambda: mx.fused_layer_norm(x.double()), "x must be"), (lambda: mx.fused_layer_norm(x[:, :0]), "at least one"),
                        (lambda: mx.fused_layer_norm(x, w[:31]), "weight must be"), (lambda: mx.fused_layer_norm(x, w.half()), "weight must be"),
                        (lambda: mx.fused_layer_norm(x, None, w[::2]), "bias must be"),
                        (lambda: mx.fused_layer_norm(x.half(), w.half(), w), "one dtype"),
                        (lambda: mx.fused_layer_norm(x, w, w, -1.0), "eps"), (lambda: mx.fused_layer_norm(x, w, w, float("nan")), "eps"),
                        (lambda: mx.FusedLayerNorm((4, 8)), "last dimension only")]:
        with pytest.raises(MxqError, match=words):
            call()


def test_token_logprobs():
    x = rand(3, 5, 40)
    x[0, 0] = -float("inf")
    x[1, 1, 3:] = -float("inf")
    t = torch.randint(0, 3, (3, 5), generator=torch.Generator().manual_seed(4))
    t[2, 2], t[2, 3] = -100, 77
    leaf = x.clone().requires_grad_()
    r = mx.token_logprobs(leaf, t, top=4, entropy=True, temperature=0.5)
    lp = (x.double() * 2).log_softmax(-1)
    ok = torch.ones(3, 5, dtype=torch.bool)
    ok[0, 0] = ok[2, 2] = ok[2, 3] = False
    want = lp.gather(-1, t.clamp(0, 39)[..., None])[..., 0]
    assert torch.allclose(r.logprobs[ok].double(), want[ok], atol=1e-5)
    assert r.logprobs[0, 0] == -float("inf") and r.logprobs[2, 2] == 0 and r.logprobs[2, 3].isnan()
    assert r.entropy[0, 0] == 0 and torch.allclose(r.entropy[1, 1].double(), -(lp[1, 1, :3].exp() * lp[1, 1, :3]).sum(), atol=1e-6)
    assert torch.equal(r.top_tokens, x.sort(dim=-1, descending=True, stable=True)[1][..., :4])
    assert not r.top_logprobs.requires_grad
    dx, = torch.autograd.grad((r.logprobs[ok].sum() + r.entropy.sum()), leaf)
    assert not dx[0, 0].any() and dx[0, 1].isfinite().all()


def test_token_logprobs_refusals():
    x, t = rand(4, 32), torch.zeros(4, dtype=torch.int64)
    for call, words in [(lambda: mx.token_logprobs(x.double(), t), "logits must be"), (lambda: mx.token_logprobs(x[:, :0], t), "at least one"),
                        (lambda: mx.token_logprobs(x, t.int()), "tokens must be"), (lambda: mx.token_logprobs(x, t[:3]), "tokens must be"),
                        (lambda: mx.token_logprobs(x, t, top=33), "top must be"), (lambda: mx.token_logprobs(x[:, :5], t, top=6), "top must be"),
                        (lambda: mx.token_logprobs(x, t, top=-1), "top must be"), (lambda: mx.token_logprobs(x), "nothing is asked"),
                        (lambda: mx.token_logprobs(x, t, temperature=0.0), "temperature"),
                        (lambda: mx.token_logprobs(x, t, temperature=float("inf")), "temperature")]:
        with pytest.raises(MxqError, match=words):
            call()


def test_c_entries_refuse_before_they_launch():
    from microxcaling_b200 import _backend
    L = _backend.lib()
    p, BAD, LARGE, UNSUPPORTED = 1 << 20, -1, -5, -2       # never dereferenced: every call below is refused
    assert L.mxq_layer_norm_fwd(p, 2, 32, p, p, 2, p, p, None, 4, 32, 1e-5, None) == BAD          # mean without rstd
    assert L.mxq_layer_norm_fwd(p, 2, 31, p, p, 2, p, p, p, 4, 32, 1e-5, None) == BAD             # rows overlap
    assert L.mxq_layer_norm_fwd(p, 2, 32, p, p, 1, p, p, p, 4, 32, 1e-5, None) == UNSUPPORTED     # bf16 with fp16 weights
    assert L.mxq_layer_norm_fwd(p, 2, 32, p, p, 2, p, p, p, 0, 32, 1e-5, None) == 0
    assert L.mxq_layer_norm_bwd(p, p, 2, 32, 32, p, 2, None, p, p, None, None, 2, None, 0, 4, 32, None) == BAD     # no statistics
    assert L.mxq_layer_norm_bwd(p, p, 2, 32, 32, p, 2, p, p, p, p, None, 2, p, 8, 4, 32, None) == BAD       # workspace too small
    assert L.mxq_token_logprobs(p, 2, 32, p, -100, 1.0, p, None, None, 33, p, p, 4, 64, None) == LARGE
    assert L.mxq_token_logprobs(p, 2, 64, p, -100, 1.0, p, None, None, 3, None, p, 4, 64, None) == BAD
    assert L.mxq_token_logprobs(p, 2, 64, p, -100, 0.0, p, None, None, 0, None, None, 4, 64, None) == BAD
    assert L.mxq_token_logprobs_grad(p, 2, 64, None, -100, 1.0, p, None, p, None, p, 4, 64, None) == BAD   # gradient without tokens
    assert L.mxq_token_logprobs_grad(p, 2, 64, p, -100, 1.0, p, None, p, p, p, 4, 64, None) == BAD         # g_entropy without entropy
