"""Log probabilities of tokens under a model's logits: what perplexity, likelihood scores and policy gradients are made of.

The framework's softmax emulates a vector format step by step; here nothing is emulated: fp32 arithmetic on the logits as they
are, one pass over a row for the log probability, the entropy and the alternatives, one more for the gradient.  No counterpart
in the reference."""
import collections

import torch
from torch.autograd.function import once_differentiable

from . import _backend
from ._backend import LOGPROBS_MAX_TOP, MxqError

_FLOATS = (torch.float32, torch.float16, torch.bfloat16)
TokenLogprobs = collections.namedtuple("TokenLogprobs", "logprobs entropy top_logprobs top_tokens")


def _run(x, tokens, top, entropy, inv_t, ignore_index, want_stats):
    """(rows of x, tokens, statistics, entropy as the kernel wrote them; the outputs in the shape of x's leading dimensions)"""
    x2 = _backend.rows_of(x)
    t = None if tokens is None else tokens.reshape(-1).contiguous()
    lp, h, stats, tlp, tok = _backend.token_logprobs(x2, t, ignore_index, inv_t, entropy, top, want_stats)
    out = (lp, h, tlp, tok)
    if x.dim() != 2:
        out = tuple(None if o is None else o.view(x.shape[:-1] + o.shape[1:]) for o in out)
    return x2, t, stats, h, out


class TokenLogprobsFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, tokens, top, entropy, inv_t, ignore_index):
        x2, t, stats, h, out = _run(x, tokens, top, entropy, inv_t, ignore_index, True)
        ctx.save_for_backward(x2, t, stats, h)
        ctx.args = (inv_t, ignore_index, x.shape)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(*out[2:])
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_h, g_tlp, g_tok):
        x2, t, stats, h = ctx.saved_tensors
        inv_t, ignore_index, shape = ctx.args
        if g_lp is None and g_h is None:
            return (None,) * 6
        flat = [None if g is None else g.reshape(-1).contiguous() for g in (g_lp, g_h)]
        dx = _backend.token_logprobs_grad(x2, t, ignore_index, inv_t, stats, h, *flat)
        return dx.view(shape), None, None, None, None, None


def _host(x, tokens, top, entropy, inv_t, ignore_index):
    """The definition as torch operations (differentiable)."""
    v = x.float() * inv_t
    V = v.shape[-1]
    empty = (v == -float("inf")).all(-1, keepdim=True)
    lp = v.masked_fill(empty, 0.0).log_softmax(-1)
    out = [None] * 4
    if tokens is not None:
        inside = (tokens >= 0) & (tokens < V)
        got = lp.gather(-1, tokens.where(inside, torch.zeros_like(tokens))[..., None])[..., 0]
        got = got.masked_fill(~inside, float("nan")).masked_fill(tokens == ignore_index, 0.0)
        out[0] = got.masked_fill(empty[..., 0] & inside & (tokens != ignore_index), -float("inf"))
    if entropy:
        p = lp.exp()
        out[1] = -(p * lp.masked_fill(p == 0, 0.0)).sum(-1).masked_fill(empty[..., 0], 0.0)
    if top:
        i = x.detach().sort(dim=-1, descending=True, stable=True)[1][..., :top]
        out[2] = lp.detach().gather(-1, i).masked_fill(empty, -float("inf"))
        out[3] = i
    return out


def token_logprobs(logits, tokens=None, top=0, entropy=False, temperature=1.0, ignore_index=-100):
    """Log probabilities under softmax(logits / temperature) over the last dimension: TokenLogprobs of

    logprobs      [...] float32: those of `tokens` [...] (int64; None without tokens).  ignore_index gives 0 and takes no part in
                  the gradient; any other index outside the vocabulary gives NaN
    entropy       [...] float32, with entropy=True
    top_logprobs  [..., top] float32 and top_tokens [..., top] int64: the `top` (at most 32) largest logits, largest first, the lowest
                  index first among equals; not differentiable
    logprobs and entropy are differentiable with respect to the logits.  -inf logits have probability 0; a row of nothing else has
    log probability -inf, entropy 0 and gradient 0; a NaN or +inf makes its row NaN."""
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _FLOATS:
        raise MxqError("logits must be a float32, float16 or bfloat16 tensor")
    if logits.dim() == 0 or logits.shape[-1] == 0:
        raise MxqError("logits need at least one value along the last dimension")
    if tokens is not None and (tokens.dtype != torch.int64 or tokens.shape != logits.shape[:-1] or tokens.device != logits.device):
        raise MxqError("tokens must be an int64 tensor of shape %s on the logits' device" % (list(logits.shape[:-1]),))
    if not 0 <= top <= min(LOGPROBS_MAX_TOP, logits.shape[-1]):
        raise MxqError("top must be between 0 and %d, and not above the vocabulary" % LOGPROBS_MAX_TOP)
    if tokens is None and not top and not entropy:
        raise MxqError("nothing is asked for: give tokens, top or entropy")
    if not 0 < temperature < float("inf"):
        raise MxqError("temperature must be positive and finite")
    args = (logits, tokens, int(top), bool(entropy), 1.0 / temperature, int(ignore_index))
    if not logits.is_cuda:
        return TokenLogprobs(*_host(*args))
    if logits.requires_grad and torch.is_grad_enabled():
        return TokenLogprobs(*TokenLogprobsFunction.apply(*args))
    if logits.requires_grad or logits.dim() != 2:
        with torch.no_grad():
            return TokenLogprobs(*_run(*args, False)[4])
    return TokenLogprobs(*_run(*args, False)[4])
