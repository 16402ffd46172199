"""The embedding head's autograd forms and refusals, where no GPU is needed: the calls that would launch kernels are
replaced by plain formulas, or are refused before they touch the device."""

import pytest

torch = pytest.importorskip("torch")

from hessboost_b200 import head  # noqa: E402


def plain(monkeypatch):
    """head's forward and backward calls as torch formulas on the CPU, as unknown to autograd as kernels are."""

    def embed_forward(tokens, table, *, row_ptr=None, scale=1.0):
        return table[tokens].sum(1) * scale

    def embed_backward(grad, tokens, n_tokens, *, row_ptr=None, scale=1.0):
        out = grad.new_zeros(n_tokens, grad.shape[1])
        return out.index_add(0, tokens.reshape(-1), grad.repeat_interleave(tokens.shape[1], 0) * scale)

    def layer_norm_forward(x, weight=None, bias=None, *, eps=1e-5):
        mean, rstd = x.mean(1), 1 / (x.var(1, unbiased=False) + eps).sqrt()
        return (x - mean[:, None]) * rstd[:, None] * weight + bias, mean, rstd

    def layer_norm_backward(dy, x, weight, mean, rstd, *, params=True):
        xh, g = (x - mean[:, None]) * rstd[:, None], dy * weight
        dx = rstd[:, None] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        return dx, (dy * xh).sum(0), dy.sum(0)

    def linear_xent_forward(x, weight, labels):
        z = x @ weight.T
        lse = torch.logsumexp(z, 1)
        return lse - z.gather(1, labels[:, None])[:, 0], lse

    def linear_xent_backward(dloss, x, weight, labels, lse):
        g = torch.exp(x @ weight.T - lse[:, None])
        g.scatter_add_(1, labels[:, None], -torch.ones_like(g[:, :1]))
        g *= dloss[:, None]
        return g @ weight, g.T @ x

    for f in (embed_forward, embed_backward, layer_norm_forward, layer_norm_backward, linear_xent_forward, linear_xent_backward):
        monkeypatch.setattr(head, f.__name__, torch.no_grad()(f))


def forms():
    g = torch.Generator().manual_seed(0)
    x, w, b = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((5, 6), (7, 6), (6,)))
    tok, labels = torch.randint(7, (5, 3), generator=g), torch.randint(7, (5,), generator=g)
    fn = torch.nn.functional
    return {
        "embed": (lambda w: head.embed(tok, w, scale=0.5), lambda w: fn.embedding(tok, w).sum(1) * 0.5, [w]),
        "layer_norm": (head.layer_norm, lambda x, w, b: fn.layer_norm(x, (6,), w, b), [x, w[0], b]),
        "linear_xent": (lambda x, w: head.linear_xent(x, w, labels),
                        lambda x, w: fn.cross_entropy(x @ w.T, labels, reduction="none"), [x, w]),
    }


@pytest.mark.parametrize("name", ["embed", "layer_norm", "linear_xent"])
def test_gradients_are_differentiable_once(monkeypatch, name):
    plain(monkeypatch)
    own, torchs, leaves = forms()[name]
    p = [t.clone().requires_grad_() for t in leaves]
    q = [t.clone().requires_grad_() for t in leaves]
    first = torch.autograd.grad(own(*p).square().sum(), p)
    for a, b in zip(first, torch.autograd.grad(torchs(*q).square().sum(), q)):
        assert torch.allclose(a, b, rtol=1e-9, atol=1e-12)
    # a gradient penalty beside another term: without its own part it would be wrong, so it has to raise
    grads = torch.autograd.grad(own(*p).square().sum(), p, create_graph=True)
    penalty = sum(t.square().sum() for t in grads) + sum(t.square().sum() for t in p)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        penalty.backward()
