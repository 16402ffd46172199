"""The embedding head's autograd forms and refusals, where no GPU is needed: the calls that would launch kernels are
replaced by plain formulas, or are refused before they touch the device."""

import ctypes

import pytest

import hessboost_b200 as H

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


P = 0x10000  # addresses that no call reads


@pytest.mark.parametrize("ins,outs,refused", [
    ([0, 0], [0, 0], "two outputs overlap"),                       # a tensor listed twice, in place
    ([0, 40], [0, 20], "two outputs overlap"),
    ([400, 800], [60, 56], "two outputs overlap"),
    ([0, 400], [4, 800], "not its own"),                           # an output one element off its input
    ([0, 400], [800, 20], "not its own"),                          # over another tensor's input
    ([400, 0], [20, 800], "not its own"),
    ([0, 40], [0, 40], None),                                      # in place, side by side
    ([40, 0], [40, 0], None),
    ([0, 0], [80, 40], None),                                      # one input twice, apart from the outputs
    ([0, 20], [120, 160], None),
    ([0, 80], [0, 40], None),                                      # one in place, one not
])
def test_clip_refuses_outputs_that_overlap(ins, outs, refused):
    # two tensors of 10 f32: the chunks of a call run in no order, so an element written twice would be scaled by chance
    L = H.lib()
    a, b = (ctypes.c_void_p * 2)(*[P + i for i in ins]), (ctypes.c_void_p * 2)(*[P + o for o in outs])
    sizes, types = (ctypes.c_uint64 * 2)(10, 10), (ctypes.c_int32 * 2)(0, 0)
    # a call that passes is refused for its workspace, the next thing looked at
    assert L.hb_clip_grad_norm(0, 2, a, b, sizes, types, 1.0, P, None, 0, None) == H.HB_INVALID_ARGUMENT
    assert (refused or "workspace") in L.hb_head_last_error().decode()


def test_clip_of_empty_tensors_overlaps_nothing():
    L = H.lib()
    a, types = (ctypes.c_void_p * 2)(P, P), (ctypes.c_int32 * 2)(0, 0)
    for sizes in ((10, 0), (0, 10), (0, 0)):
        assert L.hb_clip_grad_norm(0, 2, a, a, (ctypes.c_uint64 * 2)(*sizes), types, 1.0, P, None, 0, None) == H.HB_INVALID_ARGUMENT
        assert "workspace" in L.hb_head_last_error().decode()
