"""The embedding head's example step (examples/bin_head.py) on the framework's binned matrices, against the same step in
64 bits."""

import importlib.util
import os

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import hessboost_b200 as H  # noqa: E402
from hessboost_b200 import head  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("bin_head", os.path.join(ROOT, "examples", "bin_head.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _tokens64(x, off, cuts):
    """Global bins by their definition: the number of the feature's cuts not above the value (the last bin at most)."""
    out = np.full(x.shape, -1, np.int64)
    for f in range(x.shape[1]):
        c = cuts[off[f]:off[f + 1]]
        there = ~np.isnan(x[:, f])
        out[there, f] = off[f] + np.minimum(np.searchsorted(c, x[there, f], side="right"), len(c) - 1)
    return out


def test_bin_tokens_of_dense_and_sparse_matrices():
    rng = np.random.default_rng(3)
    x = rng.standard_normal((300, 7)).astype(np.float32)
    full = H.BinnedMatrix.from_dense(x, max_bin=16)
    tok, ptr = head.bin_tokens(full, device="cpu")
    assert ptr is None and tok.dtype == torch.int32
    np.testing.assert_array_equal(tok.numpy(), _tokens64(x, full.feature_offset.astype(int), full.cut_values))
    x[rng.random(x.shape) < 0.2] = np.nan
    m = H.BinnedMatrix.from_dense(x, max_bin=16)
    tok, ptr = head.bin_tokens(m, device="cpu")
    want = _tokens64(x, m.feature_offset.astype(int), m.cut_values)
    np.testing.assert_array_equal(tok.numpy(), want)
    # the same cells as CSR
    there = ~np.isnan(x)
    indptr = np.concatenate([[0], np.cumsum(there.sum(1))])
    s = H.BinnedMatrix.from_csr(indptr.astype(np.uint64), np.nonzero(there)[1].astype(np.uint32), x[there], 7, 16)
    tok, ptr = head.bin_tokens(s, device="cpu")
    np.testing.assert_array_equal(ptr.numpy(), indptr)
    np.testing.assert_array_equal(tok.numpy(), want[there])


@pytest.mark.gpu
@pytest.mark.parametrize("sparse", [False, True])
@pytest.mark.parametrize("classes", [7, 300])
def test_step_against_64_bits(example, sparse, classes):
    x, y = example.make_rows(700, 9, classes, seed=classes)
    m = H.BinnedMatrix.from_dense(x, max_bin=16)
    if sparse:
        there = ~np.isnan(x)
        indptr = np.concatenate([[0], np.cumsum(there.sum(1))]).astype(np.uint64)
        m = H.BinnedMatrix.from_csr(indptr, np.nonzero(there)[1].astype(np.uint32), x[there], x.shape[1], 16)
    tokens, ptr = head.bin_tokens(m)
    labels = torch.from_numpy(y).cuda()
    labels[::11] = -1
    model = example.BinHead(int(m.feature_offset[-1]), classes, width=24)
    p = [t.double().requires_grad_() for t in model.parameters()]
    fn = torch.nn.functional
    tok = torch.from_numpy(_tokens64(x, m.feature_offset.astype(int), m.cut_values)).cuda()
    e = (p[0][tok.clamp(0)] * (tok >= 0)[..., None]).sum(1) * 0.2
    logits = fn.layer_norm(e, (24,), p[1], p[2]) @ p[3].T
    loss = fn.cross_entropy(logits, labels, ignore_index=-1, reduction="none")
    want = torch.autograd.grad(loss.sum() / (labels >= 0).sum(), p)
    got_loss = model.loss(tokens, labels, ptr)
    got = model.gradients()
    # f32 sums of a few hundred terms, each off by U of its magnitude, through three layers
    tol = 256 * 2.0**-24
    loss = loss.detach()
    assert float((got_loss.double() - loss).norm() / loss.norm()) <= tol
    for a, b in zip(got, want):
        assert float((a.double() - b).norm() / b.norm()) <= tol
    norm = head.clip_grad_norm(got, 0.01)
    full = torch.sqrt(sum(b.square().sum() for b in want))
    assert abs(float(norm) - float(full)) <= tol * float(full)
    for a, b in zip(got, want):
        assert float((a.double() - b * (0.01 / full)).norm()) <= 2 * tol * float((b * (0.01 / full)).norm()) + 1e-9


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_example_learns(example, dtype):
    losses = example.main(["--rows", "4000", "--classes", "100", "--steps", "40", "--dtype", dtype])
    assert losses[0] > 3.0 and losses[-1] < 0.5 * losses[0]
