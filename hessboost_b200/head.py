"""Operators of an embedding head on the binned matrix's tokens, on torch tensors.

A row of the binned matrix is a list of tokens, its global bins: cell (row, f)
of a dense index is ``feature_offset[f] + bin`` (-1 where the value is
missing), and a CSR index (``row_ptr``, ``row_bins``) holds them as they are.
A head sums the tokens' embeddings, norms the sum and takes the softmax cross
entropy of a linear layer over the classes (any number of them, where
``multi:softmax`` grows a tree per class and stops at 64). These are its
operators, each a forward and a backward call, and the clipping of its
gradients; ``embed``, ``layer_norm`` and ``linear_xent`` are the same calls
under autograd, once: differentiating their gradients raises RuntimeError.

All tensors are on one CUDA device; the kernels run on torch's current stream
of it, nothing synchronises, and outputs are new contiguous tensors. A wrong
argument raises ValueError before anything runs, a call that the library
refuses raises HbError. Results do not change from run to run.
"""

import array
import ctypes
import operator

import torch
from torch.autograd.function import once_differentiable

from . import HB_OK, HbError, lib

__all__ = [
    "bin_tokens",
    "embed_forward",
    "embed_backward",
    "layer_norm_forward",
    "layer_norm_backward",
    "linear_xent_forward",
    "linear_xent_backward",
    "grad_norm",
    "clip_grad_norm",
    "embed",
    "layer_norm",
    "linear_xent",
]

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_INTS = {torch.int32: 0, torch.int64: 1}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(index):
    return _raw_stream(index) if _raw_stream else torch.cuda.current_stream(index).cuda_stream


def _check(status, where):
    if status != HB_OK:
        raise HbError(status, where, (lib().hb_head_last_error() or b"").decode())


def _need(ok, what):
    if not ok:
        raise ValueError(what)


def _device(t, *others):
    """The CUDA device index all the tensors share."""
    _need(t.is_cuda, "tensors must be on a CUDA device")
    d = t.device
    for o in others:
        _need(o is None or o.device == d, "tensors must be on one device")
    return d.index


def _type(t, name):
    v = _TYPES.get(t.dtype)
    _need(v is not None, f"{name} must be float32, float16 or bfloat16")
    return v


def _int(t, name):
    v = _INTS.get(t.dtype)
    _need(v is not None, f"{name} must be int32 or int64")
    return v


def _rows(t):
    """`t` as 2-D rows of consecutive elements; a copy where its strides do not allow a view of that form."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    n, d = t.shape
    if (d > 1 and t.stride(1) != 1) or (n > 1 and t.stride(0) < d):
        t = t.contiguous()
    return t


def _workspace(fn, device, *sizes):
    b = ctypes.c_uint64()
    _check(fn(*sizes, b), fn.__name__)
    return torch.empty(b.value, dtype=torch.uint8, device=device), b.value


# ---------------------------------------------------------------- tokens
def bin_tokens(matrix, device="cuda"):
    """(tokens, row_ptr) of a ``BinnedMatrix`` on `device`: [rows, features] int32 global bins with -1 where a value
    is missing and row_ptr None (dense index), or the CSR index's cells and their int64 row offsets."""
    if matrix.columns is None:
        cells = torch.from_numpy(matrix.row_bins.astype("int32"))
        return cells.to(device), torch.from_numpy(matrix.row_ptr.astype("int64")).to(device)
    cols = torch.from_numpy(matrix.columns).to(device)
    tok = cols.to(torch.int32) + torch.from_numpy(matrix.feature_offset[:-1].astype("int32")).to(device)[:, None]
    if matrix.missing is not None and not matrix.dense:
        words = torch.from_numpy(matrix.missing.view("uint8").reshape(matrix.n_cols, -1).copy()).to(device)
        bits = (words[:, :, None] >> torch.arange(8, device=device, dtype=torch.uint8)) & 1
        tok = torch.where(bits.reshape(matrix.n_cols, -1)[:, : matrix.n_rows].bool(), -1, tok)
    return tok.T.contiguous(), None


# ------------------------------------------------------------- embedding
def _cells(tokens, row_ptr):
    """(tokens, rows, row_ptr) checked: rows from row_ptr, else from tokens' first axis."""
    _int(tokens, "tokens")
    if row_ptr is None:
        _need(tokens.dim() in (1, 2), "tokens must be [rows] or [rows, cells], or 1-D with row_ptr")
        return tokens.contiguous(), tokens.shape[0], None
    _need(tokens.dim() == 1, "tokens must be 1-D with row_ptr")
    _need(row_ptr.dim() == 1 and row_ptr.dtype == torch.int64 and row_ptr.numel() >= 1,
          "row_ptr must be a 1-D int64 tensor of rows + 1 offsets")
    return tokens.contiguous(), row_ptr.numel() - 1, row_ptr.contiguous()


def embed_forward(tokens, table, *, row_ptr=None, scale=1.0):
    """out[n] = scale * the sum of table[t] over row n's tokens t, [rows, width] of table's type.

    tokens: int32 or int64, [rows, cells] or [rows] (one token a row), or 1-D with `row_ptr` (rows + 1 ascending int64
    offsets into it). A token outside [0, len(table)) is a missing cell and contributes nothing."""
    dt = _type(table, "table")
    _need(table.dim() == 2 and table.shape[0] > 0 and table.shape[1] > 0, "table must be 2-D and not empty")
    tokens, rows, ptr = _cells(tokens, row_ptr)
    table = _rows(table)
    dev = _device(table, tokens, ptr)
    n_tokens, width = table.shape
    out = table.new_empty((rows, width))
    _check(lib().hb_embed_forward(dev, tokens.data_ptr(), _INTS[tokens.dtype], None if ptr is None else ptr.data_ptr(),
                                  rows, tokens.numel(), table.data_ptr(), dt, n_tokens, width,
                                  max(table.stride(0), width), scale, out.data_ptr(), _stream(dev)), "hb_embed_forward")
    return out


def embed_backward(grad, tokens, n_tokens, *, row_ptr=None, scale=1.0):
    """The table's gradient, [n_tokens, width] of grad's type: scale * the sum of grad's rows over each token's cells,
    in cell order; 0 for tokens that do not occur."""
    dt = _type(grad, "grad")
    _need(grad.dim() == 2 and grad.shape[1] > 0, "grad must be [rows, width]")
    _need(n_tokens >= 1, "n_tokens must be at least 1")
    tokens, rows, ptr = _cells(tokens, row_ptr)
    _need(grad.shape[0] == rows, "grad must have a row for each row of tokens")
    width = grad.shape[1]
    if width > 1 and grad.stride(1) != 1 or rows > 1 and grad.stride(0) < width and grad.stride(0) != 0:
        grad = grad.contiguous()
    dev = _device(grad, tokens, ptr)
    L = lib()
    dtable = grad.new_empty((n_tokens, width))
    ws, size = _workspace(L.hb_embed_backward_workspace, grad.device, rows, tokens.numel(), n_tokens, width)
    _check(L.hb_embed_backward(dev, tokens.data_ptr(), _INTS[tokens.dtype], None if ptr is None else ptr.data_ptr(),
                               rows, tokens.numel(), grad.data_ptr(), dt, grad.stride(0), n_tokens, width, scale,
                               dtable.data_ptr(), ws.data_ptr(), size, _stream(dev)), "hb_embed_backward")
    return dtable


# ------------------------------------------------------------ layer norm
def _params(x, weight, bias):
    """The type code of weight and bias, which is x's or float32."""
    width = x.shape[-1]
    kind = None
    for p in (weight, bias):
        if p is None:
            continue
        _need(p.dim() == 1 and p.shape[0] == width, "weight and bias must be [width]")
        _need(p.dtype == x.dtype or p.dtype == torch.float32, "weight and bias must be of x's type or float32")
        _need(kind is None or kind == p.dtype, "weight and bias must be of one type")
        kind = p.dtype
    return _TYPES[x.dtype if kind is None else kind]


def layer_norm_forward(x, weight=None, bias=None, *, eps=1e-5):
    """(y, mean, rstd): y = (x - mean) * rstd * weight + bias over x's last axis, y of x's shape and type; mean and
    rstd = 1 / sqrt(variance + eps) are float32, one of each a row, for the backward call."""
    dt = _type(x, "x")
    _need(x.dim() >= 1 and x.shape[-1] > 0, "x must have a last axis that is not empty")
    _need(eps >= 0, "eps must be >= 0")
    pt = _params(x, weight, bias)
    rows = _rows(x)
    dev = _device(rows, weight, bias)
    n, width = rows.shape
    w = None if weight is None else weight.contiguous()
    b = None if bias is None else bias.contiguous()
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = torch.empty(n, dtype=torch.float32, device=x.device)
    rstd = torch.empty_like(mean)
    _check(lib().hb_layer_norm_forward(dev, rows.data_ptr(), dt, max(rows.stride(0), width), n, width,
                                       None if w is None else w.data_ptr(), None if b is None else b.data_ptr(), pt,
                                       eps, y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), _stream(dev)),
           "hb_layer_norm_forward")
    return y, mean, rstd


def layer_norm_backward(dy, x, weight, mean, rstd, *, params=True):
    """(dx, dweight, dbias) from the forward call's mean and rstd; dx of x's type, dweight and dbias of weight's type
    (x's where weight is None), both None with params=False."""
    dt = _type(x, "x")
    _need(dy.shape == x.shape and dy.dtype == x.dtype, "dy must have x's shape and type")
    _need(x.dim() >= 1 and x.shape[-1] > 0, "x must have a last axis that is not empty")
    pt = _params(x, weight, None)
    width = x.shape[-1]
    xr, gr = _rows(x), _rows(dy)
    n = xr.shape[0]
    _need(mean.dtype == rstd.dtype == torch.float32 and mean.numel() == rstd.numel() == n
          and mean.is_contiguous() and rstd.is_contiguous(), "mean and rstd must be the forward call's")
    dev = _device(xr, gr, weight, mean, rstd)
    w = None if weight is None else weight.contiguous()
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dw = db = ws = None
    size = 0
    L = lib()
    if params:
        dw, db = torch.empty((2, width), dtype=x.dtype if weight is None else weight.dtype, device=x.device).unbind(0)
        ws, size = _workspace(L.hb_layer_norm_backward_workspace, x.device, n, width)
    _check(L.hb_layer_norm_backward(dev, gr.data_ptr(), max(gr.stride(0), width), xr.data_ptr(),
                                    max(xr.stride(0), width), dt, n, width, None if w is None else w.data_ptr(), pt,
                                    mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(),
                                    None if dw is None else dw.data_ptr(), None if db is None else db.data_ptr(),
                                    None if ws is None else ws.data_ptr(), size, _stream(dev)),
           "hb_layer_norm_backward")
    return dx, dw, db


# --------------------------------------- softmax cross entropy of a layer
def _xent(x, weight, labels):
    dt = _type(x, "x")
    _need(x.dtype != torch.float16, "x and weight must be float32 or bfloat16")
    _need(x.dim() == 2 and weight.dim() == 2 and x.shape[1] == weight.shape[1] and x.shape[1] > 0
          and weight.shape[0] > 0, "x must be [rows, width] and weight [classes, width]")
    _need(weight.dtype == x.dtype, "x and weight must be of one type")
    _int(labels, "labels")
    _need(labels.dim() == 1 and labels.shape[0] == x.shape[0], "labels must be [rows]")
    x, weight, labels = _rows(x), _rows(weight), labels.contiguous()
    return dt, x, weight, labels, _device(x, weight, labels)


def linear_xent_forward(x, weight, labels):
    """(loss, lse), float32 [rows]: lse = log sum exp of a row's logits x @ weight.T, loss = lse - the label's logit.
    The logits are not kept. labels: int32 or int64; one outside [0, classes) is a row without a label: its loss is 0."""
    dt, x, weight, labels, dev = _xent(x, weight, labels)
    (n, width), v = x.shape, weight.shape[0]
    L = lib()
    loss = torch.empty(n, dtype=torch.float32, device=x.device)
    lse = torch.empty_like(loss)
    xs, wst = max(x.stride(0), width), max(weight.stride(0), width)
    ws, size = _workspace(L.hb_linear_xent_forward_workspace, x.device, dev, x.data_ptr(), xs, weight.data_ptr(), wst, dt,
                          n, width, v)
    _check(L.hb_linear_xent_forward(dev, x.data_ptr(), xs, weight.data_ptr(), wst, dt, labels.data_ptr(), _INTS[labels.dtype], n, width,
                                    v, loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), size, _stream(dev)),
           "hb_linear_xent_forward")
    return loss, lse


def linear_xent_backward(dloss, x, weight, labels, lse):
    """(dx, dweight), of x's type, of the sum over the rows of dloss * loss; dloss float32 [rows] (an expanded scalar
    will do), lse the forward call's. Rows without a label get 0 and add nothing."""
    dt, x, weight, labels, dev = _xent(x, weight, labels)
    (n, width), v = x.shape, weight.shape[0]
    _need(dloss.dtype == torch.float32 and dloss.dim() == 1 and dloss.shape[0] == n, "dloss must be float32 [rows]")
    _need(lse.dtype == torch.float32 and lse.dim() == 1 and lse.shape[0] == n and lse.is_contiguous(),
          "lse must be the forward call's")
    _device(x, dloss, lse)
    L = lib()
    dx, dw = x.new_empty((n, width)), x.new_empty((v, width))
    xs, wst = max(x.stride(0), width), max(weight.stride(0), width)
    ws, size = _workspace(L.hb_linear_xent_backward_workspace, x.device, dev, x.data_ptr(), xs, weight.data_ptr(), wst, dt,
                          n, width, v)
    _check(L.hb_linear_xent_backward(dev, dloss.data_ptr(), dloss.stride(0), x.data_ptr(), xs,
                                     weight.data_ptr(), wst, dt, labels.data_ptr(),
                                     _INTS[labels.dtype], lse.data_ptr(), n, width, v, dx.data_ptr(), dw.data_ptr(),
                                     ws.data_ptr(), size, _stream(dev)), "hb_linear_xent_backward")
    return dx, dw


# -------------------------------------------------------------- clipping
_dtype = operator.attrgetter("dtype")
_Tensor = torch.Tensor


def _tensor_list(tensors):
    """(n, addresses, elements, type codes, device) of a list of contiguous tensors on one device, the middle three as
    host arrays. (Hundreds of tensors: each question is asked of all of them in one call.)"""
    _need(len(tensors) > 0, "tensors is empty")
    devices = set(map(_Tensor.get_device, tensors))
    _need(devices != {-1}, "tensors must be on a CUDA device")
    _need(len(devices) == 1, "tensors must be on one device")
    _need(all(map(_Tensor.is_contiguous, tensors)), "tensors must be contiguous")
    dtypes = list(map(_dtype, tensors))
    _need(_TYPES.keys() >= set(dtypes), "tensors must be float32, float16 or bfloat16")
    return (len(tensors), array.array("Q", map(_Tensor.data_ptr, tensors)), array.array("Q", map(_Tensor.numel, tensors)),
            array.array("i", map(_TYPES.__getitem__, dtypes)), devices.pop())


def _address(a):
    return a.buffer_info()[0]


def grad_norm(tensors):
    """The 2-norm of all the tensors' elements together, a float32 scalar tensor on their device."""
    tensors = list(tensors)
    n, ptrs, sizes, types, dev = _tensor_list(tensors)
    L = lib()
    norm = torch.empty((), dtype=torch.float32, device=tensors[0].device)
    ws, size = _workspace(L.hb_grad_norm_workspace, norm.device, dev, n)
    _check(L.hb_grad_norm(dev, n, _address(ptrs), _address(sizes), _address(types), norm.data_ptr(), ws.data_ptr(),
                          size, _stream(dev)), "hb_grad_norm")
    return norm


def clip_grad_norm(tensors, max_norm, *, out=None):
    """The tensors' norm (as grad_norm), after scaling each tensor by min(1, max_norm / (norm + 1e-6)): in place, or
    into `out`, a list of as many contiguous tensors of the same sizes and types. Outputs that overlap (a tensor listed
    twice, in place) are refused. A norm that is not finite passes into the results through that factor."""
    tensors = list(tensors)
    _need(max_norm >= 0, "max_norm must be >= 0")
    n, ptrs, sizes, types, dev = _tensor_list(tensors)
    outs = ptrs
    if out is not None:
        out = list(out)
        _need(len(out) == n, "out must have a tensor for each of tensors")
        _, outs, out_sizes, out_types, out_dev = _tensor_list(out)
        _need(out_dev == dev and out_sizes == sizes and out_types == types,
              "out must be tensors of the same sizes and types on the same device")
    L = lib()
    norm = torch.empty((), dtype=torch.float32, device=tensors[0].device)
    ws, size = _workspace(L.hb_grad_norm_workspace, norm.device, dev, n)
    _check(L.hb_clip_grad_norm(dev, n, _address(ptrs), _address(outs), _address(sizes), _address(types), max_norm,
                               norm.data_ptr(), ws.data_ptr(), size, _stream(dev)), "hb_clip_grad_norm")
    # written through addresses: a graph that has saved one of them is to notice
    torch.autograd.graph.increment_version(tensors if out is None else out)
    return norm


# --------------------------------------------------------------- autograd
# The backward calls are kernels without a graph of their own: a gradient that
# is differentiated again (create_graph) raises.
class _Embed(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, table, row_ptr, scale):
        ctx.save_for_backward(tokens, row_ptr)
        ctx.n_tokens, ctx.scale = table.shape[0], scale
        return embed_forward(tokens, table, row_ptr=row_ptr, scale=scale)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        tokens, row_ptr = ctx.saved_tensors
        return None, embed_backward(grad, tokens, ctx.n_tokens, row_ptr=row_ptr, scale=ctx.scale), None, None


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm_forward(x, weight, bias, eps=eps)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.has_bias = bias is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = layer_norm_backward(dy, x, weight, mean, rstd, params=weight is not None or ctx.has_bias)
        return dx, None if weight is None else dw, db if ctx.has_bias else None, None


class _LinearXent(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, labels):
        loss, lse = linear_xent_forward(x, weight, labels)
        ctx.save_for_backward(x, weight, labels, lse)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss):
        dx, dw = linear_xent_backward(dloss, *ctx.saved_tensors)
        return dx, dw, None


def embed(tokens, table, *, row_ptr=None, scale=1.0):
    """embed_forward under autograd: the gradient of `table` is embed_backward's."""
    return _Embed.apply(tokens, table, row_ptr, scale)


def layer_norm(x, weight=None, bias=None, *, eps=1e-5):
    """layer_norm_forward's y under autograd (where `bias` is given without `weight`, it must be of x's type)."""
    return _LayerNorm.apply(x, weight, bias, eps)


def linear_xent(x, weight, labels):
    """linear_xent_forward's loss (one a row) under autograd."""
    return _LinearXent.apply(x, weight, labels)
