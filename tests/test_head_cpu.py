"""Refusals of the embedding-head operators that need no GPU: every entry point checks its arguments before it touches
the device, and says which one is wrong."""

import ctypes

import pytest

import hessboost_b200 as H

torch = pytest.importorskip("torch")

from hessboost_b200 import head  # noqa: E402

P, Q = 0x1000, 0x2000  # aligned addresses that no refused call reads


def refused(name, args, what):
    L = H.lib()
    assert getattr(L, name)(*args) == H.HB_INVALID_ARGUMENT
    assert what in L.hb_head_last_error().decode()


def put(args, at, v):
    args = list(args)
    args[at] = v
    return args


def test_embed_refusals():
    ok = [0, P, 0, None, 4, 12, P, 0, 10, 8, 8, 1.0, Q, None]
    for at, v, what in ((7, 3, "element type"), (2, 2, "token type"), (9, 0, "width"), (8, 0, "n_tokens"),
                        (8, 2**32, "n_tokens"), (4, 2**32, "rows"), (5, 13, "row_ptr"), (1, None, "tokens is NULL"),
                        (1, P + 2, "aligned"), (3, P + 4, "row_ptr"), (6, None, "NULL"), (12, None, "NULL"),
                        (10, 7, "table_stride"), (6, P + 2, "aligned"), (12, Q + 1, "aligned")):
        refused("hb_embed_forward", put(ok, at, v), what)
    ok = [0, P, 0, None, 4, 12, P, 0, 8, 10, 8, 1.0, Q, P, 1 << 30, None]
    for at, v, what in ((7, -1, "element type"), (6, None, "NULL"), (12, None, "NULL"), (8, 7, "grad_stride"),
                        (13, None, "workspace"), (14, 0, "workspace"), (13, P + 8, "workspace"), (6, P + 1, "aligned")):
        refused("hb_embed_backward", put(ok, at, v), what)
    refused("hb_embed_backward_workspace", [1, 1, 1, 1, None], "bytes")
    refused("hb_embed_backward_workspace", [1, 2**32, 1, 1, ctypes.c_uint64()], "out of range")


def test_norm_refusals():
    ok = [0, P, 0, 8, 4, 8, None, None, 0, 1e-5, Q, P, P, None]
    for at, v, what in ((2, 5, "element type"), (8, 1, "type"), (5, 0, "width"), (1, None, "NULL"), (10, None, "NULL"),
                        (11, None, "NULL"), (12, None, "NULL"), (3, 7, "x_stride"), (9, -1.0, "eps"), (9, float("nan"), "eps"),
                        (6, P + 2, "aligned"), (1, P + 2, "aligned")):
        refused("hb_layer_norm_forward", put(ok, at, v), what)
    ok = [0, P, 8, P, 8, 0, 4, 8, None, 0, P, P, Q, Q, Q, P, 1 << 30, None]
    for at, v, what in ((5, 5, "element type"), (7, 0, "width"), (0 + 1, None, "NULL"), (12, None, "NULL"), (2, 7, "stride"),
                        (4, 7, "stride"), (15, None, "workspace"), (16, 8, "workspace"), (13, Q + 1, "aligned")):
        refused("hb_layer_norm_backward", put(ok, at, v), what)
    refused("hb_layer_norm_backward_workspace", [1, 0, ctypes.c_uint64()], "width")


def test_xent_refusals():
    ok = [0, P, 8, P, 8, 0, P, 0, 4, 8, 100, Q, Q, P, 1 << 30, None]
    for at, v, what in ((5, 1, "f32 or bf16"), (7, 2, "label type"), (9, 0, "width"), (9, 2**21, "width"), (10, 0, "n_classes"),
                        (10, 2**31, "n_classes"), (8, 2**31, "rows"), (1, None, "NULL"), (3, None, "NULL"), (6, None, "NULL"),
                        (2, 7, "x_stride"), (4, 7, "w_stride"), (1, P + 2, "aligned"), (11, None, "NULL"), (12, Q + 2, "aligned"),
                        (13, None, "workspace"), (14, 1, "workspace")):
        refused("hb_linear_xent_forward", put(ok, at, v), what)
    ok = [0, P, 1, P, 8, P, 8, 0, P, 0, P, 4, 8, 100, Q, Q, P, 1 << 30, None]
    for at, v, what in ((7, 1, "f32 or bf16"), (1, None, "NULL"), (10, None, "NULL"), (14, None, "NULL"), (15, None, "NULL"),
                        (1, P + 2, "aligned"), (16, None, "workspace"), (17, 1, "workspace")):
        refused("hb_linear_xent_backward", put(ok, at, v), what)
    refused("hb_linear_xent_forward_workspace", [0, P, 8, P, 8, 0, 1, 8, 1, None], "bytes")
    refused("hb_linear_xent_backward_workspace", [0, P, 8, P, 8, 0, 2**31, 8, 1, ctypes.c_uint64()], "rows")


def test_clip_refusals():
    one, types = (ctypes.c_void_p * 1)(P), (ctypes.c_int32 * 1)(0)
    size = (ctypes.c_uint64 * 1)(4)
    ok = [0, 1, one, one, size, types, 1.0, Q, P, 1 << 20, None]
    for at, v, what in ((1, -1, "negative"), (2, None, "NULL"), (3, None, "NULL"), (6, -1.0, "max_norm"),
                        (6, float("nan"), "max_norm"), (7, None, "norm"), (8, None, "workspace"), (9, 0, "workspace"),
                        (2, (ctypes.c_void_p * 1)(None), "NULL"), (2, (ctypes.c_void_p * 1)(P + 2), "aligned"),
                        (3, (ctypes.c_void_p * 1)(P + 2), "aligned"), (5, (ctypes.c_int32 * 1)(7), "type"),
                        (4, (ctypes.c_uint64 * 1)(2**50), "large")):
        refused("hb_clip_grad_norm", put(ok, at, v), what)
    refused("hb_grad_norm_workspace", [0, 1, None], "NULL")
    refused("hb_grad_norm", [0, 1, one, size, types, Q + 1, P, 1 << 20, None], "norm")


def test_last_error_is_cleared_by_a_success():
    L = H.lib()
    refused("hb_layer_norm_backward_workspace", [1, 0, ctypes.c_uint64()], "width")
    b = ctypes.c_uint64()
    assert L.hb_layer_norm_backward_workspace(1, 8, b) == H.HB_OK and b.value > 0
    assert L.hb_head_last_error() == b""


def test_python_refusals():
    t, f = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(4, 8)
    for call in (lambda: head.embed_forward(t, f), lambda: head.embed_forward(t.float(), f),
                 lambda: head.embed_forward(t, f.double()), lambda: head.embed_forward(t, f[0]),
                 lambda: head.embed_forward(t, f, row_ptr=t[0]), lambda: head.embed_forward(t[0], f, row_ptr=t[0]),
                 lambda: head.embed_backward(f, t, 4), lambda: head.embed_backward(f[:2], t, 0),
                 lambda: head.layer_norm_forward(f), lambda: head.layer_norm_forward(f.int()),
                 lambda: head.layer_norm_forward(f, f[0, :3]), lambda: head.layer_norm_forward(f, f[0].half()),
                 lambda: head.layer_norm_forward(f, eps=-1.0), lambda: head.layer_norm_forward(f, f[0], f[0].double()),
                 lambda: head.layer_norm_backward(f[:2], f, None, f[0], f[0]),
                 lambda: head.linear_xent_forward(f, f, t[0]), lambda: head.linear_xent_forward(f, f[:, :3], t[0]),
                 lambda: head.linear_xent_forward(f, f.bfloat16(), t[0]), lambda: head.linear_xent_forward(f.half(), f.half(), t[0]),
                 lambda: head.linear_xent_forward(f[:3], f, t[0].float()),
                 lambda: head.grad_norm([]), lambda: head.grad_norm([f]), lambda: head.grad_norm([t]),
                 lambda: head.clip_grad_norm([f], -1.0)):
        with pytest.raises(ValueError):
            call()
