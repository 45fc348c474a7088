"""The token operators' C entry points refuse bad arguments before any device call, and the
scratch they ask for; ops.py refuses tensors that are not on a GPU.  No kernel runs."""
import ctypes as C

import pytest
import torch

from conftest import pkg

L = pkg()._lib
CTX = C.create_string_buffer(64)  # never read: every call here is refused or has nothing to do


def call(fn, **kw):
    a = L.TOKEN_ARGS[fn](**kw)
    return getattr(L.lib(), fn)(C.addressof(CTX), C.byref(a), None)


def need(fn, **kw):
    a, n = L.TOKEN_ARGS[fn](**kw), C.c_int64(-1)
    return getattr(L.lib(), fn + "_workspace")(C.byref(a), C.byref(n)), n.value


def s3(*v):
    return (C.c_int64 * 3)(*v)


LIN = dict(dtype=1, m=100, n=40, k=30, x=64, w=64, y=64, x_stride=30, w_stride=30, y_stride=40)
GRAD = dict(dtype=1, m=100, n=40, k=30, dy=64, x=64, w=64, dx=64, dy_stride=40, x_stride=30, w_stride=30, dx_stride=30)
NORM = dict(dtype=0, m=10, c=64, eps=1e-5, x=64, y=64, x_stride=64, y_stride=64)
NGRAD = dict(dtype=0, m=10, c=64, dy=64, x=64, mean=64, rstd=64, dx=64, dw=64, dy_stride=64, x_stride=64, dx_stride=64)
ATT = dict(dtype=0, b=2, h_q=4, h_kv=2, d=64, nq=9, nk=9, scale=0.1, q=64, k=64, v=64, o=64)
AGRAD = dict(ATT, go=64, lse=64, dq=64, dk=64, dv=64)


@pytest.mark.parametrize("fn,base,bad", [
    ("yk_linear", LIN, dict(dtype=2)), ("yk_linear", LIN, dict(dtype=9)), ("yk_linear", LIN, dict(act=4)),
    ("yk_linear", LIN, dict(act=-1)), ("yk_linear", LIN, dict(k=0)), ("yk_linear", LIN, dict(n=0)),
    ("yk_linear", LIN, dict(m=-1)), ("yk_linear", LIN, dict(m=1 << 30)), ("yk_linear", LIN, dict(x=None)),
    ("yk_linear", LIN, dict(y=None)), ("yk_linear", LIN, dict(y_stride=39)), ("yk_linear", LIN, dict(x_stride=-30)),
    ("yk_linear", LIN, dict(res=64, res_rows=0, res_stride=40)), ("yk_linear", LIN, dict(res=64, res_rows=101, res_stride=40)),
    ("yk_linear", LIN, dict(m=1 << 29, n=1 << 29, y_stride=1 << 29)),
    ("yk_linear", dict(LIN, k=4096, x_stride=4096, w_stride=4096), dict(ws=68, ws_bytes=16)),
    ("yk_linear_backward", GRAD, dict(dtype=2)), ("yk_linear_backward", GRAD, dict(m=0)),
    ("yk_linear_backward", GRAD, dict(act=2)), ("yk_linear_backward", GRAD, dict(w=None)),
    ("yk_linear_backward", GRAD, dict(dx_stride=29)), ("yk_linear_backward", GRAD, dict(dres=64, res_rows=101)),
    ("yk_linear_backward", GRAD, dict(act=2, z=64, z_stride=40)),  # dz needs scratch
    ("yk_layer_norm", NORM, dict(dtype=2)), ("yk_layer_norm", NORM, dict(c=0)), ("yk_layer_norm", NORM, dict(eps=-1.0)),
    ("yk_layer_norm", NORM, dict(eps=float("nan"))), ("yk_layer_norm", NORM, dict(x=None)),
    ("yk_layer_norm", NORM, dict(y_stride=63)), ("yk_layer_norm_backward", NGRAD, {}),  # dw needs scratch
    ("yk_layer_norm_backward", NGRAD, dict(mean=None, dw=None)), ("yk_layer_norm_backward", NGRAD, dict(dx_stride=3, dw=None)),
    ("yk_attention", ATT, dict(dtype=2)), ("yk_attention", ATT, dict(h_q=3)), ("yk_attention", ATT, dict(h_kv=0)),
    ("yk_attention", ATT, dict(d=0)), ("yk_attention", ATT, dict(d=129)), ("yk_attention", ATT, dict(scale=0.0)),
    ("yk_attention", ATT, dict(scale=float("inf"))), ("yk_attention", ATT, dict(scale=float("nan"))),
    ("yk_attention", ATT, dict(nk=1 << 30)), ("yk_attention", ATT, dict(nq=1 << 29)), ("yk_attention", ATT, dict(v=None)),
    ("yk_attention", ATT, dict(b=1 << 30)), ("yk_attention", dict(ATT, nq=1, nk=9000), dict(ws=64, ws_bytes=8)),
    ("yk_attention_backward", AGRAD, {}), ("yk_attention_backward", AGRAD, dict(nk=0)),
    ("yk_attention_backward", AGRAD, dict(lse=None)), ("yk_attention_backward", AGRAD, dict(ws=68, ws_bytes=1 << 20)),
])
def test_refused_before_any_device_call(fn, base, bad):
    assert call(fn, **{**base, **bad}) == L.YK_ERR_ARG, (fn, bad)
    assert fn.encode() in L.lib().yk_last_error()


def test_nothing_to_do():
    assert call("yk_linear", **{**LIN, "m": 0, "x": None}) == L.YK_OK
    assert call("yk_layer_norm", **{**NORM, "m": 0, "x": None}) == L.YK_OK
    assert call("yk_attention", **{**ATT, "nq": 0}) == L.YK_OK
    assert call("yk_attention", **{**ATT, "b": 0}) == L.YK_OK
    assert call("yk_linear_backward", dtype=1, m=3, n=4, k=5) == L.YK_OK
    assert call("yk_layer_norm_backward", dtype=1, m=3, c=4) == L.YK_OK


def test_null_arguments():
    for fn in L.TOKEN_ARGS:
        assert getattr(L.lib(), fn)(None, None, None) == L.YK_ERR_ARG
        if fn != "yk_layer_norm":
            assert getattr(L.lib(), fn + "_workspace")(None, None) == L.YK_ERR_ARG


def test_workspace_sizes():
    """Scratch: none for products with enough tiles, float32 sums where K or the keys are split."""
    assert need("yk_linear", **LIN)[0] == 0
    assert need("yk_linear", dtype=0, m=8, n=2048, k=512) == (0, 0)
    assert need("yk_linear", dtype=0, m=40960, n=4096, k=1024) == (0, 0)
    rc, n = need("yk_linear", dtype=0, m=100, n=40, k=4096)
    assert rc == 0 and n > 0 and n % (100 * 40 * 4) == 0
    rc, n = need("yk_linear_backward", dtype=0, act=2, m=100, n=40, k=30, dx=64, dw=64)
    assert rc == 0 and n >= 100 * 40 * 2
    assert need("yk_attention", **{**ATT, "nq": 1280, "nk": 1280, "b": 8, "h_q": 8, "h_kv": 8}) == (0, 0)
    rc, n = need("yk_attention", **{**ATT, "nq": 1, "nk": 20480})
    assert rc == 0 and n > 0
    assert need("yk_attention_backward", **AGRAD) == (0, 2 * 2 * 4 * 9 * 4)


def test_packed_arguments_match_the_structs():
    """ops.py hands the argument structs over as packed bytes: same size, same place of the scratch."""
    ops = pkg().ops
    for fn, s in (("yk_linear", ops._LINEAR), ("yk_linear_backward", ops._LINEAR_GRAD), ("yk_layer_norm_backward", ops._NORM_GRAD),
                  ("yk_attention", ops._ATTENTION), ("yk_attention_backward", ops._ATTENTION_GRAD)):
        t = L.TOKEN_ARGS[fn]
        assert s.size == t.ws.offset and s.size + ops._WS.size == C.sizeof(t), fn
    assert ops._NORM.size == C.sizeof(L.LayerNormArgs)
    a = L.LinearArgs.from_buffer_copy(ops._LINEAR.pack(*range(1, 20)) + ops._WS.pack(20, 21))
    assert [getattr(a, n) for n, _ in a._fields_] == list(range(1, 22))


def test_no_gpu_tensors():
    ops = pkg().ops
    x = torch.zeros(4, 8)
    with pytest.raises(pkg().YKError, match="GPU"):
        ops.linear(x, x)
    with pytest.raises(pkg().YKError, match="GPU"):
        ops.layer_norm(x)
    with pytest.raises(pkg().YKError, match="GPU"):
        ops.attention(x.view(1, 4, 1, 8), x.view(1, 4, 1, 8), x.view(1, 4, 1, 8))
    with pytest.raises(ValueError):
        ops.linear([1.0], x)


def test_rows_of_a_tensor():
    rows = pkg().ops._rows
    t = torch.zeros(4, 5, 12)
    assert rows(t, "t") == (20, 12, 12)
    assert rows(t[..., 2:7], "t") == (20, 5, 12)
    assert rows(t[:, 0], "t") == (4, 12, 60)
    assert rows(t[0, 0], "t") == (1, 12, 12)
    assert rows(t[:1].expand(3, 5, 12)[:, :1], "t") == (3, 12, 0)
    assert rows(torch.zeros(0, 3), "t")[0] == 0
    for bad in (t.transpose(1, 2), t.transpose(0, 1), t[:, :4], torch.zeros(()), torch.zeros(3, 0)):
        with pytest.raises(ValueError):
            rows(bad, "t")
