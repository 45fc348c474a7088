"""Token operators on device tensors: the matrix product with its fused epilogue, layer norm and
attention of a transformer layer over the cells of a feature map, each with its gradients.

The kernels are those the detector program runs for an ``AIFI`` row of a model YAML (model.py);
here they take torch tensors (float32, bfloat16 or float16, on one GPU).  Calls are enqueued on
the tensors' device's current stream, allocate their outputs and scratch from torch and never
synchronise, so they can be captured into a graph.  No autograd graph is built: a call whose
inputs require gradients raises while gradients are enabled, and the ``*_backward`` functions return
the gradients.  Sums are float32 and outputs are rounded once; equal calls give equal bits.

A tensor's last dimension must be contiguous; what precedes it must step evenly from row to row
(any row stride, so a channel slice of a wider tensor is fine).  Anything else raises ValueError.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib as L

ACTS = {"none": 0, "silu": 1, "gelu": 2, "relu": 3}
_DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 3}  # yk_act_dtype


def _tensor(t, name, like=None, dtypes=None):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires grad: no autograd graph is built here (detach it, or torch.no_grad())")
    if like is None:
        if t.dtype not in _DTYPES:
            raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
        if t.device.type != "cuda":
            raise L.YKError(f"{name} is on {t.device}: the token operators run on an AMD GPU only (no CPU fallback)")
    else:
        if t.device != like.device:
            raise ValueError(f"{name} is on {t.device}, expected {like.device}")
        if t.dtype not in (dtypes or (like.dtype,)):
            raise ValueError(f"{name} has dtype {t.dtype}, expected {' or '.join(str(d) for d in dtypes or (like.dtype,))}")
    return t


def _rows(t, name, cols=None):
    """(rows, columns, row stride) of a tensor as a matrix of its last dimension."""
    if t.dim() < 1 or t.shape[-1] < 1:
        raise ValueError(f"{name} must have a last dimension of at least 1")
    c = t.shape[-1]
    if cols is not None and c != cols:
        raise ValueError(f"{name} has {c} columns, expected {cols}")
    if c > 1 and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    rows, stride = 1, c
    first = True
    for n, s in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if n == 1:
            continue
        if first:
            stride, first = s, False
        elif s != stride * rows:
            raise ValueError(f"{name}: rows must be evenly spaced (shape {tuple(t.shape)}, strides {t.stride()})")
        rows *= n
    return rows, c, stride


def _vector(t, name, n, like):
    """A parameter of n elements: the tensors' dtype or float32, contiguous."""
    _tensor(t, name, like, (like.dtype, torch.float32))
    if t.shape != (n,) or not (n == 1 or t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous vector of {n} elements, got {tuple(t.shape)}")
    return t


def _p(t):
    return None if t is None else t.data_ptr()


def _call(fn, args, like):
    dev = like.device.index
    lib = L.lib()
    ws = None
    if fn != "yk_layer_norm":
        need = C.c_int64()
        rc = getattr(lib, fn + "_workspace")(C.byref(args), C.byref(need))
        if rc:
            L.check(rc, fn)
        if need.value:
            ws = torch.empty(need.value, dtype=torch.uint8, device=like.device)
            args.ws, args.ws_bytes = ws.data_ptr(), need.value
    rc = getattr(lib, fn)(L.context(dev), C.byref(args), torch.cuda.current_stream(dev).cuda_stream)
    if rc:
        L.check(rc, fn)


def _act(name):
    if name not in ACTS:
        raise ValueError(f"act must be one of {sorted(ACTS)}, got {name!r}")
    return ACTS[name]


def linear(x, weight, bias=None, *, act="none", residual=None, return_preact=False):
    """act(x weight^T + bias) + residual, in one kernel (two where few tiles split a long K).

    x [..., K]; weight [N, K]; bias [N] in x's dtype or float32; act "none", "silu", "gelu" (exact)
    or "relu"; residual [..., N] with any R <= rows(x) rows, row m of the result taking row m % R (R
    tokens shared by the images of a batch).  Returns [..., N], with return_preact also act's
    argument, which linear_backward needs unless act is "none"."""
    _tensor(x, "x")
    m, k, xs = _rows(x, "x")
    _tensor(weight, "weight", x)
    if weight.dim() != 2:
        raise ValueError("weight must be [N, K]")
    n, _, ws = _rows(weight, "weight", k)
    if n < 1:
        raise ValueError("weight must have at least one row")
    a = L.LinearArgs(dtype=_DTYPES[x.dtype], act=_act(act), m=m, n=n, k=k, x=_p(x), w=_p(weight), x_stride=xs, w_stride=ws)
    if bias is not None:
        a.bias, a.bias_f32 = _p(_vector(bias, "bias", n, x)), bias.dtype == torch.float32
    if residual is not None and m:
        r, _, rs = _rows(_tensor(residual, "residual", x), "residual", n)
        if not 1 <= r <= m:
            raise ValueError(f"residual has {r} rows, x has {m}: expected 1 to that many")
        a.res, a.res_rows, a.res_stride = _p(residual), r, rs
    y = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=x.device)
    z = torch.empty_like(y) if return_preact else None
    a.y, a.y_stride, a.z, a.z_stride = _p(y), n, _p(z), n
    if m:
        _call("yk_linear", a, x)
    return (y, z) if return_preact else y


def linear_backward(dy, x, weight, bias=None, *, act="none", preact=None, residual=None):
    """Gradients of linear() from dy [..., N]: (dx, dweight, dbias, dresidual), the last two None
    without bias / residual.  preact is linear's second result (needed unless act is "none");
    residual's shape and dtype are what counts of it.  Where it has a row per row of x its gradient
    is dy itself."""
    _tensor(x, "x")
    m, k, xs = _rows(x, "x")
    n, _, ws = _rows(_tensor(weight, "weight", x), "weight", k)
    md, _, ds = _rows(_tensor(dy, "dy", x), "dy", n)
    if weight.dim() != 2 or md != m:
        raise ValueError("weight must be [N, K] and dy have a row for every row of x")
    a = L.LinearGradArgs(dtype=_DTYPES[x.dtype], act=_act(act), m=m, n=n, k=k, dy=_p(dy), x=_p(x), w=_p(weight),
                         dy_stride=ds, x_stride=xs, w_stride=ws)
    if a.act:
        if preact is None:
            raise ValueError(f"act {act!r} needs preact, the second result of linear(..., return_preact=True)")
        mz, _, zs = _rows(_tensor(preact, "preact", x), "preact", n)
        if mz != m:
            raise ValueError("preact must have a row for every row of x")
        a.z, a.z_stride = _p(preact), zs
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dw = torch.empty(weight.shape, dtype=x.dtype, device=x.device)
    db = dres = None
    if bias is not None:
        _vector(bias, "bias", n, x)
        db = torch.empty(n, dtype=bias.dtype, device=x.device)
        a.dbias, a.bias_f32 = _p(db), bias.dtype == torch.float32
    if residual is not None:
        r, _, _ = _rows(_tensor(residual, "residual", x), "residual", n)
        if not 1 <= r <= max(m, 1):
            raise ValueError(f"residual has {r} rows, x has {m}: expected 1 to that many")
        if r == m and residual.shape == dy.shape:
            dres = dy
        else:
            dres = torch.empty(residual.shape, dtype=x.dtype, device=x.device)
            a.dres, a.dres_stride, a.res_rows = _p(dres), n, r
    if not m:
        for t in (dw, db, dres):
            if t is not None:
                t.zero_()
        return dx, dw, db, dres
    a.dx, a.dw, a.dx_stride, a.dw_stride = _p(dx), _p(dw), k, k
    _call("yk_linear_backward", a, x)
    return dx, dw, db, dres


def layer_norm(x, weight=None, bias=None, *, eps=1e-5, return_stats=False):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension (biased variance).

    weight / bias [C]: both in x's dtype or both float32; None: 1 / 0.  With return_stats also
    mean and 1 / sqrt(var + eps), float32 of x's leading shape, for layer_norm_backward."""
    _tensor(x, "x")
    m, c, xs = _rows(x, "x")
    a = L.LayerNormArgs(dtype=_DTYPES[x.dtype], m=m, c=c, eps=eps, x=_p(x), x_stride=xs, y_stride=c)
    _norm_params(a, weight, bias, c, x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    a.y = _p(y)
    mean = rstd = None
    if return_stats:
        mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
        rstd = torch.empty_like(mean)
        a.mean, a.rstd = _p(mean), _p(rstd)
    if not eps >= 0:
        raise ValueError("eps must be >= 0")
    if m:
        _call("yk_layer_norm", a, x)
    return (y, mean, rstd) if return_stats else y


def _norm_params(a, weight, bias, c, x):
    given = [t for t in (weight, bias) if t is not None]
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _vector(t, name, c, x)
    if len(given) == 2 and weight.dtype != bias.dtype:
        raise ValueError("weight and bias must have one dtype")
    a.w, a.param_f32 = _p(weight), bool(given) and given[0].dtype == torch.float32
    if bias is not None and hasattr(a, "b"):
        a.b = _p(bias)


def layer_norm_backward(dy, x, weight, mean, rstd):
    """Gradients of layer_norm() from dy, x and its mean and rstd: (dx, dweight, dbias), the last
    two in weight's dtype (float32 where weight is None)."""
    _tensor(x, "x")
    m, c, xs = _rows(x, "x")
    md, _, ds = _rows(_tensor(dy, "dy", x), "dy", c)
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        _tensor(t, name, x, (torch.float32,))
        if t.numel() != m or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous tensor with an element for every row of x")
    if md != m:
        raise ValueError("dy must have a row for every row of x")
    a = L.LayerNormGradArgs(dtype=_DTYPES[x.dtype], m=m, c=c, dy=_p(dy), x=_p(x), mean=_p(mean), rstd=_p(rstd),
                            dy_stride=ds, x_stride=xs, dx_stride=c)
    _norm_params(a, weight, None, c, x)
    pd = torch.float32 if weight is None else weight.dtype
    a.param_f32 = pd == torch.float32
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dw, db = torch.empty(c, dtype=pd, device=x.device), torch.empty(c, dtype=pd, device=x.device)
    a.dx, a.dw, a.db = _p(dx), _p(dw), _p(db)
    _call("yk_layer_norm_backward", a, x)
    return dx, dw, db


def _heads(t, name, like, shape=None):
    _tensor(t, name, like)
    if t.dim() != 4 or (shape is not None and tuple(t.shape) != shape):
        raise ValueError(f"{name} must be [batch, tokens, heads, size]" +
                         (f" = {list(shape)}" if shape is not None else "") + f", got {list(t.shape)}")
    if t.shape[3] > 1 and t.stride(3) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return t.stride()[:3]


def _attention_args(cls, q, k, v, scale, causal, q_lengths, lengths):
    qs = _heads(q, "q", None)
    b, nq, h, d = q.shape
    ks = _heads(k, "k", q)
    nk, hk = k.shape[1], k.shape[2]
    vs = _heads(v, "v", q, (b, nk, hk, d))
    if k.shape[0] != b or k.shape[3] != d:
        raise ValueError(f"k must be [{b}, tokens, heads, {d}], got {list(k.shape)}")
    if h < 1 or hk < 1 or h % hk:
        raise ValueError(f"q's heads ({h}) must be a multiple of k's ({hk})")
    if not 1 <= d <= 128:
        raise ValueError(f"head size must be in [1, 128], got {d}")
    scale = d ** -0.5 if scale is None else float(scale)
    if not 0 < scale < float("inf"):
        raise ValueError("scale must be positive and finite")
    for t, name in ((q_lengths, "q_lengths"), (lengths, "lengths")):
        if t is not None:
            _tensor(t, name, q, (torch.int32,))
            if t.shape != (b,) or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 tensor [{b}]")
    s3 = C.c_int64 * 3
    return cls(dtype=_DTYPES[q.dtype], causal=bool(causal), b=b, h_q=h, h_kv=hk, d=d, nq=nq, nk=nk, scale=scale,
               q=_p(q), k=_p(k), v=_p(v), q_lengths=_p(q_lengths), lengths=_p(lengths), q_stride=s3(*qs), k_stride=s3(*ks),
               v_stride=s3(*vs))


def attention(q, k, v, *, scale=None, causal=False, lengths=None, q_lengths=None, return_lse=False):
    """softmax(scale q k^T) v per head: q [B, Nq, H, D], k and v [B, Nk, Hk, D] with H a multiple
    of Hk (neighbouring heads of q share a key head), D <= 128; scale D^-0.5 by default.

    lengths / q_lengths (int32 [B] on the device): keys / queries in use, the rest of a padded
    batch; keys behind a length are never read, queries behind one give 0.  causal: query i
    sees keys j <= i + length - q_length, so one new token sees its whole cache.  A query that sees
    no key gives 0.  Returns o like q, with return_lse also ln of the softmax's denominators,
    float32 [B, H, Nq] (-inf where no key is seen), for attention_backward."""
    a = _attention_args(L.AttentionArgs, q, k, v, scale, causal, q_lengths, lengths)
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    a.o, a.o_stride = _p(o), (C.c_int64 * 3)(*o.stride()[:3])
    lse = torch.empty(q.shape[0], q.shape[2], q.shape[1], dtype=torch.float32, device=q.device) if return_lse else None
    a.lse = _p(lse)
    if o.numel():
        _call("yk_attention", a, q)
    return (o, lse) if return_lse else o


def attention_backward(do, q, k, v, o, lse, *, scale=None, causal=False, lengths=None, q_lengths=None):
    """Gradients of attention() with the same arguments, from do and its two results: (dq, dk, dv),
    dk and dv summed over the heads that share a key head, 0 behind the lengths."""
    a = _attention_args(L.AttentionGradArgs, q, k, v, scale, causal, q_lengths, lengths)
    s3 = C.c_int64 * 3
    a.go_stride, a.o_stride = s3(*_heads(do, "do", q, tuple(q.shape))), s3(*_heads(o, "o", q, tuple(q.shape)))
    _tensor(lse, "lse", q, (torch.float32,))
    if lse.shape != (q.shape[0], q.shape[2], q.shape[1]) or not lse.is_contiguous():
        raise ValueError("lse must be attention's second result, contiguous [B, H, Nq]")
    dq, dk, dv = (torch.empty(t.shape, dtype=q.dtype, device=q.device) for t in (q, k, v))
    if not q.numel() or not k.numel():
        return dq.zero_(), dk.zero_(), dv.zero_()
    a.go, a.o, a.lse, a.dq, a.dk, a.dv = _p(do), _p(o), _p(lse), _p(dq), _p(dk), _p(dv)
    a.dq_stride, a.dk_stride, a.dv_stride = s3(*dq.stride()[:3]), s3(*dk.stride()[:3]), s3(*dv.stride()[:3])
    _call("yk_attention_backward", a, q)
    return dq, dk, dv
