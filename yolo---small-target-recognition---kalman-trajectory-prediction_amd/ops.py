"""Token operators on device tensors: the matrix product with its fused epilogue, layer norm and
attention of a transformer layer over the cells of a feature map, each with its gradients.

The kernels are those the detector program runs for an ``AIFI`` row of a model YAML (model.py);
here they take torch tensors (float32, bfloat16 or float16, on one GPU).  Calls are enqueued on
the tensors' device's current stream, allocate their outputs and scratch from torch and never
synchronise, so they can be captured into a graph.  No autograd graph is built: a call whose
inputs require gradients (while gradients are enabled) or carry a forward-mode tangent raises, and so
does one under torch.jit.trace, which would record its empty outputs; the ``*_backward`` functions
return the gradients.  Sums are float32 and an output is rounded once; what else a 16-bit type rounds are
operands of its matrix products (attention's P and dS, linear's dz) and the preactivation that linear
returns.  Equal calls give equal bits.

A tensor's last dimension must be contiguous; what precedes it must step evenly from row to row
(any row stride, so a channel slice of a wider tensor is fine).  Anything else raises ValueError.
"""
from __future__ import annotations

import ctypes as C
import struct

import torch
from torch.autograd import forward_ad as _fwd

from . import _lib as L

ACTS = {"none": 0, "silu": 1, "gelu": 2, "relu": 3}
_DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 3}  # yk_act_dtype
_F32 = torch.float32
_F32_MIN, _F32_MAX, _INF = 2.0 ** -149, torch.finfo(_F32).max, float("inf")
_empty, _empty_like, _grad_enabled, _tracing = torch.empty, torch.empty_like, torch.is_grad_enabled, torch._C._is_tracing

# The C argument structs as packed bytes (a ctypes struct costs three times as long to fill); the
# last two fields, scratch and its size, are appended once the size is known.
_LINEAR = struct.Struct("4i 3q 6Q 6q")
_LINEAR_GRAD = struct.Struct("4i 3q 8Q 8q")
_NORM = struct.Struct("2i 2q f i 6Q 2q")
_NORM_GRAD = struct.Struct("2i 2q 8Q 3q")
_ATTENTION = struct.Struct("6i 2q f i 7Q 12q")
_ATTENTION_GRAD = struct.Struct("6i 2q f i 11Q 24q")
_WS = struct.Struct("Q q")
_NO_WS = _WS.pack(0, 0)
_raw_stream = torch._C._cuda_getCurrentRawStream  # (torch.cuda.current_stream builds an object around it)
_entry: dict = {}    # entry point -> its ctypes function
_scratch: dict = {}  # (entry point, sizes) -> bytes of scratch


def _input(t, name):
    """The operator's first tensor: sets the type and the GPU.  Returns (yk_act_dtype, device index)."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if _tracing():
        raise L.YKError("torch.jit.trace records torch operations only: this call's result would be an empty tensor")
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if not t.is_cuda:
        raise L.YKError(f"{name} is on {t.device}: the token operators run on an AMD GPU only (no CPU fallback)")
    if t.requires_grad or _fwd._current_level >= 0:
        _no_derivative(t, name)
    return code, t.get_device()


def _no_derivative(t, name):
    if t.requires_grad and _grad_enabled():
        raise ValueError(f"{name} requires grad: no autograd graph is built here (detach it, or torch.no_grad())")
    if _fwd.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} has a forward-mode tangent, which would be lost: pass unpack_dual({name}).primal")


def _like(t, name, dev, dtype, other=None):
    """Another tensor of the call: on the same GPU, of the given type (or the other one)."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor")
    if t.get_device() != dev:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{dev}")
    if t.dtype is not dtype and t.dtype is not other:
        raise ValueError(f"{name} has dtype {t.dtype}, expected {dtype}" + (f" or {other}" if other else ""))
    if t.requires_grad or _fwd._current_level >= 0:
        _no_derivative(t, name)
    return t


def _fresh(t):
    """An uninitialised contiguous tensor like t (empty_like is the faster call where that is one)."""
    return _empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _rows(t, name, cols=None):
    """(rows, columns, row stride) of a tensor as a matrix of its last dimension."""
    shape = t.shape
    if not shape or shape[-1] < 1:
        raise ValueError(f"{name} must have a last dimension of at least 1")
    c = shape[-1]
    if cols is not None and c != cols:
        raise ValueError(f"{name} has {c} columns, expected {cols}")
    if t.is_contiguous():
        return t.numel() // c, c, c
    strides = t.stride()
    if c > 1 and strides[-1] != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    rows, stride = 1, None
    for n, s in zip(shape[-2::-1], strides[-2::-1]):
        if n == 1:
            continue
        if stride is None:
            stride = s
        elif s != stride * rows:
            raise ValueError(f"{name}: rows must be evenly spaced (shape {tuple(shape)}, strides {strides})")
        rows *= n
    return rows, c, c if stride is None else stride


def _vector(t, name, n, dev, dtype):
    """A parameter of n elements, contiguous, of the tensors' type or float32: (address, 1 if float32)."""
    _like(t, name, dev, dtype, _F32)
    if t.shape != (n,) or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {n} elements, got {tuple(t.shape)}")
    return t.data_ptr(), int(t.dtype is _F32)


def _call(fn, packed, dev, sizes=None):
    """Enqueue an entry point on the device's current stream, with the scratch that `sizes` (all its
    size depends on) needs."""
    call = _entry.get(fn)
    if call is None:
        call = _entry[fn] = getattr(L.lib(), fn)
    if sizes is not None:
        need = _scratch.get((fn, sizes))
        if need is None:
            n = C.c_int64()
            L.check(getattr(L.lib(), fn + "_workspace")(packed + _NO_WS, C.byref(n)), fn)
            if len(_scratch) >= 4096:
                _scratch.clear()
            need = _scratch[(fn, sizes)] = n.value
        if need:
            ws = _empty(need, dtype=torch.uint8, device=torch.device("cuda", dev))
            packed += _WS.pack(ws.data_ptr(), need)
        else:
            packed += _NO_WS
    rc = call(L.context(dev), packed, _raw_stream(dev))
    if rc:
        L.check(rc, fn)


def _act(name):
    code = ACTS.get(name)
    if code is None:
        raise ValueError(f"act must be one of {sorted(ACTS)}, got {name!r}")
    return code


def _residual(residual, m, n, dev, dtype):
    """(address, rows, row stride) of linear()'s residual."""
    r, _, rs = _rows(_like(residual, "residual", dev, dtype), "residual", n)
    if not 1 <= r <= max(m, 1):
        raise ValueError(f"residual has {r} rows, x has {m}: expected 1 to that many")
    return residual.data_ptr(), r, rs


def linear(x, weight, bias=None, *, act="none", residual=None, return_preact=False):
    """act(x weight^T + bias) + residual, in one kernel (two where few tiles split a long K).

    x [..., K]; weight [N, K]; bias [N] in x's dtype or float32; act "none", "silu", "gelu" (exact)
    or "relu"; residual [..., N] with any R <= rows(x) rows, row m of the result taking row m % R (R
    tokens shared by the images of a batch).  Returns [..., N], with return_preact also act's
    argument, which linear_backward needs unless act is "none"."""
    dt, dev = _input(x, "x")
    dtype = x.dtype
    m, k, xs = _rows(x, "x")
    n, _, ws = _rows(_like(weight, "weight", dev, dtype), "weight", k)
    if weight.dim() != 2 or n < 1:
        raise ValueError("weight must be [N, K]")
    a = _act(act)
    b, bf = (0, 0) if bias is None else _vector(bias, "bias", n, dev, dtype)
    r, rows, rs = (0, 0, 0) if residual is None or not m else _residual(residual, m, n, dev, dtype)
    y = x.new_empty((*x.shape[:-1], n))
    z = _empty_like(y) if return_preact else None
    if m:
        _call("yk_linear", _LINEAR.pack(dt, a, bf, 0, m, n, k, x.data_ptr(), weight.data_ptr(), b, r, y.data_ptr(),
                                        0 if z is None else z.data_ptr(), xs, ws, rs, rows, n, n),
              dev, (dt, m, n, k))
    return (y, z) if return_preact else y


def linear_backward(dy, x, weight, bias=None, *, act="none", preact=None, residual=None):
    """Gradients of linear() from dy [..., N]: (dx, dweight, dbias, dresidual), the last two None
    without bias / residual.  preact is linear's second result (needed unless act is "none");
    residual's shape and dtype are what counts of it.  Where it has dy's shape its gradient is dy
    itself."""
    dt, dev = _input(x, "x")
    dtype = x.dtype
    m, k, xs = _rows(x, "x")
    n, _, ws = _rows(_like(weight, "weight", dev, dtype), "weight", k)
    md, _, ds = _rows(_like(dy, "dy", dev, dtype), "dy", n)
    if weight.dim() != 2 or md != m:
        raise ValueError("weight must be [N, K] and dy have a row for every row of x")
    a = _act(act)
    z, zs = 0, 0
    if a:
        if preact is None:
            raise ValueError(f"act {act!r} needs preact, the second result of linear(..., return_preact=True)")
        mz, _, zs = _rows(_like(preact, "preact", dev, dtype), "preact", n)
        if mz != m:
            raise ValueError("preact must have a row for every row of x")
        z = preact.data_ptr()
    dx, dw = _fresh(x), _fresh(weight)
    db = dres = None
    pb = bf = pr = rows = 0
    if bias is not None:
        _, bf = _vector(bias, "bias", n, dev, dtype)
        db = bias.new_empty(n)
        pb = db.data_ptr()
    if residual is not None:
        _, rows, _ = _residual(residual, m, n, dev, dtype)
        if residual.shape == dy.shape:
            dres, rows = dy, 0
        else:
            dres = x.new_empty(residual.shape)
            pr = dres.data_ptr()
    if m:
        _call("yk_linear_backward",
              _LINEAR_GRAD.pack(dt, a, bf, 0, m, n, k, dy.data_ptr(), x.data_ptr(), weight.data_ptr(), z, dx.data_ptr(),
                                dw.data_ptr(), pb, pr, ds, xs, ws, zs, k, k, n, rows),
              dev, (dt, a, m, n, k, pb != 0, rows))
    else:
        for t in (dw, db, dres):
            if t is not None:
                t.zero_()
    return dx, dw, db, dres


def _norm_params(weight, bias, c, dev, dtype):
    """(address of weight, of bias, 1 if they are float32)"""
    w, wf = (0, 0) if weight is None else _vector(weight, "weight", c, dev, dtype)
    b, bf = (0, wf) if bias is None else _vector(bias, "bias", c, dev, dtype)
    if weight is not None and bf != wf:
        raise ValueError("weight and bias must have one dtype")
    return w, b, bf


def layer_norm(x, weight=None, bias=None, *, eps=1e-5, return_stats=False):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension (biased variance).

    weight / bias [C]: both in x's dtype or both float32; None: 1 / 0.  With return_stats also
    mean and 1 / sqrt(var + eps), float32 of x's leading shape, for layer_norm_backward."""
    dt, dev = _input(x, "x")
    m, c, xs = _rows(x, "x")
    w, b, pf = _norm_params(weight, bias, c, dev, x.dtype)
    if not eps >= 0 or _F32_MAX < eps < _INF:
        raise ValueError("eps must be >= 0, in float32's range")
    y = _fresh(x)
    mean = rstd = None
    if return_stats:
        mean = x.new_empty(x.shape[:-1], dtype=_F32)
        rstd = _empty_like(mean)
    if m:
        _call("yk_layer_norm", _NORM.pack(dt, pf, m, c, eps, 0, x.data_ptr(), w, b, y.data_ptr(),
                                          mean.data_ptr() if return_stats else 0, rstd.data_ptr() if return_stats else 0,
                                          xs, c), dev)
    return (y, mean, rstd) if return_stats else y


def layer_norm_backward(dy, x, weight, mean, rstd):
    """Gradients of layer_norm() from dy, x and its mean and rstd: (dx, dweight, dbias), the last
    two in weight's dtype (float32 where weight is None)."""
    dt, dev = _input(x, "x")
    m, c, xs = _rows(x, "x")
    md, _, ds = _rows(_like(dy, "dy", dev, x.dtype), "dy", c)
    for t, name in ((mean, "mean"), (rstd, "rstd")):
        if _like(t, name, dev, _F32).numel() != m or not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous tensor with an element for every row of x")
    if md != m:
        raise ValueError("dy must have a row for every row of x")
    w, _, pf = _norm_params(weight, None, c, dev, x.dtype)
    dw = x.new_empty(c, dtype=_F32) if weight is None else weight.new_empty(c)
    dx, db = _fresh(x), _empty_like(dw)
    _call("yk_layer_norm_backward",
          _NORM_GRAD.pack(dt, int(dw.dtype is _F32), m, c, dy.data_ptr(), x.data_ptr(), w, mean.data_ptr(), rstd.data_ptr(),
                          dx.data_ptr(), dw.data_ptr(), db.data_ptr(), ds, xs, c),
          dev, (dt, m, c))
    return dx, dw, db


def _heads(t, name, shape):
    """Strides of [batch, tokens, heads, size]."""
    if t.shape != shape:
        raise ValueError(f"{name} must be [batch, tokens, heads, size] = {list(shape)}, got {list(t.shape)}")
    s = t.stride()
    if s[3] != 1 and shape[3] > 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")
    return s[:3]


def _attention_args(q, k, v, scale, causal, q_lengths, lengths):
    """(device, sizes that open the C struct, addresses of q k v, of the lengths, strides of q k v)"""
    dt, dev = _input(q, "q")
    dtype = q.dtype
    _like(k, "k", dev, dtype)
    _like(v, "v", dev, dtype)
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError(f"q and k must be [batch, tokens, heads, size], got {list(q.shape)} and {list(k.shape)}")
    b, nq, h, d = q.shape
    nk, hk = k.shape[1:3]
    qs, ks, vs = _heads(q, "q", q.shape), _heads(k, "k", (b, nk, hk, d)), _heads(v, "v", (b, nk, hk, d))
    if h < 1 or hk < 1 or h % hk:
        raise ValueError(f"q's heads ({h}) must be a multiple of k's ({hk})")
    if not 1 <= d <= 128:
        raise ValueError(f"head size must be in [1, 128], got {d}")
    scale = d ** -0.5 if scale is None else float(scale)
    if not _F32_MIN <= scale <= _F32_MAX:
        raise ValueError("scale must be positive and finite, in float32's range")
    if max(b, h) >= 1 << 31:
        raise ValueError("more batch elements or heads than 2^31")
    lens = [0, 0]
    for i, (t, name) in enumerate(((q_lengths, "q_lengths"), (lengths, "lengths"))):
        if t is not None:
            if _like(t, name, dev, torch.int32).shape != (b,) or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 tensor [{b}]")
            lens[i] = t.data_ptr()
    return dev, (dt, int(bool(causal)), b, h, hk, d, nq, nk, scale, 0), (q.data_ptr(), k.data_ptr(), v.data_ptr()), lens, \
        (*qs, *ks, *vs)


def attention(q, k, v, *, scale=None, causal=False, lengths=None, q_lengths=None, return_lse=False):
    """softmax(scale q k^T) v per head: q [B, Nq, H, D], k and v [B, Nk, Hk, D] with H a multiple
    of Hk (neighbouring heads of q share a key head), D <= 128; scale D^-0.5 by default.

    lengths / q_lengths (int32 [B] on the device): keys / queries in use, the rest of a padded
    batch; keys behind a length are never read, queries behind one give 0.  causal: query i
    sees keys j <= i + length - q_length, so one new token sees its whole cache.  A query that sees
    no key gives 0.  (What causality alone hides takes part as a factor of 0: a NaN or infinity in v, or
    in k, q or do backward, may show as NaN there; behind the lengths none does.)  Returns o like q, with return_lse also ln of the softmax's denominators,
    float32 [B, H, Nq] (-inf where no key is seen), for attention_backward."""
    dev, head, qkv, lens, strides = _attention_args(q, k, v, scale, causal, q_lengths, lengths)
    o = _fresh(q)
    lse = q.new_empty((q.shape[0], q.shape[2], q.shape[1]), dtype=_F32) if return_lse else None
    if o.numel():
        _call("yk_attention", _ATTENTION.pack(*head, *qkv, *lens, o.data_ptr(), lse.data_ptr() if return_lse else 0, *strides,
                                              *o.stride()[:3]), dev, head)
    return (o, lse) if return_lse else o


def attention_backward(do, q, k, v, o, lse, *, scale=None, causal=False, lengths=None, q_lengths=None):
    """Gradients of attention() with the same arguments, from do and its two results: (dq, dk, dv),
    dk and dv summed over the heads that share a key head, 0 behind the lengths."""
    dev, head, qkv, lens, strides = _attention_args(q, k, v, scale, causal, q_lengths, lengths)
    gs = _heads(_like(do, "do", dev, q.dtype), "do", q.shape)
    os = _heads(_like(o, "o", dev, q.dtype), "o", q.shape)
    if _like(lse, "lse", dev, _F32).shape != (q.shape[0], q.shape[2], q.shape[1]) or not lse.is_contiguous():
        raise ValueError("lse must be attention's second result, contiguous [B, H, Nq]")
    dq, dk, dv = _fresh(q), _fresh(k), _fresh(v)
    if not q.numel() or not k.numel():
        return dq.zero_(), dk.zero_(), dv.zero_()
    _call("yk_attention_backward",
          _ATTENTION_GRAD.pack(*head, do.data_ptr(), *qkv, o.data_ptr(), lse.data_ptr(), *lens, dq.data_ptr(), dk.data_ptr(),
                               dv.data_ptr(), *gs, *strides, *os, *dq.stride()[:3], *dk.stride()[:3], *dv.stride()[:3]),
          dev, head)
    return dq, dk, dv
