"""The token operators (ops.py) on the GPU where their other tests do not reach: gradients at the ends of
fp16's range, rows with exact means, more
rows than one launch holds, sizes that take the kernels of large calls (which those are,
test_token_ops_paths_cpu.py checks), refusals.  Element by element against float64 within the bounds of token_helpers.py."""
import pytest
import torch
from torch.autograd import forward_ad

import token_helpers as R
import token_kernels as K
from conftest import pkg
from test_token_ops_gpu import run_attention

pytestmark = pytest.mark.gpu
DT = R.DTYPES


@pytest.fixture(scope="module")
def ops():
    return pkg().ops


def rn(*shape, dt="fp32", std=1.0, seed=0):
    g = torch.Generator().manual_seed(seed + sum((i + 1) * s for i, s in enumerate(shape)))
    return (torch.randn(*shape, generator=g) * std).to(DT[dt]).cuda()


# ---- attention's gradients in fp16 -------------------------------------------------------------
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,nq,nk,h,hk,dd,sq,sk,sv,sg,scale", [
    (1, 40, 8192, 1, 1, 8, 0.01, 100, 1, 6e-5, 1.0),      # dS of 2e-8: what fp16 rounds to 0
    (1, 8192, 4096, 1, 1, 8, 100, 0.01, 1, 6e-5, 1.0),    # the same for sums over rows
    (1, 3, 81920, 2, 1, 8, 1, 1, 1, 10, None),            # P of 1e-5: dv of few rows
    (2, 100, 40, 6, 3, 64, 0.01, 0.01, 60, 2000, None),   # dS past 65504, gradients that fit
    (4, 515, 515, 16, 16, 96, 0.3, 0.3, 1, 1e-4, None),   # two tiles a wave
])
def test_attention_backward_keeps_fp16s_digits(ops, causal, b, nq, nk, h, hk, dd, sq, sk, sv, sg, scale):
    """P and dS enter a 16-bit product each with half a step of its own value, small or large.  The
    kernels take powers of two out of both: half of fp16's subnormal step is 2^-40 of P, and of dS at
    most 2^-34 of its column's largest, which here is below 2^-6, and below 2^17 where dS is large."""
    q, k, v, do = (rn(b, n, hh, dd, dt="fp16", std=s, seed=i)
                   for i, (n, hh, s) in enumerate(((nq, h, sq), (nk, hk, sk), (nk, hk, sv), (nq, h, sg))))
    ref = R.attention(q, k, v, scale, causal, do=do, grad_tiny=(2.0 ** -40, 2.0 ** -40 if sg < 100 else 2.0 ** -17))
    o, lse = ops.attention(q, k, v, scale=scale, causal=causal, return_lse=True)
    got = ops.attention_backward(do, q, k, v, o, lse, scale=scale, causal=causal)
    again = ops.attention_backward(do, q, k, v, o, lse, scale=scale, causal=causal)
    for name, g, a in zip(("dq", "dk", "dv"), got, again):
        R.check(g, *ref[name], name)
        assert torch.equal(g, a)


# ---- layer norm ----------------------------------------------------------------------------------
@pytest.mark.parametrize("dt,at", [("fp32", 1000.0), ("bf16", 144.0), ("fp16", 1000.0)])
@pytest.mark.parametrize("m,c", [(3, 64), (300, 256), (5, 640), (4, 1024), (2, 8192), (2, 16384), (8200, 256)])
def test_layer_norm_gradients_of_rows_with_exact_means(ops, dt, at, m, c):
    """Rows of one value: the mean is that value (all sums are whole numbers below 2^24, c a divisor), so
    x - mean is zero, y is the bias, and the weight's gradient, a sum of dy 0, is zero exactly; dx is
    rstd (g - mean g), a sum of c terms and three roundings."""
    x = torch.full((m, c), at, dtype=DT[dt], device="cuda")
    w, b, dy = rn(c, std=0.1) + 1, rn(c, seed=1), rn(m, c, dt=dt, seed=2)
    y, mean, rstd = ops.layer_norm(x, w, b, return_stats=True)
    assert torch.equal(y, b.to(DT[dt]).expand(m, c))
    dx, dw, db = ops.layer_norm_backward(dy, x, w, mean, rstd)
    assert not dw.any()
    g, r = dy.double() * w.double(), rstd.double()[:, None]
    want = r * (g - g.mean(1, keepdim=True))
    R.check(dx, want, R._final(want, r * ((c + 8) * R.F * g.abs().mean(1, keepdim=True) + 8 * R.F * (g.abs() + g.mean(1, keepdim=True).abs())),
                               DT[dt]), "dx")
    R.check(db, dy.double().sum(0), (m + 8) * R.F * dy.double().abs().sum(0), "db")


# ---- more workgroups than one launch holds ---------------------------------------------------------
def test_layer_norm_of_more_rows_than_a_launch_holds(ops):
    """2^28 rows of 16 per workgroup of 256 threads: parts, each row the bits of a smaller call."""
    m, c = 2 ** 28 + 37, 8
    x = rn(2 ** 16 + 3, c, dt="bf16").repeat(m // (2 ** 16 + 3) + 1, 1)[:m]
    w, b = rn(c, seed=1), rn(c, seed=2)
    y, mean, rstd = ops.layer_norm(x, w, b, return_stats=True)
    for lo, hi in ((0, 2 ** 20), (2 ** 28 - 5000, m)):
        got = ops.layer_norm(x[lo:hi], w, b, return_stats=True)
        for g, t in zip(got, (y, mean, rstd)):
            assert torch.equal(g, t[lo:hi])
    want, e = R.layer_norm(x[-99:], w, b, 1e-5)
    R.check(y[-99:], want, e, "y")


def test_residual_gradient_of_more_rows_than_a_launch_holds(ops):
    r, n = 2 ** 24 + 3, 16
    dy = rn(2 ** 16 + 1, n, dt="bf16").repeat(r // (2 ** 16 + 1) + 1, 1)[:r + 5]
    x, w = torch.zeros(r + 5, 1, dtype=dy.dtype, device="cuda"), rn(n, 1, dt="bf16")
    dres = ops.linear_backward(dy, x, w, residual=dy[:r])[3]
    assert torch.equal(dres[5:], dy[5:r])
    assert torch.equal(dres[:5], (dy[:5].float() + dy[r:].float()).to(dy.dtype))


def test_few_rows_of_more_columns_than_a_launch_holds(ops):
    n = 2 ** 27 + 5
    x, w = rn(2, 1, dt="bf16"), rn(2 ** 16 + 1, 1, dt="bf16").repeat(n // (2 ** 16 + 1) + 1, 1)[:n]
    y = ops.linear(x, w)
    assert torch.equal(y, (x.float() * w[:, 0].float()).to(y.dtype))  # (a product of two bf16 is exact in float32)


# ---- refusals ------------------------------------------------------------------------------------
def test_forward_mode_tangents_are_refused(ops):
    """A tangent would be lost without a word: every argument that carries one is refused."""
    x, w, b = rn(4, 8), rn(8, 8), rn(8)
    q, o = rn(1, 4, 2, 8), rn(1, 4, 2, 8)
    lse, m = rn(1, 2, 4), rn(4)
    calls = [(ops.linear, (x, w, b), {"residual": x}), (ops.linear_backward, (x, x, w, b), {"act": "gelu", "preact": x, "residual": x}),
             (ops.layer_norm, (x, b, b), {}), (ops.layer_norm_backward, (x, x, b, m, m), {}),
             (ops.attention, (q, q, q), {}), (ops.attention_backward, (q, q, q, q, o, lse), {})]
    with forward_ad.dual_level():
        for f, args, kw in calls:
            f(*args, **kw)  # nothing carries one
            for i, t in enumerate(args):
                d = forward_ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(ValueError, match="tangent"):
                    f(*args[:i], d, *args[i + 1:], **kw)
            for n, t in kw.items():
                if isinstance(t, torch.Tensor):
                    with pytest.raises(ValueError, match="tangent"):
                        f(*args, **{**kw, n: forward_ad.make_dual(t, torch.ones_like(t))})


def test_values_outside_float32_are_refused(ops):
    q, x = rn(1, 4, 2, 8), rn(4, 8)
    for scale in (1e39, 1e-50, -1.0, float("nan")):
        with pytest.raises(ValueError, match="scale"):
            ops.attention(q, q, q, scale=scale)
    for eps in (1e39, -1e-9, float("nan")):
        with pytest.raises(ValueError, match="eps"):
            ops.layer_norm(x, eps=eps)
    y = ops.layer_norm(x, eps=torch.finfo(torch.float32).max)
    R.check(y, *R.layer_norm(x, None, None, torch.finfo(torch.float32).max), "y")
    many = q[:, :1].expand(2 ** 31, 1, 2, 8)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.attention(many, many, many)


def test_tracing_is_refused(ops):
    x, w = rn(4, 8), rn(6, 8)
    with pytest.raises(pkg().YKError, match="jit.trace"):
        torch.jit.trace(lambda t: ops.linear(t, w), (x,))


def test_an_earlier_error_of_the_runtime_is_not_the_calls(ops):
    """A HIP call of the caller that failed leaves its code as the runtime's last error: the operators
    neither report it as a launch of theirs nor take it away."""
    import ctypes as C

    x, w, q = rn(4, 8), rn(6, 8), rn(1, 4, 2, 8)
    want = ops.linear(x, w), ops.layer_norm(x), ops.attention(q, q, q)
    torch.cuda.synchronize()
    loaded = {line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line}
    hip = C.CDLL(loaded.pop())
    assert not loaded and hip.hipSetDevice(4096) != 0  # no such device
    try:
        got = ops.linear(x, w), ops.layer_norm(x), ops.attention(q, q, q)
    finally:
        left = hip.hipGetLastError()
    assert left != 0
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_the_first_call_may_be_a_captured_one(ops, monkeypatch):
    """The device's context is made by the first call: inside a capture too."""
    x, w, q = rn(300, 64), rn(40, 64), rn(2, 200, 4, 64, dt="fp16")
    want = ops.linear(x, w, act="gelu"), ops.attention(q, q, q)
    monkeypatch.setattr(pkg()._lib, "_ctx", {})
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y, o = ops.linear(x, w, act="gelu"), ops.attention(q, q, q)
    for _ in range(3):
        y.zero_(), o.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(o, want[1])


# ---- the detector's report ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_profile_names_the_kernels_of_an_aifi_row(dtype):
    """profile() names what its batch launches: 80 cells of 2 images are above the few rows' 64 and
    one image's attention below its 128; a batch of 20-cell images takes the few-rows kernel."""
    import importlib

    import numpy as np

    from aifi_helpers import aifi_dict

    P = pkg()
    A, W, M = (importlib.import_module(f"{P.__name__}.{n}") for n in ("arch", "weights", "model"))
    ar = A.parse_arch(aifi_dict("n"))
    sd = W.synthetic_state_dict(ar, 0)
    t = {"fp32": "F32", "bf16": "B16"}[dtype]
    many = "gemm_f32_kernel<false, false, 64>" if dtype == "fp32" else f"gemm_kernel<yk::tok::{t}, false, false, "
    for hw, linear, attention in (((256, 320), many, "attn_split_kernel<yk::tok::" + t), ((128, 160), "rows_kernel<yk::tok::" + t, "attn_split_"),
                                  ((384, 640), many, "attn_kernel<yk::tok::" + t)):
        dm = M.DeviceModel(M.Program(ar, sd, hw[0], hw[1], max(hw), 2, dtype))
        frames = torch.from_numpy(np.zeros((2, *hw, 3), np.uint8)).cuda()
        dm.detect(frames, 0.25, 0.7, 300)
        names = {kind: [n for _, k, n, _ in dm.profile(frames) if k == kind] for kind in (M.YK_K_LINEAR, M.YK_K_LAYER_NORM, M.YK_K_ATTENTION)}
        assert len(names[M.YK_K_LINEAR]) == 4 and all(n.startswith(linear) for n in names[M.YK_K_LINEAR]), names
        assert all(n.startswith("norm_kernel<yk::tok::" + t) for n in names[M.YK_K_LAYER_NORM]), names
        assert all(n.startswith(attention) for n in names[M.YK_K_ATTENTION]), names


# ---- kernels that large calls take ------------------------------------------------------------------
@pytest.mark.parametrize("dt,form,m,k,n", K.PRODUCTS)
def test_products_of_large_tiles(ops, dt, form, m, k, n):
    """Whole tiles and remainders of every tile size and operand order, split or not."""
    x, w, b = rn(m, k, dt=dt), rn(n, k, dt=dt, std=k ** -0.5), rn(n, dt=dt)
    if form.startswith("ff"):
        for act, res, bias in (("none", None, None), ("gelu", rn(77, n, dt=dt, seed=2), b)):
            y, z = ops.linear(x, w, bias, act=act, residual=res, return_preact=True)
            want, ey, wz, ez = R.linear(x, w, bias, act, res)
            R.check(y, want, ey, f"y {act}")
            R.check(z, wz, ez, f"z {act}")
            assert torch.equal(y, ops.linear(x, w, bias, act=act, residual=res))
        return
    dy, z = rn(m, n, dt=dt, seed=1), rn(m, n, dt=dt, seed=3)
    for act in ("none", "silu"):
        got = ops.linear_backward(dy, x, w, b, act=act, preact=z)
        again = ops.linear_backward(dy, x, w, b, act=act, preact=z)
        for (want, e), g, a, name in zip(R.linear_grads(dy, x, w, act, z), got, again, ("dx", "dw", "db")):
            R.check(g, want, R._final(want, e, b.dtype) if name == "db" else e, f"{name} {act}")
            assert torch.equal(g, a)


@pytest.mark.parametrize("dt,c", [(dt, c) for dt, cs in K.NORM_WIDTHS.items() for c in cs])
def test_layer_norm_of_many_rows(ops, dt, c):
    """Rows of 16 lanes at every number of chunks per lane, whole and with ragged ends."""
    m = K.NORM_ROWS
    x = rn(m, c, dt=dt) * 2 + rn(m, 1, dt=dt, seed=1) * 4
    w, b, dy = rn(c, dt=dt) * 0.1 + 1, rn(c, dt=dt, seed=2), rn(m, c, dt=dt, seed=3)
    for wt, bt in ((w, b), (w.float(), b.float()), (None, None)):
        y, mean, rstd = ops.layer_norm(x, wt, bt, return_stats=True)
        want, e = R.layer_norm(x, wt, bt, 1e-5)
        R.check(y, want, e, "y")
        grads = ops.layer_norm_backward(dy, x, wt, mean, rstd)
        again = ops.layer_norm_backward(dy, x, wt, mean, rstd)
        for (want, e), g, a, name in zip(R.layer_norm_grads(dy, x, wt, 1e-5), grads, again, ("dx", "dw", "db")):
            R.check(g, want, e if name == "dx" else R._final(want, e, g.dtype), name)
            assert torch.equal(g, a)


@pytest.mark.parametrize("dt", DT)
def test_layer_norm_of_many_turns(ops, dt):
    """A workgroup of the backward pass walks many rows, each fetched while one is worked on."""
    for m, c in ((60001, 24), (20003, 600)):
        x, w, dy = rn(m, c, dt=dt) + 1, rn(c, dt=dt), rn(m, c, dt=dt, seed=3)
        y, mean, rstd = ops.layer_norm(x, w, return_stats=True)
        for (want, e), g, name in zip(R.layer_norm_grads(dy, x, w, 1e-5), ops.layer_norm_backward(dy, x, w, mean, rstd), ("dx", "dw", "db")):
            R.check(g, want, e if name == "dx" else R._final(want, e, g.dtype), name)


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,n,h,hk,d", K.TWO_TILES)
def test_attention_of_two_tiles_a_wave(ops, dt, causal, b, n, h, hk, d):
    """Blocks of 128 rows with a remainder, whole batches and ragged ones, with gradients."""
    run_attention(ops, dt, b, n, n, h, hk, d, causal)
    lens = [n, 0, 1, 129, n - 1, 64, 300, 257] + [n] * (b - 8)
    run_attention(ops, dt, b, n, n, h, hk, d, causal, lengths=lens, q_lengths=lens)
    run_attention(ops, dt, b, n, n, h, hk, d, causal, lengths=[n - 3, 17, 0, 200] * (b // 4) + [n] * (b % 4))
