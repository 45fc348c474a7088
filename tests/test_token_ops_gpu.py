"""The token operators (ops.py) on the GPU against their definitions in float64, element by
element within bounds derived in token_helpers.py: types, sizes from one token, odd sizes, strides,
masks, lengths, shared heads, gradients, refusals, streams and graphs."""
import math

import pytest
import torch

import token_helpers as R
from conftest import pkg

pytestmark = pytest.mark.gpu
DT = R.DTYPES


@pytest.fixture(scope="module")
def ops():
    return pkg().ops


def rn(*shape, dt="fp32", std=1.0, seed=0):
    g = torch.Generator().manual_seed(seed + sum((i + 1) * s for i, s in enumerate(shape)))
    return (torch.randn(*shape, generator=g) * std).to(DT[dt]).cuda()


def strided(t, pad=3, off=1):
    """The same values as a channel slice of wider rows: unaligned pointer and row stride."""
    wide = torch.full((*t.shape[:-1], t.shape[-1] + pad), float("nan"), dtype=t.dtype, device=t.device)
    wide[..., off:off + t.shape[-1]] = t
    return wide[..., off:off + t.shape[-1]]


# ---- linear ----------------------------------------------------------------------------------
SIZES = [(1, 1, 1), (1, 512, 2048), (3, 40, 24), (8, 100, 33), (17, 1111, 7), (33, 64, 130), (64, 96, 65), (65, 96, 64),
         (100, 1000, 10), (129, 72, 257), (320, 320, 1024), (200, 2048, 72), (1000, 33, 129), (2560, 320, 320)]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear(ops, dt, m, k, n):
    x, w, b = rn(m, k, dt=dt), rn(n, k, dt=dt, std=k ** -0.5), rn(n, dt=dt)
    for act, res, bias in (("none", None, None), ("gelu", None, b), ("silu", rn(m, n, dt=dt, seed=1), b.float()),
                           ("relu", rn((m + 1) // 2, n, dt=dt, seed=2), b)):
        y, z = ops.linear(x, w, bias, act=act, residual=res, return_preact=True)
        want, ey, wz, ez = R.linear(x, w, bias, act, res)
        R.check(y, want, ey, f"y {act}")
        R.check(z, wz, ez, f"z {act}")
        assert torch.equal(y, ops.linear(x, w, bias, act=act, residual=res))


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("m,k,n", [(9, 48, 40), (130, 200, 136), (300, 77, 90)])
def test_linear_strided_rows_and_images(ops, dt, m, k, n):
    x, w, b, res = rn(m, k, dt=dt), rn(n, k, dt=dt), rn(n, dt=dt), rn(m, n, dt=dt, seed=3)
    want, ey, _, _ = R.linear(x, w, b, "silu", res)
    R.check(ops.linear(strided(x), strided(w), b, act="silu", residual=strided(res)), want, ey, "unaligned")
    x8 = strided(x, pad=8 + (-k) % 8, off=8)
    R.check(ops.linear(x8, w, b, act="silu", residual=res), want, ey, "aligned slice")
    # tokens of several images, a table of one image's tokens as the residual; one row for all rows of x
    xi = torch.stack([x, x + 1])
    want, ey, _, _ = R.linear(xi, w, b, "none", res)
    R.check(ops.linear(xi, w, b, residual=res), want, ey, "images")
    xe = x[:1].expand(m, k)
    want, ey, _, _ = R.linear(xe, w, None, "none", None)
    R.check(ops.linear(xe, w), want, ey, "expanded")


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 64, 48), (5, 24, 40), (65, 96, 64), (129, 72, 257), (300, 1000, 17),
                                   (1031, 33, 70), (2560, 128, 320), (4096, 64, 64)])
@pytest.mark.parametrize("act", ["none", "gelu", "silu", "relu"])
def test_linear_backward(ops, dt, m, k, n, act):
    x, w, b, dy = rn(m, k, dt=dt), rn(n, k, dt=dt, std=k ** -0.5), rn(n, dt=dt), rn(m, n, dt=dt, seed=1)
    rows = max(1, m // 3)
    _, z = ops.linear(x, w, b, act=act, return_preact=True)
    bias = b if m % 2 else b.float()
    got = ops.linear_backward(dy, x, w, bias, act=act, preact=z, residual=rn(rows, n, dt=dt))
    again = ops.linear_backward(dy, x, w, bias, act=act, preact=z, residual=rn(rows, n, dt=dt))
    for (want, e), g, a, name in zip(R.linear_grads(dy, x, w, act, z, rows), got, again, ("dx", "dw", "db", "dres")):
        if name == "db":
            e = R._final(want, e, bias.dtype)
        R.check(g, want, e, f"{name} {act}")
        assert torch.equal(g, a)


@pytest.mark.parametrize("dt", DT)
def test_linear_backward_strided(ops, dt):
    m, k, n = 150, 60, 44
    x, w, b, dy = rn(m, k, dt=dt), rn(n, k, dt=dt), rn(n, dt=dt), rn(m, n, dt=dt, seed=1)
    _, z = ops.linear(x, w, b, act="gelu", return_preact=True)
    got = ops.linear_backward(strided(dy), strided(x), strided(w), b, act="gelu", preact=strided(z), residual=dy)
    for (want, e), g in zip(R.linear_grads(dy, x, w, "gelu", z), got):
        R.check(g, want, R._final(want, e, b.dtype) if g.dim() == 1 else e, "strided")
    assert got[3] is not None and torch.equal(got[3], dy)


# ---- layer norm --------------------------------------------------------------------------------
WIDTHS = [(1, 1), (1, 320), (5, 8), (7, 24), (300, 40), (33, 129), (10, 256), (320, 320), (64, 513), (50, 640), (9, 1027),
          (6, 2048), (5, 2056), (4, 5001), (3, 8192), (2, 8200), (2, 20001), (3000, 64)]


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("m,c", WIDTHS)
def test_layer_norm(ops, dt, m, c):
    x = rn(m, c, dt=dt) * 2 + rn(m, 1, dt=dt, seed=1) * 4
    w, b, dy = rn(c, dt=dt) * 0.1 + 1, rn(c, dt=dt, seed=2), rn(m, c, dt=dt, seed=3)
    for wt, bt, eps in ((w, b, 1e-5), (w.float(), b.float(), 1e-3), (None, None, 1e-5), (w, None, 1e-5)):
        y, mean, rstd = ops.layer_norm(x, wt, bt, eps=eps, return_stats=True)
        want, e = R.layer_norm(x, wt, bt, eps)
        R.check(y, want, e, "y")
        assert torch.equal(y, ops.layer_norm(x, wt, bt, eps=eps))
        grads = ops.layer_norm_backward(dy, x, wt, mean, rstd)
        again = ops.layer_norm_backward(dy, x, wt, mean, rstd)
        for (want, e), g, a, name in zip(R.layer_norm_grads(dy, x, wt, eps), grads, again, ("dx", "dw", "db")):
            R.check(g, want, e if name == "dx" else R._final(want, e, g.dtype), name)
            assert torch.equal(g, a)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("c", [24, 320, 1027, 2049])
def test_layer_norm_strided(ops, dt, c):
    x, w, b, dy = rn(40, c, dt=dt), rn(c, dt=dt), rn(c, dt=dt, seed=1), rn(40, c, dt=dt, seed=2)
    y, mean, rstd = ops.layer_norm(strided(x), w, b, return_stats=True)
    want, e = R.layer_norm(x, w, b, 1e-5)
    R.check(y, want, e, "y")
    for (want, e), g in zip(R.layer_norm_grads(dy, x, w, 1e-5), ops.layer_norm_backward(strided(dy), strided(x), w, mean, rstd)):
        R.check(g, want, R._final(want, e, g.dtype) if g.dim() == 1 else e, "grads")


def test_layer_norm_of_large_offsets(ops):
    """A row's offset costs the digits of its mean, not the square's: 1000 + noise keeps a unit norm."""
    x = rn(64, 500) + 1000.0
    y = ops.layer_norm(x)
    want, e = R.layer_norm(x, None, None, 1e-5)
    R.check(y, want, e, "y")
    assert abs(float(y.double().var(1, correction=0).mean()) - 1) < 1e-3


# ---- attention ------------------------------------------------------------------------------------
def run_attention(ops, dt, b, nq, nk, h, hk, dd, causal=False, lengths=None, q_lengths=None, scale=None, grads=True,
                  poison=True, wrap=lambda t: t):
    q, k, v, do = (rn(b, n, hh, dd, dt=dt, seed=s) for n, hh, s in ((nq, h, 1), (nk, hk, 2), (nk, hk, 3), (nq, h, 4)))
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda")
    qn = None if q_lengths is None else torch.tensor(q_lengths, dtype=torch.int32, device="cuda")
    ref = R.attention(q, k, v, scale, causal, lengths, q_lengths, do if grads else None)
    if poison:  # what lies behind the lengths is never read
        for t, lens in ((k, lengths), (v, lengths), (q, q_lengths), (do, q_lengths)):
            for i, n in enumerate(lens or []):
                t[i, max(n, 0):] = float("nan") if i % 2 else float("inf")
    kw = dict(scale=scale, causal=causal, lengths=ln, q_lengths=qn)
    q, k, v, do = wrap(q), wrap(k), wrap(v), wrap(do)
    o, lse = ops.attention(q, k, v, return_lse=True, **kw)
    R.check(o, *ref["o"], "o")
    R.check(lse, *ref["lse"], "lse")
    assert torch.equal(o, ops.attention(q, k, v, **kw))
    if grads:
        got = ops.attention_backward(do, q, k, v, o, lse, **kw)
        again = ops.attention_backward(do, q, k, v, o, lse, **kw)
        for name, g, a in zip(("dq", "dk", "dv"), got, again):
            R.check(g, *ref[name], name)
            assert torch.equal(g, a)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("b,nq,nk,h,hk,dd", [
    (1, 1, 1, 1, 1, 1), (2, 1, 7, 2, 1, 8), (1, 5, 3, 1, 1, 24), (2, 33, 65, 4, 2, 40), (1, 64, 64, 2, 2, 64),
    (2, 130, 129, 3, 1, 72), (1, 200, 77, 2, 2, 96), (1, 65, 200, 2, 1, 100), (1, 97, 128, 2, 2, 128), (3, 320, 320, 8, 8, 40),
    (1, 300, 260, 4, 4, 3), (2, 40, 1000, 2, 1, 33)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention(ops, dt, b, nq, nk, h, hk, dd, causal):
    run_attention(ops, dt, b, nq, nk, h, hk, dd, causal)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dd", [16, 64, 128])
def test_attention_ragged(ops, dt, causal, dd):
    """Padded batches with lengths of zero and one, poison behind them; queries that see nothing."""
    run_attention(ops, dt, 5, 90, 90, 4, 2, dd, causal, lengths=[90, 0, 1, 64, 33], q_lengths=[90, 0, 1, 64, 33])
    run_attention(ops, dt, 4, 70, 150, 2, 2, dd, causal, lengths=[150, 20, 0, 65])
    run_attention(ops, dt, 3, 70, 40, 2, 1, dd, causal, q_lengths=[70, 3, 0])
    run_attention(ops, dt, 3, 9, 40, 2, 1, dd, causal, lengths=[-5, 1000, 40], q_lengths=[9, 100, -1], poison=False)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("h,hk,dd,nq", [(8, 8, 64, 1), (16, 4, 64, 1), (8, 1, 128, 1), (4, 4, 80, 3), (6, 2, 24, 5), (32, 2, 96, 2)])
def test_attention_of_one_token(ops, dt, h, hk, dd, nq):
    """Few queries against a long cache: the keys are split over workgroups and joined."""
    run_attention(ops, dt, 3, nq, 3001, h, hk, dd, True, lengths=[3001, 1, 1777], grads=False)
    run_attention(ops, dt, 1, nq, 5000, h, hk, dd, False, grads=False)


@pytest.mark.parametrize("dt", DT)
def test_attention_strides_and_scale(ops, dt):
    # heads before tokens, unaligned rows, heads sliced from one qkv tensor
    run_attention(ops, dt, 2, 70, 90, 4, 2, 40, wrap=lambda t: t.transpose(1, 2).contiguous().transpose(1, 2))
    run_attention(ops, dt, 2, 70, 90, 4, 2, 40, True, wrap=strided)
    run_attention(ops, dt, 1, 2, 900, 4, 2, 64, scale=0.7, wrap=strided)
    q = rn(2, 50, 3 * 4 * 32, dt=dt).view(2, 50, 3, 4, 32)
    ref = R.attention(q[:, :, 0], q[:, :, 1], q[:, :, 2])
    R.check(ops.attention(q[:, :, 0], q[:, :, 1], q[:, :, 2]), *ref["o"], "qkv")
    # one cache shared by the batch
    k = rn(1, 60, 2, 32, dt=dt)
    qq = rn(3, 60, 2, 32, dt=dt, seed=5)
    ref = R.attention(qq, k.expand(3, -1, -1, -1), k.expand(3, -1, -1, -1))
    R.check(ops.attention(qq, k.expand(3, -1, -1, -1), k.expand(3, -1, -1, -1)), *ref["o"], "shared")


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_attention_extreme_scores(ops, dt):
    """Scores of hundreds: the running maximum keeps P finite, rows that one key wins stay exact."""
    q, k, v = rn(1, 100, 2, 64, dt=dt) * 20, rn(1, 300, 2, 64, dt=dt) * 5, rn(1, 300, 2, 64, dt=dt)
    ref = R.attention(q, k, v)
    o, lse = ops.attention(q, k, v, return_lse=True)
    R.check(o, *ref["o"], "o")
    R.check(lse, *ref["lse"], "lse")


def test_attention_offsets_beyond_32_bits(ops):
    """A cache whose rows lie more than 2^31 elements apart."""
    nk, dd = 130, 64
    step = 2 ** 31 // 64 + 8
    big = torch.empty(nk * step + dd, dtype=torch.float16, device="cuda")
    k = big.as_strided((1, nk, 1, dd), (0, step, dd, 1))
    kk = rn(1, nk, 1, dd, dt="fp16")
    k.copy_(kk)
    q = rn(1, 80, 1, dd, dt="fp16", seed=1)
    ref = R.attention(q, kk, kk)
    R.check(ops.attention(q, k, k), *ref["o"], "o")
    R.check(ops.attention(q[:, :1], k, k), *R.attention(q[:, :1], kk, kk)["o"], "token")


# ---- gradients against differences -----------------------------------------------------------------
def directional(f, args, dirs, dy, h=1e-5):
    """(f(x + h e) - f(x - h e)) . dy / 2h in float64."""
    up = f(*[a.double() + h * e for a, e in zip(args, dirs)])
    dn = f(*[a.double() - h * e for a, e in zip(args, dirs)])
    return float(((up - dn) * dy.double()).sum() / (2 * h))


def agree(grads, bounds, dirs, diff):
    got = sum(float((g.double() * e).sum()) for g, e in zip(grads, dirs))
    slack = sum(float((b * e.abs()).sum()) for b, e in zip(bounds, dirs))
    # the difference's own error: h^2 and the cancellation of float64, far below 1e-6 of the terms
    scale = sum(float((g.double() * e).abs().sum()) for g, e in zip(grads, dirs))
    assert abs(got - diff) <= slack + 1e-6 * scale + 1e-9, (got, diff, slack)


def test_gradients_against_differences(ops):
    x, w, b, dy = rn(20, 30), rn(12, 30, std=0.2), rn(12), rn(20, 12, seed=1)
    e = [rn(*t.shape, seed=7).double() for t in (x, w, b)]
    for act in ("gelu", "silu", "none"):
        _, z = ops.linear(x, w, b, act=act, return_preact=True)
        g = ops.linear_backward(dy, x, w, b, act=act, preact=z)[:3]
        want = R.linear_grads(dy, x, w, act, z)
        diff = directional(lambda x, w, b: R.act64(x @ w.t() + b, act), (x, w, b), e, dy)
        # z was rounded to float32: act'' is below 1
        slack = [2 * bd + 1e-6 * v.abs().max() for v, bd in want]
        agree(g, slack, e, diff)
    y, mean, rstd = ops.layer_norm(x, w[0], w[1], return_stats=True)
    g = ops.layer_norm_backward(x.flip(0).contiguous(), x, w[0], mean, rstd)
    e = [rn(20, 30, seed=8).double(), rn(30, seed=9).double(), rn(30, seed=10).double()]

    def norm(x, w, b):
        c = x - x.mean(1, keepdim=True)
        return c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt() * w + b

    diff = directional(norm, (x, w[0], w[1]), e, x.flip(0))
    agree(g, [bd for _, bd in R.layer_norm_grads(x.flip(0), x, w[0], 1e-5)], e, diff)
    q, k, v, do = (rn(1, n, 2, 16, seed=s) for n, s in ((9, 1), (13, 2), (13, 3), (9, 4)))
    e = [rn(*t.shape, seed=11).double() for t in (q, k, v)]
    for causal in (False, True):
        o, lse = ops.attention(q, k, v, causal=causal, return_lse=True)
        g = ops.attention_backward(do, q, k, v, o, lse, causal=causal)

        def att(q, k, v):
            s = torch.einsum("bihd,bjhd->bhij", q, k) / 4
            if causal:
                s = s.masked_fill(torch.ones(9, 13, dtype=torch.bool, device="cuda").triu(5), -math.inf)
            return torch.einsum("bhij,bjhd->bihd", torch.softmax(s, 3), v)

        ref = R.attention(q, k, v, None, causal, do=do)
        agree(g, [ref[n][1] for n in ("dq", "dk", "dv")], e, directional(att, (q, k, v), e, do))


# ---- refusals, empty inputs -------------------------------------------------------------------------
def test_refusals(ops):
    x, w = rn(4, 8), rn(6, 8)
    bad = [lambda: ops.linear(x, rn(6, 7)), lambda: ops.linear(x, w.half()), lambda: ops.linear(x, w, rn(5)),
           lambda: ops.linear(x, w, act="tanh"), lambda: ops.linear(x, w, residual=rn(5, 6)),
           lambda: ops.linear(x, w, residual=rn(4, 5)), lambda: ops.linear(x.t(), rn(6, 4)),
           lambda: ops.linear(x.double(), w.double()), lambda: ops.linear(x, rn(2, 3, 8)), lambda: ops.linear(x, w, w[0].half()),
           lambda: ops.linear(x.view(2, 2, 8).transpose(0, 1)[:, :, :], w), lambda: ops.linear(rn(4, 8)[:, :0], w[:, :0]),
           lambda: ops.linear(x, w.requires_grad_()), lambda: ops.linear_backward(rn(4, 6), x, w.detach(), act="gelu"),
           lambda: ops.linear_backward(rn(3, 6), x, w.detach()), lambda: ops.layer_norm(x, rn(7)),
           lambda: ops.layer_norm(x, rn(8), rn(8).half()), lambda: ops.layer_norm(x, eps=-1.0),
           lambda: ops.layer_norm_backward(x, x, None, rn(3), rn(4)), lambda: ops.layer_norm_backward(x[:3], x, None, rn(4), rn(4))]
    q, k = rn(2, 5, 4, 16), rn(2, 7, 2, 16)
    ln = torch.tensor([1, 2], device="cuda")
    bad += [lambda: ops.attention(q, rn(2, 7, 3, 16), rn(2, 7, 3, 16)), lambda: ops.attention(q, k, rn(2, 6, 2, 16)),
            lambda: ops.attention(rn(1, 5, 2, 136), rn(1, 5, 2, 136), rn(1, 5, 2, 136)),
            lambda: ops.attention(q, k, k, scale=0.0), lambda: ops.attention(q, k, k, scale=math.inf),
            lambda: ops.attention(q, k, k, lengths=ln), lambda: ops.attention(q, k, k, lengths=ln[:1].int()),
            lambda: ops.attention(q, k, k, lengths=ln.int().cpu()), lambda: ops.attention(q[0], k, k),
            lambda: ops.attention(q.transpose(2, 3), k, k), lambda: ops.attention(q, k.half(), k),
            lambda: ops.attention_backward(q, q, k, k, q, rn(2, 5, 4)), lambda: ops.attention_backward(q[:1], q, k, k, q, rn(2, 4, 5))]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was not refused")
    with pytest.raises(pkg().YKError):
        ops.linear(x.cpu(), w.detach().cpu())
    with torch.no_grad():
        ops.linear(x, w)


def test_empty_inputs(ops):
    x, w, b = rn(0, 8), rn(6, 8), rn(6)
    assert ops.linear(x, w, b, act="gelu", residual=rn(0, 6)).shape == (0, 6)
    g = ops.linear_backward(rn(0, 6), x, w, b)
    assert g[0].shape == (0, 8) and not g[1].any() and not g[2].any()
    y, mean, rstd = ops.layer_norm(x, return_stats=True)
    assert y.shape == (0, 8) and mean.shape == (0,)
    g = ops.layer_norm_backward(x, x, w[0].contiguous(), mean, rstd)
    assert g[0].shape == (0, 8) and not g[1].any() and not g[2].any()
    for nq, nk in ((3, 0), (0, 3), (40, 0)):
        q, k = rn(2, nq, 2, 16), rn(2, nk, 2, 16)
        o, lse = ops.attention(q, k, k, return_lse=True)
        assert o.shape == q.shape and not o.any() and bool((lse == -math.inf).all())
        dq, dk, dv = ops.attention_backward(q, q, k, k, o, lse)
        assert not dq.any() and not dk.any() and not dv.any()


# ---- a run of them: a transformer layer's training step -----------------------------------------------
def layer_step(ops, p, x, gy, heads, lengths=None):
    """Post-norm transformer layer over [B, T, C]: attention, its projection with the residual in the
    epilogue, norm, GELU feed-forward, norm; then every gradient."""
    b, t, c = x.shape
    kw = dict(lengths=lengths, q_lengths=lengths)
    qkv = ops.linear(x, p["wqkv"], p["bqkv"], residual=p["pos"])
    q, k, v = (s.unflatten(-1, (heads, c // heads)) for s in qkv.chunk(3, -1))
    o, lse = ops.attention(q, k, v, return_lse=True, **kw)
    h1 = ops.linear(o.flatten(2), p["wo"], p["bo"], residual=x)
    n1, m1, r1 = ops.layer_norm(h1, p["g1"], p["s1"], return_stats=True)
    a, z = ops.linear(n1, p["w1"], p["b1"], act="gelu", return_preact=True)
    h2 = ops.linear(a, p["w2"], p["b2"], residual=n1)
    y, m2, r2 = ops.layer_norm(h2, p["g2"], p["s2"], return_stats=True)
    dh2, dg2, ds2 = ops.layer_norm_backward(gy, h2, p["g2"], m2, r2)
    da, dw2, db2, _ = ops.linear_backward(dh2, a, p["w2"], p["b2"])
    dn1, dw1, db1, _ = ops.linear_backward(da, n1, p["w1"], p["b1"], act="gelu", preact=z)
    dh1, dg1, ds1 = ops.layer_norm_backward(dn1 + dh2, h1, p["g1"], m1, r1)
    do, dwo, dbo, _ = ops.linear_backward(dh1, o.flatten(2), p["wo"], p["bo"])
    dq, dk, dv = ops.attention_backward(do.view_as(o), q, k, v, o, lse, **kw)
    dqkv = torch.cat([dq.flatten(2), dk.flatten(2), dv.flatten(2)], -1)
    dx, dwqkv, dbqkv, dpos = ops.linear_backward(dqkv, x, p["wqkv"], p["bqkv"], residual=p["pos"])
    return {"y": y, "x": dx + dh1, "wqkv": dwqkv, "bqkv": dbqkv, "pos": dpos, "wo": dwo, "bo": dbo, "w1": dw1, "b1": db1,
            "w2": dw2, "b2": db2, "g1": dg1, "s1": ds1, "g2": dg2, "s2": ds2}


def layer_inputs(dt, b=2, t=75, c=48, f=80):
    p = {"wqkv": rn(3 * c, c, dt=dt, std=c ** -0.5), "bqkv": rn(3 * c, dt=dt, std=0.1), "pos": rn(t, 3 * c, dt=dt, std=0.3),
         "wo": rn(c, c, dt=dt, std=c ** -0.5), "bo": rn(c, dt=dt, std=0.1), "w1": rn(f, c, dt=dt, std=c ** -0.5),
         "b1": rn(f, dt=dt, std=0.1), "w2": rn(c, f, dt=dt, std=f ** -0.5), "b2": rn(c, dt=dt, std=0.1, seed=1)}
    for n in ("1", "2"):
        p["g" + n], p["s" + n] = rn(c, dt=dt, std=0.1, seed=2) + 1, rn(c, dt=dt, std=0.1, seed=3)
    return p, rn(b, t, c, dt=dt), rn(b, t, c, dt=dt, seed=4)


def layer_autograd(p, x, gy, heads):
    """The same layer in float64 torch operations on the CPU, differentiated by autograd."""
    p = {n: t.double().cpu().requires_grad_() for n, t in p.items()}
    x = x.double().cpu().requires_grad_()
    b, t, c = x.shape

    def norm(v, g, s):
        u = v - v.mean(-1, keepdim=True)
        return u / (u.square().mean(-1, keepdim=True) + 1e-5).sqrt() * g + s

    qkv = x @ p["wqkv"].t() + p["bqkv"] + p["pos"]
    q, k, v = (s.reshape(b, t, heads, c // heads).transpose(1, 2) for s in qkv.chunk(3, -1))
    o = torch.softmax(q @ k.transpose(2, 3) / math.sqrt(c // heads), -1) @ v
    h1 = o.transpose(1, 2).reshape(b, t, c) @ p["wo"].t() + p["bo"] + x
    n1 = norm(h1, p["g1"], p["s1"])
    h2 = R.act64(n1 @ p["w1"].t() + p["b1"], "gelu") @ p["w2"].t() + p["b2"] + n1
    y = norm(h2, p["g2"], p["s2"])
    y.backward(gy.double().cpu())
    return {"y": y.detach(), "x": x.grad, **{n: t.grad for n, t in p.items()}}


@pytest.mark.parametrize("dt", DT)
def test_transformer_layer_step(ops, dt):
    """Forward and every gradient of a layer against float64 autograd.  A value passes some 12
    roundings on its way (each at most u relative to the terms it is summed from); terms are of the
    size of their tensor's root mean square, so 12 u of it, times 8 for the largest of the elements
    and the norms' division, bounds the elements; float32 has sums of up to 240 terms in place of the
    roundings of operands."""
    p, x, gy = layer_inputs(dt)
    got, want = layer_step(ops, p, x, gy, 4), layer_autograd(p, x, gy, 4)
    u = R.half_step(DT[dt]) if dt != "fp32" else 16 * R.F
    for n in want:
        rms = float(want[n].square().mean().sqrt())
        err = float((got[n].double().cpu().reshape(want[n].shape) - want[n]).abs().max())
        assert err <= 12 * 8 * u * rms, (n, err / (u * rms))


def test_layer_step_captured(ops):
    """The step captured into a graph, replayed with eager work and other inputs in between, equals
    the eager step bit for bit; two graphs hold scratch of their own."""
    p, x, gy = layer_inputs("bf16")
    ln = torch.tensor([75, 40], dtype=torch.int32, device="cuda")
    eager = layer_step(ops, p, x, gy, 4, ln)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        layer_step(ops, p, x, gy, 4, ln)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = layer_step(ops, p, x, gy, 4, ln)
        graphs.append((g, out))
    keep = x.clone()
    for i in range(4):
        x.copy_(keep * (1 + i))
        want = layer_step(ops, p, x, gy, 4, ln)
        for g, _ in graphs:
            g.replay()
        if i % 2:
            layer_step(ops, p, keep, gy, 4, ln)
            torch.cuda.synchronize()
        for _, out in graphs:
            for n in want:
                assert torch.equal(out[n], want[n]), (i, n)
    x.copy_(keep)
    graphs[0][0].replay()
    for n in eager:
        assert torch.equal(graphs[0][1][n], eager[n]), n


def test_calls_on_two_streams(ops):
    """Calls in flight on two streams at once use scratch of their own."""
    x, w, dy = rn(300, 2048, dt="bf16"), rn(72, 2048, dt="bf16", std=0.02), rn(300, 72, dt="bf16")
    q, k = rn(2, 1, 8, 64, dt="bf16"), rn(2, 4000, 8, 64, dt="bf16")
    want = [ops.linear(x, w), ops.attention(q, k, k), *ops.linear_backward(dy, x, w)[:2]]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append([ops.linear(x, w), ops.attention(q, k, k), *ops.linear_backward(dy, x, w)[:2]])
    torch.cuda.synchronize()
    for o in outs:
        for a, b in zip(o, want):
            assert torch.equal(a, b)


def test_linear_fp32_of_infinite_and_huge_values(ops):
    """float32 products run as sums of bf16 parts, which cannot hold infinity nor what rounds to it:
    sums they break are taken again, so infinities, NaN and values next to the largest come out as
    the plain product's, in every direction and split."""
    big = 3.4e38
    for m, k, n in ((70, 96, 80), (300, 1500, 40)):
        x, w, dy = rn(m, k), rn(n, k, std=k ** -0.5), rn(m, n, seed=1)
        x[1, 2], x[2, 3], x[3, 4], x[5, 0], w[6, 7] = math.inf, -math.inf, math.nan, big, math.inf
        w[8, 0], w[9, 9] = 2.0 ** -20, 0.0
        x[10, 9] = math.inf  # times zero
        want = x.double() @ w.double().t()
        y = ops.linear(x, w)
        fits = torch.where(want.abs() > torch.finfo(torch.float32).max, want.sign() * math.inf, want)
        R.check(y, fits, (k + 8) * R.F * (x.double().abs() @ w.double().abs().t()).nan_to_num(posinf=0) * 2 + R.TINY, "y")
        dx, dw, _, _ = ops.linear_backward(dy, x, w)
        for got, a, b in ((dx, dy, w), (dw, dy.t(), x)):
            g = a.double() @ b.double()
            mag = (a.double().abs() @ b.double().abs()).nan_to_num(posinf=0)
            R.check(got, torch.where(g.abs() > torch.finfo(torch.float32).max, g.sign() * math.inf, g), (m + n + 8) * R.F * mag * 2 + R.TINY,
                    "gradient")


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_few_keys_many_rows(ops, dt, causal):
    """Few key blocks against many rows: the rows are split and their sums of dk and dv joined."""
    run_attention(ops, dt, 2, 700, 30, 6, 2, 40, causal)
    run_attention(ops, dt, 3, 333, 333, 6, 2, 24, causal, lengths=[333, 0, 170], q_lengths=[333, 0, 170])
    run_attention(ops, dt, 1, 600, 100, 3, 3, 96, causal, lengths=[70])


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("m,k,n", [(100, 9000, 24), (16000, 100, 100), (70, 4000, 1000)])
def test_linear_split_products(ops, dt, m, k, n):
    """Products whose K is split: the join's lanes and orders, forward and backward."""
    x, w, b, dy = rn(m, k, dt=dt), rn(n, k, dt=dt, std=k ** -0.5), rn(n, dt=dt), rn(m, n, dt=dt, seed=1)
    y, z = ops.linear(x, w, b, act="silu", return_preact=True)
    want, ey, wz, ez = R.linear(x, w, b, "silu", None)
    R.check(y, want, ey, "y")
    R.check(z, wz, ez, "z")
    assert torch.equal(y, ops.linear(x, w, b, act="silu"))
    got = ops.linear_backward(dy, x, w, b, act="silu", preact=z)
    again = ops.linear_backward(dy, x, w, b, act="silu", preact=z)
    for (want, e), g, a in zip(R.linear_grads(dy, x, w, "silu", z), got, again):
        R.check(g, want, R._final(want, e, g.dtype) if g.dim() == 1 else e, "grads")
        assert torch.equal(g, a)


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_few_rows_many_keys_backward(ops, dt, causal):
    """A token or a few against many keys, trained: the keys are split and their sums of dq joined."""
    run_attention(ops, dt, 2, 1, 1500, 4, 2, 80, causal)
    run_attention(ops, dt, 3, 5, 700, 2, 1, 24, causal, lengths=[700, 0, 129], q_lengths=[5, 2, 0])
    run_attention(ops, dt, 1, 40, 900, 2, 2, 128, causal, lengths=[333])


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("act", ["none", "gelu", "silu", "relu"])
@pytest.mark.parametrize("m,k,n", [(4136, 64, 4096), (2560, 72, 1032)])
def test_linear_whole_and_partial_tiles(ops, dt, act, m, k, n):
    """Products of many tiles, most of them whole: the epilogue with and without a residual of
    fewer rows, and their gradients."""
    x, w, b, res = rn(m, k, dt=dt), rn(n, k, dt=dt, std=k ** -0.5), rn(n, dt=dt), rn(77, n, dt=dt, seed=2)
    for bias, r in ((b, res), (None, None)):
        y, z = ops.linear(x, w, bias, act=act, residual=r, return_preact=True)
        want, ey, wz, ez = R.linear(x, w, bias, act, r)
        R.check(y, want, ey, f"y {act}")
        R.check(z, wz, ez, f"z {act}")
        assert torch.equal(y, ops.linear(x, w, bias, act=act, residual=r))
    dy = rn(m, n, dt=dt, seed=3)
    for (want, e), g, name in zip(R.linear_grads(dy, x, w, act, z), ops.linear_backward(dy, x, w, b, act=act, preact=z), ("dx", "dw", "db")):
        R.check(g, want, R._final(want, e, b.dtype) if name == "db" else e, f"{name} {act}")


@pytest.mark.parametrize("dt", DT)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("b,nq,nk,h,hk,dd", [(2, 100, 2300, 4, 2, 72), (1, 150, 2111, 2, 2, 33), (2, 300, 3100, 1, 1, 128)])
def test_attention_row_blocks_with_split_keys(ops, dt, causal, b, nq, nk, h, hk, dd):
    """Too few row blocks to fill the chip: their keys in ranges, joined."""
    run_attention(ops, dt, b, nq, nk, h, hk, dd, causal)
    run_attention(ops, dt, b, nq, nk, h, hk, dd, causal, lengths=[nk - 5, 70][:b], q_lengths=[nq - 1, nq][:b])
