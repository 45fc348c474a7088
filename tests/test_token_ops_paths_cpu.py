"""What the token operators refuse, where that shows without a GPU."""
import ctypes as C

import pytest
import torch
from torch.autograd import forward_ad

import token_kernels as K
from conftest import pkg

L = pkg()._lib
CTX = C.create_string_buffer(64)  # never read: every call here is refused


def test_forward_mode_tangents_are_refused():
    like = pkg().ops._like
    t = torch.zeros(3)
    with forward_ad.dual_level():
        like(t, "t", -1, torch.float32)
        like(t.int(), "t", -1, torch.int32)
        with pytest.raises(ValueError, match="tangent"):
            like(forward_ad.make_dual(t, t), "t", -1, torch.float32)


def test_tracing_is_refused():
    ops, x = pkg().ops, torch.zeros(4, 8)
    for f in (lambda t: ops.linear(t, t), lambda t: ops.layer_norm(t)):
        with pytest.raises(pkg().YKError, match="jit.trace"):
            torch.jit.trace(f, (x,))


@pytest.mark.parametrize("fn,args", [
    ("yk_linear", dict(dtype=0, m=1 << 28, n=1 << 13, k=8, x=64, w=64, y=64, x_stride=8, w_stride=8, y_stride=1 << 13)),
    ("yk_linear_backward", dict(dtype=0, m=1 << 28, n=8, k=1 << 13, dy=64, x=64, w=64, dx=64, dy_stride=8, x_stride=1 << 13,
                                w_stride=1 << 13, dx_stride=1 << 13, ws=64, ws_bytes=1 << 50)),
    ("yk_attention", dict(dtype=0, b=1 << 24, h_q=1, h_kv=1, d=8, nq=1, nk=9, scale=1.0, q=64, k=64, v=64, o=64)),
    ("yk_attention", dict(dtype=1, b=1 << 20, h_q=2, h_kv=2, d=8, nq=513, nk=9, scale=1.0, q=64, k=64, v=64, o=64)),
    ("yk_attention_backward", dict(dtype=0, b=1 << 20, h_q=2, h_kv=2, d=8, nq=129, nk=9, scale=1.0, q=64, k=64, v=64, o=64, go=64,
                                   lse=64, dq=64, dk=64, dv=64, ws=64, ws_bytes=1 << 50)),
    ("yk_attention_backward", dict(dtype=0, b=1 << 20, h_q=2, h_kv=2, d=8, nq=1, nk=513, scale=1.0, q=64, k=64, v=64, o=64, go=64,
                                   lse=64, dq=64, dk=64, dv=64, ws=64, ws_bytes=1 << 50)),
])
def test_more_workgroups_than_a_launch_holds(fn, args):
    """A launch holds fewer than 2^32 threads: refused with nothing launched."""
    a = L.TOKEN_ARGS[fn](**args)
    assert getattr(L.lib(), fn)(C.addressof(CTX), C.byref(a), None) == L.YK_ERR_ARG
    assert b"than a launch holds" in L.lib().yk_last_error()


# ---- the sizes of test_token_ops_paths_gpu.py reach the kernels that they are there for --------------
@pytest.mark.parametrize("dt,form,m,k,n", K.PRODUCTS)
def test_sizes_reach_the_products_of_large_tiles(dt, form, m, k, n):
    names = {"ff": K.linear_kernels(dt, m, k, n), **dict(zip(("ft", "tt"), K.linear_grad_kernels(dt, m, k, n)))}
    assert K.product_form(dt, names[form[:2]]) == form


@pytest.mark.parametrize("dt", K.NORM_WIDTHS)
def test_sizes_reach_every_norm_of_16_lanes(dt):
    t, got = K.TRAIT[dt], set()
    for c in K.NORM_WIDTHS[dt]:
        fwd, bwd = K.norm_kernels(dt, K.NORM_ROWS, c)
        got |= {fwd[0], bwd[0]}
    assert {f"norm_kernel<{t}, 16, {i}>" for i in range(2, 9)} | {f"norm_grad_kernel<{t}, 16, 2>"} <= got


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("b,n,h,hk,d", K.TWO_TILES)
def test_sizes_reach_two_tiles_a_wave(dt, b, n, h, hk, d):
    t, dp = K.TRAIT[dt], (d + 31) // 32 * 32
    fwd, bwd = K.attention_kernels(dt, b, n, n, h, hk, d)
    assert fwd == [f"attn_kernel<{t}, {dp}, 2, true>"]
    assert f"attn_dq_kernel<{t}, {dp}, 2, true>" in bwd
    assert f"attn_dkv_kernel<{t}, {dp}, {2 if dp == 96 else 1}, true>" in bwd


def test_kernels_are_reported_for_good_arguments_only():
    with pytest.raises(pkg().YKError, match="activation"):
        K.kernels("yk_linear", "bf16", **{"m": 4, "n": 4, "k": 4, "act": 9})


@pytest.mark.parametrize("args", [[64, 8, 0, "nn.ReLU"], [64, 8, 0, "nn.GELU", True], [64, 0], [64, -8], [0, 8], [64.5, 8], ["64", 8]])
def test_aifi_arguments_that_change_the_layer_are_refused(args):
    """An activation or a norm order that the layer does not have, sizes that no layer has."""
    import importlib

    from aifi_helpers import aifi_dict

    d = aifi_dict("s")
    d["backbone"][10][3] = args
    parse = importlib.import_module(pkg().__name__ + ".arch").parse_arch
    with pytest.raises(ValueError, match="AIFI"):
        parse(d)
    d["backbone"][10][3] = [64, 8, 0.1]  # a dropout is of training only
    assert parse(d).layers[10].args == {"hidden": 64, "heads": 8}
