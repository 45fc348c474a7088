"""Which kernels a token operator's call launches (yk_token_kernels, include/yk_diag.h), and calls whose
sizes reach kernels that only large ones take.  Nothing runs."""
import ctypes as C

from conftest import pkg

DTYPE = {"bf16": 0, "fp32": 1, "fp16": 3}
TRAIT = {"bf16": "B16", "fp32": "F32", "fp16": "H16"}
PTR = 64  # an address that is 16-byte aligned and never followed
ROOM = dict(ws=PTR, ws_bytes=1 << 50)


def kernels(fn, dt, **args):
    """Names of the kernels of a call, without their namespace."""
    L = pkg()._lib
    a = L.TOKEN_ARGS[fn](dtype=DTYPE[dt], **args)
    f, buf = L.lib().yk_token_kernels, C.create_string_buffer(4096)
    f.argtypes = [C.c_int, C.c_void_p, C.c_char_p, C.c_int]
    L.check(f(12 + list(L.TOKEN_ARGS).index(fn), C.addressof(a), buf, len(buf)), fn)
    return [n.replace("yk::tok::", "") for n in buf.value.decode().split("\n")[:-1]]


def linear_kernels(dt, m, k, n, **kw):
    return kernels("yk_linear", dt, m=m, n=n, k=k, x=PTR, w=PTR, y=PTR, x_stride=k, w_stride=k, y_stride=n, **{**ROOM, **kw})


def linear_grad_kernels(dt, m, k, n, **kw):
    """dx and dw alone, one list each."""
    a = dict(m=m, n=n, k=k, dy=PTR, x=PTR, w=PTR, dy_stride=n, x_stride=k, w_stride=k, dx_stride=k, dw_stride=k, **{**ROOM, **kw})
    return kernels("yk_linear_backward", dt, dx=PTR, **a), kernels("yk_linear_backward", dt, dw=PTR, **a)


def norm_kernels(dt, m, c):
    a = dict(m=m, c=c, x=PTR, x_stride=c)
    return (kernels("yk_layer_norm", dt, y=PTR, y_stride=c, **a),
            kernels("yk_layer_norm_backward", dt, dy=PTR, mean=PTR, rstd=PTR, dx=PTR, dw=PTR, dy_stride=c, dx_stride=c, **a, **ROOM))


def attention_kernels(dt, b, nq, nk, h, hk, d, causal=False):
    """(forward, backward) of contiguous tensors."""
    s3, q, k = C.c_int64 * 3, (nq * h * d, h * d, d), (nk * hk * d, hk * d, d)
    a = dict(causal=int(causal), b=b, h_q=h, h_kv=hk, d=d, nq=nq, nk=nk, scale=1.0, q=PTR, k=PTR, v=PTR, o=PTR, lse=PTR, q_stride=s3(*q),
             k_stride=s3(*k), v_stride=s3(*k), o_stride=s3(*q), **ROOM)
    return kernels("yk_attention", dt, **a), kernels("yk_attention_backward", dt, go=PTR, dq=PTR, dk=PTR, dv=PTR, go_stride=s3(*q),
                                                     dq_stride=s3(*q), dk_stride=s3(*k), dv_stride=s3(*k), **a)


# Products (m, k, n) by the tile that one of their three takes: forward "ff", dx "ft" and dw "tt" (which
# operands lie transposed), the tile, "a" with rows aligned for loads straight to LDS, "+" with K split.
PRODUCTS_16 = [("ff256a", 2104, 264, 4200), ("ff256a+", 136, 16392, 4104), ("ff128a", 2104, 136, 2072), ("ff128a+", 1080, 4104, 1048),
               ("ft128a", 2104, 2072, 136), ("ft128a+", 1080, 1048, 4104), ("ft256a+", 2104, 2072, 8200), ("tt128a", 136, 2104, 2072),
               ("tt128a+", 4184, 1032, 2056), ("tt256a+", 4104, 2104, 2072), ("ff128", 2101, 137, 2077), ("ft128", 2101, 2077, 137),
               ("tt128", 137, 2101, 2077), ("ff128+", 1033, 4105, 1051), ("ft128+", 1033, 1051, 4105), ("tt128+", 4105, 1033, 2101)]
PRODUCTS_32 = [("ff128", 2101, 136, 2072), ("ff128+", 1033, 1048, 1051), ("ft128", 2104, 2077, 136), ("ft128+", 1033, 1048, 1051),
               ("tt128", 136, 2101, 2072), ("tt128+", 1033, 1048, 1051)]
PRODUCTS = [(dt, *p) for dt, ps in (("bf16", PRODUCTS_16), ("fp16", PRODUCTS_16), ("fp32", PRODUCTS_32)) for p in ps]


def product_form(dt, names):
    """The same shorthand of a product's kernels."""
    head, args = names[0].rstrip(">").split("<")
    args = args.split(", ")
    if dt == "fp32":
        assert head == "gemm_f32_kernel"
        form = args[0][0] + args[1][0] + args[2]
    else:
        assert head == "gemm_kernel" and args[0] == TRAIT[dt]
        form = args[1][0] + args[2][0] + args[3] + ("a" if args[-1] == "true" else "")
    return form + ("+" if len(names) > 1 and names[1].startswith("split_sum_kernel") else "")


# Rows of 16 lanes, which take many rows: widths by their chunks per lane (forward 1 to 8, backward 1 and 2)
NORM_ROWS = 8203
NORM_WIDTHS = {"bf16": [24, 129, 200, 256, 257, 390, 640, 703, 777, 1023], "fp16": [100, 160, 255, 384, 450, 513, 700, 770, 1000],
               "fp32": [65, 100, 128, 130, 200, 257, 320, 350, 390, 511]}

# Two tiles a wave: batch, tokens, heads, key heads, head size
TWO_TILES = [(8, 515, 8, 8, 40), (8, 515, 8, 8, 64), (9, 500, 16, 8, 96), (8, 515, 8, 8, 128), (16, 600, 4, 4, 24)]
