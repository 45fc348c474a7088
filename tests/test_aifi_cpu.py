"""AIFI rows of a model YAML: parsing, parameters, lowering to token ops, the engine-file checks."""
import importlib

import numpy as np
import pytest
import torch

from aifi_helpers import aifi_dict
from conftest import pkg

P = pkg()
A = importlib.import_module(P.__name__ + ".arch")
W = importlib.import_module(P.__name__ + ".weights")
M = importlib.import_module(P.__name__ + ".model")


def program(dtype="bf16", **kw):
    ar = A.parse_arch(aifi_dict(**kw))
    return M.Program(ar, W.synthetic_state_dict(ar, 0), 256, 320, 320, 2, dtype)


def test_parse():
    ar = A.parse_arch(aifi_dict("s", 1024, 8))
    L = ar.layers[10]
    assert (L.kind, L.c1, L.c2, L.args) == ("AIFI", 320, 320, {"hidden": 1024, "heads": 8})
    assert A.detect_strides(ar) == [4, 8, 16, 32] and ar.layers[-1].f == [19, 16, 22, 25]
    sd = W.synthetic_state_dict(ar, 0)
    for name, shape in A.encoder_specs(ar):
        assert tuple(sd[name].shape) == shape
    assert len(A.encoder_specs(ar)) == 12


@pytest.mark.parametrize("heads,n", [(7, 1), (1, 1), (8, 4)])
def test_refused_rows(heads, n):
    """320 channels: no 7 heads, no head of 320; several layers in a row."""
    d = aifi_dict("s", 64, heads)
    d["backbone"][10][1] = n
    with pytest.raises(ValueError, match="AIFI"):
        A.parse_arch(d)


def test_repeats_follow_the_depth_gain():
    """Two repeats at the s scale's depth of 0.67 are one layer, as for every other row."""
    d = aifi_dict("s")
    d["backbone"][10][1] = 2
    assert A.parse_arch(d).layers[10].kind == "AIFI"


def test_lowering():
    prog = program()
    kinds = [op.kind for op in prog.ops if op.kind >= M.YK_K_LINEAR]
    assert kinds == [M.YK_K_LINEAR, M.YK_K_ATTENTION, M.YK_K_LINEAR, M.YK_K_LAYER_NORM, M.YK_K_LINEAR, M.YK_K_LINEAR,
                     M.YK_K_LAYER_NORM]
    c, T = 192, 8 * 10
    lin = [(op, n) for op, n in zip(prog.ops, prog.op_flops(1)) if op.kind == M.YK_K_LINEAR]
    assert [n for _, n in lin] == [2 * T * a * b for a, b in ((3 * c, c), (c, c), (256, c), (c, 256))]
    # the first product's table: positions through the query and key weights, nothing for the values
    op = lin[0][0]
    tab = np.frombuffer(bytes(prog.blob[op.t_off:op.t_off + T * 3 * c * 2]), np.int16)
    tab = torch.from_numpy(tab.copy()).view(torch.bfloat16).float().view(T, 3 * c)
    w = prog.sd["model.10.ma.in_proj_weight"]
    want = torch.from_numpy(M.sincos_positions(8, 10, c)) @ w[:2 * c].t()
    assert torch.allclose(tab[:, :2 * c], want, rtol=2 ** -8, atol=1e-5) and not tab[:, 2 * c:].any()


def test_position_table():
    t = M.sincos_positions(3, 5, 8)
    assert t.shape == (15, 8)
    # row 7: column 2, row 1, frequencies 1 and 1 / 100
    want = [np.sin(2), np.sin(.02), np.cos(2), np.cos(.02), np.sin(1), np.sin(.01), np.cos(1), np.cos(.01)]
    assert np.allclose(t[7], want, atol=1e-6)


def test_fp8_and_concat_refused():
    with pytest.raises(ValueError, match="AIFI"):
        program("fp8")
    d = aifi_dict()
    d["head"][1], row = d["head"][1], d["head"][1]
    d["head"].insert(2, [-1, 1, "AIFI", [64, 8]])
    assert row[2] == "Concat"
    ar = A.parse_arch({**d, "head": d["head"][:3] + [[[-1], 1, "Detect", ["nc"]]]})
    with pytest.raises(ValueError, match="one output map"):
        M.Program(ar, W.synthetic_state_dict(ar, 0, planted=False), 256, 320, 320, 1, "bf16")


def test_engine_file_checks(tmp_path):
    """An engine with token ops is written and read back by the host checks; broken ones are refused
    before any device call (there is none here: an accepted one fails at the GPU)."""
    import ctypes as C

    L = P._lib
    prog = program()
    first = next(i for i, op in enumerate(prog.ops) if op.kind == M.YK_K_LINEAR)

    def load(change=None):
        keep = bytes(prog.ops[first]), bytes(prog.ops[first + 1])
        if change:
            change(prog.ops[first], prog.ops[first + 1])
        path = str(tmp_path / "m.ykengine")
        prog.export_engine(path)
        C.memmove(C.addressof(prog.ops[first]), keep[0], len(keep[0]))
        C.memmove(C.addressof(prog.ops[first + 1]), keep[1], len(keep[1]))
        ctx, out = C.create_string_buffer(64), C.c_void_p()
        if not change and torch.cuda.is_available():
            return L.YK_ERR_HIP  # (the checks are the CPU's; a real context loads it in test_aifi_gpu.py)
        return L.lib().yk_model_load(C.addressof(ctx), path.encode(), C.byref(out))

    assert load() == L.YK_ERR_HIP, L.lib().yk_last_error()
    bad = [lambda a, b: setattr(a, "act", 4), lambda a, b: setattr(a, "has_res", 3), lambda a, b: setattr(a, "cout", 0),
           lambda a, b: setattr(a, "w_off", len(prog.blob) - 8), lambda a, b: setattr(a, "t_off", len(prog.blob) - 8),
           lambda a, b: setattr(a, "b_off", 1), lambda a, b: setattr(a.dst, "buf", a.src[0].buf),
           lambda a, b: setattr(a.src[0], "h", 999), lambda a, b: setattr(a, "kind", 7), lambda a, b: setattr(a, "n_src", 2),
           lambda a, b: setattr(b, "ksize", 7), lambda a, b: setattr(b, "ksize", 0), lambda a, b: setattr(b, "ksize", 1)]
    for i, f in enumerate(bad):
        assert load(f) == L.YK_ERR_ARG, i
