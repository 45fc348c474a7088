"""A detector with an AIFI layer behind SPPF: the P2 topology with one row more."""
import copy
import importlib

from conftest import pkg


def aifi_dict(scale="n", hidden=256, heads=8):
    A = importlib.import_module(pkg().__name__ + ".arch")
    d = copy.deepcopy(A.YOLOV8_SMALL)
    d["scale"] = scale
    d["backbone"].append([-1, 1, "AIFI", [hidden, heads]])
    up = lambda f: [up(x) for x in f] if isinstance(f, list) else f + 1 if f >= 9 else f  # noqa: E731
    d["head"] = [[up(f), n, m, a] for f, n, m, a in d["head"]]
    return d


def layer_list(ar):
    return [(L.i, L.f, L.kind, {**L.args, **({"c": int(L.c2 * 0.5)} if L.kind == "C2f" else {})}) for L in ar.layers]
