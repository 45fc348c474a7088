"""A detector with an AIFI layer on the GPU against the torch-CPU oracle: the layer's activations and
what follows it, the graph path, the batch, and predict() from a YAML file."""
import importlib

import numpy as np
import pytest
import torch

from aifi_helpers import aifi_dict, layer_list
from conftest import pkg
from oracle import detector_ref as D

pytestmark = pytest.mark.gpu


def build(dtype, scale="n", hw=(256, 320), B=2, **kw):
    P = pkg()
    A, W, M = (importlib.import_module(f"{P.__name__}.{n}") for n in ("arch", "weights", "model"))
    ar = A.parse_arch(aifi_dict(scale, **kw))
    sd = W.synthetic_state_dict(ar, 0)
    sc = P.synth.Scene(seed=1, n_targets=8, n_frames=B, height=hw[0], width=hw[1])
    frames = [sc.frame(t) for t in range(B)]
    dm = M.DeviceModel(M.Program(ar, sd, hw[0], hw[1], max(hw), B, dtype))
    ref = D.RefDetector(layer_list(ar), sd, A.detect_strides(ar))
    return dm, ref, frames, torch.from_numpy(np.stack(frames)).cuda()


def rel(a, b):
    return float((a.double() - b.double()).abs().max() / b.double().abs().max())


def same(a, b):
    """Equal detections: counts, and the rows in use (the others are not written)."""
    return torch.equal(a[1], b[1]) and all(torch.equal(x[:n], y[:n]) for x, y, n in zip(a[0], b[0], a[1].tolist()))


@pytest.mark.parametrize("dtype,tol", [("fp32", 1e-4), ("fp16", 0.02), ("bf16", 0.15)])
@pytest.mark.parametrize("scale,hidden,heads", [("n", 256, 8), ("s", 1024, 8), ("n", 100, 3)])
def test_layers_match_the_oracle(dtype, tol, scale, hidden, heads):
    """fp32 as the other layers' bound; the 16-bit programs round every layer on the way (26 of them
    before the last, each by u relative to its terms)."""
    dm, ref, frames, ft = build(dtype, scale, hidden=hidden, heads=heads)
    dm.detect(ft, 0.25, 0.7, 300)
    ref.forward(D.preprocess(frames, 320), keep_all=True)
    for layer in (9, 10, 13, 25):
        got, want = dm.layer_nchw(layer, 2), ref.outputs[layer]
        assert got.shape == want.shape
        assert rel(got, want) < tol, (layer, rel(got, want))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_graph_lanes_and_batches(dtype):
    """Captured and replayed, on several lanes, and an image alone: the same bits."""
    dm, _, _, ft = build(dtype, B=3)
    want = dm.detect(ft, 0.001, 0.7, 50)
    for lanes in (1, 3):
        dm.set_lanes(lanes)
        for _ in range(3):
            got = dm.detect(ft, 0.001, 0.7, 50, graph=True)
            torch.cuda.synchronize()
            assert same(got, want)
            dm.detect(ft, 0.001, 0.7, 50)
    layer = dm.layer_nchw(10, 3)
    dm.detect(ft[1:2].contiguous(), 0.001, 0.7, 50)
    # (the products of one image take smaller tiles: sums in another order)
    assert rel(dm.layer_nchw(10, 1)[0], layer[1]) < (1e-5 if dtype == "fp32" else 0.05)
    assert len(dm.profile(ft)) == len(dm.prog.ops) + 1


def test_candidates_match_the_oracle():
    """fp32: the box and score of every anchor before NMS (whose decisions a score's last digits may
    turn on random weights), within the other detectors' 1e-4 of the largest."""
    dm, ref, frames, ft = build("fp32")
    dm.detect(ft, 0.0, 0.7, 300)
    cand, cnt = dm.candidates(2)
    y, _ = ref.forward(D.preprocess(frames, 320))
    for b in range(2):
        assert cnt[b] == dm.prog.n_anchors == y.shape[2]
        rows = torch.from_numpy(cand[b])[torch.from_numpy(cand[b][:, 5].view(np.int32).astype(np.int64)).argsort()]
        xywh = y[b, :4].t()
        want = torch.cat([xywh[:, :2] - xywh[:, 2:] / 2, xywh[:, :2] + xywh[:, 2:] / 2, y[b, 4:5].t()], 1)
        assert rel(rows[:, :4], want[:, :4]) < 1e-4 and rel(rows[:, 4], want[:, 4]) < 1e-4


def test_predict_from_a_yaml_file(tmp_path):
    """YOLO(yaml)(frame) runs the layer: the detections of the program lowered from the same rows."""
    import yaml

    P = pkg()
    A, W, M = (importlib.import_module(f"{P.__name__}.{n}") for n in ("arch", "weights", "model"))
    d = aifi_dict("n")
    d.pop("scale")
    path = tmp_path / "yolov8n-aifi.yaml"
    path.write_text(yaml.safe_dump(d))
    ar = A.parse_arch(A.load_model_dict(str(path)))
    assert ar.layers[10].kind == "AIFI"
    sd = W.synthetic_state_dict(ar, 0)
    frame = P.synth.Scene(seed=2, n_targets=8, n_frames=1, height=256, width=320).frame(0)
    got = P.YOLO(str(path), weights=sd, dtype="fp32")(frame, conf=0.0005, imgsz=320)[0].boxes.data
    dm = M.DeviceModel(M.Program(ar, sd, 256, 320, 320, 1, "fp32"))
    dets, counts = dm.detect(torch.from_numpy(frame[None]).cuda(), 0.0005, 0.7, 300)
    assert len(got) == int(counts[0]) > 0 and torch.allclose(got.cpu(), dets[0, :len(got)].cpu(), rtol=1e-4, atol=1e-3)


def test_engine_file_roundtrip(tmp_path):
    """A C host's load of the exported engine detects the same bits."""
    P = pkg()
    M = importlib.import_module(P.__name__ + ".model")
    dm, _, _, ft = build("bf16")
    dm.prog.export_engine(str(tmp_path / "m.ykengine"))
    assert same(M.EngineModel(str(tmp_path / "m.ykengine")).detect(ft, 0.001), dm.detect(ft, 0.001))
