"""Serving endpoint (runners/serve.py): health + micro-batched predict on a
tiny CPU model."""

import io

import numpy as np
import pytest
import torch
from PIL import Image


@pytest.fixture(scope="module")
def client():
    from starlette.testclient import TestClient

    from deepfake_detection_amd.runners.serve import InferenceEngine, create_app

    class TinyEngine(InferenceEngine):
        def __init__(self):
            # bypass the B7-scale constructor: tiny conv net with the same
            # (B, 12, 600, 600) -> (B, 2) contract
            self.device = "cpu"
            self.dtype = torch.float32
            self.model = torch.nn.Sequential(
                torch.nn.Conv2d(12, 4, 3, stride=8), torch.nn.AdaptiveAvgPool2d(1),
                torch.nn.Flatten(), torch.nn.Linear(4, 2), torch.nn.Softmax(-1)).eval()
            self.max_batch = 4
            self.batch_window_s = 0.005
            import asyncio

            self._queue = asyncio.Queue()
            self._worker = None

    engine = TinyEngine()
    with TestClient(create_app(engine)) as c:
        yield c


def _png_bytes():
    img = Image.fromarray((np.random.rand(64, 48, 3) * 255).astype(np.uint8))
    buf = io.BytesIO()
    img.save(buf, format="PNG")
    return buf.getvalue()


def test_health(client):
    r = client.get("/health")
    assert r.status_code == 200
    assert r.json()["status"] == "ok"


def test_predict(client):
    r = client.post("/predict", content=_png_bytes(),
                    headers={"Content-Type": "application/octet-stream"})
    assert r.status_code == 200
    body = r.json()
    assert 0.0 <= body["fake_probability"] <= 1.0
    assert body["label"] in ("fake", "real")


def test_predict_concurrent_batched(client):
    import concurrent.futures as cf

    def one(_):
        return client.post("/predict", content=_png_bytes(),
                           headers={"Content-Type": "application/octet-stream"})

    with cf.ThreadPoolExecutor(8) as ex:
        rs = list(ex.map(one, range(8)))
    assert all(r.status_code == 200 for r in rs)


# ---------------------------------------------------------------------------
# models that were trained with --group-norm
# ---------------------------------------------------------------------------

@pytest.fixture(scope="module")
def group_norm_model(tmp_path_factory):
    """(the model with its softmax, its halved checkpoint, a BatchNorm model's)"""
    import deepfake_detection_amd as dfd
    from deepfake_detection_amd.models.layers_extra import convert_groupnorm_model
    from deepfake_detection_amd.params import DeepFakeModel

    folder = tmp_path_factory.mktemp("group_norm")
    torch.manual_seed(0)
    model = dfd.create_deepfake_model_v4("efficientnet_deepfake_v4", num_classes=2, in_chans=12)
    torch.save({"state_dict": model.state_dict()}, folder / "batch.pth.tar")
    model = convert_groupnorm_model(model, 16)
    with torch.no_grad():
        for p in model.parameters():
            if p.dim() == 1:
                p.add_(torch.rand_like(p) * 0.1)
    torch.save({"state_dict": {k: v.half() for k, v in model.state_dict().items()}},
               folder / "group.pth.tar")
    model.load_state_dict({k: v.half() for k, v in model.state_dict().items()})
    return DeepFakeModel(model).eval(), str(folder / "group.pth.tar"), str(folder / "batch.pth.tar")


def served_engine(monkeypatch, *argv):
    import uvicorn

    from deepfake_detection_amd.runners import serve

    engines = []
    monkeypatch.setattr(serve, "create_app", engines.append)
    monkeypatch.setattr(uvicorn, "run", lambda app, **kw: None)
    serve.main(["--no-fp16", *argv])
    return engines[0]


def test_serve_a_group_norm_model(group_norm_model, monkeypatch):
    model, path, _ = group_norm_model
    x = torch.randn(2, 12, 96, 96)
    engine = served_engine(monkeypatch, "--checkpoint", path, "--group-norm", "16")
    with torch.no_grad():
        want = model(x)[:, 0]
    assert torch.equal(engine.forward(x), want)
    # what the flag is for: another count of groups is another model
    other = served_engine(monkeypatch, "--checkpoint", path, "--group-norm", "8")
    assert not torch.equal(other.forward(x), want)


def test_group_norm_of_the_test_command(group_norm_model, tmp_path, monkeypatch):
    from deepfake_detection_amd.params import preprocess_image
    from deepfake_detection_amd.runners import test as command

    model, path, _ = group_norm_model
    pixels = np.random.RandomState(0).randint(0, 255, (64, 48, 3), dtype=np.uint8)
    Image.fromarray(pixels).save(tmp_path / "a.png")
    scores = []
    run = command.test_img
    monkeypatch.setattr(command, "test_img", lambda *a, **kw: scores.extend(run(*a, **kw)))
    command.main([str(tmp_path / "a.png"), "--checkpoint", path, "--device", "cpu",
                  "--group-norm", "16"])
    with torch.no_grad():
        want = model(preprocess_image(pixels, device="cpu", dtype=torch.float32))[0, 0].item()
    assert scores == [(str(tmp_path / "a.png"), want)]


def test_checkpoint_of_the_other_norm(group_norm_model, monkeypatch, caplog):
    """Weights of a BatchNorm model do not run with group norms. Without the
    flag a checkpoint may lack weights, as before, but not silently."""
    from deepfake_detection_amd.runners.test import test_img

    _, path, batch = group_norm_model
    with pytest.raises(RuntimeError, match="running_mean"):
        served_engine(monkeypatch, "--checkpoint", batch, "--group-norm", "16")
    with pytest.raises(RuntimeError, match="running_mean"):
        test_img([], checkpoint_path=batch, device="cpu", group_norm=16)
    with caplog.at_level("WARNING"):
        test_img([], checkpoint_path=batch, device="cpu")
        assert not caplog.records
        test_img([], checkpoint_path=path, device="cpu")
    assert "running_mean" in caplog.text
