"""Every way in which an engine's weights change over HTTP reaches the 8-bit copies that it serves from; engines without such copies are left alone."""
import pytest
import torch

from miles_b200.engine import Engine
from miles_b200.engine.server import build_app
from miles_b200.models import ParamStore, build_model, get_config
from miles_b200.weight_sync.registry import put_bucket


@pytest.fixture
def served(monkeypatch):
    from fastapi.testclient import TestClient

    cfg = get_config("qwen3-tiny")
    store = ParamStore(cfg, "cpu", torch.float32, seed=11)
    eng = Engine(build_model(cfg, store), max_running=2, page_size=8, max_seq_len=64)
    seen = []
    first = next(iter(store.params))
    monkeypatch.setattr(eng.model, "refresh_block_scaled", lambda: seen.append(store.params[first].flatten()[0].item()), raising=False)
    monkeypatch.setattr(eng.model, "mx_kind", "fp8_block", raising=False)
    return TestClient(build_app(eng)), eng, store, first, seen


def test_updates_reach_the_copies(served, tmp_path):
    from miles_b200.weight_sync.disk_delta import DiskDeltaWriter

    c, eng, store, first, seen = served
    value = torch.full_like(store.params[first], 0.25)
    c.post("/update_weights_from_tensor", json={"bucket_id": put_bucket([(first, value)]), "weight_version": 3})
    assert seen == [0.25] and eng.weight_version == 3  # after the copy, before the version
    c.post("/update_weights_from_tensor", json={"bucket_id": put_bucket([(first, value * 2)])})
    assert seen == [0.25]  # a bucket without a version: the versions' call follows
    c.post("/update_weight_version", json={"new_version": 4})
    assert seen == [0.25, 0.5] and eng.weight_version == 4
    w = DiskDeltaWriter(str(tmp_path / "delta"), encoding="overwrite")
    w.write([(n, torch.full_like(t, 0.75)) for n, t in store.params.items()], version=1)
    c.post("/pull_weights", json={"path": str(tmp_path / "delta" / "v00000001"), "weight_version": 5})
    assert seen == [0.25, 0.5, 0.75]


@pytest.mark.parametrize("kind", [None, "mxfp8"])
def test_other_engines_are_left_alone(served, monkeypatch, kind):
    c, eng, store, first, seen = served
    if kind is None:
        monkeypatch.delattr(eng.model, "mx_kind")
    else:
        monkeypatch.setattr(eng.model, "mx_kind", kind)
    c.post("/update_weights_from_tensor", json={"bucket_id": put_bucket([(first, torch.zeros_like(store.params[first]))]), "weight_version": 3})
    assert seen == [] and eng.weight_version == 3
