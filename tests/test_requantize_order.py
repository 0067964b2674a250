"""Engines in other processes make their block-scaled copies of new weights before they go on generating."""
from types import SimpleNamespace

import pytest
import torch

from miles_b200.loop import RLLoop
from miles_b200.weight_sync.broadcast import BroadcastWeightUpdater
from miles_b200.weight_sync.disk_delta import DiskDeltaUpdater


class Engine:
    def __init__(self):
        self.posts = []

    def post(self, path, payload=None):
        self.posts.append((path, payload))
        return {}

    def post_async(self, path, payload=None):
        self.post(path, payload)
        return SimpleNamespace(result=lambda: None)


def loop(updater, fmt):
    out = object.__new__(RLLoop)
    out.args, out.ps, out.weight_updater = SimpleNamespace(rollout_engine_urls="http://127.0.0.1:9", weight_sync_quant=fmt), SimpleNamespace(world_size=1, rank=0), updater
    return out


@pytest.fixture
def actor():
    store = SimpleNamespace(version=3, params={"w": torch.ones(4)})
    return SimpleNamespace(args=SimpleNamespace(), store=store, on_gpu=False, ps=SimpleNamespace(rank=0, world_size=1))


@pytest.mark.parametrize("fmt", ["none", "mxfp8", "fp8_block"])
def test_broadcast(actor, fmt):
    engines = [Engine(), Engine()]
    updater = BroadcastWeightUpdater(actor, engines)
    updater.connected, updater._parts = True, lambda: []
    loop(updater, fmt)._update_weights()
    for e in engines:
        names = [p for p, _ in e.posts]
        assert names[0] == "/pause_generation" and names[-1] == "/continue_generation"
        assert [x for x in e.posts if x[0] == "/requantize_weights"] == ([] if fmt == "none" else [("/requantize_weights", {"format": fmt})])
        if fmt != "none":
            assert names.index("/update_weight_version") < names.index("/requantize_weights")


@pytest.mark.parametrize("fmt", ["none", "fp8_block"])
def test_disk_delta(actor, tmp_path, fmt):
    engines = [Engine()]
    loop(DiskDeltaUpdater(actor, engines, str(tmp_path)), fmt)._update_weights()
    assert [p for p, _ in engines[0].posts] == ["/pull_weights"] + ([] if fmt == "none" else ["/requantize_weights"])


def test_a_rank_without_an_updater_goes_on():
    assert loop(None, "fp8_block")._update_weights() == {}
