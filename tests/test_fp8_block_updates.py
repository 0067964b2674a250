"""No answer comes from 8-bit copies of weights that have changed since, whichever endpoint changed them; and one update quantises them once."""
import pytest
import torch

from miles_b200.engine import Engine
from miles_b200.engine.server import build_app
from miles_b200.models import ParamStore, build_model, get_config
from miles_b200.weight_sync.registry import put_bucket


class Served:
    """A CPU engine whose model reports what its copies would have been made of."""

    def __init__(self, monkeypatch):
        from fastapi.testclient import TestClient

        cfg = get_config("qwen3-tiny")
        self.store = ParamStore(cfg, "cpu", torch.float32, seed=11)
        self.eng = Engine(build_model(cfg, self.store), max_running=2, page_size=8, max_seq_len=64)
        self.first, self.seen, self.made = next(iter(self.store.params)), [], []
        note = lambda: self.seen.append(self.value())  # noqa: E731
        monkeypatch.setattr(self.eng.model, "refresh_block_scaled", note, raising=False)
        monkeypatch.setattr(self.eng.model, "enable_block_scaled", lambda kind: self.made.append(kind) or note() or 7, raising=False)
        monkeypatch.setattr(self.eng.model, "mx_kind", "fp8_block", raising=False)
        monkeypatch.setattr(self.eng.model, "mx", {0: 0, 1: 1}, raising=False)
        self.c = TestClient(build_app(self.eng), raise_server_exceptions=False)

    def value(self):
        return self.store.params[self.first].flatten()[0].item()

    def fill(self, v):
        self.store.params[self.first].fill_(v)

    def bucket(self, v):
        return put_bucket([(self.first, torch.full_like(self.store.params[self.first], v))])


@pytest.fixture
def s(monkeypatch):
    return Served(monkeypatch)


def generate(s):
    return s.c.post("/generate", json={"input_ids": [1, 2, 3], "sampling_params": {"max_new_tokens": 2, "temperature": 0.0}})


def score(s):
    return s.c.post("/generate", json={"input_ids": [1, 2, 3], "sampling_params": {"max_new_tokens": 0}})


def feed(s):
    s.eng.feed([("a", [1, 2, 3], [2])])
    s.eng.end_feed("a")


CHANGES = {
    "tensors": lambda s, m: s.c.post("/update_weights_from_tensor", json={"bucket_id": s.bucket(0.5)}),
    "tensors, end": lambda s, m: [s.c.post("/update_weights_from_tensor", json={"bucket_id": s.bucket(0.5)}), s.c.post("/end_weight_update")],
    "tensors, version": lambda s, m: s.c.post("/update_weights_from_tensor", json={"bucket_id": s.bucket(0.5), "weight_version": 3}),
    "tensors, then an unknown one": lambda s, m: s.c.post("/update_weights_from_tensor", json={"bucket_id": put_bucket([
        (s.first, torch.full_like(s.store.params[s.first], 0.5)), ("no.such.weight", torch.zeros(1))])}),
    "disk": lambda s, m: [m.setattr("miles_b200.checkpoint.load_hf", lambda cfg, store, path, strict: s.fill(0.5)),
                          s.c.post("/update_weights_from_disk", json={"model_path": "x"})],
    "distributed": lambda s, m: [m.setattr("miles_b200.weight_sync.broadcast.receive_bucket", lambda b, store: s.fill(0.5)),
                                 s.c.post("/update_weights_from_distributed", json={})],
    "delta": lambda s, m: [m.setattr("miles_b200.weight_sync.disk_delta.apply_delta_dir", lambda store, path: s.fill(0.5)),
                           s.c.post("/pull_weights", json={"path": "x"})],
    "adapter in": lambda s, m: [m.setattr("miles_b200.lora.merge_adapter_into", lambda store, t, scale: s.fill(0.5)),
                                s.c.post("/load_lora_adapter_from_tensors", json={"lora_name": "a", "bucket_id": s.bucket(0.1)})],
    "adapter out": lambda s, m: [m.setattr("miles_b200.lora.merge_adapter_into", lambda store, t, scale: s.fill(0.5 if scale < 0 else 0.1)),
                                 s.c.post("/load_lora_adapter_from_tensors", json={"lora_name": "a", "bucket_id": s.bucket(0.1)}),
                                 s.c.post("/unload_lora_adapter", json={"lora_name": "a"})],
}


@pytest.mark.parametrize("ask", [generate, score, feed])
@pytest.mark.parametrize("how", CHANGES)
def test_what_is_computed_next_reads_new_copies(s, monkeypatch, how, ask):
    CHANGES[how](s, monkeypatch)
    assert s.value() == 0.5
    ours, before = s.eng.model.forward_hidden, []
    monkeypatch.setattr(s.eng.model, "forward_hidden", lambda *a, **k: before.append(s.seen[-1:]) or ours(*a, **k))
    ask(s)
    assert before and all(b == [0.5] for b in before)
    made = len(s.seen)
    ask(s)
    assert len(s.seen) == made  # (nothing has changed since)


def test_reset_weights_reach_the_copies(s):
    s.c.post("/weights_checker", json={"action": "snapshot"})
    s.c.post("/weights_checker", json={"action": "compare"})
    assert s.seen == []
    s.c.post("/weights_checker", json={"action": "reset_tensors"})
    assert s.seen == [0.0]


def test_a_paused_engine_waits_for_the_last_bucket(s):
    s.c.post("/pause_generation", json={})
    for v in (0.25, 0.5):
        s.c.post("/update_weights_from_tensor", json={"bucket_id": s.bucket(v)})
        s.eng.step()
    assert s.seen == []
    s.c.post("/update_weight_version", json={"new_version": 2})
    s.c.post("/continue_generation")
    assert generate(s).status_code == 200 and s.seen == [0.5]


def test_one_update_quantises_once(s):
    s.c.post("/update_weights_from_tensor", json={"bucket_id": s.bucket(0.5)})
    s.c.post("/update_weight_version", json={"new_version": 2})
    assert s.c.post("/requantize_weights", json={"format": "fp8_block"}).json() == {"success": True, "num_tensors": 2}
    assert s.seen == [0.5] and s.made == []
    s.fill(0.75)  # (a write that no endpoint made)
    assert s.c.post("/requantize_weights", json={"format": "fp8_block"}).json()["num_tensors"] == 7
    s.c.post("/update_weights_from_tensor", json={"bucket_id": s.bucket(0.25)})
    s.c.post("/requantize_weights", json={"format": "fp8_block"})
    s.c.post("/update_weight_version", json={"new_version": 3})
    s.c.post("/requantize_weights", json={"format": "mxfp8"})  # another format
    assert s.seen == [0.5, 0.75, 0.25, 0.25, 0.25] and s.made == ["fp8_block", "fp8_block", "mxfp8"]
