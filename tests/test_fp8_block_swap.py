"""Quantising anew while an engine is in use: copies change as a whole, a layer is computed from one set of them, and it happens where the engine is
stepped."""
import asyncio

import pytest
import torch

from miles_b200 import _build
from miles_b200.models import ParamStore, build_model, get_config
from miles_b200.ops import fp8_block as F8


def served(preset="qwen3-smoke"):
    if _build.needs_build():
        pytest.skip("the extension has not been built here")
    model = build_model(get_config(preset), ParamStore(get_config(preset), "cpu", torch.bfloat16, seed=5), "b200")
    model.enable_block_scaled("fp8_block")
    return model


def test_copies_change_as_a_whole(monkeypatch):
    model = served()
    before, names = dict(model.mx), []
    assert len(before) == 4 * model.cfg.num_layers
    ours = F8.quantize_weight

    def between(w, halves=1):
        assert model.mx_kind == "fp8_block" and model.mx.keys() == before.keys()  # whoever computes now finds them all
        assert all(model._fp8_layer(i, 64) is not None for i in range(model.cfg.num_layers))
        names.append(w.data_ptr())
        return ours(w, halves)

    monkeypatch.setattr(F8, "quantize_weight", between)
    model.refresh_block_scaled()
    assert sorted(names) == sorted(before) and all(model.mx[k] is w for k, w in before.items())


@pytest.mark.parametrize("preset", ["qwen3-smoke", "qwen3-smoke-moe"])
def test_a_layer_is_computed_from_one_set_of_copies(preset, monkeypatch):
    """The copies are exchanged in the middle of a layer: it goes on with those that it began with."""
    model = served(preset)
    T, H = 16, model.cfg.hidden_size
    moe = model.cfg.layer_is_moe(0)
    first, second = ("moe.w1", "moe.w2") if moe else ("mlp.gate_up.weight", "mlp.down.weight")
    mine = [model.mx[model.store.params[f"layers.0.{n}"].data_ptr()] for n in ("attn.qkv.weight", "attn.o.weight", first, second)]
    read = []

    def product(x, w, *a, **k):
        read.append(w)
        model.mx = {}
        n = w.q.shape[-2]
        return torch.zeros(len(x.q if isinstance(x, F8.Fp8Rows) else x), n, dtype=torch.bfloat16)

    def gated(x, w, *a, **k):
        y = product(x, w)
        return rows(y[:, :y.shape[1] // 2])

    def rows(v):
        return F8.Fp8Rows(torch.zeros(v.shape, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(len(v), -(-v.shape[1] // 128)))

    for name, fake in (("linear", product), ("grouped_linear", product), ("gated_linear", gated), ("grouped_gated_linear", gated),
                       ("rmsnorm_rows", lambda x, w, eps, residual=None, keep=False: (rows(x), x, x)),
                       ("permute_rows", lambda x, src, num_tiles, top_k: rows(torch.zeros(len(x.q) * top_k, x.q.shape[1])))):
        monkeypatch.setattr(F8, name, fake)

    class C:
        def __getattr__(self, name):
            cfg = model.cfg
            if name.startswith("qk_norm_rope"):
                return lambda *a: (torch.zeros(T, cfg.num_q_heads, cfg.head_dim), torch.zeros(T, cfg.num_kv_heads, cfg.head_dim), None, None)
            if name == "moe_combine":
                return lambda *a: torch.zeros(T, H)
            return lambda *a, **k: 1  # (counts of launches)

    model.C = C()
    model.attention = lambda q, k, v, cu: (torch.zeros(T, model.cfg.num_q_heads, model.cfg.head_dim, dtype=torch.bfloat16), None)
    model._route = lambda *a: (None, None, None)
    ids = torch.zeros(T, max(model.cfg.moe_top_k, 1), dtype=torch.int32)
    model._permute_plan = lambda *a: type("Plan", (), dict(ids=ids, src=None, dest=None, tile_group=ids, num_tiles=None, max_rows=ids.numel()))()
    model.layer_forward(0, torch.zeros(T, H, dtype=torch.bfloat16), None, None, T)
    assert [id(w) for w in read] == [id(w) for w in mine]


def test_requantising_happens_where_the_engine_is_stepped(monkeypatch):
    from fastapi.testclient import TestClient

    from miles_b200.engine import Engine
    from miles_b200.engine.server import build_app

    cfg = get_config("qwen3-tiny")
    eng = Engine(build_model(cfg, ParamStore(cfg, "cpu", torch.float32, seed=11)), max_running=2, page_size=8, max_seq_len=64)
    seen = []

    def enable(kind):
        asyncio.get_running_loop()  # (raises in a worker thread)
        seen.append(kind)
        return 7

    monkeypatch.setattr(eng.model, "enable_block_scaled", enable, raising=False)
    c = TestClient(build_app(eng))
    assert c.post("/requantize_weights", json={"format": "fp8_block"}).json() == {"success": True, "num_tensors": 7} and seen == ["fp8_block"]
    assert not c.post("/requantize_weights", json={"format": "other"}).json()["success"] and seen == ["fp8_block"]
