"""Captured decode steps and the block-scaled copies that they read: copies of one format stay where they are, another format has the steps captured anew."""
import contextlib

import pytest
import torch

from miles_b200 import _build
from miles_b200.engine import Engine, SamplingParams
from miles_b200.models import ParamStore, build_model, get_config

KINDS = ["mxfp8", "nvfp4", "fp8_block"]


def test_steps_are_captured_anew_when_the_copies_move(monkeypatch):
    cfg = get_config("qwen3-tiny")
    eng = Engine(build_model(cfg, ParamStore(cfg, "cpu", torch.float32, seed=11)), max_running=2, page_size=8, max_seq_len=64)
    replayed = []

    class Graph:
        def replay(self):
            replayed.append(self)

    monkeypatch.setattr(torch.cuda, "CUDAGraph", Graph)
    monkeypatch.setattr(torch.cuda, "graph", lambda g, pool=None: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "graph_pool_handle", lambda: None)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    monkeypatch.setattr(eng, "_decode_body", lambda B, routes: None)
    monkeypatch.setattr(eng, "_upload_rows", lambda reqs, B: None)
    eng.on_gpu = eng.use_cuda_graph = True
    run = lambda *keys: [eng._run_decode(B, False) for B in keys] and replayed[-len(keys):]  # noqa: E731
    first = run(1, 2, 1)
    assert first[0] is first[2] and first[0] is not first[1]  # one graph for a row bound
    eng.model.mx_generation = 1
    assert not eng._graphs_current() and not eng._can_look_ahead({"reqs": []})
    eng.sync, again = object(), run(2, 1, 2)
    assert again[0] is again[2] and not set(again) & set(first) and eng._graphs_current()
    eng.model.mx_generation = 2
    assert not eng._can_launch_ahead({"reqs": []}, eng._rows_B)
    eng._graphs.clear()  # none left: nothing reads the old copies
    assert eng._graphs_current()


def test_generations_of_copies():
    """They count moves, not refreshes."""
    if _build.needs_build():
        pytest.skip("the extension has not been built here")
    cfg = get_config("qwen3-smoke")
    model = build_model(cfg, ParamStore(cfg, "cpu", torch.bfloat16, seed=5), "b200")
    assert model.mx_generation == 0
    with pytest.raises(ValueError, match="unknown block-scaled kind"):
        model.enable_block_scaled("fp6")
    assert model.mx_generation == 0 and not getattr(model, "mx", None)
    model.enable_block_scaled("fp8_block")
    first = model.mx_generation
    assert first > 0
    at = {k: (w.q.data_ptr(), w.scales.data_ptr()) for k, w in model.mx.items()}
    model.store.params["layers.0.attn.o.weight"].mul_(0.5)
    model.refresh_block_scaled()
    assert model.mx_generation == first and at == {k: (w.q.data_ptr(), w.scales.data_ptr()) for k, w in model.mx.items()}
    del model.mx[model.store.params["layers.0.attn.o.weight"].data_ptr()]
    model.refresh_block_scaled()
    assert model.mx_generation > first and model.mx.keys() == at.keys()
    second = model.mx_generation
    model.use_block_scaled("mxfp8", {})
    third = model.mx_generation
    assert third > second
    model.refresh_block_scaled()  # (kept up to date by whoever owns them)
    assert model.mx_generation == third and model.mx_kind == "mxfp8"
    model.enable_block_scaled("fp8_block")
    assert model.mx_generation > third and model.mx_kind == "fp8_block" and len(model.mx) == len(at)
    model.store.params["layers.0.attn.o.weight"].mul_(0.5)
    before = model.mx[model.store.params["layers.0.attn.o.weight"].data_ptr()].scales.clone()
    model.store.params["layers.0.attn.o.weight"].mul_(0.5)
    model.refresh_block_scaled()  # its own again
    assert not torch.equal(before, model.mx[model.store.params["layers.0.attn.o.weight"].data_ptr()].scales)


def engine(kind, graph):
    cfg = get_config("qwen3-smoke-moe")
    model = build_model(cfg, ParamStore(cfg, "cuda", torch.bfloat16, init_std=0.02, seed=5), "b200")
    if kind:
        model.enable_block_scaled(kind)
    return Engine(model, max_running=40, page_size=64, max_seq_len=256, use_cuda_graph=graph, prefix_cache=False)


def tokens(eng):
    g = torch.Generator().manual_seed(0)
    prompts = [torch.randint(0, eng.cfg.vocab_size, (20 + i,), generator=g).tolist() for i in range(40)]
    return [r["output_ids"] for r in eng.generate(prompts, [SamplingParams(temperature=0.0, max_new_tokens=8, ignore_eos=True) for _ in prompts])]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_copies_of_every_format_stay_where_they_are(kind):
    """40 running rows, captured and eager, across an update of the weights: the same tokens."""
    out = {}
    for graph in (False, True):
        eng = engine(kind, graph)
        at = {k: [t.data_ptr() for t in vars(w).values() if torch.is_tensor(t)] for k, w in eng.model.mx.items()}
        first = tokens(eng)
        eng.model.store.params["layers.1.attn.o.weight"].mul_(-3.0)
        eng.model.refresh_block_scaled()
        assert at == {k: [t.data_ptr() for t in vars(w).values() if torch.is_tensor(t)] for k, w in eng.model.mx.items()}
        out[graph] = first, tokens(eng)
        assert first != out[graph][1]
        eng.model.check_status()
    assert out[False] == out[True]


@pytest.mark.gpu
def test_another_format_reaches_captured_steps():
    """Steps captured in bf16, and then in one format after the other: every time those of an eager engine that serves the format."""
    eng = engine(None, True)
    want = {kind: tokens(engine(kind, False)) for kind in (None, *KINDS)}
    assert tokens(eng) == want[None]
    for kind in ("mxfp8", "fp8_block", "nvfp4", "fp8_block", "mxfp8"):
        assert eng.serve_block_scaled(kind) == 8
        assert tokens(eng) == want[kind], kind
    eng.model.check_status()
