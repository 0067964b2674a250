"""What block-scaled copies of the weights take, and the room that a trainer's engine leaves for them beside its cache."""
import pytest
import torch

from miles_b200 import _build
from miles_b200.models import ParamStore, build_model, get_config

PRESETS = ["qwen3-smoke", "qwen3-smoke-moe", "glm4moe-smoke"]


def held(model):
    return sum(t.numel() * t.element_size() for w in model.mx.values() for t in vars(w).values() if torch.is_tensor(t))


def check(preset, kind, device):
    cfg = get_config(preset)
    store = ParamStore(cfg, device, torch.bfloat16, seed=5)
    model = build_model(cfg, store, "b200")
    model.enable_block_scaled(kind)
    said = model.block_scaled_bytes(store.specs, kind)
    assert held(model) <= said + 8 * len(model.mx) and said <= 1.01 * held(model)  # (NVFP4 has two fp32 numbers a tensor)
    assert model.block_scaled_bytes(store.specs, "none") == 0


@pytest.mark.parametrize("preset", PRESETS)
def test_bytes_of_copies(preset):
    if _build.needs_build():
        pytest.skip("the extension has not been built here")
    check(preset, "fp8_block", "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["mxfp8", "nvfp4", "fp8_block"])
@pytest.mark.parametrize("preset", PRESETS)
def test_bytes_of_copies_on_the_device(preset, kind):
    check(preset, kind, "cuda")


def loop(preset, kind, *more):
    from miles_b200.loop import RLLoop
    from miles_b200.utils.arguments import parse_args

    return RLLoop(parse_args(["--model-preset", preset, "--rollout-batch-size", "8", "--n-samples-per-prompt", "4", "--rollout-max-response-len", "16",
                              "--rollout-max-prompt-len", "32", "--rm-type", "parity", "--lr", "1e-5", "--eps-clip", "0.2", "--micro-batch-size", "8",
                              "--weight-decay", "0.0", "--colocate", "--num-rollout", "2", "--actor-num-gpus-per-node", "1",
                              "--rollout-quantization", kind, *more]))


def held_by(kind):
    cfg = get_config("qwen3-smoke")
    model = build_model(cfg, ParamStore(cfg, "cuda", torch.bfloat16, seed=5), "b200")
    model.enable_block_scaled(kind)
    return held(model)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["mxfp8", "fp8_block"])
def test_the_cache_leaves_room_for_the_copies(kind, monkeypatch):
    """8 MB free beside the reserve, where the cache wants 7.8 and the copies take 4.7: what they take is not given to the cache."""
    from miles_b200.loop import RLLoop

    free, build, size = 8 << 20, RLLoop._build_engine, {}

    def tight(self):
        with monkeypatch.context() as m:
            total = torch.cuda.mem_get_info()[1]
            m.setattr(torch.cuda, "mem_get_info", lambda *a: (total // 7 + free, total))
            build(self)

    monkeypatch.setattr(RLLoop, "_build_engine", tight)
    for k in ("none", kind):
        e = loop("qwen3-smoke", k, "--no-share-kv-grad-memory").engine
        size[k] = e.num_pages * e.page_size * e.layout.bytes_per_slot()
    assert size["none"] <= free and 0 < size[kind] <= free - held_by(kind)


@pytest.mark.gpu
@pytest.mark.parametrize("preset", ["qwen3-smoke", "qwen3-smoke-moe"])
def test_the_trainer_rolls_out_from_8_bit_copies(preset):
    """Two steps with --rollout-quantization fp8_block: 32 running rows decode from the copies, which follow every update; the trainer's own
    model stays in bf16."""
    made = loop(preset, "fp8_block", "--check-weight-update-equal")
    model = made.engine.model
    assert model is not made.actor.model and not getattr(made.actor.model, "mx", None) and model.mx_kind == "fp8_block"
    first = {k: w.q.view(torch.uint8).clone() for k, w in model.mx.items()}
    hist = made.run()
    torch.cuda.synchronize()
    assert len(hist) == 2 and all(m["train/grad_norm"] > 0 for m in hist) and made.engine.weight_version == made.actor.store.version == 2
    assert any(not torch.equal(first[k], w.q.view(torch.uint8)) for k, w in model.mx.items())
    from miles_b200.ops.fp8_block import quantize_weight

    for name, w in model.store.params.items():
        if w.data_ptr() in model.mx:
            kept = model.mx[w.data_ptr()]
            fresh = quantize_weight(w, kept.halves)
            assert torch.equal(kept.q.view(torch.uint8), fresh.q.view(torch.uint8)) and torch.equal(kept.scales, fresh.scales), name


GB = 10 ** 9


def plan(copies, host, total=190 * GB, experts=28 * GB):
    from miles_b200.trainer.actor import choose_memory_plan

    return choose_memory_plan(total, GB, experts, kv_bytes=0, state="bf16", host_bytes=host, copy_bytes=copies)


def test_copies_displace_optimizer_state():
    """190 GB, of which 84 % hold 12 of replicated parameters, 56 of expert weights and 56 of gradients: 35.6 are left for 168 of state, 13 of 64 chunks; with
    30 of copies 2 of 64; and where the host takes 150, of the 168 at least 18: 7 of 64. Where the state without copies would have been placed it is placed."""
    state = 6 * 28 * GB
    assert plan(0, None)["resident_frac"] == plan(0, 200 * GB)["resident_frac"] == 13 / 64
    assert plan(30 * GB, None)["resident_frac"] == plan(30 * GB, 200 * GB)["resident_frac"] == 2 / 64
    tight = plan(30 * GB, 150 * GB)
    assert tight["resident_frac"] == 7 / 64 and state * (1 - 7 / 64) <= 150 * GB < state * (1 - 6 / 64)
    assert plan(30 * GB, int(state * (1 - 13 / 64)))["resident_frac"] == 13 / 64
    for copies in (0, 30 * GB):  # what cannot be placed without copies cannot with them
        with pytest.raises(MemoryError):
            plan(copies, int(state * (1 - 13 / 64)) - GB)
    assert plan(0, 0, total=400 * GB) == plan(30 * GB, 0, total=400 * GB) and not plan(0, 0, total=400 * GB)["offload"]


@pytest.mark.gpu
def test_the_optimizer_plan_is_told_of_the_copies(monkeypatch):
    from miles_b200.trainer import actor

    seen, ours = {}, actor.choose_memory_plan
    for kind in ("none", "fp8_block"):
        monkeypatch.setattr(actor, "choose_memory_plan", lambda *a, **k: seen.setdefault(kind, k["copy_bytes"]) and None or ours(*a, **k))
        loop("qwen3-smoke", kind)
    assert seen["none"] == 0 and abs(seen["fp8_block"] - held_by("fp8_block")) <= 1024
