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
