"""Models whose weights are split over ranks, served from E4M3 copies with a scale for each 128 x 128: what each product reads."""
import pytest
import torch

from miles_b200 import _build
from miles_b200.models import ParamStore, build_model, get_config
from miles_b200.models.b200_impl import MoeCtx


def make(preset, device, **kw):
    if device == "cpu" and _build.needs_build():
        pytest.skip("the extension has not been built here")
    cfg = get_config(preset)
    return build_model(cfg, ParamStore(cfg, device, torch.bfloat16, init_std=0.05, seed=5), "b200", **kw)


def test_experts_behind_an_exchange_are_multiplied_in_bf16():
    """The plans of the expert-parallel exchanges: without expert ids (decode steps), or with those of a padded receive buffer (prompts)."""
    model = make("qwen3-smoke-moe", "cpu")
    model.enable_block_scaled("fp8_block")
    P, cfg = model.store.params, model.cfg
    w1, w2 = P["layers.0.moe.w1"], P["layers.0.moe.w2"]
    calls = []

    class C:
        def __getattr__(self, name):
            return lambda *a, **k: calls.append(name) or torch.zeros(64, w2.shape[2], dtype=torch.bfloat16)

    model.C = C()
    offsets = torch.zeros(cfg.num_experts + 1, dtype=torch.int32)
    for ids in (None, torch.zeros(64, 1, dtype=torch.int32)):
        plan = MoeCtx(ids, None, None, offsets, None, None, torch.zeros(1, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 64, pairs=32)
        _, _, yp = model._experts_fwd(torch.zeros(64, cfg.hidden_size, dtype=torch.bfloat16), plan, w1, w2, keep=False)
        assert yp.shape == (64, cfg.hidden_size) and calls == ["grouped_gemm_rows", "swiglu_fwd", "grouped_gemm_rows"]
        calls.clear()


def test_no_copies_of_experts_behind_an_exchange():
    model = make("qwen3-smoke-moe", "cpu", ep=object())
    model.enable_block_scaled("fp8_block")
    served = {n for n, w in model.store.params.items() if w.data_ptr() in model.mx}
    assert served == {n for n in model.store.params if n.endswith(("attn.qkv.weight", "attn.o.weight"))}


@pytest.mark.gpu
def test_rows_of_an_exchange_give_what_bf16_gives():
    out = []
    for kind in (None, "fp8_block"):
        model = make("qwen3-smoke-moe", "cuda")
        if kind:
            model.enable_block_scaled(kind)
        cfg, P = model.cfg, model.store.params
        g = torch.Generator().manual_seed(3)
        h = torch.randn(40, cfg.hidden_size, generator=g).bfloat16().cuda()
        ids = torch.stack([torch.randperm(cfg.num_experts, generator=g)[:cfg.moe_top_k] for _ in range(40)]).int().cuda()
        plan = model._permute_plan(ids, cfg.num_experts)
        plan.ids = None
        xp = model.C.moe_permute(h, plan.src, plan.num_tiles, cfg.moe_top_k)
        out.append(model._experts_fwd(xp, plan, P["layers.0.moe.w1"], P["layers.0.moe.w2"], keep=False)[2][plan.dest.long()])
        model.check_status()
    assert torch.equal(*out)
