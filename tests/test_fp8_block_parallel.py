"""Models whose weights are split over ranks, served from E4M3 copies with a scale for each 128 x 128: what each product reads."""
import dataclasses

import pytest
import torch

from miles_b200 import _build
from miles_b200.models import ParamStore, build_model, get_config
from miles_b200.models.b200_impl import MoeCtx


def make(preset, device, ffn=None, **kw):
    if device == "cpu" and _build.needs_build():
        pytest.skip("the extension has not been built here")
    cfg = get_config(preset)
    if ffn is not None:
        cfg = dataclasses.replace(cfg, ffn_hidden_size=ffn)
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


class Whole:
    """What tensor parallelism asks of its exchange, for one rank that holds everything."""
    n = 2

    def __init__(self, C):
        self.C = C

    def linear_allreduce(self, a, w, b_mn=False, residual=None, gemm_status=None):
        y = (a.float() @ w.float().t()).to(torch.bfloat16)
        return y if residual is None else y + residual


LAYERS = [("qwen3-smoke", dict()), ("qwen3-smoke", dict(tp=Whole(None))), ("glm4-smoke", dict()), ("glm4moe-smoke", dict(ep=object()))]


@pytest.mark.parametrize("ffn", [1024, 304, 1008])
@pytest.mark.parametrize("preset,kw", LAYERS)
def test_gate_up_blocks_are_those_that_the_layer_reads(preset, kw, ffn):
    """A gated product reads gate and up rows with blocks of their own; under tensor or expert parallelism and with sandwich norms the product is an
    ungated one, which reads those of one matrix (the halves of 304 and 1008 rows end inside a block)."""
    model = make(preset, "cpu", ffn, **kw)
    model.enable_block_scaled("fp8_block")
    w = model.mx[model.store.params["layers.0.mlp.gate_up.weight"].data_ptr()]
    assert w.halves == (2 if preset == "qwen3-smoke" and not kw else 1)
    assert w.whole == (w.halves == 1 or ffn % 128 == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("ffn", [1024, 304, 1008])
@pytest.mark.parametrize("preset,kw", LAYERS[:3])
def test_every_layer_answers_whatever_its_width(preset, kw, ffn):
    """Prompts, decode-sized passes and passes that keep activations, through dense layers whose gate and up rows end inside a block. 8 bits are off by
    0.04 a product, as one value in 8 bits by 0.03 at most; three products follow one another at most and gates count once more: 0.04 sqrt(7) = 0.11."""
    model = make(preset, "cuda", ffn, **kw)
    x = torch.randn(150, model.cfg.hidden_size, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    pos = torch.arange(150, dtype=torch.int32, device="cuda")
    for T in (9, 150):
        cu = torch.tensor([0, T], dtype=torch.int32, device="cuda")
        model.mx = {}
        want = model.layer_forward(0, x[:T], pos[:T], cu, T)
        wide = x.repeat(20, 1) if T == 150 else x[:T]
        bf16 = model._gated(wide, model.store.params["layers.0.mlp.gate_up.weight"], keep=True)
        model.enable_block_scaled("fp8_block")
        calls = []
        linear = model._fp8_linear
        model._fp8_linear = lambda *a: calls.append(1) or linear(*a)
        got = model.layer_forward(0, x[:T], pos[:T], cu, T)
        del model._fp8_linear
        assert len(calls) >= (2 if kw else 3)  # (rows of a sharded product are exchanged in bf16)
        added = (want.float() - x[:T].float()).norm()
        assert 0 < (got.float() - want.float()).norm() <= 0.15 * added
        kept = model._gated(wide, model.store.params["layers.0.mlp.gate_up.weight"], keep=True)
        for a, b in zip(kept, bf16):
            assert (a.float() - b.float()).norm() <= 0.15 * b.float().norm()
    model.check_status()
