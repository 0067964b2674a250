"""Models that serve from E4M3 copies of their weights with a scale for each 128 x 128 (``enable_block_scaled("fp8_block")``)."""
import pytest
import torch

from miles_b200.engine import Engine, SamplingParams
from miles_b200.models import ParamStore, build_model, get_config
from miles_b200.ops import fp8_block as F8

pytestmark = pytest.mark.gpu
PRESETS = ["qwen3-smoke", "qwen3-smoke-moe", "llama3-smoke", "mixtral-smoke", "glm4moe-smoke", "glm4-smoke", "qwen2moe-smoke"]


def make(preset, std=0.05):
    store = ParamStore(get_config(preset), "cuda", torch.bfloat16, init_std=std, seed=5)
    return build_model(store.cfg, store, "b200")


def scores(model, lens=(150, 90)):
    T = sum(lens)
    tokens = torch.randint(0, model.cfg.vocab_size, (T,), generator=torch.Generator().manual_seed(1)).cuda().int()
    pos = torch.cat([torch.arange(n) for n in lens]).cuda().int()
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    rows = torch.arange(0, T - 1).cuda()
    lp, _ = model.forward_logprobs(tokens, pos, cu, rows, tokens[(rows + 1).long()], 1.0)
    model.check_status()
    return lp


class Formulas:
    """The operators from their definitions in 64 bits, with the types and roundings of `ops.fp8_block`."""

    @staticmethod
    def wide(w):
        one = lambda q, s: q.double() * s.double().repeat_interleave(128, 0)[:q.shape[0]].repeat_interleave(128, 1)[:, :q.shape[1]]  # noqa: E731
        return torch.cat([one(q, s) for q, s in zip(w.q.chunk(w.halves), w.scales.chunk(w.halves))])

    @staticmethod
    def rows(v):
        blocks = -(-v.shape[1] // 128)
        s = torch.stack([b.abs().amax(1) for b in v.split(128, 1)], 1).clamp_min(1e-10).div(448).float()
        assert s.shape[1] == blocks
        return F8.Fp8Rows((v / s.double().repeat_interleave(128, 1)[:, :v.shape[1]]).float().clamp(-448, 448).to(torch.float8_e4m3fn), s)

    @classmethod
    def values(cls, x):
        x = x if isinstance(x, F8.Fp8Rows) else cls.rows(x.double())
        return x.q.double() * x.scales.double().repeat_interleave(128, 1)[:, :x.q.shape[1]]

    @classmethod
    def linear(cls, x, w, residual=None, out=None, status=None):
        y = cls.values(x) @ cls.wide(w).t()
        return (y if residual is None else y + residual.double()).bfloat16()

    @classmethod
    def by_expert(cls, x, w, tile_group, num_tiles):
        v = cls.values(x)
        y = v.new_zeros(v.shape[0], w.q.shape[1])
        for e, first, n, _ in tile_group[:int(num_tiles[0])].tolist():
            y[first:first + n] = v[first:first + n] @ cls.wide(F8.Fp8Weight(w.q[e], w.scales[e], w.halves)).t()
        return y

    @classmethod
    def grouped_linear(cls, x, w, tile_group, num_tiles, out=None, status=None):
        return cls.by_expert(x, w, tile_group, num_tiles).bfloat16()

    @classmethod
    def gated(cls, y):
        g, u = y.chunk(2, 1)
        return cls.rows(g * torch.sigmoid(g) * u)

    @classmethod
    def gated_linear(cls, x, w, status=None):
        return cls.gated(cls.values(x) @ cls.wide(w).t())

    @classmethod
    def grouped_gated_linear(cls, x, w, tile_group, num_tiles, status=None):
        return cls.gated(cls.by_expert(x, w, tile_group, num_tiles))

    @classmethod
    def rmsnorm_rows(cls, x, weight, eps, residual=None, keep=False):
        h = x if residual is None else (x.double() + residual.double()).bfloat16()
        y = h.double() / (h.double().square().mean(1, keepdim=True) + eps).sqrt() * weight.double()
        return cls.rows(y), h, y.bfloat16() if keep else None

    @classmethod
    def permute_rows(cls, x, src, num_tiles, top_k):
        at = (src.long().clamp_min(0) // top_k)
        return F8.Fp8Rows(x.q.view(torch.uint8)[at].view(torch.float8_e4m3fn), x.scales[at])


def tokens_of(model, lens=(150, 90)):
    tokens = torch.randint(0, model.cfg.vocab_size, (sum(lens),), generator=torch.Generator().manual_seed(1)).cuda()
    pos = torch.cat([torch.arange(n) for n in lens]).cuda().int()
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    return model.store.params["embed.weight"][tokens].contiguous(), pos, cu


def off(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm().clamp_min(1e-300)).item()


@pytest.mark.parametrize("preset", PRESETS)
def test_operators_inside_a_forward_are_the_formulas(preset, monkeypatch):
    """Every call that a model makes of an operator, against the formula on the same operands. Results part where a value lies at a border of its
    rounding: never by more than a step of bf16, 2^-7 of the value, and scales, which are fp32, by the sums' error of 2^-18."""
    model = make(preset)
    assert model.enable_block_scaled("fp8_block") >= 4 * (model.cfg.num_layers - 1)
    calls = []

    def watch(name, ours, formula):
        def call(*a, **k):
            got = ours(*a, **k)
            want = formula(*a, **{n: v for n, v in k.items() if n != "status"})
            for g, w in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
                live = slice(0, int(a[3][0]) and int(sum(a[2][:int(a[3][0]), 2])) if name.startswith("grouped") else None)
                if isinstance(g, F8.Fp8Rows):
                    assert off(g.scales[live], w.scales[live]) <= 2.0 ** -18 and off(g.q.float()[live], w.q.float()[live]) <= 2.0 ** -6
                elif g is not None:
                    assert off(g[live], w[live]) <= 2.0 ** -8
            calls.append(name)
            return got
        return call

    x, pos, cu = tokens_of(model)
    with monkeypatch.context() as m:
        for name in ("linear", "grouped_linear", "gated_linear", "grouped_gated_linear", "rmsnorm_rows", "permute_rows"):
            m.setattr(F8, name, watch(name, getattr(F8, name), getattr(Formulas, name)))
        for i in range(model.cfg.num_layers):
            x = model.layer_forward(i, x, pos, cu, 150)
    model.check_status()
    per = {"rmsnorm_rows", "linear"} if not model.cfg.post_norms else {"linear"}
    moe = {model.cfg.layer_is_moe(i) for i in range(model.cfg.num_layers)}
    assert per <= set(calls) and (True not in moe or {"permute_rows", "grouped_gated_linear", "grouped_linear"} <= set(calls))
    assert False not in moe or model.cfg.post_norms or "gated_linear" in calls


@pytest.mark.parametrize("preset", PRESETS)
def test_layers_stay_close_to_bf16(preset):
    """What a layer adds to the residual stream, from 8-bit operands and from bf16. A value rounded to E4M3 is off by 2^-4 / sqrt(3) of itself in the
    mean square at most, about 0.03, so a product of two such operands by 0.04; three products follow one another on the longest way (gates
    count once more), and attention mixes values of as much noise: 0.04 sqrt(7) = 0.11. A wrong operand would be off by more than 1."""
    model = make(preset, 0.02)
    x, pos, cu = tokens_of(model)
    for i in range(model.cfg.num_layers):
        model.mx = {}
        a, b = [], []
        want = model.layer_forward(i, x, pos, cu, 150, record=a)
        model.enable_block_scaled("fp8_block")
        y = model.layer_forward(i, x, pos, cu, 150, record=b)
        same = torch.ones(x.shape[0], dtype=torch.bool, device="cuda")
        for u, v in zip(a, b):  # (rows whose experts differ are not compared)
            same &= (u.sort(1).values == v.sort(1).values).all(1)
        assert same.float().mean() >= 0.5 and off((y.float() - x.float())[same], (want.float() - x.float())[same]) <= 0.15
        x = want
    model.check_status()


def test_training_passes_of_few_rows_and_other_formats():
    model = make("qwen3-smoke-moe")
    model.enable_block_scaled("fp8_block")
    few = scores(model, (5, 3))  # up to SMALL_T rows stay with the bf16 weights
    model.mx = {}
    assert torch.equal(few, scores(model, (5, 3)))
    ref = scores(model)
    model.enable_block_scaled("fp8_block")
    fp8 = scores(model)
    model.enable_block_scaled("mxfp8")
    mx = scores(model)
    model.enable_block_scaled("fp8_block")
    assert torch.equal(scores(model), fp8) and not torch.equal(mx, fp8) and not torch.equal(ref, fp8)


@pytest.mark.parametrize("preset", ["qwen3-smoke", "qwen3-smoke-moe"])
def test_weight_updates_reach_the_copies_where_they_are(preset):
    model = make(preset)
    model.enable_block_scaled("fp8_block")
    at = {k: (w.q.data_ptr(), w.scales.data_ptr()) for k, w in model.mx.items()}
    before = scores(model)
    model.store.params["layers.0.attn.o.weight"].mul_(0.5)
    model.refresh_block_scaled()
    assert at == {k: (w.q.data_ptr(), w.scales.data_ptr()) for k, w in model.mx.items()}
    after = scores(model)
    assert (after - before).abs().max().item() > 0
    fresh = make(preset)
    fresh.store.params["layers.0.attn.o.weight"].mul_(0.5)
    fresh.enable_block_scaled("fp8_block")
    assert torch.equal(scores(fresh), after)


@pytest.mark.parametrize("preset", ["qwen3-smoke", "qwen3-smoke-moe"])
def test_engine_decodes_with_captured_graphs_across_a_weight_update(preset):
    """20 running rows: decode steps take the 8-bit products. Captured steps give the tokens of eager ones, before and after an update."""
    out = {}
    for graph in (False, True):
        model = make(preset, 0.02)
        model.enable_block_scaled("fp8_block")
        eng = Engine(model, max_running=20, page_size=64, max_seq_len=256, use_cuda_graph=graph, prefix_cache=False)
        g = torch.Generator().manual_seed(0)
        prompts = [torch.randint(0, model.cfg.vocab_size, (20 + 3 * i,), generator=g).tolist() for i in range(20)]
        sps = [SamplingParams(temperature=0.0, max_new_tokens=12, ignore_eos=True) for _ in prompts]
        first = [r["output_ids"] for r in eng.generate(prompts, sps)]
        model.store.params["layers.1.attn.o.weight"].mul_(-3.0)
        model.refresh_block_scaled()
        second = [r["output_ids"] for r in eng.generate(prompts, sps)]
        model.check_status()
        assert first != second
        out[graph] = (first, second)
    assert out[False] == out[True]


def test_server_and_trainer_name_the_format():
    from miles_b200.engine.server import build_from_args

    eng, _, _ = build_from_args(["--model-preset", "qwen3-smoke-moe", "--quantization", "fp8_block", "--max-running-requests", "4", "--context-length", "256",
                                 "--mem-fraction-static", "0.2"])
    assert eng.model.mx_kind == "fp8_block" and len(eng.model.mx) == 8
