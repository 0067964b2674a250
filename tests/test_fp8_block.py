"""Calls of the block-scaled 8-bit operators that cannot be answered are refused with a message before anything is launched: shapes and types
first, wherever the tensors lie, then the device."""
import pytest
import torch

from miles_b200 import _build
from miles_b200.ops import reference as R

E4 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def C():
    from miles_b200.ops import _ext

    if _build.needs_build():
        pytest.skip("the extension has not been built here")
    return _ext.load(required=True)


def q8(*shape):
    return torch.zeros(shape, dtype=torch.uint8).view(E4)


def f32(*shape):
    return torch.zeros(shape)


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def i32(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def linear(C, **over):
    a = dict(xq=q8(4, 256), xs=f32(4, 2), wq=q8(64, 256), ws=f32(1, 2), halves=1) | over
    return C.fp8_linear(**a)


@pytest.mark.parametrize("over,words", [
    (dict(), "CUDA tensor"),
    (dict(xq=bf(4, 256)), "float8_e4m3fn matrix"),
    (dict(xq=q8(4, 2, 128)), "float8_e4m3fn matrix"),
    (dict(xq=q8(256, 4).t()), "contiguous rows"),
    (dict(xq=q8(4, 250), xs=f32(4, 2), wq=q8(64, 250)), "multiple of 16 wide"),
    (dict(xq=q8(4, 0), xs=f32(4, 0), wq=q8(64, 0), ws=f32(1, 0)), "multiple of 16 wide"),
    (dict(xq=q8(4, 264)[:, :256]), "16 bytes apart"),
    (dict(xq=q8(1, 256).expand(4, 256)), "16 bytes apart"),
    (dict(xs=f32(4, 3)), "x: scales"),
    (dict(xs=f32(2, 4).t()), "x: scales"),
    (dict(xs=f32(4, 2).double()), "x: scales"),
    (dict(wq=q8(64, 128)), "x is 256 wide"),
    (dict(wq=q8(2, 64, 256)), "weight must be"),
    (dict(wq=q8(64, 512)[:, :256]), "weight must be"),
    (dict(ws=f32(2, 2)), "weight: scales"),
    (dict(ws=f32(1, 1)), "weight: scales"),
    (dict(halves=2), "reads one matrix"),
    (dict(halves=3), "halves is 1"),
    (dict(residual=bf(4, 63)), "residual must be"),
    (dict(tile_group=i32(1, 4)), "given together"),
    (dict(tile_group=i32(1, 4), num_tiles=i32(1)), "weight must be"),
    (dict(tile_group=i32(1, 3), num_tiles=i32(1), wq=q8(2, 64, 256), ws=f32(2, 1, 2)), "tile_group must be"),
    (dict(tile_group=i32(1, 4).long(), num_tiles=i32(1), wq=q8(2, 64, 256), ws=f32(2, 1, 2)), "tile_group must be"),
    (dict(tile_group=i32(1, 4), num_tiles=i32(0), wq=q8(2, 64, 256), ws=f32(2, 1, 2)), "num_tiles"),
    (dict(status=f32(1)), "status"),
])
def test_linear_refusals(C, over, words):
    if "residual" in over:  # (looked at after the operands' device: on the CPU that is what is refused)
        words = "CUDA tensor"
    with pytest.raises(RuntimeError, match=words):
        linear(C, **over)


@pytest.mark.parametrize("over,words", [
    (dict(), "CUDA tensor"),
    (dict(wq=q8(63, 256)), "even number"),
    (dict(wq=q8(40, 256), ws=f32(2, 2)), "multiple of 16 wide"),
    (dict(halves=1), "reads a gate-up weight"),
    (dict(ws=f32(1, 2)), "weight: scales"),
])
def test_gated_refusals(C, over, words):
    a = dict(xq=q8(4, 256), xs=f32(4, 2), wq=q8(64, 256), ws=f32(2, 2), halves=2) | over
    if over.get("wq") is not None and over["wq"].shape[0] == 63:
        words = "halves is 1, or 2"
    with pytest.raises(RuntimeError, match=words):
        C.fp8_gated_linear(**a)


@pytest.mark.parametrize("call,words", [
    (lambda C: C.fp8_quantize_rows(bf(4, 128)), "CUDA tensor"),
    (lambda C: C.fp8_quantize_rows(f32(4, 128)), "bf16 matrix"),
    (lambda C: C.fp8_quantize_rows(bf(4, 120)), "multiple of 16 wide"),
    (lambda C: C.fp8_quantize_rows(bf(1, 128).expand(4, 128)), "overlap"),
    (lambda C: C.fp8_quantize_rows(bf(128, 4).t()), "contiguous rows"),
    (lambda C: C.fp8_rmsnorm_rows(bf(4, 32784), bf(32784), 1e-6), "at most 32768"),
    (lambda C: C.fp8_rmsnorm_rows(bf(4, 128), bf(64), 1e-6), "weight must be"),
    (lambda C: C.fp8_rmsnorm_rows(bf(4, 128), f32(128), 1e-6), "weight must be"),
    (lambda C: C.fp8_rmsnorm_rows(bf(4, 128), bf(128), 1e-6, bf(3, 128)), "residual must be"),
    (lambda C: C.fp8_permute_rows(q8(4, 128), f32(4, 1), i32(8).long(), i32(2), 2), "src must be"),
    (lambda C: C.fp8_permute_rows(q8(4, 128), f32(4, 1), i32(8), i32(1), 2), "num_tiles"),
    (lambda C: C.fp8_permute_rows(q8(4, 128), f32(4, 1), i32(8), i32(2), 0), "top_k"),
    (lambda C: C.fp8_permute_rows(q8(4, 128), f32(4, 1), i32(8), i32(2), 2), "CUDA tensor"),
])
def test_row_refusals(C, call, words):
    with pytest.raises(RuntimeError, match=words):
        call(C)


@pytest.mark.parametrize("shape,halves", [((64,), 1), ((64, 120), 1), ((63, 128), 2), ((64, 128), 3), ((0, 128), 1)])
def test_weights_that_are_refused(shape, halves):
    from miles_b200.ops.fp8_block import quantize_weight

    with pytest.raises(ValueError, match="weights are"):
        quantize_weight(bf(*shape), halves)


@pytest.mark.parametrize("shape,halves,blocks", [((300, 272), 1, (3, 3)), ((320, 144), 2, (4, 2)), ((5, 96, 128), 2, (5, 2, 1)), ((5, 256, 128), 1, (5, 2, 1))])
def test_blocks_of_a_weight(shape, halves, blocks):
    from miles_b200.ops.fp8_block import quantize_weight

    w = torch.randn(shape, generator=torch.Generator().manual_seed(1)).bfloat16()
    r = quantize_weight(w, halves)
    assert r.q.shape == shape and r.q.dtype == E4 and r.scales.shape == blocks
    v = r.dequantize().double()
    # half a step of E4M3, below its normal values 2^-10 scales, and the two fp32 roundings of a quotient and a product
    assert ((v - w.double()).abs() <= (2.0 ** -4 + 2.0 ** -22) * w.double().abs() + 2.0 ** -10 * r.scales.max().item()).all()
    if halves == 2:
        half = quantize_weight(w[..., :shape[-2] // 2, :])
        assert torch.equal(half.scales, r.scales[..., :blocks[-2] // 2, :])


def test_rows_of_the_oracle():
    x = torch.randn(5, 272, generator=torch.Generator().manual_seed(2)) * 3
    x[1] = 0
    q, s = R.fp8_rows_quant(x)
    assert q.shape == (5, 272) and s.shape == (5, 3) and (s[1] == torch.tensor(1e-10) / 448).all()
    assert ((R.fp8_rows_dequant(q, s) - x).abs() <= (2.0 ** -4 + 2.0 ** -22) * x.abs() + 2.0 ** -10 * s.max()).all()
