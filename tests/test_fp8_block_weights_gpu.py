"""Weights of more rows than 65535 blocks of 128: experts together are one matrix for the quantiser."""
import pytest
import torch

from miles_b200.ops import fp8_block as F8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(65536 * 128 + 48, 16), (65540, 128, 16)])
def test_every_block_is_quantised(shape):
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
    r = F8.quantize_weight(w)
    rows = w.view(-1, 16)
    padded = torch.nn.functional.pad(rows, (0, 0, 0, -rows.shape[0] % 128)).view(-1, 128 * 16).float()
    scales = padded.abs().amax(1).clamp_min(1e-10) / 448
    assert (r.scales.flatten() / scales - 1).abs().max().item() <= 2.0 ** -22  # (a quotient, here by a reciprocal: two roundings of 2^-24 each)
    values = r.q.view(-1, 16).float() * r.scales.flatten().repeat_interleave(128)[:rows.shape[0], None]
    # half a step of E4M3, below its normal values 2^-10 scales, and the fp32 roundings of reciprocal, quotient and product
    limit = (2.0 ** -4 + 2.0 ** -21) * rows.float().abs() + 2.0 ** -10 * r.scales.flatten().repeat_interleave(128)[:rows.shape[0], None]
    assert ((values - rows.float()).abs() <= limit).all()
