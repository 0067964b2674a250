"""What a product adds to and writes is looked at before the device, like its other operands."""
import pytest
import torch

from miles_b200 import _build

E4 = torch.float8_e4m3fn


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("name", ["residual", "out"])
@pytest.mark.parametrize("bad,words", [
    (bf(4, 63), "must be a CUDA tensor \\[4, 64\\], got \\[4, 63\\]"),
    (bf(5, 64), "must be a CUDA tensor \\[4, 64\\], got \\[5, 64\\]"),
    (bf(4, 64).float(), "must be a bf16 matrix"),
    (bf(4, 64, 1), "must be a bf16 matrix"),
    (bf(64, 4).t(), "must be a bf16 matrix"),
    (bf(1, 64).expand(4, 64), "rows must not overlap"),
    (bf(4, 64), "must be a CUDA tensor on the device"),
])
def test_residual_and_out(name, bad, words):
    from miles_b200.ops import _ext

    if _build.needs_build():
        pytest.skip("the extension has not been built here")
    z = torch.zeros
    who = "x " if "on the device" in words else f"{name}:? "
    with pytest.raises(RuntimeError, match=who + words):
        _ext.load(required=True).fp8_linear(z(4, 256, dtype=torch.uint8).view(E4), z(4, 2), z(64, 256, dtype=torch.uint8).view(E4), z(1, 2), 1, **{name: bad})
