"""The largest number of rows, and which kernel is chosen up to it."""
import pytest
import torch

from miles_b200 import _build

LIMIT = 2 ** 31 - 256


@pytest.fixture(scope="module")
def C():
    from miles_b200.ops import _ext

    if _build.needs_build():
        pytest.skip("the extension has not been built here")
    return _ext.load(required=True)


def rows(n):
    return torch.empty(n, 16, dtype=torch.float8_e4m3fn, device="meta"), torch.empty(n, 1, device="meta")


@pytest.mark.parametrize("n,words", [(LIMIT, "CUDA tensor"), (LIMIT + 1, "2\\^31 - 256 rows"), (2 ** 31 - 129, "2\\^31 - 256 rows"), (2 ** 31 + 5, "2\\^31 - 256 rows")])
def test_rows_that_tiles_cannot_reach_are_refused(C, n, words):
    q, s = rows(n)
    weight = torch.empty(32, 16, dtype=torch.float8_e4m3fn, device="meta"), torch.empty(1, 1, device="meta")
    gate_up = weight[0], torch.empty(2, 1, device="meta")
    i32 = lambda *shape: torch.empty(shape, dtype=torch.int32, device="meta")  # noqa: E731
    for call in (lambda: C.fp8_linear(q, s, *weight, 1), lambda: C.fp8_gated_linear(q, s, *gate_up, 2), lambda: C.fp8_permute_rows(q, s, i32(4), i32(2), 1)):
        with pytest.raises(RuntimeError, match=words):
            call()


def test_many_rows_an_expert_go_to_pairs(C):
    """Up to the limit: an average of rows is formed from half as many again."""
    for n in (2 ** 20, 2 ** 30, 3 * 2 ** 29, LIMIT):
        assert C.fp8_grouped_launches(n, 8, 2048, 768, False, 1 << 23) == 2
