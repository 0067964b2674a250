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


@pytest.mark.gpu
@pytest.mark.parametrize("K", [16, 144, 2048])
def test_entries_of_no_token_leave_zeros(K):
    """Rows of the expert order that belong to no token: zeros, with the scale of an empty block."""
    from miles_b200.ops import fp8_block as F8

    T, top_k = 5, 2
    x = F8.quantize_rows(torch.randn(T, K, generator=torch.Generator().manual_seed(4)).bfloat16().cuda())
    src = torch.tensor([3, -1, 9, 0, -7, -1, 4, 2, -1], dtype=torch.int32)
    live = 8
    y = F8.permute_rows(x, src.cuda(), torch.tensor([1, live], dtype=torch.int32, device="cuda"), top_k)
    for i, pair in enumerate(src[:live].tolist()):
        q, s = y.q[i].float(), y.scales[i]
        if pair < 0:
            assert (q == 0).all() and torch.equal(s, torch.full_like(s, 1e-10) / torch.full_like(s, 448.0))
        else:
            assert torch.equal(q, x.q[pair // top_k].float()) and torch.equal(s, x.scales[pair // top_k])
