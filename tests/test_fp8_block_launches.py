"""How many kernels a product by expert is: what the engines' launch counts say of it."""
import pytest
import torch

from miles_b200 import _build

# rows, experts, N, K, gated: both sides of the choice between the kernels, the gated limit on rows and the ungated one
SIZES = [(64 * 8, 128, 1536, 2048, True), (64 * 8, 128, 2048, 768, False), (48 * 128, 128, 1536, 2048, True), (48 * 128, 128, 2048, 768, False),
         (128 * 128, 128, 1536, 2048, True), (128 * 128, 128, 2048, 768, False), (72, 128, 2048, 768, False), (300, 8, 512, 272, True), (300, 8, 272, 512, False)]


def C():
    from miles_b200.ops import _ext

    if not torch.cuda.is_available() and _build.needs_build():
        pytest.skip("the extension has not been built here")
    return _ext.load(required=True)


def tiles_of(rows, experts):
    per = [rows // experts + (e < rows % experts) for e in range(experts)]
    tiles, first = [], 0
    for e, n in enumerate(per):
        tiles += [(e, first + a, min(128, n - a), 0) for a in range(0, n, 128)]
        first += n
    return tiles


def test_the_sizes_decide():
    said = {s: C().fp8_grouped_launches(*s, len(tiles_of(*s[:2]))) for s in SIZES}
    assert set(said.values()) == {1, 2}
    assert said[SIZES[2]] == said[SIZES[4]] == said[SIZES[5]] == 2 and said[SIZES[0]] == said[SIZES[6]] == 1
    assert C().fp8_grouped_launches(0, 8, 512, 256, False, 4) == C().fp8_grouped_launches(64, 8, 512, 256, False, 0) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("size", SIZES)
def test_as_many_kernels_as_it_says(size):
    from cuda.bindings import runtime

    from miles_b200.ops import fp8_block as F8

    rows, experts, n, k, gated = size
    tiles = tiles_of(rows, experts)
    tg, nt = torch.tensor(tiles, dtype=torch.int32, device="cuda"), torch.tensor([len(tiles), rows], dtype=torch.int32, device="cuda")
    x = F8.Fp8Rows(torch.zeros(rows, k, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn), torch.ones(rows, -(-k // 128), device="cuda"))
    w = F8.quantize_weight(torch.zeros(experts, n, k, dtype=torch.bfloat16, device="cuda"), 2 if gated else 1)
    call = lambda: (F8.grouped_gated_linear if gated else F8.grouped_linear)(x, w, tg, nt)  # noqa: E731
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        call()
    err, _, count = runtime.cudaGraphGetNodes(g.raw_cuda_graph(), 0)
    assert int(err) == 0 and count == C().fp8_grouped_launches(rows, experts, n, k, gated, len(tiles))
