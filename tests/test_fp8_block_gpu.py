"""Serving in block-scaled 8 bits against the definitions in 64 bits.

Tolerances, all from the roundings: a value rounded to 8 bits is off by half a step, 2^-4 of itself or (below the smallest normal value) 2^-10
scales; to bf16 by 2^-8 of itself. A sum over K in fp32 is off by at most 2^-23 of the sum of the magnitudes for each addition on the way of a
term: the 128 of its block and one for each block. What comes of these in a quotient or a product is added where it is used.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
U8, TINY8, UBF = 2.0 ** -4, 2.0 ** -10, 2.0 ** -8


@pytest.fixture(scope="module")
def F8():
    from miles_b200.ops import fp8_block

    return fp8_block


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def acts(rows, k, g):
    channel = torch.randn(k, generator=g, device=DEV).exp()
    return (torch.randn(rows, k, generator=g, device=DEV) * channel).bfloat16()


def rows64(r):
    return r.q.double() * r.scales.double().repeat_interleave(128, 1)[:, :r.q.shape[1]]


def weight64(w):
    def one(q, s):
        return q.double() * s.double().repeat_interleave(128, 0)[:q.shape[0]].repeat_interleave(128, 1)[:, :q.shape[1]]

    qs, ss = (w.q, w.scales) if w.q.dim() == 3 else (w.q[None], w.scales[None])
    out = torch.stack([torch.cat([one(a, b) for a, b in zip(q.chunk(w.halves), s.chunk(w.halves))]) for q, s in zip(qs, ss)])
    return out if w.q.dim() == 3 else out[0]


def check_rows(got, want, err=0.0):
    """``got`` are 8-bit rows of ``want`` (64 bits), which the kernel knew up to ``err`` (a number or a matrix)."""
    T, K = want.shape
    assert got.q.shape == (T, K) and got.scales.shape == (T, -(-K // 128)) and got.q.dtype == torch.float8_e4m3fn
    err = err if torch.is_tensor(err) else torch.full_like(want, err)
    for b in range(got.scales.shape[1]):
        c = slice(b * 128, (b + 1) * 128)
        s = got.scales[:, b].double()
        true = want[:, c].abs().amax(1).clamp_min(1e-10) / 448
        slack = err[:, c].amax(1) / 448 + 2.0 ** -22 * true
        assert ((s - true).abs() <= slack).all(), ((s - true).abs() / slack).max().item()
        off = (got.q[:, c].double() * s[:, None] - want[:, c]).abs()
        most = U8 * want[:, c].abs() + TINY8 * s[:, None] + 1.1 * err[:, c] + 2.0 ** -20 * want[:, c].abs()
        assert (off <= most).all(), (off / most).max().item()


def product64(x, w):
    """The product in 64 bits, and what its fp32 sum may be off by."""
    a, b = rows64(x), weight64(w)
    c = (128 + x.scales.shape[1] + 4) * 2.0 ** -23
    return a @ b.t(), c * (a.abs() @ b.abs().t())


def check_bf16(y, want, err):
    off = (y.double() - want).abs()
    most = UBF * want.abs() + 1.01 * err + 1e-30
    assert torch.isfinite(y).all() and (off <= most).all(), (off / most).max().item()


def gated64(y, err):
    """silu(gate) * up and its error: |d silu| <= 1.1 |dg|, and eight roundings of its own."""
    (g, u), (eg, eu) = y.chunk(2, 1), err.chunk(2, 1)
    si = g * torch.sigmoid(g)
    return si * u, 1.1 * eg * u.abs() + si.abs() * eu + 1.1 * eg * eu + (8 + g.abs() / 4) * 2.0 ** -23 * (si * u).abs()


# ------------------------------------------------------------------------------------------------ rows
@pytest.mark.parametrize("T,K", [(1, 16), (3, 128), (5, 144), (77, 2048), (2, 2064), (9, 9728), (1, 32784), (0, 256)])
def test_quantize_rows(F8, T, K):
    from miles_b200.ops import reference as R

    x = acts(T, K, gen(K))
    if T:
        x[0, :min(K, 128)] = 0
    got = F8.quantize_rows(x)
    check_rows(got, x.double())
    q, s = R.fp8_rows_quant(x.cpu())
    assert torch.equal(got.scales.cpu(), s) and torch.equal(got.q.cpu().view(torch.uint8), q.view(torch.uint8))  # the formula's values bit for bit


def test_quantize_rows_apart_and_extremes(F8):
    wide = acts(7, 512, gen(1))
    x = wide[:, 128:400]
    assert torch.equal(F8.quantize_rows(x).q.view(torch.uint8), F8.quantize_rows(x.contiguous()).q.view(torch.uint8))
    top = torch.finfo(torch.bfloat16).max
    x = torch.tensor([[top, -top, 1.0, 0.0] * 64, [1e-40, -2e-39, 0.0, 3e-38] * 64], device=DEV).bfloat16()
    check_rows(F8.quantize_rows(x), x.double())
    x = torch.ones(2, 256, device=DEV).bfloat16()
    x[0, 3], x[1, 200] = float("nan"), float("-inf")
    r = F8.quantize_rows(x)
    assert r.scales[0, 0].isnan() and r.scales[1, 1].isinf() and r.scales[0, 1].cpu() == r.scales[1, 0].cpu() == torch.tensor(1.0) / 448
    v = rows64(r)
    # (448 times the fp32 number next to 1 / 448, which is off by 2^-24 of itself)
    assert v[0, :128].isnan().all() and v[1, 128:].isnan().all() and ((v[0, 128:] - 1).abs() <= 2.0 ** -24).all() and ((v[1, :128] - 1).abs() <= 2.0 ** -24).all()


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("T,H", [(1, 16), (2, 2048), (3, 2560), (129, 1040), (300, 4096), (5, 8192), (4, 8208), (2, 32768), (0, 2048)])
def test_rmsnorm_rows(F8, T, H, residual):
    g = gen(H + residual)
    x, w = acts(T, H, g), (1 + 0.2 * torch.randn(H, generator=g, device=DEV)).bfloat16()
    res = acts(T, H, g) if residual else None
    rows, h, y = F8.rmsnorm_rows(x, w, 1e-6, res, keep=True)
    if residual:
        want = x.double() + res.double()
        assert ((h.double() - want).abs() <= UBF * want.abs()).all()
    else:
        assert h.data_ptr() == x.data_ptr()
    h64 = h.double()
    y64 = h64 / (h64.square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
    # the mean of squares adds up 8 VPT terms a thread, 5 + 32 partial sums: under 80 additions, halved by the root; five more roundings
    rel = 45 * 2.0 ** -24
    assert ((y.double() - y64).abs() <= (UBF + 2 * rel) * y64.abs()).all()
    check_rows(rows, y64, rel * y64.abs())
    again = F8.rmsnorm_rows(x, w, 1e-6, res)
    assert again[2] is None and torch.equal(again[0].q.view(torch.uint8), rows.q.view(torch.uint8))


def test_rmsnorm_rows_apart_and_zero_rows(F8):
    g = gen(5)
    wide, w = acts(6, 1024, g), torch.ones(512, device=DEV).bfloat16()
    res = acts(6, 1536, g)[:, 512:1024]
    a = F8.rmsnorm_rows(wide[:, 256:768], w, 1e-6, res)
    b = F8.rmsnorm_rows(wide[:, 256:768].contiguous(), w, 1e-6, res.contiguous())
    assert torch.equal(a[0].q.view(torch.uint8), b[0].q.view(torch.uint8)) and torch.equal(a[1], b[1]) and torch.equal(a[0].scales, b[0].scales)
    z = F8.rmsnorm_rows(torch.zeros(3, 512, device=DEV).bfloat16(), w, 1e-6)[0]
    assert (z.q.float() == 0).all() and (z.scales.cpu() == torch.tensor(1e-10) / 448).all()  # (the quotient; on a GPU torch multiplies by 1 / 448)


@pytest.mark.parametrize("T,K,top_k,E", [(1, 16, 1, 4), (37, 144, 3, 8), (200, 2048, 8, 128)])
def test_permute_rows(F8, ext, T, K, top_k, E):
    g = gen(T)
    x = F8.quantize_rows(acts(T, K, g))
    ids = torch.rand(T, E, generator=g, device=DEV).topk(top_k, 1).indices.int()
    _, _, dest, src, _, nt = ext.moe_build_permutation(ids, E, T * top_k + 40, 1)
    p = F8.permute_rows(x, src, nt, top_k)
    live = int(nt[1])
    assert live == T * top_k
    at = dest.view(T, top_k).long()
    for k in range(top_k):
        assert torch.equal(p.q.view(torch.uint8)[at[:, k]], x.q.view(torch.uint8)) and torch.equal(p.scales[at[:, k]], x.scales)


# ------------------------------------------------------------------------------------------------ products
SIZES = [(1, 128, 128), (1, 5120, 2048), (2, 16, 16), (7, 1, 144), (16, 136, 1040), (17, 300, 400), (33, 547, 512), (64, 2048, 4096), (100, 129, 9728), (128, 256, 256),
         (129, 257, 272), (300, 1000, 1040), (513, 768, 2048), (2000, 2560, 512), (4100, 1304, 144)]


@pytest.mark.parametrize("T,N,K", SIZES)
def test_linear(F8, T, N, K):
    g = gen(T + N)
    x = F8.quantize_rows(acts(T, K, g))
    w = F8.quantize_weight((torch.randn(N, K, generator=g, device=DEV) * torch.randn(N, 1, generator=g, device=DEV).exp()).bfloat16())
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    want, err = product64(x, w)
    check_bf16(F8.linear(x, w, status=status), want, err)
    res = acts(T, N, g)
    check_bf16(F8.linear(x, w, res, status=status), want + res.double(), err + 2.0 ** -23 * (want.abs() + res.double().abs()))
    assert int(status) == 0


def test_linear_scales_of_any_value(F8):
    """Every block of both operands has a scale of another magnitude, so that a wrong one shows at once."""
    g = gen(9)
    T, N, K = 200, 400, 1040
    x = (torch.randn(T, K, generator=g, device=DEV) * torch.exp(2 * torch.randn(T, 9, generator=g, device=DEV)).repeat_interleave(128, 1)[:, :K]).bfloat16()
    mag = torch.exp(2 * torch.randn(4, 9, generator=g, device=DEV)).repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    x, w = F8.quantize_rows(x), F8.quantize_weight((torch.randn(N, K, generator=g, device=DEV) * mag).bfloat16())
    for rows in (slice(None), slice(0, 20)):
        part = F8.Fp8Rows(x.q[rows], x.scales[rows])
        check_bf16(F8.linear(part, w), *product64(part, w))


@pytest.mark.parametrize("T", [5, 40, 300])
@pytest.mark.parametrize("N", [250, 256])
def test_linear_operands_apart(F8, T, N):
    """Rows of x, the residual and the result that are apart, results that are not 16-byte aligned, the residual as the result."""
    g = gen(T)
    K = 272
    x = F8.quantize_rows(acts(T, K, g))
    w = F8.quantize_weight(torch.randn(N, K, generator=g, device=DEV).bfloat16())
    wide = torch.zeros(T, K + 48, dtype=torch.uint8, device=DEV)
    wide[:, 32:32 + K] = x.q.view(torch.uint8)
    apart = F8.Fp8Rows(wide.view(torch.float8_e4m3fn)[:, 32:32 + K], x.scales)
    want, err = product64(x, w)
    for first, more in ((0, 8), (3, 7), (8, 3)):
        buf = torch.full((T, N + first + more), 7.0, device=DEV).bfloat16()
        res = acts(T, N + 5, g)[:, 2:2 + N]
        got = F8.linear(apart, w, res, out=buf[:, first:first + N])
        check_bf16(got, want + res.double(), err + 2.0 ** -23 * (want.abs() + res.double().abs()))
        assert (buf[:, :first] == 7).all() and (buf[:, first + N:] == 7).all()
    y = res.clone()
    assert torch.equal(F8.linear(x, w, y, out=y), F8.linear(x, w, res))


@pytest.mark.parametrize("T", [257, 300, 511])
@pytest.mark.parametrize("N", [8, 200, 264, 1001])
def test_linear_into_part_of_a_wide_result(F8, T, N):
    """The last rows and columns end inside a box of 32 x 64 that leaves at once; what lies around the result stays."""
    g = gen(T + N)
    x, w = F8.quantize_rows(acts(T, 400, g)), F8.quantize_weight(torch.randn(N, 400, generator=g, device=DEV).bfloat16())
    want, err = product64(x, w)
    pad = -N % 8
    for residual in (False, True):
        buf = torch.full((T + 40, N + pad + 80), 7.0, device=DEV).bfloat16()
        res = acts(T, N, g) if residual else None
        got = F8.linear(x, w, res, out=buf[3:3 + T, 16:16 + N])
        if residual:
            check_bf16(got, want + res.double(), err + 2.0 ** -23 * (want.abs() + res.double().abs()))
        else:
            check_bf16(got, want, err)
        buf[3:3 + T, 16:16 + N] = 7.0
        assert (buf == 7).all()


@pytest.mark.parametrize("T", [2945, 2970])
@pytest.mark.parametrize("N,first,apart", [(968, 16, 16), (968, 3, 8), (1001, 8, 15), (1000, 8, 7)])
def test_linear_of_many_rows_into_part_of_a_wide_result(F8, T, N, first, apart):
    """The same where pairs of CTAs compute it: results and residuals whose rows are or are not multiples of 16 bytes apart, the residual as the result."""
    g = gen(T + N)
    x, w = F8.quantize_rows(acts(T, 144, g)), F8.quantize_weight(torch.randn(N, 144, generator=g, device=DEV).bfloat16())
    want, err = product64(x, w)
    buf = torch.full((T + 33, N + first + apart), 7.0, device=DEV).bfloat16()
    out = buf[1:1 + T, first:first + N]
    check_bf16(F8.linear(x, w, out=out), want, err)
    for res in (acts(T, N, g), acts(T, N + 8, g)[:, 8:], acts(T, N + 3, g)[:, 2:2 + N]):
        check_bf16(F8.linear(x, w, res, out=out), want + res.double(), err + 2.0 ** -23 * (want.abs() + res.double().abs()))
    out.copy_(res)
    there = F8.linear(x, w, out, out=out).clone()
    assert torch.equal(there, F8.linear(x, w, res))
    out.fill_(7.0)
    assert (buf == 7).all()


def test_linear_of_no_rows_and_bf16_rows(F8):
    w = F8.quantize_weight(torch.randn(64, 128, device=DEV).bfloat16())
    assert F8.linear(F8.quantize_rows(torch.zeros(0, 128, device=DEV).bfloat16()), w).shape == (0, 64)
    x = acts(30, 128, gen(2))
    assert torch.equal(F8.linear(x, w), F8.linear(F8.quantize_rows(x), w))


def test_offsets_beyond_32_bits(F8):
    """Rows, results and weights whose places pass 2^31 elements: the last ones are right, and so are the first."""
    g = gen(8)
    T, N = 270000, 8192
    x = F8.quantize_rows(torch.randn(T, 128, generator=g, device=DEV).bfloat16())
    w = F8.quantize_weight(torch.randn(N, 128, generator=g, device=DEV).bfloat16())
    y = F8.linear(x, w)
    for rows in (slice(0, 60), slice(T - 60, T)):
        part = F8.Fp8Rows(x.q[rows], x.scales[rows])
        check_bf16(y[rows], *product64(part, w))
    r = F8.quantize_rows(y)
    normed, _, _ = F8.rmsnorm_rows(y, torch.ones(N, device=DEV).bfloat16(), 1e-6)
    for rows in (slice(0, 20), slice(T - 20, T)):
        check_rows(F8.Fp8Rows(r.q[rows], r.scales[rows]), y[rows].double())
        h = y[rows].double()
        want = h / (h.square().mean(1, keepdim=True) + 1e-6).sqrt()
        check_rows(F8.Fp8Rows(normed.q[rows], normed.scales[rows]), want, 45 * 2.0 ** -24 * want.abs())
    del y, r, normed
    E, N, K = 260, 2048, 4096  # 2.2 GB of weights
    q = torch.randint(0, 120, (E, N, K), generator=g, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn)
    w = F8.Fp8Weight(q, torch.rand(E, N // 128, K // 128, generator=g, device=DEV))
    for count in (3, 140):  # by either kernel
        x = F8.quantize_rows(acts(count * E, K, g))
        tiles = torch.tensor(tiles_of([count] * E), dtype=torch.int32, device=DEV)
        y = F8.grouped_linear(x, w, tiles, torch.tensor([len(tiles)], dtype=torch.int32, device=DEV))
        for e in (0, E - 1):
            rows = slice(e * count, (e + 1) * count)
            check_bf16(y[rows], *product64(F8.Fp8Rows(x.q[rows], x.scales[rows]), F8.Fp8Weight(w.q[e], w.scales[e])))


@pytest.mark.parametrize("T", [6, 300])
def test_the_status_word_is_left_alone(F8, T):
    """A code that another kernel left stays for the model to report."""
    g = gen(T)
    w = F8.quantize_weight(torch.randn(384, 256, generator=g, device=DEV).bfloat16(), 2)
    status = torch.full((1,), 17, dtype=torch.int32, device=DEV)
    F8.gated_linear(acts(T, 256, g), w, status)
    assert int(status) == 17


def test_linear_keeps_nan_and_infinities_in_their_rows(F8):
    g = gen(3)
    for T in (20, 200):
        x = acts(T, 256, g)
        w = F8.quantize_weight(torch.randn(130, 256, generator=g, device=DEV).bfloat16())
        clean = F8.linear(x, w)
        x[3, 5], x[11, 200] = float("nan"), float("inf")
        y = F8.linear(x, w)
        bad = torch.zeros(T, dtype=torch.bool, device=DEV)
        bad[[3, 11]] = True
        assert y[bad].isnan().all() and torch.equal(y[~bad], clean[~bad])


@pytest.mark.parametrize("T,I,K", [(1, 128, 128), (1, 768, 2048), (3, 16, 16), (20, 144, 400), (64, 768, 2048), (65, 300 // 16 * 16, 144), (130, 368, 1040), (700, 2048, 512),
                                   (3000, 1296, 272)])
def test_gated_linear(F8, T, I, K):
    g = gen(T + I)
    x = F8.quantize_rows(acts(T, K, g))
    w = F8.quantize_weight((torch.randn(2 * I, K, generator=g, device=DEV) * 2 / K ** 0.5).bfloat16(), halves=2)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = F8.gated_linear(x, w, status)
    check_rows(got, *gated64(*product64(x, w)))
    assert int(status) == 0


def test_gated_linear_of_large_gates(F8):
    """Gates far below zero leave zeros, far above the product; one that is NaN takes its block along."""
    x = F8.quantize_rows(torch.ones(4, 128, device=DEV).bfloat16())
    w = torch.ones(256, 128, device=DEV).bfloat16()
    w[:64], w[64:128] = -40.0, 40.0
    got = F8.gated_linear(x, F8.quantize_weight(w, halves=2))
    v = rows64(got)
    # (a product of 128 equal terms is exact; e^-5120 is zero)
    assert (v[:, :64] == 0).all() and ((v[:, 64:] - 5120 * 128.0).abs() <= 2.0 ** -20 * 5120 * 128).all()
    s = x.scales.clone()
    s[2] = float("nan")
    v = rows64(F8.gated_linear(F8.Fp8Rows(x.q, s), F8.quantize_weight(w, halves=2)))
    assert v[2].isnan().all() and v[[0, 1, 3]].isfinite().all()


def tiles_of(counts, first=0):
    out = []
    for g, c in enumerate(counts):
        out += [[g, first + a, min(128, c - a), 0] for a in range(0, c, 128)]
        first += c
    return out


GROUPS = {"few": [3, 0, 1, 0, 17, 2, 0, 9], "none": [0, 0, 0, 0], "many": [130, 0, 256, 1, 300, 127], "one": [0, 0, 1], "long": [0, 1500, 3],
          "wide": [2] * 100 + [0] * 20 + [40] * 8}


@pytest.mark.parametrize("name", GROUPS)
@pytest.mark.parametrize("N,K", [(256, 128), (2048, 768), (200, 272)])
def test_grouped_linear_and_rows_outside_tiles(F8, name, N, K):
    counts = GROUPS[name]
    g = gen(len(name) + N)
    lead, T = 5, sum(counts)  # five rows before the first expert's, six behind the last's: in no tile
    x = F8.quantize_rows(acts(lead + T + 6, K, g))
    w = F8.quantize_weight(torch.randn(len(counts), N, K, generator=g, device=DEV).bfloat16())
    tiles = tiles_of(counts, lead)
    tg = torch.tensor(tiles + [[len(counts) + 3, 1 << 30, 128, 0], [0, lead, 128, 0]], dtype=torch.int32, device=DEV)  # dead tiles are not looked at
    nt = torch.tensor([len(tiles)], dtype=torch.int32, device=DEV)
    out = torch.full((lead + T + 6, N), 7.0, device=DEV).bfloat16()
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    y = F8.grouped_linear(x, w, tg, nt, out=out, status=status)
    assert y.data_ptr() == out.data_ptr() and (y[:lead] == 7).all() and (y[lead + T:] == 7).all() and int(status) == 0
    at = lead
    for e, c in enumerate(counts):
        part = F8.Fp8Rows(x.q[at:at + c], x.scales[at:at + c])
        check_bf16(y[at:at + c], *product64(part, F8.Fp8Weight(w.q[e], w.scales[e])))
        at += c


@pytest.mark.parametrize("name", GROUPS)
@pytest.mark.parametrize("I,K", [(128, 128), (768, 2048), (80, 272)])
def test_grouped_gated_linear(F8, name, I, K):
    counts = GROUPS[name]
    g = gen(len(name) + I)
    T = sum(counts)
    x = F8.quantize_rows(acts(T + 6, K, g))
    w = F8.quantize_weight((torch.randn(len(counts), 2 * I, K, generator=g, device=DEV) * 2 / K ** 0.5).bfloat16(), halves=2)
    tiles = tiles_of(counts)
    tg = torch.tensor(tiles + [[0, 0, 0, 0]], dtype=torch.int32, device=DEV)
    nt = torch.tensor([len(tiles)], dtype=torch.int32, device=DEV)
    got = F8.grouped_gated_linear(x, w, tg, nt)
    at = 0
    for e, c in enumerate(counts):
        part = F8.Fp8Rows(x.q[at:at + c], x.scales[at:at + c])
        want = gated64(*product64(part, F8.Fp8Weight(w.q[e], w.scales[e], 2)))
        check_rows(F8.Fp8Rows(got.q[at:at + c], got.scales[at:at + c]), *want)
        at += c


# ------------------------------------------------------------------------------------------------ together
def experts_block(F8, ext, b):
    """A decoder layer's second half: norm with residual, routed experts, their sum back into the residual stream."""
    rows, h, y = F8.rmsnorm_rows(b["x"], b["norm"], 1e-6, b["res"], keep=True)
    logits = y.float() @ b["router"].t()
    ids, wts, _ = ext.moe_router_topk(logits, None, 4, True, True)
    E, T = b["router"].shape[0], b["x"].shape[0]
    _, _, dest, src, tg, nt = ext.moe_build_permutation(ids, E, T * 4, 1)
    p = F8.permute_rows(rows, src, nt, 4)
    act = F8.grouped_gated_linear(p, b["w1"], tg, nt, b["status"])
    yp = F8.grouped_linear(act, b["w2"], tg, nt, status=b["status"])
    return rows, h, ids, wts, dest, p, act, yp, ext.moe_combine(yp, dest, wts, T, 4, h)


def block_inputs(F8, T, seed):
    g = gen(seed)
    H, I, E = 512, 256, 16
    return dict(x=acts(T, H, g), res=acts(T, H, g), norm=(1 + 0.1 * torch.randn(H, generator=g, device=DEV)).bfloat16(),
                router=torch.randn(E, H, generator=g, device=DEV) * 0.2, w1=F8.quantize_weight((torch.randn(E, 2 * I, H, generator=g, device=DEV) * 0.05).bfloat16(), 2),
                w2=F8.quantize_weight((torch.randn(E, H, I, generator=g, device=DEV) * 0.05).bfloat16()), status=torch.zeros(1, dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("T", [1, 33, 700])
def test_operators_together(F8, ext, T):
    b = block_inputs(F8, T, T)
    rows, h, ids, wts, dest, p, act, yp, out = experts_block(F8, ext, b)
    at = dest.view(T, 4).long()
    for k in range(4):
        assert torch.equal(p.q.view(torch.uint8)[at[:, k]], rows.q.view(torch.uint8)) and torch.equal(p.scales[at[:, k]], rows.scales)
        for e in ids[:, k].unique().tolist():
            r = at[:, k][ids[:, k] == e]
            pick = lambda t: F8.Fp8Rows(t.q.view(torch.uint8)[r].view(torch.float8_e4m3fn), t.scales[r])  # noqa: E731
            check_rows(pick(act), *gated64(*product64(pick(p), F8.Fp8Weight(b["w1"].q[e], b["w1"].scales[e], 2))))
            check_bf16(yp[r], *product64(pick(act), F8.Fp8Weight(b["w2"].q[e], b["w2"].scales[e])))
    parts = [wts[:, k:k + 1].double() * yp[at[:, k]].double() for k in range(4)]
    want, most = h.double() + sum(parts), h.double().abs() + sum(t.abs() for t in parts)
    assert ((out.double() - want).abs() <= UBF * want.abs() + 8 * 2.0 ** -24 * most).all()
    assert int(b["status"]) == 0


@pytest.mark.parametrize("T", [3, 300])
def test_captured_and_on_other_streams(F8, ext, T):
    """Replays of a captured run on new inputs, and two runs at once on two streams, leave what single runs leave."""
    b, c = block_inputs(F8, T, 1), block_inputs(F8, T, 2)
    last = lambda r: [r[0].q.view(torch.uint8), r[6].scales, r[7], r[8]]  # noqa: E731
    want_b, want_c = ([t.clone() for t in last(experts_block(F8, ext, i))] for i in (b, c))
    torch.cuda.synchronize()
    still = dict(b, x=b["x"].clone(), res=b["res"].clone())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        experts_block(F8, ext, still)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = last(experts_block(F8, ext, still))
    for i in (c, b, c):
        still["x"].copy_(i["x"])
        still["res"].copy_(i["res"])
        graph.replay()
        torch.cuda.synchronize()
        if i is b:
            assert all(torch.equal(x, y) for x, y in zip(out, want_b))
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(one):
            got_b = last(experts_block(F8, ext, b))
        with torch.cuda.stream(two):
            got_c = last(experts_block(F8, ext, c))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got_b + got_c, want_b + want_c))
    assert int(b["status"]) == int(c["status"]) == 0


def test_refusals_of_operands_on_the_device(F8):
    x, w = F8.quantize_rows(acts(4, 256, gen(1))), F8.quantize_weight(torch.randn(64, 256, device=DEV).bfloat16())
    wide = torch.zeros(4 * 256 + 64, dtype=torch.uint8, device=DEV)
    off = lambda n: wide[n:n + 1024].view(torch.float8_e4m3fn).view(4, 256)  # noqa: E731
    for call, words in ((lambda: F8.linear(F8.Fp8Rows(off(8), x.scales), w), "16-byte aligned"),
                        (lambda: F8.linear(F8.Fp8Rows(x.q, x.scales.cpu()), w), "on the device"),
                        (lambda: F8.linear(x, w, acts(4, 63, gen(2))), "residual must be"),
                        (lambda: F8.linear(x, w, out=torch.empty(4, 64, device=DEV)), "out must be"),
                        (lambda: F8.linear(x, w, out=torch.empty(1, 64, device=DEV).bfloat16().expand(4, 64)), "overlap"),
                        (lambda: F8.quantize_rows(acts(4, 264, gen(3))[:, 4:260]), "16-byte aligned"),
                        (lambda: F8.rmsnorm_rows(acts(4, 256, gen(4)), torch.ones(256, device=DEV).bfloat16(), 1e-6, acts(4, 260, gen(5))[:, :256]), "16-byte aligned"),
                        (lambda: F8.gated_linear(x, F8.quantize_weight(torch.randn(96, 256, device=DEV).bfloat16())), "gate-up weight")):
        with pytest.raises(RuntimeError, match=words):
            call()
    assert F8.linear(x, w).isfinite().all()  # (a refused call leaves nothing behind)


# ------------------------------------------------------------------------------------------------ weights
@pytest.mark.parametrize("shape,halves", [((128, 128), 1), ((300, 272), 1), ((3, 200, 144), 1), ((4, 256, 128), 1), ((320, 144), 2), ((2, 96, 256), 2), ((512, 128), 2)])
def test_quantize_weight(F8, shape, halves):
    w = (torch.randn(shape, generator=gen(sum(shape)), device=DEV)).bfloat16()
    a, b = F8.quantize_weight(w, halves), F8.quantize_weight(w.cpu(), halves)
    assert a.scales.shape == b.scales.shape and torch.equal(a.scales.cpu(), b.scales)
    v = weight64(a).view(shape)
    s = (a.scales.double().max()).item()
    # half a step, and the rounding of the reciprocal that the quantiser multiplies with
    assert ((v - w.double()).abs() <= (U8 + 2.0 ** -22) * w.double().abs() + TINY8 * s).all()
    assert torch.allclose(a.dequantize().double(), v, rtol=2.0 ** -23, atol=0)
