"""Serving in block-scaled 8 bits (`csrc/fp8_rows.cu`, `csrc/fp8_gemm.cu`): the format of FP8 checkpoints with ``weight_block_size`` [128, 128].

Activations are "8-bit rows": E4M3 values with one fp32 scale for each row and 128 columns, ``max(amax, 1e-10) / 448``. Weights are E4M3 with
one fp32 scale for each 128 x 128 (`weight_sync.quantize`, format ``fp8_block``). Scales may have any value, unlike those of `ops.mx_gemm`.

* `quantize_rows`, `rmsnorm_rows`, `permute_rows` leave such rows: of bf16 activations, of a norm with the residual's addition, of rows in expert order;
* `linear` and `grouped_linear` multiply them with a weight, or by expert over row tiles: bf16 results;
* `gated_linear` and `grouped_gated_linear` multiply them with a gate-up weight and leave ``silu(gate) * up`` as 8-bit rows again.

Rows are a multiple of 16 wide, and at most 2^31 - 256; nothing else about the sizes has to be even, rows of `x` may be apart, and no rows are
fine. Row tiles are those of the router's sort (``moe_build_permutation``): int32 ``{expert, first row, rows (at most 128), 0}`` of which the first ``num_tiles[0]``
are live; each row of the result belongs to at most one tile, and rows that belong to none are left unwritten. A block that holds NaN or
an infinity gets that scale, and what is multiplied with it becomes NaN. Everything runs on the current stream without a wait of the host, and the
list of joined row tiles that products by expert of many rows need is the allocator's, so calls can be captured and run beside one another.
Inference only: weights that are trained stay in bf16.

``status`` is the models' device status word: it receives a code should a wait inside a kernel ever run out.

Reference counterpart: the FP8 rollout recipes, whose engines multiply block-quantised weights
(miles/backends/megatron_utils/megatron_to_hf/processors/quantizer_fp8.py, miles/utils/fp8_kernel.py:24-79).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Union

import torch

from . import _ext
from . import reference as R

BLOCK = 128


@dataclass
class Fp8Rows:
    q: torch.Tensor        # float8_e4m3fn [T, K]
    scales: torch.Tensor   # fp32 [T, ceil(K / 128)]

    def dequantize(self) -> torch.Tensor:
        return R.fp8_rows_dequant(self.q, self.scales)


@dataclass
class Fp8Weight:
    q: torch.Tensor        # float8_e4m3fn [N, K], or [experts, N, K]
    scales: torch.Tensor   # fp32 [halves * ceil(N / halves / 128), ceil(K / 128)], or [experts, ...]
    halves: int = 1        # 2: a gate-up weight whose halves have blocks of their own (they do anyway if they are multiples of 128)

    @property
    def whole(self) -> bool:
        """Whether its blocks are also those of one matrix of all its rows, so that the ungated products read it."""
        return self.halves == 1 or self.q.shape[-2] // 2 % BLOCK == 0

    def dequantize(self) -> torch.Tensor:
        def split(t):
            return t.unflatten(-2, (self.halves, t.shape[-2] // self.halves))

        return R.fp8_block128_dequant(split(self.q), split(self.scales)).flatten(-3, -2)


def quantize_weight(w: torch.Tensor, halves: int = 1) -> Fp8Weight:
    """A bf16 weight ``[N, K]``, or one for each expert ``[experts, N, K]``; ``halves`` 2: gate rows, then as many up rows."""
    if w.dim() not in (2, 3) or halves not in (1, 2) or w.shape[-2] % halves or w.shape[-1] % 16 or w.numel() == 0:
        raise ValueError(f"weights are [N, K] or [experts, N, K] with K % 16 == 0 and, in two halves, N % 2 == 0; got {tuple(w.shape)} in {halves}")
    N, K = w.shape[-2:]
    wb = w.to(torch.bfloat16).contiguous()
    per = N // halves
    mats = wb.view(-1, K) if per % BLOCK == 0 else wb.view(-1, per, K)  # full blocks: all matrices lie in one grid of them
    one = _ext.load(required=True).quant_fp8_block128 if w.is_cuda else R.fp8_block128_quant
    if mats.dim() == 2:
        q, s = one(mats, False)
    else:
        q, s = (torch.stack(t) for t in zip(*(one(m, False) for m in mats)))
    q = q.view(torch.float8_e4m3fn) if q.dtype == torch.uint8 else q
    return Fp8Weight(q.reshape(w.shape), s.reshape(*w.shape[:-2], halves * -(-per // BLOCK), -(-K // BLOCK)), halves)


def quantize_rows(x: torch.Tensor) -> Fp8Rows:
    """8-bit rows of bf16 activations ``[T, K]``."""
    return Fp8Rows(*_ext.load(required=True).fp8_quantize_rows(x))


def rmsnorm_rows(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: Optional[torch.Tensor] = None, keep: bool = False):
    """``(8-bit rows of RMSNorm(h) * weight, h, the normalised rows in bf16 if keep)`` with ``h = x + residual`` rounded to bf16 (``x`` itself
    without a residual). The statistics are those of the rounded ``h``; the 8-bit rows are rounded once, from 32 bits."""
    q, s, h, y = _ext.load(required=True).fp8_rmsnorm_rows(x, weight, eps, residual, keep)
    return Fp8Rows(q, s), h, y


def permute_rows(x: Fp8Rows, src: torch.Tensor, num_tiles: torch.Tensor, top_k: int) -> Fp8Rows:
    """Rows in expert order: row i is token ``src[i] // top_k``'s (negative: zeros); ``src`` and ``num_tiles`` as ``moe_build_permutation`` leaves
    them, rows past the ``num_tiles[1]`` live ones stay unwritten."""
    return Fp8Rows(*_ext.load(required=True).fp8_permute_rows(x.q, x.scales, src, num_tiles, top_k))


def _rows(x: Union[Fp8Rows, torch.Tensor]) -> Fp8Rows:
    return x if isinstance(x, Fp8Rows) else quantize_rows(x)


def linear(x: Union[Fp8Rows, torch.Tensor], w: Fp8Weight, residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
           status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``x @ w^T (+ residual)`` in bf16, rounded once; ``x`` as 8-bit rows, or in bf16 (quantised first). ``out`` may be the residual itself,
    and shares no memory with the operands otherwise."""
    x = _rows(x)
    return _ext.load(required=True).fp8_linear(x.q, x.scales, w.q, w.scales, w.halves, residual, None, None, out, status)


def grouped_linear(x: Union[Fp8Rows, torch.Tensor], w: Fp8Weight, tile_group: torch.Tensor, num_tiles: torch.Tensor,
                   out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Every row tile of ``x`` times its expert's weight, in bf16."""
    x = _rows(x)
    return _ext.load(required=True).fp8_linear(x.q, x.scales, w.q, w.scales, w.halves, None, tile_group, num_tiles, out, status)


def gated_linear(x: Union[Fp8Rows, torch.Tensor], w: Fp8Weight, status: Optional[torch.Tensor] = None) -> Fp8Rows:
    """8-bit rows of ``silu(gate) * up`` for a gate-up weight ``[2 I, K]``, kept in 32 bits from the products to the rounding."""
    x = _rows(x)
    return Fp8Rows(*_ext.load(required=True).fp8_gated_linear(x.q, x.scales, w.q, w.scales, w.halves, None, None, status))


def grouped_gated_linear(x: Union[Fp8Rows, torch.Tensor], w: Fp8Weight, tile_group: torch.Tensor, num_tiles: torch.Tensor,
                         status: Optional[torch.Tensor] = None) -> Fp8Rows:
    """The same by expert: ``w`` is ``[experts, 2 I, K]``."""
    x = _rows(x)
    return Fp8Rows(*_ext.load(required=True).fp8_gated_linear(x.q, x.scales, w.q, w.scales, w.halves, tile_group, num_tiles, status))
