"""Numbers in 8 bits: e4m3 with float32 scales, as the kernels of ``csrc/fp8_rows.cu`` and ``csrc/linear_fp8.cu`` write and read them.

Rows (activations) have a scale for every 128 columns, weights one for every block of 128 x 128 (the blocks of the checkpoints that the
reference reads, src/quanta/minimax/loader.py:223-247).  A block of numbers v with the largest |v| = a is held as ``q = e4m3(v * 448 / a)`` and
the scale ``a / 448``; a counts as at least 2^-100.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from . import kernels

BLOCK = kernels.FP8_BLOCK
TOP = 448.0                   # the largest e4m3
SMALLEST = 2.0 ** -100        # the least a block's largest number counts as


@dataclass(frozen=True)
class Fp8Rows:
    """Rows ``q`` ``[n, columns]`` (float8_e4m3fn) with ``scales`` ``[ceil(columns / 128), n]``."""
    q: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self):
        return self.q.shape


@dataclass(frozen=True)
class Fp8Weight:
    """A matrix ``q`` ``[N, K]`` (float8_e4m3fn) with ``scales`` ``[ceil(N / 128), ceil(K / 128)]``."""
    q: torch.Tensor
    scales: torch.Tensor

    @property
    def shape(self):
        return self.q.shape

    def dequantized(self) -> torch.Tensor:
        """The numbers it stands for, float32 (for tools; the kernels read the matrix as it is)."""
        n, k = self.q.shape
        return self.q.float() * self.scales.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]


def empty_rows(n: int, columns: int, device) -> Fp8Rows:
    return Fp8Rows(torch.empty((n, columns), dtype=torch.float8_e4m3fn, device=device),
                   torch.empty((-(-columns // BLOCK), n), dtype=torch.float32, device=device))


def quantize_rows(x: torch.Tensor) -> Fp8Rows:
    """``x`` ``[n, K]`` (float32 or bfloat16, on the GPU) in 8 bits, in one launch."""
    out = empty_rows(x.shape[0], x.shape[1], x.device)
    kernels.rows_to_fp8(x, out.q, out.scales)
    return out


def quantize_weight(w: torch.Tensor, rows_at_a_time: int = 32 * BLOCK) -> Fp8Weight:
    """``w`` ``[N, K]`` in 8 bits, on its device; once, when a model is loaded.  ``rows_at_a_time`` (a multiple of 128) bounds the float32 copy."""
    n, k = w.shape
    if rows_at_a_time % BLOCK:
        raise ValueError(f"quantize_weight: {rows_at_a_time} rows at a time are no whole blocks of {BLOCK}")
    q = torch.empty((n, k), dtype=torch.float8_e4m3fn, device=w.device)
    scales = torch.empty((-(-n // BLOCK), -(-k // BLOCK)), dtype=torch.float32, device=w.device)
    for r0 in range(0, n, rows_at_a_time):
        part = w[r0: r0 + rows_at_a_time].float()
        rows = part.shape[0]
        part = torch.nn.functional.pad(part, (0, -k % BLOCK, 0, -rows % BLOCK))
        blocks = part.view(-1, BLOCK, part.shape[1] // BLOCK, BLOCK)
        scale = blocks.abs().amax((1, 3)).clamp_min(SMALLEST) / TOP
        if not bool(torch.isfinite(scale).all()):
            raise ValueError("quantize_weight: the matrix holds a NaN or an infinity")
        scales[r0 // BLOCK: r0 // BLOCK + scale.shape[0]] = scale
        q[r0: r0 + rows] = (blocks / scale[:, None, :, None]).clamp(-TOP, TOP).reshape(part.shape)[:rows, :k].to(q.dtype)
    return Fp8Weight(q, scales)
