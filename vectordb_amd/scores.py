"""Dense scores on device tensors: rows held in 8 bits, their block-scaled product, and what is laid over score rows.

    base = quantize_rows(vectors)                        # once: f32 / f16 / bf16 tensor [n, dim] -> Q8Rows
    q = quantize_rows(queries)                           # per batch
    s = score_rows(q, base, DistanceMetric.Cosine)       # [nq, n] f32
    s = adjust_scores(s, DistanceMetric.Cosine, pass_bits=bits, boost=boost, seen=seen, seen_offsets=offsets, frequency=f)

Each call is one entry point of the library (vdb_q8_quantize_dev, vdb_q8_score_dev, vdb_score_adjust_dev: include/vdbmi.h has
the formulas and the layout), enqueued on the current stream of the tensors' device; nothing waits.  Tensors must live on one
GPU; what a call cannot take is refused with ArgumentError before anything is launched, or VectorLengthMismatch for rows of two lengths.
The calls have no gradient: while gradients are recorded a tensor that requires one is refused, as are tensors with tangents and
negated views; a tensor written through `out` counts as changed in place, so that a backward pass which saved it says so.
The calls themselves are in the module _tensors (csrc/tensors.cpp): a small one is over in the time of a few Python statements.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import api as _api, load_library
from .capi import ArgumentError, DistanceMetric, Q8RowsC, VectorLengthMismatch

try:
    from ._tensors import adjust_scores, bind, check_rows, quantize_rows, rows_struct, score_rows
except ModuleNotFoundError as e:
    raise ImportError("vectordb_amd/_tensors.so is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` or "
                      "`make -C vectordb_amd/csrc`; there is no other form of these calls") from e

BLOCK = 128                               # columns that share one scale


class Q8Rows:
    """Rows of `dim` columns as e4m3 codes (uint8 [n, >= dim, a multiple of 16]), one power-of-two scale per block of 128
    columns (uint8 [n, >= blocks, a multiple of 4]: exponent + 127) and squared norms (f32 [n], or None: dot products only).
    The attributes may be set anew: every call reads and checks the tensors that are there when it is made."""
    __slots__ = ("codes", "scales", "norms2", "dim")

    def __init__(self, codes, scales, norms2, dim):
        self.codes, self.scales, self.norms2, self.dim = codes, scales, norms2, int(dim)
        check_rows(codes, scales, norms2, self.dim)

    @property
    def _c(self):
        """The tensors of this moment as the struct of the C ABI."""
        return Q8RowsC(*rows_struct(self.codes, self.scales, self.norms2, self.dim))

    @classmethod
    def empty(cls, n, dim, device):
        """Room for n rows."""
        if dim < 1 or n < 0:
            raise ArgumentError("empty rows")
        wide, blocks = -(-dim // 16) * 16, -(-dim // (4 * BLOCK)) * 4
        return cls(torch.empty((n, wide), dtype=torch.uint8, device=device), torch.empty((n, blocks), dtype=torch.uint8, device=device),
                   torch.empty(n, dtype=torch.float32, device=device), dim)

    def __len__(self):
        return self.codes.shape[0]

    def __getitem__(self, rows):
        """A range of rows, sharing memory."""
        if not isinstance(rows, slice) or rows.step not in (None, 1):
            raise ArgumentError("rows are taken by ranges")
        return Q8Rows(self.codes[rows], self.scales[rows], None if self.norms2 is None else self.norms2[rows], self.dim)


def _bind():
    library, a = load_library(), _api()

    def address(entry):
        return C.cast(getattr(library, entry), C.c_void_p).value
    # the current stream's handle alone, without a Stream object around it (2 us a call), where torch offers it
    stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
    bind(address("vdb_q8_quantize_on"), address("vdb_q8_score_on"), address("vdb_score_adjust_on"), Q8Rows, a.check, ArgumentError, VectorLengthMismatch, torch.OutOfMemoryError, stream,
             frozenset(int(m) for m in DistanceMetric))


_bind()
