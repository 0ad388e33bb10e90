"""Dense scores on device tensors: rows held in 8 bits, their block-scaled product, and what is laid over score rows.

    base = quantize_rows(vectors)                        # once: f32 / f16 / bf16 tensor [n, dim] -> Q8Rows
    q = quantize_rows(queries)                           # per batch
    s = score_rows(q, base, DistanceMetric.Cosine)       # [nq, n] f32
    s = adjust_scores(s, DistanceMetric.Cosine, pass_bits=bits, boost=boost, seen=seen, seen_offsets=offsets, frequency=f)

Each call is one entry point of the C ABI (vdb_q8_quantize_dev, vdb_q8_score_dev, vdb_score_adjust_dev: include/vdbmi.h has
the formulas and the layout), enqueued on the current stream of the tensors' device; nothing waits.  Tensors must live on one
GPU; what a call cannot take is refused with ArgumentError before anything is launched, or VectorLengthMismatch for rows of two lengths.
"""
from __future__ import annotations

import ctypes as C

import torch

from .capi import ArgumentError, DistanceMetric, Q8RowsC, ScoreAdjustC, VectorLengthMismatch

BLOCK = 128                               # columns that share one scale
_Tensor = torch.Tensor
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_METRICS = frozenset(int(m) for m in DistanceMetric)


_lib = None


def _api():
    global _lib
    if _lib is None:
        from . import api
        _lib = api()
    return _lib


# the handle alone, without a Stream object around it (2 us a call), where torch offers it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _refuse(why):
    raise ArgumentError(why)


def _check(t, what, dtype, ndim, device=None):
    """A tensor of one type and rank whose last axis is dense; -> elements from row to row."""
    if not isinstance(t, _Tensor) or t.dtype is not dtype or t.dim() != ndim:
        _refuse(f"{what}: expected a {ndim}-d {dtype} tensor")
    if device is not None and t.device != device:
        _refuse(f"{what} is on {t.device}, not on {device}")
    width = t.shape[-1]
    if t.is_contiguous():
        return width
    stride = t.stride()
    if width > 1 and stride[-1] != 1:
        _refuse(f"{what}: the last axis must be dense")
    if ndim == 2 and t.shape[0] > 1:
        if stride[0] < width:
            _refuse(f"{what}: rows overlap")
        return stride[0]
    return width


def _on_gpu(t, what):
    if not isinstance(t, _Tensor) or not t.is_cuda:
        _refuse(f"{what} must be a tensor on the GPU")


def _metric(m):
    if m not in _METRICS:
        _refuse("unknown metric")
    return int(m)


def _out(out, nq, n, device):
    if out is None:
        return torch.empty((nq, n), dtype=torch.float32, device=device), n
    stride = _check(out, "out", torch.float32, 2, device)
    if out.shape != (nq, n):
        _refuse(f"out: expected shape {(nq, n)}")
    return out, stride


class Q8Rows:
    """Rows of `dim` columns as e4m3 codes (uint8 [n, >= dim, a multiple of 16]), one power-of-two scale per block of 128
    columns (uint8 [n, >= blocks, a multiple of 4]: exponent + 127) and squared norms (f32 [n], or None: dot products only).
    The attributes may be set anew: every call reads and checks the tensors that are there when it is made."""
    __slots__ = ("codes", "scales", "norms2", "dim")

    def __init__(self, codes, scales, norms2, dim):
        self.codes, self.scales, self.norms2, self.dim = codes, scales, norms2, int(dim)
        self._c

    @property
    def _c(self):
        """The tensors of this moment as the struct of the C ABI."""
        codes, scales, norms2, dim = self.codes, self.scales, self.norms2, self.dim
        _on_gpu(codes, "codes")
        dev = codes.device
        cs, ss = _check(codes, "codes", torch.uint8, 2), _check(scales, "scales", torch.uint8, 2, dev)
        (n, wide), (m, blocks) = codes.shape, scales.shape
        if dim < 1 or wide < -(-dim // 16) * 16 or blocks < -(-dim // (4 * BLOCK)) * 4:
            _refuse("codes or scales are narrower than a row")
        if m != n:
            _refuse("codes and scales hold different numbers of rows")
        norms = None
        if norms2 is not None:
            _check(norms2, "norms2", torch.float32, 1, dev)
            if norms2.shape[0] != n:
                _refuse("codes and norms2 hold different numbers of rows")
            norms = norms2.data_ptr()
        return Q8RowsC(codes.data_ptr(), scales.data_ptr(), norms, n, dim, cs, ss)

    @classmethod
    def empty(cls, n, dim, device):
        """Room for n rows."""
        if dim < 1 or n < 0:
            _refuse("empty rows")
        wide, blocks = -(-dim // 16) * 16, -(-dim // (4 * BLOCK)) * 4
        self = cls.__new__(cls)
        self.codes, self.scales = torch.empty((n, wide), dtype=torch.uint8, device=device), torch.empty((n, blocks), dtype=torch.uint8, device=device)
        self.norms2, self.dim = torch.empty(n, dtype=torch.float32, device=device), dim
        _on_gpu(self.codes, "a Q8Rows")
        return self

    def __len__(self):
        return self.codes.shape[0]

    def __getitem__(self, rows):
        """A range of rows, sharing memory."""
        if not isinstance(rows, slice) or rows.step not in (None, 1):
            _refuse("rows are taken by ranges")
        return Q8Rows(self.codes[rows], self.scales[rows], None if self.norms2 is None else self.norms2[rows], self.dim)


def quantize_rows(rows, out=None):
    """f32 / f16 / bf16 rows [n, dim] -> Q8Rows (into `out` where given: appending is quantize_rows(new, out=room[n:n + k]))."""
    _on_gpu(rows, "rows")
    kind = _DTYPES.get(rows.dtype)
    if kind is None:
        _refuse("rows: expected f32, f16 or bf16")
    stride = _check(rows, "rows", rows.dtype, 2)
    (n, dim), dev = rows.shape, rows.device
    if out is None:
        out = Q8Rows.empty(n, dim, dev)
    elif not isinstance(out, Q8Rows):
        _refuse("out is a Q8Rows")
    to = out._c
    if to.n != n or to.dim != dim or out.codes.device != dev:
        _refuse(f"out: expected {n} rows of {dim} columns on {dev}")
    api = _api()
    api.check(api.fn.q8_quantize_dev(rows.data_ptr(), kind, stride, C.byref(to), _raw_stream(dev.index)))
    return out


def score_rows(queries, base, metric, out=None):
    """Scores [nq, n] of every query (Q8Rows) against every row (Q8Rows)."""
    if not isinstance(queries, Q8Rows) or not isinstance(base, Q8Rows):
        _refuse("queries and base are Q8Rows")
    q, b, dev = queries._c, base._c, base.codes.device
    if queries.codes.device != dev:
        _refuse(f"queries are on {queries.codes.device}, not on {dev}")
    if q.dim != b.dim:
        raise VectorLengthMismatch(f"Vector length mismatch: expected {b.dim}, got {q.dim}")
    out, stride = _out(out, q.n, b.n, dev)
    api = _api()
    api.check(api.fn.q8_score_dev(C.byref(q), C.byref(b), _metric(metric), out.data_ptr(), stride, _raw_stream(dev.index)))
    return out


def adjust_scores(scores, metric, *, pass_bits=None, boost=None, seen=None, seen_offsets=None, repeat=None, frequency=None, presence=None, out=None):
    """What vdb_score_adjust describes, over scores [nq, n] f32 (a tensor of its own, or `out`; out=scores works in place).

    pass_bits: int32 [words] or [1 or nq, words], words = ceil(n / 32); boost: f32 [n] or [1 or nq, n]; seen: int32 columns of all
    queries behind each other (read as unsigned; those >= n are passed over), seen_offsets: int64 [nq + 1]; repeat / frequency / presence: f32 [nq]."""
    _on_gpu(scores, "scores")
    dev = scores.device
    stride = _check(scores, "scores", torch.float32, 2)
    nq, n = scores.shape
    metric = _metric(metric)
    how = ScoreAdjustC()

    def per_query(t, what, dtype, width):
        if isinstance(t, torch.Tensor) and t.dim() == 1:
            _check(t, what, dtype, 1, dev)
            rows, s = 1, 0
        else:
            s, rows = _check(t, what, dtype, 2, dev), t.shape[0]
        if t.shape[-1] < width or rows not in (1, nq):
            _refuse(f"{what}: expected 1 or {nq} rows of {width}")
        return t.data_ptr(), s if rows > 1 else 0

    if pass_bits is not None:
        how.pass_bits, how.pass_stride = per_query(pass_bits, "pass_bits", torch.int32, -(-n // 32))
    if boost is not None:
        how.boost, how.boost_stride = per_query(boost, "boost", torch.float32, n)
    if (seen is None) != (seen_offsets is None):
        _refuse("seen and seen_offsets come together")
    if seen is not None:
        _check(seen, "seen", torch.int32, 1, dev)
        _check(seen_offsets, "seen_offsets", torch.int64, 1, dev)
        if seen_offsets.shape[0] != nq + 1:
            _refuse(f"seen_offsets: expected {nq + 1}")
        how.n_seen = seen.shape[0]
        if how.n_seen:
            how.seen, how.seen_offsets = seen.data_ptr(), seen_offsets.data_ptr()
    for what, t in (("repeat", repeat), ("frequency", frequency), ("presence", presence)):
        if t is None:
            continue
        _check(t, what, torch.float32, 1, dev)
        if seen is None:
            _refuse(f"{what} without seen")
        if t.shape[0] != nq:
            _refuse(f"{what}: expected {nq}")
        setattr(how, what, t.data_ptr())
    out, out_stride = _out(out, nq, n, dev)
    api = _api()
    api.check(api.fn.score_adjust_dev(scores.data_ptr(), stride, nq, n, metric, C.byref(how), out.data_ptr(), out_stride, _raw_stream(dev.index)))
    return out
