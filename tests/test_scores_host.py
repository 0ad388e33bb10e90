"""8-bit rows and score rows: what the entry points refuse, on the host, before a device is touched (CPU-safe)."""
import ctypes as C

import numpy as np
import pytest

from vectordb_amd.capi import Q8RowsC, ScoreAdjustC

P = 1 << 20                                                    # an aligned address that no refused call reads
GIB = 1 << 30


def rows(n=10, dim=200, codes=P, scales=P + GIB, norms2=P + 2 * GIB, code_stride=208, scale_stride=4):
    return Q8RowsC(codes, scales, norms2, n, dim, code_stride, scale_stride)


def quantize(vdb, d_rows=P + 3 * GIB, dtype=0, stride=200, **kw):
    vdb.check(vdb.fn.q8_quantize_dev(d_rows, dtype, stride, C.byref(rows(**kw)), None))


def score(vdb, a, b, metric=1, out=P + 8 * GIB, out_stride=10):
    vdb.check(vdb.fn.q8_score_dev(C.byref(a), C.byref(b), metric, out, out_stride, None))


def other(**kw):
    d = dict(codes=P + 4 * GIB, scales=P + 5 * GIB, norms2=P + 6 * GIB)
    d.update(kw)
    return rows(**d)


def adjust(vdb, scores=P, stride=100, nq=4, n=100, metric=1, out=P + GIB, out_stride=100, **how):
    h = ScoreAdjustC(**how)
    vdb.check(vdb.fn.score_adjust_dev(scores, stride, nq, n, metric, C.byref(h), out, out_stride, None))


def test_strides(vdb):
    a, b = C.c_size_t(0), C.c_size_t(0)
    for dim, cs, ss in ((1, 16, 4), (16, 16, 4), (17, 32, 4), (128, 128, 4), (512, 512, 4), (513, 528, 8), (960, 960, 8), (1 << 24, 1 << 24, 1 << 17)):
        vdb.check(vdb.fn.q8_strides(dim, C.byref(a), C.byref(b)))
        assert (a.value, b.value) == (cs, ss)
    for dim in (0, (1 << 24) + 1):
        with pytest.raises(vdb.ArgumentError):
            vdb.check(vdb.fn.q8_strides(dim, C.byref(a), C.byref(b)))
    with pytest.raises(vdb.ArgumentError):
        vdb.check(vdb.fn.q8_strides(8, None, C.byref(b)))


@pytest.mark.parametrize("bad", [dict(dim=0), dict(dim=(1 << 24) + 1, code_stride=(1 << 24) + 16, scale_stride=1 << 18, stride=1 << 25), dict(n=1 << 32),
                                 dict(code_stride=200), dict(code_stride=192), dict(scale_stride=2), dict(scale_stride=0), dict(dim=600, code_stride=608, scale_stride=4, stride=600),
                                 dict(codes=None), dict(scales=None), dict(codes=P + 8), dict(scales=P + GIB + 2), dict(norms2=P + 2 * GIB + 1), dict(stride=199),
                                 dict(dtype=3), dict(dtype=-1), dict(d_rows=None), dict(d_rows=P + 3 * GIB + 2), dict(d_rows=P + 3 * GIB + 1, dtype=2),
                                 dict(d_rows=P), dict(d_rows=P + GIB), dict(d_rows=P + 2 * GIB - 256), dict(scales=P + 16), dict(norms2=P + GIB),
                                 dict(code_stride=(1 << 64) - 16), dict(stride=1 << 62), dict(n=1 << 31, code_stride=1 << 40)])
def test_the_quantiser_refuses(vdb, bad):
    with pytest.raises(vdb.ArgumentError):
        quantize(vdb, **bad)


def test_the_quantiser_needs_a_target(vdb):
    with pytest.raises(vdb.ArgumentError):
        vdb.check(vdb.fn.q8_quantize_dev(P, 0, 8, None, None))


@pytest.mark.parametrize("call", [
    lambda v: score(v, rows(), other(), metric=3), lambda v: score(v, rows(), other(), metric=-1),
    lambda v: score(v, rows(), other(), out=None), lambda v: score(v, rows(), other(), out=P + 8 * GIB + 2), lambda v: score(v, rows(), other(), out_stride=9),
    lambda v: score(v, rows(norms2=None), other(), metric=0), lambda v: score(v, rows(), other(norms2=None), metric=2),
    lambda v: score(v, rows(), other(), out=P), lambda v: score(v, rows(), other(), out=P + 5 * GIB), lambda v: score(v, rows(), other(), out=P + 6 * GIB + 36, metric=2),
    lambda v: score(v, rows(), other(), out_stride=1 << 62), lambda v: score(v, rows(code_stride=200), other()), lambda v: score(v, rows(), other(scale_stride=3)),
    lambda v: v.check(v.fn.q8_score_dev(None, C.byref(rows()), 1, P, 10, None))])
def test_the_product_refuses(vdb, call):
    with pytest.raises(vdb.ArgumentError):
        call(vdb)


def test_the_product_refuses_rows_of_two_lengths(vdb):
    with pytest.raises(vdb.VectorLengthMismatch) as e:
        score(vdb, rows(dim=199), other())
    assert (e.value.expected, e.value.actual) == (200, 199)
    with pytest.raises(vdb.VectorLengthMismatch):
        vdb.q8_score_scan(np.zeros((1, 3), np.float32), np.zeros((1, 4), np.float32), 1)


@pytest.mark.parametrize("bad", [dict(metric=3), dict(n=1 << 32, stride=1 << 33, out_stride=1 << 33), dict(nq=1 << 32), dict(stride=99), dict(out_stride=99), dict(scores=None), dict(out=None),
                                 dict(scores=P + 2), dict(out=P + GIB + 1), dict(pass_bits=P + 2 * GIB, pass_stride=3), dict(pass_bits=P + 2 * GIB + 2), dict(boost=P + 2 * GIB, boost_stride=99),
                                 dict(n_seen=5), dict(n_seen=5, seen=P + 2 * GIB), dict(n_seen=5, seen_offsets=P + 2 * GIB), dict(n_seen=5, seen=P + 2 * GIB, seen_offsets=P + 3 * GIB + 4),
                                 dict(out=P + 4), dict(out=P, out_stride=104), dict(out=P + 1200), dict(boost=P + GIB), dict(pass_bits=P + GIB + 1596),
                                 dict(n_seen=5, seen=P + GIB, seen_offsets=P + 3 * GIB), dict(n_seen=5, seen=P + 2 * GIB, seen_offsets=P + 3 * GIB, presence=P + GIB + 400),
                                 dict(stride=1 << 61), dict(pass_bits=P + 2 * GIB, pass_stride=1 << 61)])
def test_the_adjustment_refuses(vdb, bad):
    with pytest.raises(vdb.ArgumentError):
        adjust(vdb, **bad)


def test_the_adjustment_needs_its_description(vdb):
    with pytest.raises(vdb.ArgumentError):
        vdb.check(vdb.fn.score_adjust_dev(P, 8, 1, 8, 1, None, P + GIB, 8, None))


def test_nothing_to_do_is_no_error(vdb):
    quantize(vdb, n=0)
    quantize(vdb, n=0, codes=None, scales=None, norms2=None, d_rows=None)
    score(vdb, rows(n=0), other(), out=None)
    score(vdb, rows(), other(n=0), out=None, out_stride=0)
    adjust(vdb, nq=0, scores=None, out=None)
    adjust(vdb, n=0, stride=0, out_stride=0)
    assert vdb.q8_score_scan(np.zeros((0, 4), np.float32), np.zeros((3, 4), np.float32), 1).shape == (0, 3)
    assert vdb.q8_score_scan(np.zeros((2, 4), np.float32), np.zeros((0, 4), np.float32), 0).shape == (2, 0)


@pytest.mark.parametrize("q,b", [((2, 0), (3, 0)), ((4,), (3, 4))])
def test_the_host_scan_refuses(vdb, q, b):
    with pytest.raises(vdb.ArgumentError):
        vdb.q8_score_scan(np.zeros(q, np.float32), np.zeros(b, np.float32), 1)


def test_without_a_gpu_the_calls_fail_with_a_device_error(vdb):
    if vdb.fn.device_count() > 0:
        pytest.skip("a GPU is present")
    for call in (lambda: quantize(vdb), lambda: score(vdb, rows(), other()), lambda: adjust(vdb),
                 lambda: vdb.q8_score_scan(np.zeros((2, 4), np.float32), np.zeros((3, 4), np.float32), 1)):
        with pytest.raises(vdb.DeviceError):
            call()


def test_the_tensor_calls_refuse_host_tensors(vdb):
    torch = pytest.importorskip("torch")
    from vectordb_amd import scores as S
    with pytest.raises(vdb.ArgumentError):
        S.quantize_rows(torch.zeros(2, 4))
    with pytest.raises(vdb.ArgumentError):
        S.Q8Rows(torch.zeros(2, 16, dtype=torch.uint8), torch.zeros(2, 4, dtype=torch.uint8), None, 4)
    with pytest.raises(vdb.ArgumentError):
        S.adjust_scores(torch.zeros(2, 4), 1)
    with pytest.raises(vdb.ArgumentError):
        S.score_rows(torch.zeros(2, 4), torch.zeros(2, 4), 1)
