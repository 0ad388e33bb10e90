"""The tensor calls on 8-bit rows and score rows on the GPU: which tensors they use, and what they refuse."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from vectordb_amd import scores as S  # noqa: E402
from vectordb_amd.capi import ArgumentError, DistanceMetric as M  # noqa: E402


def gauss(n, dim, seed):
    return torch.randn(n, dim, generator=torch.Generator().manual_seed(seed)).cuda()


def same(a, b):
    return torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and torch.equal(a.norms2, b.norms2)


# ---------------------------------------------------------------- the tensors of the moment

def test_rows_whose_tensors_were_replaced(vdb):
    """Scores are those of the tensors that are there now, and the quantiser writes those and no others."""
    q, first, second = S.quantize_rows(gauss(3, 100, 1)), S.quantize_rows(gauss(50, 100, 2)), S.quantize_rows(gauss(70, 100, 3))
    old = (first.codes, first.scales, first.norms2)
    kept = [t.clone() for t in old]
    r = S.Q8Rows(*old, 100)
    r.codes, r.scales, r.norms2 = second.codes, second.scales, second.norms2
    assert len(r) == 70 and torch.equal(S.score_rows(q, r, M.Cosine), S.score_rows(q, second, M.Cosine))
    assert torch.equal(S.score_rows(r, q, M.Cosine), S.score_rows(second, q, M.Cosine))
    x = gauss(70, 100, 4)
    S.quantize_rows(x, out=r)
    assert same(second, S.quantize_rows(x))
    assert all(torch.equal(a, b) for a, b in zip(old, kept))


def test_rows_whose_tensors_were_resized(vdb):
    r = S.Q8Rows.empty(4, 100, "cuda")
    r.codes.resize_(300, 112); r.scales.resize_(300, 4); r.norms2.resize_(300)
    x = gauss(300, 100, 5)
    assert S.quantize_rows(x, out=r) is r and same(r, S.quantize_rows(x))
    q = S.quantize_rows(gauss(2, 100, 6))
    assert S.score_rows(q, r, M.Dot).shape == (2, 300)
    r.scales.resize_(4, 4)                                     # no longer as many as codes
    with pytest.raises(ArgumentError):
        S.score_rows(q, r, M.Dot)
    with pytest.raises(ArgumentError):
        S.quantize_rows(x, out=r)


def test_norms_that_come_later(vdb):
    full, q = S.quantize_rows(gauss(20, 64, 1)), S.quantize_rows(gauss(3, 64, 2))
    r = S.Q8Rows(full.codes, full.scales, None, 64)
    with pytest.raises(ArgumentError):
        S.score_rows(q, r, M.Cosine)
    r.norms2 = full.norms2
    assert torch.equal(S.score_rows(q, r, M.Cosine), S.score_rows(q, full, M.Cosine))
    r.norms2 = None
    with pytest.raises(ArgumentError):
        S.score_rows(q, r, M.Cosine)


@pytest.mark.parametrize("change", [lambda r: setattr(r, "codes", r.codes.cpu()), lambda r: setattr(r, "codes", None), lambda r: setattr(r, "scales", r.scales.cpu()), lambda r: setattr(r, "norms2", r.norms2.double()),
                                    lambda r: setattr(r, "dim", 113), lambda r: setattr(r, "dim", 0), lambda r: setattr(r, "codes", r.codes[:19]), lambda r: setattr(r, "norms2", r.norms2[:19]),
                                    lambda r: setattr(r, "codes", r.codes.t()), lambda r: setattr(r, "codes", r.codes[:, :96])])
def test_rows_that_no_longer_fit_are_refused(vdb, change):
    r = S.quantize_rows(gauss(20, 100, 1))
    q = S.quantize_rows(gauss(3, 100, 2))
    change(r)
    with pytest.raises(ArgumentError):
        S.score_rows(q, r, M.Dot)


# ---------------------------------------------------------------- the call itself

def test_a_small_adjustment_costs_about_one_torch_operation(vdb):
    """Boosts on a thousand scores: a launch and little else, as the addition that it is.  The shortest of blocks taken in turn."""
    import time
    s, boost = torch.randn(1, 1000, device="cuda"), torch.randn(1000, device="cuda")
    assert torch.equal(S.adjust_scores(s, M.Dot, boost=boost), s + boost)

    def block(f, calls=300):
        torch.cuda.synchronize()
        t = time.perf_counter()
        for _ in range(calls):
            f()
        torch.cuda.synchronize()
        return time.perf_counter() - t
    both = [(block(lambda: S.adjust_scores(s, M.Dot, boost=boost)), block(lambda: s + boost)) for _ in range(40)]
    ours, torchs = min(a for a, _ in both), min(b for _, b in both)
    assert ours <= 1.3 * torchs, (ours, torchs)


def test_metrics_of_every_form(vdb):
    import numpy as np
    s = torch.randn(2, 40, device="cuda")
    boost = torch.randn(40, device="cuda")
    for m, want in ((0, s - boost), (1, s + boost), (2, s - boost)):
        for form in (m, M(m), float(m), np.int64(m)):
            assert torch.equal(S.adjust_scores(s, form, boost=boost), want)
    for bad in (3, -1, 1 << 70, 0.5, None, "dot", [1], float("nan"), torch.tensor(1)):
        with pytest.raises(ArgumentError):
            S.adjust_scores(s, bad)


def test_a_result_beyond_the_memory_is_torchs_own_error(vdb):
    """Three terabytes of scores: refused by the allocator, and the next call works."""
    q, b = S.Q8Rows.empty(200_000, 16, "cuda"), S.Q8Rows.empty(4_000_000, 16, "cuda")
    with pytest.raises(torch.OutOfMemoryError):
        S.score_rows(q, b, M.Dot)
    x = gauss(3, 16, 1)
    assert S.score_rows(S.quantize_rows(x), S.quantize_rows(x), M.Dot).shape == (3, 3)
