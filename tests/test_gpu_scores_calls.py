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
