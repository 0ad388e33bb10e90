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


# ---------------------------------------------------------------- gradients

def test_what_requires_a_gradient_is_refused_while_gradients_are_recorded(vdb):
    x = gauss(4, 32, 1).requires_grad_()
    want = S.quantize_rows(x.detach())
    with pytest.raises(ArgumentError, match="gradient"):
        S.quantize_rows(x)
    with pytest.raises(ArgumentError, match="gradient"):
        S.quantize_rows(x * 2)
    with torch.no_grad():
        assert same(S.quantize_rows(x), want)
    with torch.inference_mode():
        assert same(S.quantize_rows(x), want)
    # norms, scores and everything that is laid over them
    r = S.Q8Rows(want.codes, want.scales, want.norms2, 32)
    r.norms2 = want.norms2.clone().requires_grad_()
    with pytest.raises(ArgumentError, match="gradient"):
        S.score_rows(want, r, M.Cosine)
    s, ones = torch.randn(4, 40, device="cuda"), torch.ones(4, device="cuda")
    seen, off = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.arange(5, device="cuda")
    lists = dict(seen=seen, seen_offsets=off)
    kws = [dict(boost=torch.randn(40, device="cuda")), dict(repeat=ones, **lists), dict(frequency=ones, **lists), dict(presence=ones, **lists), dict(out=torch.empty_like(s))]
    plain = [S.adjust_scores(s, M.Dot, **kw).clone() for kw in kws]
    with pytest.raises(ArgumentError, match="gradient"):
        S.adjust_scores(s.clone().requires_grad_(), M.Dot)
    for kw, value in zip(kws, plain):
        name = next(k for k in kw if k not in lists)
        kw = {**kw, name: kw[name].clone().requires_grad_()}
        with pytest.raises(ArgumentError, match="gradient"):
            S.adjust_scores(s, M.Dot, **kw)
        with torch.no_grad():
            assert torch.equal(S.adjust_scores(s.clone().requires_grad_(), M.Dot, **kw), value)


def test_an_output_that_a_backward_pass_saved_counts_as_changed(vdb):
    a = torch.randn(3, 20, device="cuda", requires_grad=True)
    s = a * 2
    y = (s * s).sum()                                          # saves s
    d = s.detach()
    S.adjust_scores(d, M.Dot, boost=torch.ones(20, device="cuda"), out=d)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


def test_versions_of_outputs(vdb):
    x = gauss(5, 40, 1)
    r, s = S.quantize_rows(x), torch.empty(5, 5, device="cuda")
    before = [t._version for t in (r.codes, r.scales, r.norms2, s, x)]
    S.quantize_rows(x, out=r)
    S.score_rows(r, r, M.Dot, out=s)
    assert [t._version for t in (r.codes, r.scales, r.norms2, s, x)] == [v + 1 for v in before[:4]] + before[4:]
    S.adjust_scores(s, M.Dot)
    assert s._version == before[3] + 1
    S.quantize_rows(x, out=S.Q8Rows(r.codes, r.scales, None, 40))
    assert r.codes._version == before[0] + 2 and r.norms2._version == before[2] + 1
    with torch.inference_mode():                               # such tensors have no versions
        room, t = S.Q8Rows.empty(5, 40, "cuda"), torch.empty(5, 5, device="cuda")
        S.quantize_rows(x, out=room)
    S.score_rows(room, r, M.Dot, out=t)
    assert same(room, S.quantize_rows(x)) and torch.equal(t, S.score_rows(r, r, M.Dot))


def test_negated_views_and_tangents_are_refused(vdb):
    import torch.autograd.forward_ad as fwad
    x = gauss(4, 32, 1)
    with pytest.raises(ArgumentError):
        S.quantize_rows(torch._neg_view(x))
    assert same(S.quantize_rows(torch._neg_view(x).resolve_neg()), S.quantize_rows(-x))
    with pytest.raises(ArgumentError):
        S.adjust_scores(x, M.Dot, out=torch._neg_view(x.clone()))
    with fwad.dual_level():
        with pytest.raises(ArgumentError):
            S.adjust_scores(fwad.make_dual(x, torch.ones_like(x)), M.Dot)
        with pytest.raises(ArgumentError):
            S.adjust_scores(x, M.Dot, boost=fwad.make_dual(x[0], torch.ones_like(x[0])))


def test_tensors_without_memory_are_refused(vdb):
    x = gauss(4, 32, 1)
    with pytest.raises(ArgumentError):
        S.quantize_rows(torch.sparse_coo_tensor([[0], [1]], [1.0], (4, 32), device="cuda"))
    with pytest.raises(ArgumentError):
        torch.func.vmap(lambda t: S.adjust_scores(t, M.Dot))(torch.stack([x, x]))
    with pytest.raises(ArgumentError):
        torch.func.grad(lambda t: S.adjust_scores(t, M.Dot).sum())(x)
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        with pytest.raises(ArgumentError):
            S.quantize_rows(torch.empty(4, 32, device="cuda"))


def test_a_scan_beyond_the_memory_leaves_nothing_behind(vdb):
    """A terabyte of rows is refused by the allocator before anything is read, and the next calls know nothing of it."""
    import numpy as np
    x = gauss(3, 64, 1)
    want = S.score_rows(S.quantize_rows(x), S.quantize_rows(x), M.Dot)
    room = np.zeros((4, 64), np.float32)
    for _ in range(2):
        with pytest.raises(vdb.DeviceError):
            vdb.check(vdb.fn.q8_score_scan(room.ctypes.data, 1, room.ctypes.data, 4_000_000_000, 64, 1, 0, room.ctypes.data))
        assert torch.equal(S.score_rows(S.quantize_rows(x), S.quantize_rows(x), M.Dot), want)
        h = x.cpu().numpy()
        assert np.array_equal(vdb.q8_score_scan(h, h, 1), want.cpu().numpy())
