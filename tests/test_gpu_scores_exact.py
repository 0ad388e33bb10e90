"""The block-scaled product on rows whose scores are whole numbers below 2^24: exact products added in 32 bits give them exactly, in any
order, so a lost bit anywhere shows.  Every kernel and tile size.

Tolerances of the other two metrics, u = 2^-24 (roots and reciprocals of the hardware are one step, 2 u, off at most):
  cosine     two roots (4 u), their product and the 1e-10 (2 u), a reciprocal or two (4 u), a product or two (2 u) of |cos|; one u of 1 - cos
  euclidean  |q|^2 + |r|^2 - 2 dot is exact below 2^24, else off by one rounding of |q|^2 + |r|^2; half of its own u, and the root's 2 u
"""
import pytest

torch = pytest.importorskip("torch")

from vectordb_amd import scores as S  # noqa: E402
from vectordb_amd.capi import DistanceMetric as M  # noqa: E402

U = 2.0 ** -24
SHAPES = [(1, 20001, 100), (16, 20000, 128),                   # up to 16 queries: rows of one block
          (3, 3000, 4096), (16, 2001, 960), (1, 300, 8000),    # the columns split over a workgroup
          (8, 30001, 960), (16, 14400, 8000), (8, 70001, 960),   # workgroups that walk through the rows, two and three blocks on their way
          (20, 20000, 100), (31, 20001, 960), (17, 30000, 2000),   # up to 32 queries
          (20, 500, 960), (33, 300, 4096), (200, 77, 640),     # few tiles of 32 x 32, split columns
          (129, 25001, 960), (40, 33001, 2000),                # tiles of 64 x 64
          (64, 150001, 300),                                   # 128 x 64
          (128, 30001, 960), (250, 9001, 4096),                # 128 x 128
          (300, 60003, 960),                                   # 256 x 128
          (256, 65537, 300)]                                   # 256 x 256


def codes_of(v):
    """Whole numbers that e4m3 holds -> codes, zero up to a multiple of 16 columns."""
    n, dim = v.shape
    c = torch.zeros(n, -(-dim // 16) * 16, dtype=torch.uint8, device=v.device)
    e = v.to(torch.float8_e4m3fn)
    assert torch.equal(e.to(v.dtype), v)
    c[:, :dim] = e.view(torch.uint8)
    return c


def rows_of(v, exponents=None):
    """Q8Rows that hold v * 2^exponent of the block; squared norms of v itself."""
    n, dim = v.shape
    nb = -(-dim // 128)
    scales = torch.full((n, -(-nb // 4) * 4), 127, dtype=torch.uint8, device=v.device)
    if exponents is not None:
        scales[:, :nb] = (exponents + 127).to(torch.uint8)
    return S.Q8Rows(codes_of(v), scales, v.double().square().sum(1).float(), dim)


def signs(n, dim, g):
    return torch.randint(0, 2, (n, dim), generator=g, device=g.device).float().mul_(2).sub_(1)


def large_beside_small(n, dim, large, g, pattern=9):
    """+-1, and +-large in one column of each eight: the same columns for all rows, so that large meets large."""
    v = signs(n, dim, g)
    at = torch.arange(0, dim, 8) + torch.randint(0, 8, (-(-dim // 8),), generator=torch.Generator().manual_seed(pattern))
    v[:, at[at < dim].to(v.device)] *= large
    return v


def products(q, b):
    """-> q b^T in 64 bits; the largest sum of magnitudes stays below 2^24, whatever the order of the additions."""
    qd, bt = q.double(), b.double().t().contiguous()
    assert float(torch.mm(qd.abs(), bt.abs()).max()) < 2 ** 24
    return torch.mm(qd, bt)


def generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.gpu
@pytest.mark.parametrize("nq,n,dim", SHAPES)
def test_large_products_beside_small_ones(vdb, nq, n, dim):
    """2^14 beside 1 in every eight columns: the 1 counts."""
    g = generator(nq + n + dim)
    q, b = large_beside_small(nq, dim, 128, g), large_beside_small(n, dim, 128, g)
    b[n // 2] = q[nq - 1]                                      # a row that is a query, and one beside it
    b[n - 1] = q[0]; b[n - 1, dim - 1] *= -1
    want = products(q, b)
    rq, rb = rows_of(q), rows_of(b)
    assert torch.equal(S.score_rows(rq, rb, M.Dot).double(), want)
    nq2, nb2 = q.double().square().sum(1)[:, None], b.double().square().sum(1)
    cos = want / (nq2.sqrt() * nb2.sqrt() + 1e-10)
    assert bool(((S.score_rows(rq, rb, M.Cosine).double() - (1 - cos)).abs() <= 12 * U * cos.abs() + 1.01 * U * (1 - cos).abs()).all())
    both = nq2 + nb2
    d = (both - 2 * want).clamp(min=0)
    off = torch.where(both < 2 ** 24, 0.0, U * both)
    root = d.sqrt()
    got = S.score_rows(rq, rb, M.Euclidean).double()
    assert bool(((got - root).abs() <= 3 * U * root + off / torch.maximum(root, off.sqrt()).clamp(min=1e-300)).all())
    if float(both.max()) < 2 ** 24:
        assert float(got[nq - 1, n // 2]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("nq,n,dim", SHAPES)
def test_blocks_of_different_scales(vdb, nq, n, dim):
    """Blocks between 2^-60 and 2^60 whose products meet at 2^-2, 1 and 2^2: small blocks count beside large ones."""
    g = generator(nq * n + dim)
    nb = -(-dim // 128)
    q, b = large_beside_small(nq, dim, 32, g), large_beside_small(n, dim, 32, g)
    eq = torch.randint(-58, 59, (nb,), generator=g, device="cuda")
    together = torch.randint(-1, 2, (nb,), generator=g, device="cuda") * 2
    unit = torch.exp2(together.double() + 2).repeat_interleave(128)[:dim]                  # in units of 2^-2
    want = products(q.double() * unit, b)
    got = S.score_rows(rows_of(q, eq.expand(nq, nb)), rows_of(b, (together - eq).expand(n, nb)), M.Dot)
    assert torch.equal(got.double() * 4, want)


@pytest.mark.gpu
@pytest.mark.parametrize("nq,n,dim", SHAPES + [(1, 40, 131072), (2, 33, 100000), (16, 20001, 4000)])
def test_long_sums_of_positive_products(vdb, nq, n, dim):
    g = generator(dim)
    q, b = (torch.randint(1, 16, (k, dim), generator=g, device="cuda").float() for k in (nq, n))
    assert torch.equal(S.score_rows(rows_of(q), rows_of(b), M.Dot).double(), products(q, b))


@pytest.mark.gpu
@pytest.mark.parametrize("metric", list(M))
@pytest.mark.parametrize("nq,n,dim", [(600, 100003, 300), (300, 200001, 960), (1000, 60001, 272), (640, 100000, 256)])
def test_large_score_matrices_whose_rows_share_lines(vdb, nq, n, dim, metric):
    """Scores beyond the last-level cache, in rows that begin anywhere in a line: those of dense aligned rows, and nothing between them."""
    g = generator(7)
    q, b = (S.quantize_rows(torch.randn(k, dim, generator=g, device="cuda")) for k in (nq, n))
    wide = -(-n // 32) * 32 + 64
    aligned = torch.full((nq, wide), -5.0, device="cuda")
    S.score_rows(q, b, metric, out=aligned[:, :n])
    assert torch.equal(S.score_rows(q, b, metric), aligned[:, :n])
    for at, apart in ((1, n + 3), (7, n + 8 + -n % 8)):
        room = torch.full((nq, apart + 8), -5.0, device="cuda")
        S.score_rows(q, b, metric, out=room[:, at:at + n])
        assert torch.equal(room[:, at:at + n], aligned[:, :n])
        assert bool((room[:, :at] == -5).all()) and bool((room[:, at + n:] == -5).all())
    assert bool((aligned[:, n:] == -5).all())


def test_a_window_of_13_bits_would_show():
    """The inputs above against a sum that keeps, of each eight products, 13 bits below the largest: nearly every score is another."""
    g = torch.Generator().manual_seed(1)
    q, b = large_beside_small(4, 960, 128, g), large_beside_small(50, 960, 128, g)
    p = (q[:, None, :] * b[None]).double().view(4, 50, 120, 8)
    unit = torch.exp2(torch.floor(torch.log2(p.abs().amax(-1, keepdim=True))) - 13)
    windowed = (torch.trunc(p / unit) * unit).sum((-1, -2))
    assert float((windowed != p.sum((-1, -2))).double().mean()) > 0.9
