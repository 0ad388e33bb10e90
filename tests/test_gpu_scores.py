"""8-bit rows, their block-scaled product and score rows on the GPU, against plain 64-bit forms.

Tolerances count roundings (u = 2^-24, half a step of f32):
  norms2    a lane's chain of at most 8 per block, 5 exchanges and 15 further sums of non-negative terms: (8 blocks + 20) u of the sum
  dot       exact products; one rounding of at most a whole step (2 u) per addition: 2 u 128 blocks of sum |q_i r_i|
  cosine    that over |q||r|, and eight roundings of values no larger than 1 + |cos|
  euclidean the square: twice the dot's, and four roundings of |q|^2 + |r|^2; the root: one step more
  adjust    four roundings of the sum of the magnitudes that enter
"""
import ctypes as C

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from vectordb_amd import scores as S  # noqa: E402
from vectordb_amd.capi import ArgumentError, DistanceMetric as M, Q8RowsC, ScoreAdjustC, VectorLengthMismatch  # noqa: E402

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- plain forms (numpy, 64 bits)

def e4m3_values():
    """The values of the 127 non-negative codes below NaN, in order."""
    v = []
    for c in range(127):
        e, f = c >> 3, c & 7
        v.append(f * 2.0 ** -9 if e == 0 else (8 + f) * 2.0 ** (e - 10))
    return np.array(v)


E4M3 = e4m3_values()


def to_code(x):
    """Nearest code, ties to the even one; -0 and what rounds to it keep their sign; nonfinite -> 0x7F."""
    ax = np.where(np.isfinite(x), np.abs(x), 0)
    hi = np.clip(np.searchsorted(E4M3, ax), 1, 126)
    lo = hi - 1
    dl, dh = ax - E4M3[lo], E4M3[hi] - ax
    c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    c = c | np.where(np.signbit(x), 0x80, 0)
    return np.where(np.isfinite(x), c, 0x7F).astype(np.uint8)


def plain_quantize(x):
    """-> codes [n, up16], scales [n, up4], held values [n, dim] of float64 rows."""
    n, dim = x.shape
    nb, wide = -(-dim // 128), -(-dim // 16) * 16
    codes, scales = np.zeros((n, wide), np.uint8), np.full((n, -(-nb // 4) * 4), 127, np.uint8)
    vals = np.zeros((n, dim))
    table = np.concatenate([E4M3, [np.nan], -E4M3, [np.nan]])
    for b in range(nb):
        p = x[:, b * 128:(b + 1) * 128]
        a = np.where(np.isfinite(p), np.abs(p), 0).max(1)
        e = np.zeros(n, np.int64)
        for i in range(n):
            if a[i] > 0:
                k = -100
                while a[i] > 448 * 2.0 ** k:
                    k += 1
                e[i] = k
        scales[:, b] = e + 127
        top = np.where(e == 120, 240.0, 448.0)[:, None]                             # no value rounds up to 2^128
        c = p / 2.0 ** e[:, None]
        c = to_code(np.where(np.isfinite(c), np.clip(c, -top, top), c))
        codes[:, b * 128:b * 128 + p.shape[1]] = c
        vals[:, b * 128:b * 128 + p.shape[1]] = table[c] * 2.0 ** e[:, None]
    return codes, scales, vals


def held(r):
    """The values that rows hold, float64 on the CPU."""
    codes, scales = r.codes.cpu().numpy(), r.scales.cpu().numpy().astype(np.int64)
    table = np.concatenate([E4M3, [np.nan], -E4M3, [np.nan]])
    return table[codes[:, :r.dim]] * np.exp2((scales - 127).astype(np.float64)).repeat(128, 1)[:, :r.dim]


def check_scores(got, q, b, metric, dim):
    """got [nq, n] against held values q, b (float64)."""
    got = got.double().cpu().numpy()
    dot, mag = q @ b.T, np.abs(q) @ np.abs(b).T
    off = 2 * U * 128 * -(-dim // 128) * mag
    nq, nb = (q * q).sum(1)[:, None], (b * b).sum(1)[None]
    norm_off = (8 * -(-dim // 128) + 20) * U
    if metric == M.Dot:
        assert np.all(np.abs(got - dot) <= off + 2.0 ** -149)
    elif metric == M.Cosine:
        den = np.sqrt(nq * nb) + 1e-10
        assert np.all(np.abs(got - (1 - dot / den)) <= off / den + (8 * U + norm_off) * (1 + np.abs(dot) / den))
    else:
        sq = np.maximum(nq + nb - 2 * dot, 0)
        assert np.all(np.abs(got * got - sq) <= 2 * off + (4 * U + norm_off) * (nq + nb) + 4 * U * sq)


def gauss(n, dim, seed, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, dim, generator=g)
    return x * torch.exp(spread * torch.randn(n, 1, generator=g))


# ---------------------------------------------------------------- quantiser

@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,dim", [(1, 1), (3, 3), (9, 16), (5, 17), (33, 100), (8, 127), (7, 128), (17, 129), (2, 511), (3, 513), (6, 960), (2, 4100), (600, 300), (2049, 260), (2200, 129), (700, 90),
                                    # rows by groups of 4, 8, 16 and 32 lanes, by wavefronts and by workgroups, with and without a ragged end
                                    (70, 4), (70, 5), (70, 7), (70, 8), (70, 12), (70, 15), (70, 31), (70, 32), (70, 33), (70, 63), (70, 64), (70, 65), (70, 112), (1, 2),
                                    (2050, 511), (2050, 512), (2051, 513), (2060, 700), (2050, 960), (2051, 1667), (2049, 2048), (2049, 8400), (40, 8400)])
def test_quantised_rows_equal_the_definition(vdb, kind, n, dim):
    x = gauss(n, dim, n * 1000 + dim).to(TYPES[kind])
    r = S.quantize_rows(x.cuda())
    codes, scales, vals = plain_quantize(x.double().numpy())
    assert np.array_equal(r.codes.cpu().numpy(), codes)
    assert np.array_equal(r.scales.cpu().numpy(), scales)
    want = (vals * vals).sum(1)
    assert np.all(np.abs(r.norms2.cpu().numpy() - want) <= (8 * -(-dim // 128) + 20) * U * want)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,dim", [(50, 3), (50, 20), (50, 40), (50, 70), (50, 130), (2100, 130), (2100, 600), (2100, 1030)])
def test_special_values_in_every_kernel(vdb, kind, n, dim):
    """Infinities, NaN, the largest values and signed zeros beside ordinary rows, wherever a row ends."""
    t = TYPES[kind]
    at = torch.arange(n)
    x = gauss(n, dim, dim)
    x[at % 11 == 10] *= 1e-6                                                        # f16: subnormals
    x = x.to(t)
    for i, v in enumerate((float("inf"), -float("inf"), float("nan"), torch.finfo(t).max, -torch.finfo(t).max, torch.finfo(t).smallest_normal, -0.0)):
        rows = at[at % 11 == i]
        x[rows, (rows * 7) % dim] = v
        x[rows[::3], dim - 1] = v
    x[at % 11 == 9] = 0
    r = S.quantize_rows(x.cuda())
    codes, scales, vals = plain_quantize(x.double().numpy())
    assert np.array_equal(r.codes.cpu().numpy(), codes)
    assert np.array_equal(r.scales.cpu().numpy(), scales)
    with np.errstate(over="ignore", invalid="ignore"):
        want = (vals * vals).sum(1)
        got = r.norms2.cpu().numpy().astype(np.float64)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        ok = ~np.isnan(want) & (want < 2.0 ** 127)
        assert np.all(np.abs(got - want)[ok] <= (8 * -(-dim // 128) + 20) * U * want[ok] + 2.0 ** -140)
        assert np.all(got[want > 2.0 ** 129] == np.inf)


def test_special_values(vdb):
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(14, 130)
    x[1, :4] = torch.tensor([inf, -inf, nan, 3.0]); x[2] = nan                       # no finite value at all
    x[3, 0] = 1e-45; x[3, 1] = -1e-45; x[4, 0] = 2.0 ** -126; x[4, 5] = 2.0 ** -149    # subnormal rows
    x[5, 0] = 3.4028234e38; x[5, 1] = -1e38; x[5, 2] = 1.0                             # the largest float
    x[6, 0] = 448.0; x[7, 0] = float(np.nextafter(np.float32(448), np.float32(1e9))); x[8, 0] = float(np.nextafter(np.float32(448), np.float32(0)))
    x[9, 0] = 448.0; x[9, 1:9] = torch.tensor([17.0, 19.0, -17.0, 18.0, 21.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -9 * 1.5])   # ties; half the smallest code
    x[10, :2] = torch.tensor([-0.0, 0.0]); x[11, 128] = -7.0; x[12, 0] = 1e-30; x[12, 129] = 1e30; x[13] = -1.0
    r = S.quantize_rows(x.cuda())
    codes, scales, vals = plain_quantize(x.double().numpy())
    assert np.array_equal(r.codes.cpu().numpy(), codes)
    assert np.array_equal(r.scales.cpu().numpy(), scales)
    n2 = r.norms2.cpu().numpy()
    assert np.isnan(n2[1]) and np.isnan(n2[2]) and n2[0] == 0 and n2[10] == 0 and n2[13] == np.float32(130)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("at,pad", [(0, 0), (0, 5), (1, 3), (4, 4), (2, 6)])
def test_rows_of_any_alignment_and_stride(vdb, kind, at, pad):
    wide = gauss(19, at + 150 + pad, 5).to(TYPES[kind]).cuda()
    x = wide[:, at:at + 150]
    a, b = S.quantize_rows(x), S.quantize_rows(x.clone())
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales) and torch.equal(a.norms2, b.norms2)


def test_rows_written_into_a_larger_room_leave_the_rest_alone(vdb):
    room = S.Q8Rows(torch.full((20, 192), 0xAB, dtype=torch.uint8, device="cuda"), torch.full((20, 12), 0xCD, dtype=torch.uint8, device="cuda"),
                    torch.full((20,), -1.0, device="cuda"), 150)
    x = gauss(7, 150, 8).cuda()
    S.quantize_rows(x, out=room[5:12])
    want = S.quantize_rows(x)
    assert torch.equal(room.codes[5:12, :160], want.codes) and torch.equal(room.scales[5:12, :4], want.scales) and torch.equal(room.norms2[5:12], want.norms2)
    assert bool((room.codes[:5] == 0xAB).all()) and bool((room.codes[12:] == 0xAB).all()) and bool((room.codes[:, 160:] == 0xAB).all())
    assert bool((room.scales[:, 4:] == 0xCD).all()) and bool((room.scales[12:] == 0xCD).all()) and bool((room.norms2[12:] == -1).all())
    # the product reads rows with these strides, and nothing behind them
    s = S.score_rows(room[5:8], room[5:12], M.Cosine)
    check_scores(s, held(want)[:3], held(want), M.Cosine, 150)


def test_norms_may_be_left_out(vdb):
    x = gauss(5, 64, 3).cuda()
    room = S.Q8Rows.empty(5, 64, x.device)
    bare = S.Q8Rows(room.codes, room.scales, None, 64)
    S.quantize_rows(x, out=bare)
    assert torch.equal(bare.codes, S.quantize_rows(x).codes)
    check_scores(S.score_rows(bare, bare, M.Dot), held(bare), held(bare), M.Dot, 64)
    with pytest.raises(ArgumentError):
        S.score_rows(bare, bare, M.Euclidean)


def test_more_rows_than_a_grid_holds(vdb):
    n = (8 << 20) + 77
    x = torch.arange(n, dtype=torch.float32, device="cuda").remainder_(449).unsqueeze(1)
    r = S.quantize_rows(x)
    want = S.quantize_rows(torch.arange(449, dtype=torch.float32, device="cuda").unsqueeze(1))
    at = torch.arange(n, device="cuda") % 449
    assert torch.equal(r.codes, want.codes[at]) and torch.equal(r.scales, want.scales[at]) and torch.equal(r.norms2, want.norms2[at])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,dim", [(19, 5), (19, 40), (19, 70), (2100, 150), (2100, 600), (2100, 520)])
def test_any_alignment_and_a_larger_room_in_every_kernel(vdb, kind, n, dim):
    """Rows at odd places of a wider table into rows of a wider room: the codes of dense rows, and nothing beside them."""
    for at, pad in ((0, 0), (1, 2), (3, 8), (5, 0)):
        wide = gauss(n, at + dim + pad, 5).to(TYPES[kind]).cuda()
        wide[:, :at] = float("nan"); wide[:, at + dim:] = float("nan")
        want = S.quantize_rows(wide[:, at:at + dim].clone())
        w, sc = want.codes.shape[1], want.scales.shape[1]
        room = S.Q8Rows(torch.full((n + 9, w + 16), 0xAB, dtype=torch.uint8, device="cuda"), torch.full((n + 9, sc + 4), 0xCD, dtype=torch.uint8, device="cuda"),
                        torch.full((n + 9,), -1.0, device="cuda"), dim)
        S.quantize_rows(wide[:, at:at + dim], out=room[4:4 + n])
        assert torch.equal(room.codes[4:4 + n, :w], want.codes) and torch.equal(room.scales[4:4 + n, :sc], want.scales) and torch.equal(room.norms2[4:4 + n], want.norms2)
        assert bool((room.codes[:4] == 0xAB).all()) and bool((room.codes[4 + n:] == 0xAB).all()) and bool((room.codes[:, w:] == 0xAB).all())
        assert bool((room.scales[:4] == 0xCD).all()) and bool((room.scales[4 + n:] == 0xCD).all()) and bool((room.scales[:, sc:] == 0xCD).all())
        assert bool((room.norms2[:4] == -1).all()) and bool((room.norms2[4 + n:] == -1).all())


def test_more_long_rows_than_a_grid_holds(vdb):
    """4.3 million rows of 520 bf16 values: more wavefronts than are launched, and bytes beyond 32 bits."""
    n, dim, period = (4 << 20) + 99_991, 520, 1021
    few = gauss(period, dim, 9).to(torch.bfloat16).cuda()
    x = few[torch.arange(n, device="cuda") % period]
    r, want = S.quantize_rows(x), S.quantize_rows(few.repeat(3, 1))                  # 3063 rows: the same kernel
    del x
    for lo in range(0, n, 1 << 20):
        hi = min(n, lo + (1 << 20))
        at = torch.arange(lo, hi, device="cuda") % period
        assert torch.equal(r.codes[lo:hi], want.codes[at]) and torch.equal(r.scales[lo:hi], want.scales[at]) and torch.equal(r.norms2[lo:hi], want.norms2[at])
    q = S.quantize_rows(gauss(40, dim, 4).cuda())                                    # tiles: the last rows against all of them
    s = S.score_rows(q, r, M.Euclidean)
    assert torch.equal(s[:, n - 3000:], S.score_rows(q, r, M.Euclidean)[:, n - 3000:])
    check_scores(s[:, n - 200:], held(q), held(r[n - 200:]), M.Euclidean, dim)


# ---------------------------------------------------------------- product

SHAPES = [(1, 1, 1), (1, 15, 16), (2, 16, 17), (16, 17, 127), (17, 33, 128), (15, 64, 129), (3, 100, 100), (1, 1000, 960), (8, 1000, 960), (16, 999, 513),
          (31, 257, 260), (33, 513, 130), (64, 300, 640), (65, 255, 96), (100, 511, 300), (128, 256, 128), (129, 700, 1000), (200, 1000, 64), (256, 256, 512),
          (257, 1025, 768), (300, 77, 2000), (513, 600, 144), (1000, 130, 960), (7, 50, 9000), (5, 40, 4096), (16, 40000, 640), (3, 40, 4097), (2, 33, 4100), (70, 90, 4100), (130, 260, 4224), (1, 70000, 32), (500, 5000, 112),
          # each tile size of the tiled kernel, whole tiles and ragged ones
          (70, 20001, 300), (128, 12800, 64), (300, 60003, 70), (384, 51200, 128), (129, 50001, 200), (512, 25600, 192), (256, 65536, 16), (1000, 20003, 130),
          (40, 150001, 70), (64, 153600, 48), (333, 2049, 200), (128, 8192, 128), (512, 131072, 16), (2000, 40001, 50), (128, 25600, 256),
          (33, 262145, 200), (64, 262144, 100), (128, 262144, 512), (90, 240001, 512),
          # up to 32 queries
          (17, 30000, 100), (32, 16000, 128), (31, 20001, 960), (17, 15000, 129), (32, 40000, 4096), (20, 33333, 300), (25, 14401, 4090),
          # few queries of many columns
          (1, 300, 8192), (3, 33000, 8190), (16, 40001, 5000), (2, 70, 8193), (16, 14400, 8192), (1, 40, 131072), (1, 40, 131073)]


@pytest.mark.parametrize("metric", list(M))
@pytest.mark.parametrize("nq,n,dim", SHAPES)
def test_scores_against_64_bits(vdb, metric, nq, n, dim):
    q, b = S.quantize_rows(gauss(nq, dim, 1).cuda()), S.quantize_rows(gauss(n, dim, 2).cuda())
    check_scores(S.score_rows(q, b, metric), held(q), held(b), metric, dim)


@pytest.mark.parametrize("metric", list(M))
@pytest.mark.parametrize("nq,n", [(1, 333), (20, 333), (70, 333), (300, 333), (100, 20011), (129, 50001), (300, 60003), (600, 120000), (512, 131072), (200, 8001), (64, 150000), (40, 262145), (20, 20011), (32, 16000)])
def test_score_rows_lie_apart_and_what_is_between_stays(vdb, nq, n, metric):
    q, b = S.quantize_rows(gauss(nq, 200, 1).cuda()), S.quantize_rows(gauss(n, 200, 2).cuda())
    want = S.score_rows(q, b, metric)
    for at, wide in ((0, n + 3), (1, n + 7), (3, n + 2), (8, n + 8 + -n % 8)):
        room = torch.full((nq, wide + 8), -5.0, device="cuda")
        S.score_rows(q, b, metric, out=room[:, at:at + n])
        assert torch.equal(room[:, at:at + n], want)
        assert bool((room[:, :at] == -5).all()) and bool((room[:, at + n:] == -5).all())


@pytest.mark.parametrize("nq,n", [(2, 9), (20, 40), (300, 12)])
def test_rows_very_far_apart(vdb, nq, n):
    """Rows 16 MiB and more apart: beyond what the offsets of the tiled kernel hold."""
    step = (1 << 24) + 16
    b = S.quantize_rows(gauss(n, 300, 2).cuda())
    room = torch.empty(n * step, dtype=torch.uint8, device="cuda").as_strided((n, 304), (step, 1))
    room.copy_(b.codes)
    far = S.Q8Rows(room, b.scales, b.norms2, 300)
    q = S.quantize_rows(gauss(nq, 300, 1).cuda())
    check_scores(S.score_rows(q, far, M.Cosine), held(q), held(b), M.Cosine, 300)
    check_scores(S.score_rows(far, q, M.Euclidean), held(b), held(q), M.Euclidean, 300)


@pytest.mark.parametrize("nq,n,dim", [(5, 40, 256), (40, 300, 256), (300, 300, 384), (100, 20000, 256), (300, 30000, 384), (200, 8001, 256), (64, 150000, 256), (500, 131072, 256), (20, 20000, 384), (32, 16000, 128)])
def test_scales_far_apart(vdb, nq, n, dim):
    """Blocks from 2^-60 to 2^60 whose products meet in the middle."""
    g = torch.Generator().manual_seed(4)
    x, y = torch.randn(nq, dim, generator=g), torch.randn(n, dim, generator=g)
    e = torch.randint(-60, 61, (dim // 128,), generator=g).repeat_interleave(128).float()
    q, b = S.quantize_rows((x * torch.exp2(e)).cuda()), S.quantize_rows((y * torch.exp2(-e)).cuda())
    check_scores(S.score_rows(q, b, M.Dot), held(q), held(b), M.Dot, dim)


@pytest.mark.parametrize("nq,n", [(3, 100), (40, 200), (200, 12000)])
@pytest.mark.parametrize("q_scale", [1e-20, 1e-7, 1e-3, 1.0, 1e9, 9e17])
@pytest.mark.parametrize("b_scale", [1e-20, 1e-4, 1.0, 9e17])
def test_small_and_large_rows(vdb, nq, n, q_scale, b_scale):
    """The 1e-10 beside small norms, and norms whose product is beyond what a reciprocal holds."""
    x, y = gauss(nq, 200, 1, 0.1), gauss(n, 200, 2, 0.1)
    x, y = x / x.norm(dim=1, keepdim=True) * 14, y / y.norm(dim=1, keepdim=True) * 14
    y[::3] *= 0.7
    q, b = S.quantize_rows((x * q_scale).cuda()), S.quantize_rows((y * b_scale).cuda())
    check_scores(S.score_rows(q, b, M.Cosine), held(q), held(b), M.Cosine, 200)
    if min(q_scale, b_scale) >= 1e-7 and max(q_scale, b_scale) <= 1e9:              # products of smaller ones are subnormal; (14 * 9e17)^2 twice is beyond f32
        check_scores(S.score_rows(q, b, M.Euclidean), held(q), held(b), M.Euclidean, 200)


@pytest.mark.parametrize("nq,n", [(2, 30), (40, 40), (300, 300), (100, 20000), (300, 60000), (200, 50000), (200, 8001), (64, 150000), (512, 131072), (33, 262145), (20, 20000)])
def test_nonfinite_rows_score_nan_and_no_others(vdb, nq, n):
    x, y = gauss(nq, 200, 1), gauss(n, 200, 2)
    x[1, 150] = float("inf"); y[3, 7] = float("nan"); y[n - 1, 199] = float("-inf")
    q, b = S.quantize_rows(x.cuda()), S.quantize_rows(y.cuda())
    for metric in M:
        s = S.score_rows(q, b, metric).cpu()
        bad = torch.zeros(nq, n, dtype=torch.bool)
        bad[1] = True; bad[:, 3] = True; bad[:, n - 1] = True
        assert torch.equal(torch.isnan(s), bad)


@pytest.mark.parametrize("nq,n", [(1, 50), (9, 3000), (20, 70), (70, 20000), (300, 30000), (20, 20000)])
def test_bytes_behind_a_row_do_not_matter(vdb, nq, n):
    """NaN codes behind the row's 16-byte pieces, any scale behind its last block."""
    dim = 150
    q, b = S.quantize_rows(gauss(nq, dim, 1).cuda()), S.quantize_rows(gauss(n, dim, 2).cuda())
    want = S.score_rows(q, b, M.Dot)

    def wide(r):
        w = S.Q8Rows(torch.full((len(r), 256), 0x7F, dtype=torch.uint8, device="cuda"), torch.full((len(r), 8), 255, dtype=torch.uint8, device="cuda"), None, dim)
        w.codes[:, :160] = r.codes
        w.scales[:, :2] = r.scales[:, :2]
        return w
    assert torch.equal(S.score_rows(wide(q), wide(b), M.Dot), want)


def test_a_scale_of_255_is_nan(vdb):
    q, b = S.quantize_rows(gauss(3, 256, 1).cuda()), S.quantize_rows(gauss(20, 256, 2).cuda())
    b.scales[4, 1] = 255
    s = S.score_rows(q, b, M.Dot)
    assert bool(torch.isnan(s[:, 4]).all()) and int(torch.isnan(s).sum()) == 3


def test_zero_rows(vdb):
    z = torch.zeros(3, 130, device="cuda")
    q = S.quantize_rows(z)
    b = S.quantize_rows(torch.cat([z, gauss(3, 130, 2).cuda()]))
    assert bool((S.score_rows(q, b, M.Dot) == 0).all()) and bool((S.score_rows(q, b, M.Cosine) == 1).all())
    d = S.score_rows(q, b, M.Euclidean)
    assert bool((d[:, :3] == 0).all()) and torch.allclose(d[0, 3:], b.norms2[3:].sqrt(), rtol=4 * U, atol=0)


@pytest.mark.parametrize("nq", [1, 20, 200])
def test_a_row_against_itself(vdb, nq):
    """|q - q|: nothing below zero under the root, and no more than the lost digits allow."""
    q = S.quantize_rows(gauss(nq, 300, 9).cuda())
    for metric in (M.Euclidean, M.Cosine):
        s = S.score_rows(q, q, metric)
        assert not bool(s.isnan().any())
        check_scores(s, held(q), held(q), metric, 300)


def test_scores_are_the_same_bits_from_call_to_call(vdb):
    q, b = S.quantize_rows(gauss(400, 700, 1).cuda()), S.quantize_rows(gauss(2000, 700, 2).cuda())
    whole = S.score_rows(q, b, M.Cosine)
    assert torch.equal(whole, S.score_rows(q, b, M.Cosine))
    for lo, hi in ((0, 1), (5, 21), (100, 140), (200, 300)):
        part = S.score_rows(q[lo:hi], b, M.Cosine)
        check_scores(part, held(q)[lo:hi], held(b), M.Cosine, 700)
        assert torch.equal(part, S.score_rows(q[lo:hi], b, M.Cosine))


def test_offsets_beyond_32_bits(vdb):
    n, dim = 4_300_000, 1000                                          # 4.3 GB of codes
    x = gauss(64, dim, 3).cuda()
    few = S.quantize_rows(x)
    room = S.Q8Rows.empty(n, dim, x.device)
    room.codes.zero_(); room.scales.fill_(127); room.norms2.zero_()
    S.quantize_rows(x, out=room[n - 64:])
    q = S.quantize_rows(gauss(3, dim, 4).cuda())
    s = S.score_rows(q, room, M.Dot)
    assert not bool(s[:, :n - 64].any())
    check_scores(s[:, n - 64:], held(q), held(few), M.Dot, dim)
    del room, s
    q, b = S.quantize_rows(gauss(4400, 16, 5).cuda()), S.quantize_rows(gauss(1_000_000, 16, 6).cuda())
    s = S.score_rows(q, b, M.Dot)                                     # 4.4e9 scores
    check_scores(s[4390:, 999_000:], held(q[4390:]), held(b[999_000:]), M.Dot, 16)
    before = s[4390:, 999_000:].clone()
    S.adjust_scores(s, M.Dot, presence=torch.ones(4400, device="cuda"), seen=torch.full((4400,), 999_999, dtype=torch.int32, device="cuda"),
                    seen_offsets=torch.arange(4401, device="cuda"), out=s)
    before[:, 999] -= 1
    assert torch.equal(s[4390:, 999_000:], before)


def test_the_host_scan_is_the_device_calls(vdb):
    q, b = gauss(20, 150, 1).numpy(), gauss(500, 150, 2).numpy()
    for metric in M:
        got = vdb.q8_score_scan(q, b, metric)
        want = S.score_rows(S.quantize_rows(torch.tensor(q).cuda()), S.quantize_rows(torch.tensor(b).cuda()), metric)
        assert np.array_equal(got, want.cpu().numpy())


# ---------------------------------------------------------------- score rows

def plain_adjust(s, metric, passing=None, boost=None, seen=None, repeat=None, frequency=None, presence=None):
    """-> (result, magnitudes that entered), float64; passing: bool [1 or nq, n]; boost [1 or nq, n]; seen: list of column lists."""
    nq, n = s.shape
    g = s.astype(np.float64) * (1 if metric == M.Dot else -1)
    mag = np.abs(g)
    for q in range(nq):
        if seen is not None:
            cols, times = np.unique([c for c in seen[q] if 0 <= c < n], return_counts=True)
            cols = cols.astype(np.int64)
            if len(cols):
                r = 1.0 if repeat is None else float(repeat[q])
                f = 0.0 if frequency is None else float(frequency[q])
                p = 0.0 if presence is None else float(presence[q])
                v = g[q, cols]
                v = np.where(v > 0, v / r, v * r)
                mag[q, cols] = np.abs(v) + np.abs(f) * times + abs(p)
                g[q, cols] = v - (f * times + p)
    if boost is not None:
        g = g + boost; mag = mag + np.abs(boost)
    if passing is not None:
        g = np.where(passing, g, -np.inf)
    return (g if metric == M.Dot else -g), mag


def words_of(passing):
    m, n = passing.shape
    w = np.zeros((m, -(-n // 32) * 32), np.uint8)
    w[:, :n] = passing
    return torch.tensor(np.packbits(w, axis=1, bitorder="little").view(np.int32).copy()).cuda()


def seen_of(lists):
    off = np.concatenate([[0], np.cumsum([len(l) for l in lists])])
    flat = np.array([c for l in lists for c in l], np.int64)
    return torch.tensor(flat.astype(np.uint32).view(np.int32)).cuda(), torch.tensor(off, dtype=torch.int64).cuda()


def check_adjusted(got, want, mag):
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    fin = np.isfinite(want)
    assert np.array_equal(np.sign(got[np.isinf(want)]), np.sign(want[np.isinf(want)]))
    assert np.all(np.abs(got[fin] - want[fin]) <= 4 * U * mag[fin])


ADJUST = [(1, 1), (1, 31), (2, 32), (3, 33), (5, 100), (1, 10000), (4, 4095), (4, 4096), (4, 4097), (7, 8191), (2, 65537), (300, 129), (1, 300001)]


@pytest.mark.parametrize("metric", list(M))
@pytest.mark.parametrize("nq,n", ADJUST)
@pytest.mark.parametrize("parts", ["pass", "boost", "seen", "all", "none"])
def test_adjusted_scores_against_64_bits(vdb, metric, nq, n, parts):
    rng = np.random.default_rng(nq * 100003 + n)
    s = (rng.standard_normal((nq, n)) * 3).astype(np.float32)
    kw, dev = {}, {}
    if parts in ("pass", "all"):
        kw["passing"] = rng.random((nq if parts == "all" else 1, n)) < 0.3
        dev["pass_bits"] = words_of(kw["passing"])
    if parts in ("boost", "all"):
        b = rng.standard_normal((1 if parts == "all" else nq, n)).astype(np.float32)
        kw["boost"], dev["boost"] = b.astype(np.float64), torch.tensor(b).cuda()
    if parts in ("seen", "all"):
        lists = [list(rng.integers(0, n + 3, size=int(rng.integers(0, 400)))) for _ in range(nq)]
        lists[0] = [n - 1] * 70 + [0] * 3 + [0xFFFFFFFF, n]
        kw["seen"] = lists
        dev["seen"], dev["seen_offsets"] = seen_of(lists)
        for name, lo, hi in (("repeat", 1.0, 2.0), ("frequency", -0.2, 0.5), ("presence", 0.0, 1.0)):
            v = rng.uniform(lo, hi, nq).astype(np.float32)
            kw[name], dev[name] = v, torch.tensor(v).cuda()
    t = torch.tensor(s).cuda()
    got = S.adjust_scores(t, metric, **dev)
    assert torch.equal(t.cpu(), torch.tensor(s))
    check_adjusted(got, *plain_adjust(s, metric, **kw))
    assert torch.equal(S.adjust_scores(t, metric, out=t, **dev), got)                       # in place


@pytest.mark.parametrize("metric", list(M))
def test_masked_columns_hide_whatever_was_there(vdb, metric):
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    s = torch.tensor([[inf, -inf, nan, low, -low, 1.0, 0.0, -0.0] * 9] * 3).cuda()
    none = torch.zeros(1, 3, dtype=torch.int32, device="cuda")
    worst = -inf if metric == M.Dot else inf
    assert bool((S.adjust_scores(s, metric, pass_bits=none) == worst).all())                # a row without a passing column
    every = torch.full((3,), -1, dtype=torch.int32, device="cuda")
    got = S.adjust_scores(s, metric, pass_bits=every)
    assert torch.equal(got.isnan(), s.isnan()) and torch.equal(got.nan_to_num(7), s.nan_to_num(7))
    got = S.adjust_scores(s, metric, boost=torch.full((72,), inf, device="cuda"), pass_bits=none)
    assert bool((got == worst).all())


def test_every_member_alone_and_neutral_values(vdb):
    s = gauss(3, 500, 1).cuda()
    seen, off = seen_of([[1, 2, 2], [], [499] * 1000])
    one, zero = torch.ones(3, device="cuda"), torch.zeros(3, device="cuda")
    assert torch.equal(S.adjust_scores(s, M.Dot), s)
    assert torch.equal(S.adjust_scores(s, M.Dot, seen=seen, seen_offsets=off), s)
    assert torch.equal(S.adjust_scores(s, M.Cosine, seen=seen, seen_offsets=off, repeat=one, frequency=zero, presence=zero), s)
    got = S.adjust_scores(s, M.Dot, seen=seen, seen_offsets=off, frequency=one)
    want = s.clone(); want[0, 1] -= 1; want[0, 2] -= 2; want[2, 499] -= 1000
    assert torch.equal(got, want)


def test_strided_scores_and_bitmaps(vdb):
    rng = np.random.default_rng(3)
    for at, wide in ((0, 1003), (1, 1003), (0, 1004), (4, 1008), (3, 1010)):
        n = 999
        room = torch.tensor(rng.standard_normal((6, wide)).astype(np.float32)).cuda()
        s = room[:, at:at + n]
        passing = rng.random((6, n)) < 0.5
        bits = torch.full((6, 40), -1, dtype=torch.int32, device="cuda"); bits[:, :32] = words_of(passing)
        boost = torch.tensor(rng.standard_normal((6, wide)).astype(np.float32)).cuda()[:, at:at + n]
        want, mag = plain_adjust(s.cpu().numpy(), M.Dot, passing=passing, boost=boost.double().cpu().numpy())
        before = room.clone()
        check_adjusted(S.adjust_scores(s, M.Dot, pass_bits=bits, boost=boost), want, mag)
        out = torch.full((6, wide + 3), 9.0, device="cuda")
        S.adjust_scores(s, M.Dot, pass_bits=bits, boost=boost, out=out[:, 1:1 + n])
        check_adjusted(out[:, 1:1 + n], want, mag)
        assert bool((out[:, 0] == 9).all()) and bool((out[:, 1 + n:] == 9).all()) and torch.equal(room, before)
        S.adjust_scores(s, M.Dot, pass_bits=bits, boost=boost, out=s)
        check_adjusted(s, want, mag)
        keep = torch.ones(wide, dtype=torch.bool, device="cuda"); keep[at:at + n] = False
        assert torch.equal(room[:, keep], before[:, keep])


def test_offsets_that_lie_are_cut(vdb):
    """Offsets beyond the list end at the list; offsets that descend give an empty list."""
    s = torch.zeros(3, 64, device="cuda")
    seen = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    off = torch.tensor([0, 1 << 40, 2, 3], dtype=torch.int64, device="cuda")
    got = S.adjust_scores(s, M.Dot, seen=seen, seen_offsets=off, presence=torch.ones(3, device="cuda"))
    want = torch.zeros(3, 64, device="cuda"); want[0, 1:4] = -1; want[2, 3] = -1
    assert torch.equal(got, want)


@pytest.mark.parametrize("n,length", [(100, 100000), (5000, 20000), (200000, 60000)])
def test_long_lists(vdb, n, length):
    rng = np.random.default_rng(n)
    s = rng.standard_normal((2, n)).astype(np.float32)
    lists = [list(rng.integers(0, n, size=length)), [5] * length]
    seen, off = seen_of(lists)
    f = np.array([0.25, 0.5], np.float32)
    want, mag = plain_adjust(s, M.Dot, seen=lists, frequency=f)
    check_adjusted(S.adjust_scores(torch.tensor(s).cuda(), M.Dot, seen=seen, seen_offsets=off, frequency=torch.tensor(f).cuda()), want, mag)


# ---------------------------------------------------------------- calls

def test_refusals_on_tensors(vdb):
    x = gauss(4, 32, 1).cuda()
    r = S.quantize_rows(x)
    for bad in (x.double(), x[0], x.t(), x.cpu(), x.int()):
        with pytest.raises(ArgumentError):
            S.quantize_rows(bad)
    for bad in (S.Q8Rows.empty(3, 32, x.device), S.Q8Rows.empty(4, 31, x.device)):
        with pytest.raises(ArgumentError):
            S.quantize_rows(x, out=bad)
    with pytest.raises(VectorLengthMismatch):
        S.score_rows(r, S.quantize_rows(gauss(4, 33, 1).cuda()), M.Dot)
    for kw in (dict(out=torch.empty(4, 5, device="cuda")), dict(out=torch.empty(4, 4)), dict(out=torch.empty(4, 4, device="cuda").t()), dict(metric=7)):
        with pytest.raises(ArgumentError):
            S.score_rows(r, r, **{"metric": M.Dot, **kw})
    for codes, scales, dim in ((r.codes, r.scales, 33), (r.codes, r.scales[:2], 32), (r.codes[:, :31], r.scales, 32), (r.codes.float(), r.scales, 32), (r.codes, r.scales, 0)):
        with pytest.raises(ArgumentError):
            S.Q8Rows(codes, scales, None, dim)
    s = torch.zeros(4, 40, device="cuda")
    i4, o4 = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(5, dtype=torch.int64, device="cuda")
    for kw in (dict(pass_bits=torch.zeros(1, dtype=torch.int32, device="cuda")), dict(pass_bits=torch.zeros(3, 2, dtype=torch.int32, device="cuda")), dict(boost=torch.zeros(39, device="cuda")),
               dict(boost=torch.zeros(40)), dict(seen=i4), dict(seen_offsets=o4), dict(seen=i4, seen_offsets=o4[:4]), dict(seen=i4.long(), seen_offsets=o4), dict(repeat=torch.ones(4, device="cuda")),
               dict(seen=i4, seen_offsets=o4, presence=torch.ones(3, device="cuda")), dict(out=s[:3]), dict(out=torch.zeros(4, 80, device="cuda")[:, ::2]), dict(boost=s[0], out=s)):
        with pytest.raises(ArgumentError):
            S.adjust_scores(s, M.Dot, **kw)


def test_host_pointers_are_refused(vdb):
    """A pageable host pointer where device memory is expected is an error, not a fault."""
    x = np.zeros((4, 128), np.float32); dev = S.quantize_rows(torch.zeros(4, 128, device="cuda"))
    with pytest.raises(ArgumentError):
        vdb.check(vdb.fn.q8_quantize_dev(x.ctypes.data, 0, 128, C.byref(dev._c), None))
    host = Q8RowsC(dev._c.codes, dev._c.scales, x.ctypes.data, 4, 128, 128, 4)
    out = torch.zeros(4, 4, device="cuda")
    with pytest.raises(ArgumentError):
        vdb.check(vdb.fn.q8_score_dev(C.byref(dev._c), C.byref(host), 0, out.data_ptr(), 4, None))
    how = ScoreAdjustC(boost=x.ctypes.data)
    with pytest.raises(ArgumentError):
        vdb.check(vdb.fn.score_adjust_dev(out.data_ptr(), 4, 4, 4, 1, C.byref(how), out.data_ptr(), 4, None))
    torch.cuda.synchronize()


def test_empty_tensors(vdb):
    e = S.quantize_rows(torch.zeros(0, 32, device="cuda"))
    r = S.quantize_rows(torch.ones(3, 32, device="cuda"))
    assert len(e) == 0 and S.score_rows(e, r, M.Cosine).shape == (0, 3) and S.score_rows(r, e, M.Cosine).shape == (3, 0)
    assert S.adjust_scores(torch.zeros(0, 5, device="cuda"), M.Dot).shape == (0, 5) and S.adjust_scores(torch.zeros(5, 0, device="cuda"), M.Dot).shape == (5, 0)


def chain(x, y, metric, **how):
    return S.adjust_scores(S.score_rows(S.quantize_rows(x), S.quantize_rows(y), metric), metric, **how)


@pytest.mark.parametrize("metric", list(M))
@pytest.mark.parametrize("nq,n,dim", [(1, 500, 96), (20, 5000, 768), (150, 3000, 200)])
def test_the_run_of_them(vdb, metric, nq, n, dim):
    """Rows quantised, scored, adjusted: against 64 bits from the held values on."""
    rng = np.random.default_rng(1)
    x, y = gauss(nq, dim, 1, 0.2), gauss(n, dim, 2, 0.2)
    passing = rng.random((1, n)) < 0.5
    boost = (rng.standard_normal((1, n)) * 0.1).astype(np.float32)
    lists = [list(rng.integers(0, n, 30)) for _ in range(nq)]
    pres = rng.random(nq).astype(np.float32)
    seen, off = seen_of(lists)
    got = chain(x.cuda(), y.cuda(), metric, pass_bits=words_of(passing), boost=torch.tensor(boost).cuda(), seen=seen, seen_offsets=off, presence=torch.tensor(pres).cuda())
    q, b = S.quantize_rows(x.cuda()), S.quantize_rows(y.cuda())
    s = S.score_rows(q, b, metric)
    check_scores(s, held(q), held(b), metric, dim)
    check_adjusted(got, *plain_adjust(s.cpu().numpy(), metric, passing=passing, boost=boost.astype(np.float64), seen=lists, presence=pres))


def test_a_segments_filter_masks_its_rows(vdb):
    """The bitmap that a segment compiles for a filter is the bitmap that score rows are masked with."""
    rng = np.random.default_rng(5)
    n, dim = 700, 64
    x = rng.standard_normal((n, dim)).astype(np.float32)
    seg = vdb.Segment(vdb.HNSWIndex(vdb.DistanceMetric.Euclidean, 8, 32, 8, dim))
    tier = rng.integers(0, 5, n)
    seg.insert_batch_columns(x, {"tier": tier})
    f = vdb.Filter.Compare("tier", vdb.ScalarComparisonOp.Lt, vdb.PayloadValue.Int(2))
    words = -(-n // 32)
    p, e = np.zeros(words, np.uint32), np.zeros(words, np.uint32)
    vdb.check(vdb.fn.segment_filter_bitmaps(seg._h, f._h, p.ctypes.data, e.ctypes.data, words))
    t = torch.tensor(x).cuda()
    s = chain(t[:4], t, M.Euclidean, pass_bits=torch.tensor(p.view(np.int32)).cuda())
    assert torch.equal(torch.isinf(s[0]).cpu(), torch.tensor(tier >= 2))


def test_two_streams_at_once(vdb):
    jobs = [(gauss(60 + 70 * i, 300, i).cuda(), gauss(4000, 300, 50 + i).cuda()) for i in range(4)]
    want = [chain(x, y, M.Cosine) for x, y in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    for _ in range(5):
        got = []
        for s, (x, y) in zip(streams, jobs):
            with torch.cuda.stream(s):
                got.append(chain(x, y, M.Cosine))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_and_replayed(vdb):
    """Two captured graphs replayed between each other and eager work: every replay equals the eager result on the same inputs."""
    nq, n, dim = 40, 3000, 200
    rng = np.random.default_rng(2)
    seen, off = seen_of([list(rng.integers(0, n, 50)) for _ in range(nq)])
    how = dict(pass_bits=words_of(rng.random((1, n)) < 0.5), seen=seen, seen_offsets=off, frequency=torch.rand(nq, device="cuda"))
    graphs = []
    for k in range(2):
        x, y = gauss(nq, dim, k).cuda(), gauss(n, dim, 10 + k).cuda()
        q, b = S.Q8Rows.empty(nq, dim, x.device), S.Q8Rows.empty(n, dim, x.device)
        s, out = torch.empty(nq, n, device="cuda"), torch.empty(nq, n, device="cuda")

        def once():
            S.quantize_rows(x, out=q); S.quantize_rows(y, out=b)
            S.score_rows(q, b, M.Euclidean, out=s)
            S.adjust_scores(s, M.Euclidean, out=out, **how)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            once()
        graphs.append((g, x, y, out))
    for turn in range(4):
        for g, x, y, out in graphs:
            x.copy_(gauss(nq, dim, 100 + turn)); y.copy_(gauss(n, dim, 200 + turn))
            g.replay()
        torch.cuda.synchronize()
        for g, x, y, out in graphs:
            assert torch.equal(out, chain(x, y, M.Euclidean, **how))


def test_host_threads_at_once(vdb):
    import threading
    x, y = gauss(30, 128, 1).cuda(), gauss(2000, 128, 2).cuda()
    want = chain(x, y, M.Dot)
    torch.cuda.synchronize()
    bad = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = chain(x, y, M.Dot)
                torch.cuda.current_stream().synchronize()
                if not torch.equal(got, want):
                    bad.append(1)
    ts = [threading.Thread(target=work) for _ in range(4)]
    [t.start() for t in ts]; [t.join() for t in ts]
    assert not bad
