"""The operators on 8-bit rows and on dense score rows: their plain forms, and the calls a user makes.

  quantize   rows -> e4m3 codes, one power-of-two scale per row and block of 128 columns, squared norms
  score      nq x n scores (dot, cosine, euclidean) of queries and rows held that way
  adjust     filter bitmaps, boosts and the demotion of rows already shown, on dense score rows

Layout of 8-bit rows: codes uint8 [n, dim rounded up to 16] (zero beyond dim), scales uint8 [n, blocks rounded up to 4]
(exponent + 127, 127 beyond the last block), norms2 float32 [n].
"""
import torch

own = False

BLOCK = 128
METRICS = ("cosine", "dot", "euclidean")
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def up(v, m):
    return -(-v // m) * m


def listed():
    return [
        # one query against ten thousand short rows: what a small collection answers per call, bound by latency
        {"name": "score 1x10k x128", "op": "score", "nq": 1, "n": 10_000, "dim": 128, "metric": "cosine"},
        # one query against a million long rows: a pass over the rows, bound by memory
        {"name": "score 1x1M x960", "op": "score", "nq": 1, "n": 1_000_000, "dim": 960, "metric": "cosine"},
        # eight queries share the pass
        {"name": "score 8x1M x960", "op": "score", "nq": 8, "n": 1_000_000, "dim": 960, "metric": "dot"},
        # a ragged batch: odd counts, rows that end inside a block
        {"name": "score 77x300007 x100", "op": "score", "nq": 77, "n": 300_007, "dim": 100, "metric": "euclidean"},
        # a batch of a thousand queries against the whole collection: matrix cores and 4 GB of scores
        {"name": "score 1000x1M x960", "op": "score", "nq": 1000, "n": 1_000_000, "dim": 960, "metric": "cosine"},
        # long rows against a vocabulary-sized table: matrix cores alone
        {"name": "score 4096x32000 x4096", "op": "score", "nq": 4096, "n": 32_000, "dim": 4096, "metric": "dot"},
        # the one query of a call
        {"name": "quantize 1 x960", "op": "quantize", "n": 1, "dim": 960, "type": "float32"},
        # rows as a half-precision embedding model hands them over, ragged
        {"name": "quantize 300007 x100 bf16", "op": "quantize", "n": 300_007, "dim": 100, "type": "bfloat16"},
        # a whole collection at once
        {"name": "quantize 1M x960", "op": "quantize", "n": 1_000_000, "dim": 960, "type": "float32"},
        # one query's scores: a narrow filter and what its user has seen
        {"name": "adjust 1x10k", "op": "adjust", "nq": 1, "n": 10_000, "metric": "dot", "seen": 50, "pass_pct": 10, "own_mask": False, "boost": False},
        # a batch over a vocabulary-sized table, every query with a mask and a long history of its own
        {"name": "adjust 64x128000", "op": "adjust", "nq": 64, "n": 128_000, "metric": "dot", "seen": 4000, "pass_pct": 50, "own_mask": True, "boost": True},
        # distances to a million rows, one filter and one boost for all queries, odd count
        {"name": "adjust 16x1000003", "op": "adjust", "nq": 16, "n": 1_000_003, "metric": "euclidean", "seen": 300, "pass_pct": 90, "own_mask": False, "boost": True},
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, even over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["score", "score", "quantize", "adjust"])
    if op == "score":
        nq, dim = _spread(rng, 1, 10_000), _spread(rng, 8, 4096)
        most = min(1_000_000, 1_000_000_000 // nq, 960_000_000 // dim, int(9.6e11) // (nq * dim))
        return {"op": op, "nq": nq, "n": _spread(rng, min(1000, most), most), "dim": dim, "metric": rng.choice(METRICS)}
    if op == "quantize":
        dim = _spread(rng, 8, 4096)
        return {"op": op, "n": _spread(rng, 1, min(1_000_000, 960_000_000 // dim)), "dim": dim, "type": rng.choice(sorted(TYPES))}
    nq = _spread(rng, 1, 256)
    n = _spread(rng, 1000, min(1_000_003, 16_000_000 // nq))
    return {"op": op, "nq": nq, "n": n, "metric": rng.choice(METRICS), "seen": rng.choice([0, _spread(rng, 1, 4000)]),
            "pass_pct": rng.choice([1, 10, 50, 100]), "own_mask": rng.random() < 0.5, "boost": rng.random() < 0.5}


# ---------------------------------------------------------------- inputs

def _rows(n, dim, metric, g):
    """Embedding-like rows: blobs around centres with non-negative coordinates for distances; blocks of differing size for products."""
    dev = g.device
    if metric == "dot":
        x = torch.randn(n, dim, generator=g, device=dev)
        return x.mul_(torch.randn(n, 1, generator=g, device=dev).mul_(0.5).exp_())
    centres = torch.rand(256, dim, generator=torch.Generator(device=dev).manual_seed(77), device=dev) * 128
    x = centres[torch.randint(256, (n,), generator=g, device=dev)]
    return x.add_(torch.randn(n, dim, generator=g, device=dev), alpha=12.0).clamp_(min=0)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "quantize":
        return {"op": "quantize", "rows": _rows(case["n"], case["dim"], "euclidean", g).to(TYPES[case["type"]])}
    if case["op"] == "score":
        side = [_quantize(_rows(k, case["dim"], case["metric"], g)) for k in (case["nq"], case["n"])]
        return {"op": "score", "queries": side[0], "base": side[1], "dim": case["dim"], "metric": case["metric"]}
    nq, n = case["nq"], case["n"]
    s = torch.randn(nq, n, generator=g, device="cuda") * 4
    if case["metric"] != "dot":
        s = s.abs_() + 0.5
    st = {"op": "adjust", "metric": case["metric"], "scores": s, "pass_bits": None, "boost": None, "seen": None, "seen_offsets": None,
          "repeat": None, "frequency": None, "presence": None}
    if case["pass_pct"] < 100:
        m, words = (nq if case["own_mask"] else 1), up(n, 32) // 32
        bits = torch.rand(m, words, 32, generator=g, device="cuda") < case["pass_pct"] / 100
        w = (bits.to(torch.int64) << torch.arange(32, device="cuda")).sum(-1)
        st["pass_bits"] = torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)
    if case["boost"]:
        st["boost"] = torch.randn(n, generator=g, device="cuda") * 0.1
    if case["seen"]:
        lens = torch.randint(case["seen"] // 2, case["seen"] + 1, (nq,), generator=g, device="cuda")
        st["seen_offsets"] = torch.cat([lens.new_zeros(1), lens.cumsum(0)])
        at = torch.rand(int(lens.sum()), generator=g, device="cuda") ** 3 * n            # some rows many times
        st["seen"] = at.to(torch.int32).clamp_(max=n - 1)
        st["repeat"] = torch.rand(nq, generator=g, device="cuda") * 0.5 + 1
        st["frequency"] = torch.rand(nq, generator=g, device="cuda") * 0.5
        st["presence"] = torch.rand(nq, generator=g, device="cuda")
    return st


# ---------------------------------------------------------------- plain forms

def _quantize(rows):
    n, dim = rows.shape
    nb = up(dim, BLOCK) // BLOCK
    x = torch.zeros(n, nb * BLOCK, device=rows.device)
    x[:, :dim] = rows
    x = x.view(n, nb, BLOCK)
    fine = torch.isfinite(x)
    a = torch.where(fine, x.abs(), 0).amax(-1)
    m, e = torch.frexp(a)                                                                # a = m 2^e, 1/2 <= m < 1
    e = torch.where(a == 0, 0, (e - 9 + (m > 0.875)).clamp(min=-100))
    half = -(e // 2)                                                                     # 2^-e in two factors that are both ordinary floats
    c = x * torch.exp2(half.float()).unsqueeze(-1) * torch.exp2((-e - half).float()).unsqueeze(-1)
    codes = torch.where(fine, c, float("nan")).to(torch.float8_e4m3fn)
    s = torch.exp2(e.float())
    norms2 = (codes.float().square().sum(-1) * s * s).sum(-1)
    scales = torch.full((n, up(nb, 4)), 127, dtype=torch.uint8, device=rows.device)
    scales[:, :nb] = (e + 127).to(torch.uint8)
    return {"codes": codes.view(n, nb * BLOCK)[:, :up(dim, 16)].contiguous().view(torch.uint8), "scales": scales, "norms2": norms2}


def _values(r, dim, dtype):
    s = torch.exp2(r["scales"][:, :up(dim, BLOCK) // BLOCK].to(dtype) - 127)
    return r["codes"].view(torch.float8_e4m3fn)[:, :dim].to(dtype) * s.repeat_interleave(BLOCK, 1)[:, :dim]


def _score(st):
    q, b = st["queries"], st["base"]
    out = _values(q, st["dim"], torch.float32) @ _values(b, st["dim"], torch.float32).T
    nq, nb = q["norms2"][:, None], b["norms2"][None, :]
    if st["metric"] == "cosine":
        return 1 - out / (nq.sqrt() * nb.sqrt() + 1e-10)
    if st["metric"] == "euclidean":
        return (nq + nb - 2 * out).clamp(min=0).sqrt()
    return out


def _adjust(st):
    nq, n = st["scores"].shape
    dev = st["scores"].device
    g = st["scores"] if st["metric"] == "dot" else -st["scores"]
    if st["seen"] is not None:
        lens = st["seen_offsets"][1:] - st["seen_offsets"][:-1]
        row = torch.repeat_interleave(torch.arange(nq, device=dev), lens, output_size=st["seen"].numel())
        count = torch.zeros(nq * n, dtype=torch.int32, device=dev)
        count.index_add_(0, row * n + st["seen"], torch.ones_like(st["seen"]))
        c = count.view(nq, n).float()
        rep = st["repeat"][:, None]
        d = torch.where(g > 0, g / rep, g * rep) - (st["frequency"][:, None] * c + st["presence"][:, None])
        g = torch.where(c > 0, d, g)
    if st["boost"] is not None:
        g = g + st["boost"]
    if st["pass_bits"] is not None:
        ok = (st["pass_bits"][:, :, None] >> torch.arange(32, device=dev, dtype=torch.int32)) & 1
        g = torch.where(ok.view(ok.shape[0], -1)[:, :n] != 0, g, float("-inf"))
    return g if st["metric"] == "dot" else -g


def _plain(st):
    if st["op"] == "quantize":
        return _quantize(st["rows"].float())
    return _score(st) if st["op"] == "score" else _adjust(st)


# ---------------------------------------------------------------- the framework's calls

def _framework(st):
    from vectordb_amd import scores as S
    if st["op"] == "quantize":
        r = S.quantize_rows(st["rows"])
        return {"codes": r.codes, "scales": r.scales, "norms2": r.norms2}
    metric = {"cosine": S.DistanceMetric.Cosine, "dot": S.DistanceMetric.Dot, "euclidean": S.DistanceMetric.Euclidean}[st["metric"]]
    if st["op"] == "score":
        return S.score_rows(S.Q8Rows(dim=st["dim"], **st["queries"]), S.Q8Rows(dim=st["dim"], **st["base"]), metric)
    return S.adjust_scores(st["scores"], metric, pass_bits=st["pass_bits"], boost=st["boost"], seen=st["seen"], seen_offsets=st["seen_offsets"],
                           repeat=st["repeat"], frequency=st["frequency"], presence=st["presence"])


def run(state):
    out = _framework(state) if own else _plain(state)
    if state["op"] == "quantize":
        out["codes"] = out["codes"].view(torch.float8_e4m3fn)
    return out


def work(case):
    if case["op"] == "quantize":
        n, dim = case["n"], case["dim"]
        size = 4 if case["type"] == "float32" else 2
        return {"bytes": n * (dim * size + dim + up(dim, BLOCK) // BLOCK + 4), "flops": 4 * n * dim}
    if case["op"] == "score":
        nq, n, dim = case["nq"], case["n"], case["dim"]
        row = dim + up(dim, BLOCK) // BLOCK + (0 if case["metric"] == "dot" else 4)
        return {"bytes": (nq + n) * row + 4 * nq * n, "flops": 2 * nq * n * dim}
    nq, n = case["nq"], case["n"]
    side = 0 if case["pass_pct"] == 100 else up(n, 32) // 8 * (nq if case["own_mask"] else 1)
    side += 4 * n if case["boost"] else 0
    side += nq * (3 * case["seen"] + 20) if case["seen"] else 0                         # lists of three quarters of the longest on average
    return {"bytes": 8 * nq * n + side, "flops": 2 * nq * n}


# ---------------------------------------------------------------- the definitions in 64 bits

def _exact_codes(x):
    """x / 2^e to the nearest value with four significant bits (three below 2^-6 lose one each), ties to even."""
    ax = x.abs()
    step = torch.exp2(torch.floor(torch.log2(ax.clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step                                                  # torch.round: halves to even


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "quantize":
        x = st["rows"].double()
        n, dim = x.shape
        nb, wide = up(dim, BLOCK) // BLOCK, up(dim, 16)
        codes, norms2 = torch.zeros(n, wide, dtype=torch.float64, device=x.device), torch.zeros(n, dtype=torch.float64, device=x.device)
        for b in range(nb):
            part = x[:, b * BLOCK:(b + 1) * BLOCK]
            a = part.abs().amax(1, keepdim=True)
            e = torch.ceil(torch.log2(a.clamp(min=2.0 ** -100) / 448))                   # the smallest e with a <= 448 2^e
            e = e + (a > 448 * torch.exp2(e)).double() - (a <= 224 * torch.exp2(e)).double()
            e = torch.where(a == 0, 0, e)
            c = _exact_codes(part * torch.exp2(-e))
            codes[:, b * BLOCK:b * BLOCK + part.shape[1]] = c
            norms2 += (c * torch.exp2(e)).square().sum(1)
        return {"codes": codes, "scales": None, "norms2": norms2}
    if case["op"] == "score":
        q, b = _values(st["queries"], st["dim"], torch.float64), _values(st["base"], st["dim"], torch.float64)
        nq, nb = st["queries"]["norms2"].double()[:, None], st["base"]["norms2"].double()
        out = torch.empty(q.shape[0], b.shape[0], dtype=torch.float64, device=q.device)
        for at in range(0, b.shape[0], 1 << 16):
            p = slice(at, at + (1 << 16))
            d = torch.mm(q, b[p].t().contiguous())
            if case["metric"] == "cosine":
                d = 1 - d / (torch.sqrt(nq * nb[p]) + 1e-10)
            elif case["metric"] == "euclidean":
                d = torch.sqrt(torch.relu(nq + nb[p] - d - d))
            out[:, p] = d
        return out
    s = st["scores"].double()
    sign = 1.0 if case["metric"] == "dot" else -1.0
    out = torch.empty_like(s)
    for i in range(s.shape[0]):
        g = s[i] * sign
        if st["seen"] is not None:
            lo, hi = st["seen_offsets"][i:i + 2].tolist()
            at, times = torch.unique(st["seen"][lo:hi].long(), return_counts=True)
            v, r = g[at], st["repeat"][i].double()
            v = torch.maximum(v, v.new_zeros(())) / r + torch.minimum(v, v.new_zeros(())) * r
            g[at] = v - times * st["frequency"][i].double() - st["presence"][i].double()
        if st["boost"] is not None:
            g += st["boost"].double()
        if st["pass_bits"] is not None:
            w = st["pass_bits"][i if case["own_mask"] else 0].long() & 0xFFFFFFFF
            j = torch.arange(s.shape[1], device=s.device)
            g[(w[j // 32] // (2 ** (j % 32))) % 2 == 0] = -float("inf")
        out[i] = g * sign
    return out
