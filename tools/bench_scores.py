"""The operators on 8-bit rows and score rows: times of whole calls, and the launches that a profile is taken of.

    python tools/bench_scores.py [--plain] [--only "NAME|NAME"]      a call of every listed case (perf/operators.py) and of a few more, us
    python tools/bench_scores.py --calls 30                         nothing but that many calls of every listed case, in order
    python tools/bench_scores.py --reduce DIR                       what rocprofv3 wrote of such runs -> profiles/q8_rows_and_score_rows_*

Profiles, each in a run of its own:
    rocprofv3 --kernel-trace --stats --output-format csv -d DIR/stats -- python3 tools/bench_scores.py --calls 30
    rocprofv3 --pmc SQ_WAVES SQ_BUSY_CU_CYCLES SQ_INSTS_VALU SQ_INSTS_VALU_MFMA_BF16 SQ_VALU_MFMA_BUSY_CYCLES SQ_INSTS_LDS SQ_LDS_BANK_CONFLICT SQ_INSTS_VMEM \\
              --kernel-trace --output-format csv -d DIR/sq -- python3 tools/bench_scores.py --calls 3
    rocprofv3 --pmc FETCH_SIZE --kernel-trace --output-format csv -d DIR/fetch -- python3 tools/bench_scores.py --calls 3
    rocprofv3 --pmc WRITE_SIZE --kernel-trace --output-format csv -d DIR/write -- python3 tools/bench_scores.py --calls 3
"""
import argparse
import csv
import glob
import importlib.util
import json
import os
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


def operators():
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def timed(once, sets, block_s=0.1, blocks=7):
    """Median over blocks of calls that follow each other, the inputs in turn, each result kept until the next is there; us."""
    import torch

    def block(n, at):
        torch.cuda.synchronize()
        t = time.perf_counter()
        for i in range(n):
            r = once(sets[(at + i) % len(sets)])  # noqa: F841
        torch.cuda.synchronize()
        return (time.perf_counter() - t) / n
    for _ in range(3):
        one = block(20, 0)
    n = max(3, min(20000, int(block_s / one)))
    return sorted(block(n, b) for b in range(blocks))[blocks // 2] * 1e6


def measure(a, m):
    import numpy as np
    import torch
    import vectordb_amd
    from vectordb_amd import scores as S

    def line(name, own, plain=None):
        print(json.dumps({"case": name, "us": round(own, 2), **({} if plain is None else {"plain_us": round(plain, 2)})}), flush=True)
    more = [{"name": "adjust 1x1000, boosts alone", "op": "adjust", "nq": 1, "n": 1000, "metric": "dot", "seen": 0, "pass_pct": 100, "own_mask": False, "boost": True},
            {"name": "adjust 16x1000003, boosts alone", "op": "adjust", "nq": 16, "n": 1000003, "metric": "dot", "seen": 0, "pass_pct": 100, "own_mask": False, "boost": True},
            {"name": "adjust 1x1000, nothing", "op": "adjust", "nq": 1, "n": 1000, "metric": "euclidean", "seen": 0, "pass_pct": 100, "own_mask": False, "boost": False},
            {"name": "adjust 64x128000 without lists", "op": "adjust", "nq": 64, "n": 128000, "metric": "dot", "seen": 0, "pass_pct": 50, "own_mask": True, "boost": True}]
    only = a.only.split("|") if a.only else None
    for case in m.listed() + more:
        if only and case["name"] not in only:
            continue
        sets = [m.prepare(case, seed) for seed in range(3)]
        m.own = True
        own = timed(m.run, sets)
        m.own = False
        line(case["name"], own, timed(m.run, sets) if a.plain else None)
        del sets
        torch.cuda.empty_cache()
    if only:
        return
    # one list of a million columns among fifteen queries without
    s = torch.randn(16, 1_000_003, device="cuda")
    seen = torch.randint(0, 1_000_003, (1_000_000,), device="cuda", dtype=torch.int32)
    for name, lens in (("one query", [1_000_000] + [0] * 15), ("all queries alike", [62_500] * 16)):
        off = torch.tensor([0] + lens, device="cuda").cumsum(0)
        line("adjust 16x1000003, a million seen columns, " + name, timed(lambda _: S.adjust_scores(s, 1, seen=seen, seen_offsets=off, out=s), [None]))
    del s
    api = vectordb_amd.api()
    for nq, n, dim in ((1, 10_000, 128), (100, 100_000, 960)):
        g = np.random.default_rng(0)
        q, b = g.standard_normal((nq, dim), np.float32), g.standard_normal((n, dim), np.float32)
        line(f"host scan {nq} x {n} x {dim}", timed(lambda _: api.q8_score_scan(q, b, 0), [None], block_s=0.3, blocks=3))


def calls(a, m):
    import torch
    m.own = True
    for case in m.listed():
        state = m.prepare(case, 1)
        for _ in range(a.calls):
            m.run(state)
        torch.cuda.synchronize()
        del state
        torch.cuda.empty_cache()


def newest(pattern):
    return max(glob.glob(pattern, recursive=True), key=os.path.getmtime)


def short(name):
    if "quantize_kernelIDF16bLi16ELb0" in name:
        return "quantize_kernel<__bf16, 16, false>"
    name = name.replace("void ", "").replace("vdb::(anonymous namespace)::", "").replace("vdb::", "")
    return name[:name.index("(")] if "(" in name else name


def reduce(a, m):
    cases = [c["name"] for c in m.listed()]
    to = os.path.join(ROOT, "profiles", "q8_rows_and_score_rows_")
    rows = sorted((r for r in csv.DictReader(open(newest(a.reduce + "/stats/**/*kernel_trace.csv"))) if "vdb" in r["Kernel_Name"]), key=lambda r: int(r["Start_Timestamp"]))
    per = len(rows) // len(cases)
    assert per * len(cases) == len(rows)
    with open(to + "kernel_times.csv", "w") as f:
        w = csv.writer(f)
        w.writerow(["case", "kernel", "workgroups", "launches", "min_us", "median_us", "max_us"])
        for i, c in enumerate(cases):
            g = rows[per * i:per * i + per]
            assert len({r["Kernel_Name"] for r in g}) == 1
            t = sorted((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3 for r in g)
            w.writerow([c, short(g[0]["Kernel_Name"]), int(g[0]["Grid_Size_X"]) // int(g[0]["Workgroup_Size_X"]), per, round(t[0], 2), round(t[per // 2], 2), round(t[-1], 2)])
    out = {}
    for group in ("sq", "fetch", "write"):
        launches = {}
        for r in csv.DictReader(open(newest(a.reduce + "/" + group + "/**/*counter_collection.csv"))):
            if "vdb" in r["Kernel_Name"]:
                launches.setdefault(int(r["Dispatch_Id"]), {"kernel": short(r["Kernel_Name"])})[r["Counter_Name"]] = float(r["Counter_Value"])
        launches = [launches[k] for k in sorted(launches)]
        per = len(launches) // len(cases)
        assert per * len(cases) == len(launches)
        for i, c in enumerate(cases):
            e = out.setdefault(c, {"kernel": launches[per * i]["kernel"]})
            e.update({k: round(v) for k, v in launches[per * i + per - 1].items() if k != "kernel"})
    for e in out.values():
        if e.get("SQ_VALU_MFMA_BUSY_CYCLES"):
            e["matrix_pipes_busy_of_cu_busy_cycles"] = round(e["SQ_VALU_MFMA_BUSY_CYCLES"] / 4 / e["SQ_BUSY_CU_CYCLES"], 3)
        e["hbm_MB"] = round((2 * e["FETCH_SIZE"] + e["WRITE_SIZE"]) * 1024 / 1e6, 1)
    with open(to + "counters.json", "w") as f:
        json.dump({"what": "one launch per case, the last of three; FETCH_SIZE / WRITE_SIZE in KiB as reported; hbm_MB = 2 x FETCH_SIZE + WRITE_SIZE (a read of 128 bytes is counted as 64)",
                   "cases": out}, f, indent=1)


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--plain", action="store_true")
    ap.add_argument("--only", default="", help="names, separated by |")
    ap.add_argument("--calls", type=int, default=0)
    ap.add_argument("--reduce", default="")
    a = ap.parse_args()
    m = operators()
    return reduce(a, m) if a.reduce else calls(a, m) if a.calls else measure(a, m)


if __name__ == "__main__":
    main()
