"""Times the position operators on the cases of perf/operators.py (one GPU).

  python scripts/position_ops_time.py                      us a call among calls, every case
  rocprofv3 --kernel-trace -f csv -d DIR -- python scripts/position_ops_time.py --seconds 0.15
  python scripts/position_ops_time.py --trace DIR          the trace by case: every kernel's median, their sum, and the period of
                                                           a pass (first kernel to first kernel)
  rocprofv3 --pmc ... --kernel-trace -f csv -d DIR -- python scripts/position_ops_time.py --passes 3 --only NAME[,NAME]
  python scripts/position_ops_time.py --counters DIR       what the counters say of each kernel

Calls go round three sets of inputs of different seeds, one after another without waiting, in every mode; what they share of the
last-level cache is what three sets leave there.  An idle card takes tens of milliseconds of work to reach its clock (a kernel of
309 us takes 375 at first): times and traces begin behind 0.1 s of it; the counters' runs do not, so they are given in cycles."""
import argparse
import collections
import csv
import glob
import os
import statistics
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
OURS = ("qk_norm_rope", "rel_attn")
CUS, XCDS = 256, 8


def states(M, case):
    return [M.prepare(case, seed) for seed in (1, 2, 3)]


def run(M, cases, passes, seconds):
    import torch
    for c in cases:
        st = states(M, c)
        n, end = 0, time.perf_counter() + (seconds or 0.0)
        while n < (passes or 30) or time.perf_counter() < end:
            for _ in range(min(30, passes or 30)):
                M.run(st[n % 3])
                n += 1
            torch.cuda.synchronize()
        print("done", c["name"], flush=True)


def time_calls(M, cases):
    import torch
    for c in cases:
        st = states(M, c)
        def took(n):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for i in range(n):
                M.run(st[i % 3])
            b.record()
            b.synchronize()
            return a.elapsed_time(b) * 1e3 / n
        n = int(max(30, min(4000, 100e3 / took(30))))
        took(n)
        got = [took(n) for _ in range(7)]
        w = M.work(c)
        us = statistics.median(got)
        print(f"{c['name']:24s} {us:9.2f} us  ({min(got):.2f} .. {max(got):.2f})  {w['bytes'] / us / 1e6:6.2f} TB/s  "
              f"{w['flops'] / us / 1e6:7.1f} TFLOP/s", flush=True)


def rows_of(where, kind):
    rows = []
    for f in sorted(glob.glob(os.path.join(where, "**", f"*{kind}.csv"), recursive=True)):
        rows += csv.DictReader(open(f))
    return rows


def short(name):
    return name.split("(")[0].replace("void ", "").replace("unsigned short", "bf16").replace("float", "fp32")


def trace(where, names):
    """kernels of other origin (the next case's inputs) part one case's launches from the next's"""
    runs, last = [], False
    for r in sorted(rows_of(where, "kernel_trace"), key=lambda r: int(r["Start_Timestamp"])):
        ours = any(o in r["Kernel_Name"] for o in OURS)
        if ours and not last:
            runs.append([])
        if ours:
            runs[-1].append((short(r["Kernel_Name"]), int(r["Start_Timestamp"]), int(r["End_Timestamp"]), r["Grid_Size_X"], r["VGPR_Count"]))
        last = ours
    for name, got in zip(names, runs):
        first = got[0][0]
        length = next((i for i in range(1, len(got)) if got[i][0] == first and len(got) % i == 0 and
                       [g[0] for g in got[i:2 * i]] == [g[0] for g in got[:i]]), len(got))
        passes = [got[i:i + length] for i in range(0, len(got), length)]
        behind = passes[0][0][1] + 100e6
        passes = [p for p in passes if p[0][1] > behind] or passes
        starts = [p[0][1] for p in passes]
        period = statistics.median([b - a for a, b in zip(starts, starts[1:])] or [0]) / 1e3
        medians = [statistics.median(p[i][2] - p[i][1] for p in passes) / 1e3 for i in range(length)]
        print(f"{name}: kernels {sum(medians):.1f} us of a period of {period:.1f}")
        for i, (k, _, _, grid, vgpr) in enumerate(passes[0]):
            lo = min(p[i][2] - p[i][1] for p in passes) / 1e3
            print(f"  {medians[i]:8.1f}  (least {lo:.1f})  grid {grid}  registers {vgpr}  {k}")


def counters(where):
    got = collections.OrderedDict()
    for r in rows_of(where, "counter_collection"):
        if any(o in r["Kernel_Name"] for o in OURS):
            got.setdefault(short(r["Kernel_Name"]) + " grid " + r["Grid_Size"], collections.OrderedDict()).setdefault(
                r["Counter_Name"], []).append(float(r["Counter_Value"]))
    for k, c in got.items():
        v = {n: statistics.median(x) for n, x in c.items()}
        cycles = v.get("GRBM_GUI_ACTIVE", 0.0) / XCDS
        print(k)
        if cycles:
            share = lambda n, per: f"{100 * v[n] / (cycles * CUS * per):.0f} %" if n in v else "-"
            print(f"  {cycles:.0f} cycles;  of the time: matrix pipes {share('SQ_VALU_MFMA_BUSY_CYCLES', 4)}, vector instructions "
                  f"{share('SQ_ACTIVE_INST_VALU', 1)}, LDS {share('SQ_LDS_IDX_ACTIVE', 1)}, its bank conflicts {share('SQ_LDS_BANK_CONFLICT', 1)}")
        print("  " + ", ".join(f"{n} {x:.4g}" for n, x in v.items()))


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--passes", type=int)
    ap.add_argument("--seconds", type=float)
    ap.add_argument("--only")
    ap.add_argument("--trace")
    ap.add_argument("--counters")
    a = ap.parse_args()
    if a.counters:
        return counters(a.counters)
    from perf import operators as M
    M.own = True
    cases = [c for c in M.listed() if not a.only or c["name"] in a.only.split(",")]
    if a.trace:
        return trace(a.trace, [c["name"] for c in cases])
    if a.passes or a.seconds:
        return run(M, cases, a.passes, a.seconds)
    time_calls(M, cases)


if __name__ == "__main__":
    main()
