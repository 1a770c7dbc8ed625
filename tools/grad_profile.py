#!/usr/bin/env python3
"""Kernel times and HBM bytes of the gradient operators, from rocprofv3, into
profiles/grad_kernel_stats.csv and profiles/grad_pmc.txt.

  python3 tools/grad_profile.py passes N [NAME ...]   what is profiled: N passes of every case of
                                                      perf/operators.py (three sets of inputs in turn)
  bash tools/grad_profile.sh DIR                      the rocprofv3 runs, on a GPU
  python3 tools/grad_profile.py tables DIR            the tables, from what they left in DIR

The first half of a case's passes warms up and is left out of the tables.  Cases
follow each other with other kernels between them (their inputs are made), which is
how the tables tell them apart.
"""
import csv
import pathlib
import re
import statistics
import subprocess
import sys

ROOT = pathlib.Path(__file__).resolve().parents[1]
sys.path[:0] = [str(ROOT / "perf"), str(ROOT / "rdma-ring-collectives_amd")]


def passes(n, names):
    import operators
    import torch
    operators.own = True
    for case in operators.listed():
        if names and case["name"] not in names:
            continue
        states = [operators.prepare(case, seed) for seed in range(3)]
        torch.cuda.synchronize()
        for i in range(n):
            operators.run(states[i % 3])
        torch.cuda.synchronize()
        print("case", case["name"], flush=True)
        del states
        torch.cuda.empty_cache()


TYPE = {"DF16b": "bf16", "DF16_": "f16", "f": "f32", "d": "f64", "float": "f32", "double": "f64"}


def short(kernel):
    """k_grad_clip<bf16, f32, 0> from either spelling of a kernel's name."""
    m = re.search(r"(k_grad_\w+?)I((?:DF16b|DF16_|f|d|L[bi]\d+E)+)E", kernel) if kernel.startswith("_ZN") else None
    if m:
        parts = re.findall(r"DF16b|DF16_|L[bi]\d+E|f|d", m[2])
        return f"{m[1]}<{', '.join(TYPE.get(p) or p[2:-1] for p in parts)}>"
    m = re.search(r"(k_grad_\w+)(?:<([^>]*)>)?", kernel)
    if not m or not m[2]:
        return m[1] if m else kernel
    parts = [TYPE.get(p, {"true": "1", "false": "0"}.get(p, p)) for p in m[2].split(", ")]
    return f"{m[1]}<{', '.join(parts)}>"


def segments(path, order):
    """Rows of the gradient kernels, one list for each case."""
    rows, found, inside = sorted(csv.DictReader(open(path)), key=lambda r: int(r[order])), [], False
    for r in rows:
        mine = "k_grad" in r["Kernel_Name"]
        if mine and not inside:
            found.append([])
        if mine:
            found[-1].append(r)
        inside = mine
    return found


def by_place(rows, value):
    """[(kernel, work-items, values)] for each launch of a pass, over the second half of the passes."""
    names = [(short(r["Kernel_Name"]), r.get("Grid_Size_X") or r["Grid_Size"]) for r in rows]
    per = next(p for p in range(1, len(names) + 1) if len(names) % p == 0 and names == names[:p] * (len(names) // p))
    n = len(names) // per
    return [(*names[k], [value(r) for r in rows[k::per][n // 2:]]) for k in range(per)]


def algorithmic(case, kernel):
    """(bytes read, bytes written) that one launch cannot do without; None where a call is more than one launch."""
    import operators
    size = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}
    es, oes = size[case["dt"]], size[case.get("out_dt", case["dt"])]
    n = case["n"] if case["kind"].startswith("fold") else sum(m for _, m in operators._sizes(case)[0])
    if "sumsq" in kernel:
        return n * es, 0
    if "fold" in kernel:
        return n * es * case["nsrc"], n * oes
    if "clip" in kernel:
        return n * (oes if case["kind"] == "fold_clip" else es), n * oes
    return None


def tables(found):
    import operators
    cases = operators.listed()
    commit = subprocess.run(["git", "rev-parse", "--short", "HEAD"], cwd=ROOT, capture_output=True, text=True).stdout.strip()
    trace = segments(found / "kt_kernel_trace.csv", "Start_Timestamp")
    assert len(trace) == len(cases), (len(trace), len(cases))
    with open(ROOT / "profiles" / "grad_kernel_stats.csv", "w") as f:
        w = csv.writer(f)
        w.writerow([f"rocprofv3 --kernel-trace at {commit}: case", "kernel", "work-items", "launches", "median us", "min us"])
        for case, rows in zip(cases, trace):
            for kernel, grid, us in by_place(rows, lambda r: (int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3):
                w.writerow([case["name"], kernel, grid, len(us), f"{statistics.median(us):.2f}", f"{min(us):.2f}"])
    lines = [f"rocprofv3 --pmc at {commit}, FETCH_SIZE, WRITE_SIZE and the SQ counters in a run each, median per launch;"
             " FETCH_SIZE x 2 (gfx950 correction)"]
    fetch, write, sq = (segments(found / f"{name}_counter_collection.csv", "Dispatch_Id") for name in ("fetch", "write", "sq"))
    for k, case in enumerate(cases):
        read = by_place(fetch[k], lambda r: float(r["Counter_Value"]) * 2048)
        wrote = by_place(write[k], lambda r: float(r["Counter_Value"]) * 1024)
        one = {c: [r for r in sq[k] if r["Counter_Name"] == c] for c in ("SQ_ACTIVE_INST_VALU", "SQ_WAVE_CYCLES")}
        valu, cycles = (by_place(v, lambda r: float(r["Counter_Value"])) for v in one.values())
        for j, (kernel, _, got) in enumerate(read):
            line = "%-18s %-36s read %8.2f MB" % (case["name"], kernel, statistics.median(got) / 1e6)
            need = algorithmic(case, kernel)
            split = sum(short(r[0]) == kernel for r in read) > 1      # more tensors than a launch holds
            if need and not split:
                line += " of %8.2f" % (need[0] / 1e6)
            line += "  written %8.2f MB" % (statistics.median(wrote[j][2]) / 1e6)
            if need and not split and need[1]:
                line += " of %8.2f" % (need[1] / 1e6)
            busy = statistics.median(valu[j][2]) / max(statistics.median(cycles[j][2]), 1)
            lines.append(line + "  VALU %.3f of the wave cycles" % busy)
    (ROOT / "profiles" / "grad_pmc.txt").write_text("\n".join(lines) + "\n")
    print("\n".join(lines))


if __name__ == "__main__":
    if sys.argv[1:2] == ["passes"]:
        passes(int(sys.argv[2]), sys.argv[3:])
    elif sys.argv[1:2] == ["tables"] and len(sys.argv) == 3:
        tables(pathlib.Path(sys.argv[2]))
    else:
        sys.exit(__doc__)
