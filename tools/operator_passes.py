"""Kernel times of the operators at the cases listed in perf/operators.py, from a kernel trace.

    cd /tmp && rocprofv3 --kernel-trace --output-format csv -d /tmp/passes -o o -- python3 <repo>/tools/operator_passes.py run 12
    python3 <repo>/tools/operator_passes.py summary /tmp/passes
`run N` makes N passes of every listed case with one set of inputs; a cauchy_() kernel marks where a case's passes begin.  `summary`
prints median and minimum of each of this library's kernels, case by case, in launch order."""
import csv
import glob
import os
import statistics
import sys

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _module():
    import importlib.util

    sys.path.insert(0, REPO)
    spec = importlib.util.spec_from_file_location("operators", os.path.join(REPO, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def run(passes):
    import torch

    m = _module()
    m.own = True
    for case in m.listed():
        state = m.prepare(case, 1)
        m.run(state)  # workspaces
        torch.empty(7, device="cuda").cauchy_()
        for _ in range(passes):
            m.run(state)
        torch.cuda.synchronize()
        print(case["name"], flush=True)


def summary(folder):
    (path,) = glob.glob(os.path.join(folder, "**", "*kernel_trace.csv"), recursive=True)
    rows = sorted(csv.DictReader(open(path)), key=lambda r: int(r["Start_Timestamp"]))
    names, at, times, left = [c["name"] for c in _module().listed()], -1, [], False
    for r in rows:
        kernel = r["Kernel_Name"].split("(")[0].replace("void ", "")
        if "cauchy" in r["Kernel_Name"]:
            at, left = at + 1, False
            times.append({})
        elif at >= 0 and not left:
            if kernel.startswith("hv_"):
                times[at].setdefault(kernel, []).append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
            elif "normal" in r["Kernel_Name"] or "uniform" in r["Kernel_Name"]:
                left = True  # the next case's inputs
    for name, kernels in zip(names, times):
        for kernel, t in kernels.items():
            print(f"{name:26s} {kernel:46s} n={len(t):3d}  median {statistics.median(t):8.2f}  min {min(t):8.2f} us")


if __name__ == "__main__":
    run(int(sys.argv[2])) if sys.argv[1] == "run" else summary(sys.argv[2])
