"""Times the operators of perf/operators.py: python3 tools/bench_operators.py [--plain] [name ...]

One line a case: microseconds a pass (passes queued one behind another), GB/s and TFLOP/s of the bytes and operations that a pass cannot do without.
Under ``rocprofv3 --kernel-trace --stats -- python3 tools/bench_operators.py`` the kernels' own times (profiles/operators_kernel_stats.csv)."""
import importlib.util
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


def main():
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    ops.own = "--plain" not in sys.argv
    names = [a for a in sys.argv[1:] if not a.startswith("--")]
    for case in ops.listed():
        if names and case["name"] not in names:
            continue
        state = ops.prepare(case, 1)
        for _ in range(3):
            ops.run(state)
        start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        n = 20
        start.record()
        for _ in range(n):
            ops.run(state)
        end.record()
        torch.cuda.synchronize()
        us, work = start.elapsed_time(end) / n * 1e3, ops.work(case)
        print("%-38s %10.1f us %8.0f GB/s %8.1f TFLOP/s" % (case["name"], us, work["bytes"] / us / 1e3, work["flops"] / us / 1e6), flush=True)
        del state


if __name__ == "__main__":
    main()
