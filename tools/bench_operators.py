"""Times the operators of perf/operators.py: python3 tools/bench_operators.py [--plain] [--more] [name ...]

``--more``: sizes besides the listed ones -- rows of few tokens, heads of few rows, a weight gradient for each tile of the kernel.  One line a case: microseconds a pass (passes queued one behind another), GB/s and TFLOP/s of the bytes and operations that a pass cannot do without.
Under ``rocprofv3 --kernel-trace --stats -- python3 tools/bench_operators.py`` the kernels' own times (profiles/operators_kernel_stats.csv)."""
import gc
import importlib.util
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)


def more(ops):
    rows = [ops._token_case(f"log_prob_{64 * 512}x{V}_{dt}{'_grad' if g else ''}", "log_prob", dt, 64, 512, V, 0, grad=g)
            for V in (18, 128, 512, 2048) for dt in ("bf16", "fp32") for g in (False, True)]
    heads = [ops._linear_case(f"linear_{N}x{D}x1_bf16", "bf16", N, D, 1, True) for N, D in ((1, 4096), (1, 65536), (64, 65536), (65536, 1024))]
    tiles = [ops._linear_case(f"linear_{N}x{D}x{O}_{dt}", dt, N, D, O, False)
             for dt, N, D, O in (("bf16", 2048, 3000, 3000), ("bf16", 4096, 2048, 500), ("bf16", 65536, 257, 13), ("fp16", 8192, 2048, 8192),
                                 ("fp32", 8192, 2048, 2048), ("fp32", 65536, 257, 13))]
    return rows + heads + tiles


def main():
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    ops.own = "--plain" not in sys.argv
    gc.disable()  # a full collection among the passes takes 100 ms
    names = [a for a in sys.argv[1:] if not a.startswith("--")]
    for case in more(ops) if "--more" in sys.argv else ops.listed():
        if names and case["name"] not in names:
            continue
        state = ops.prepare(case, 1)
        for _ in range(10):
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
