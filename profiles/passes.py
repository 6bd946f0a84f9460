"""Passes of timed cases for a profiler to look at: passes.py MODULE CASES COUNT.

MODULE: operators or more_operators (of perf/); CASES: names with commas, or all; from the repository's root, e.g.

    rocprofv3 --kernel-trace --stats -d out/ks -o run -f csv -- python3 profiles/passes.py more_operators all 10
"""
from __future__ import annotations

import importlib
import os
import sys


def main(module: str, names: str, count: str) -> None:
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    import torch
    m = importlib.import_module("perf." + module)
    m.own = True
    for case in m.listed():
        if names != "all" and case["name"] not in names.split(","):
            continue
        state = m.prepare(case, 1)
        for _ in range(int(count)):
            m.run(state)
        torch.cuda.synchronize()
        print(case["name"], flush=True)
        del state


if __name__ == "__main__":
    main(*sys.argv[1:])
