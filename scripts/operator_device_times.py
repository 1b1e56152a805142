#!/usr/bin/env python3
"""Device time of every listed case of perf/operators.py without the host: twenty passes captured into one graph, the
graph replayed.  Prints one JSON line.  scripts/operator_device_times.py > profiles/blocks_device_times.json"""
import json
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from perf import operators  # noqa: E402

PASSES, REPLAYS = 20, 15


def main():
    operators.own = True
    out = {"unit": f"us a pass, median (least, most) of {REPLAYS} replays of {PASSES} captured passes"}
    for case in operators.listed():
        state = operators.prepare(case, 1)
        operators.run(state)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = [operators.run(state) for _ in range(PASSES)]
        times = []
        for k in range(REPLAYS + 3):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            graph.replay()
            end.record()
            torch.cuda.synchronize()
            if k >= 3:
                times.append(start.elapsed_time(end) / PASSES * 1e3)
        times.sort()
        out[case["name"]] = [round(v, 2) for v in (times[REPLAYS // 2], times[0], times[-1])]
        del graph, kept, state
        torch.cuda.empty_cache()
    print(json.dumps(out))


if __name__ == "__main__":
    main()
