"""What the traces and counters of layer_ops_kernel_trace_pmc.txt were taken of: the cases of perf/operators.py and the further
ones below, CALLS times each over several sets of operands in turn (three, or with `cold` as many as exceed every cache):

    rocprofv3 --kernel-trace --stats --output-format csv -d OUT -o b -- python3 profiles/layer_ops_cases.py CALLS [cold]
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from perf import operators  # noqa: E402

operators.own = True
FURTHER = [operators._quantize("quantize-fp32-2048x4096", 2048, 4096, "fp32")]
FURTHER += [operators._matmul(f"matmul-{m}x{n}x{k}", m, n, k, "bf16", False)
            for m, n, k in ((16, 4096, 4096), (64, 4096, 4096), (128, 4096, 4096), (192, 4096, 4096), (384, 4096, 4096), (768, 4096, 4096),
                            (16, 4096, 4097), (64, 4096, 4097), (1024, 4096, 4097), (8192, 8192, 4097))]


def main():
    calls, cold = int(sys.argv[1]), "cold" in sys.argv[2:]
    for case in operators.listed() + FURTHER:
        sets = min(64, max(3, (1 << 30) // operators.work(case)["bytes"] + 1)) if cold else 3
        states = [operators.prepare(case, seed) for seed in range(sets)]
        torch.cuda.synchronize()
        for i in range(calls):
            operators.run(states[i % sets])
        torch.cuda.synchronize()
        print(case["name"], sets, flush=True)
        del states
        torch.cuda.empty_cache()


main()
