"""The calls traced in profiles/mx_kernels__operator_cases.txt: the cases of perf/operators.py, and some sizes and forms beside them, REPS times each on
up to REPS sets of inputs and weights in turn (more than the last-level cache, where they are large). A cos kernel stands before and behind every case's calls.

  python3 perf/mx_calls.py REPS
"""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from perf import operators as op  # noqa: E402

op.own = True
CACHE = 600e6   # bytes that a case's rotating states hold together, at least


def extra():
    """(name, case, call of a state) of what is traced beside the listed cases."""
    fused, quant, w4 = op._ops()
    lin = lambda name, M, N, K, act: (name, op._case(name, "linear", M, K, n=N, act=act), op.run)

    def codes(s):
        if "pair" not in s:
            s["pair"] = quant.quant_fp8_e8m0(s["x"])
        return w4.linear_fp4(s["pair"], s["w"])
    return [("W4A8 16 rows 4608 x 5120 from codes", op._case("", "linear", 16, 5120, n=4608, act="fp8"), codes),
            lin("W4A8 97 rows 5120 x 8192", 97, 5120, 8192, "fp8"), lin("W4A4 512 rows 4608 x 5120", 512, 4608, 5120, "fp4"),
            lin("W4A8 512 rows 4608 x 5120", 512, 4608, 5120, "fp8"), lin("W4A8 8192 rows 8192 x 8192", 8192, 8192, 8192, "fp8"),
            ("norm 16384 x 5120 to FP4, with y", op._case("", "norm", 16384, 5120),
             lambda s: fused.add_rmsnorm_quant(s["x"], s["res"], s["g"], op.EPS, fmt="fp4", y=True)),
            ("quantise 32768 x 5120, codes only", op._case("", "quant", 32768, 5120), lambda s: quant.quant_fp4(s["x"]))]


def mark():
    torch.cuda.synchronize()
    torch.zeros(7, device="cuda").cos_()
    torch.cuda.synchronize()


def main(reps):
    for name, case, call in [(c["name"], c, op.run) for c in op.listed()] + extra():
        n = max(2, min(reps, int(CACHE / op.work(case)["bytes"]) + 1))
        states = [op.prepare(case, seed) for seed in range(n)]
        for s in states:
            call(s)
        mark()
        for i in range(reps):
            call(states[i % n])
        mark()
        print(name, flush=True)
        del states
    print("done", flush=True)


if __name__ == "__main__":
    main(int(sys.argv[1]))
