"""One operator case of perf/operators.py, passes of the framework's kernels: the program that tools/operators_profile.sh profiles.

usage: operators_pass.py CASE [PASSES]      CASE may also be R,V,d[,f32]: loss and gradients of that size, dw in bf16 or added in fp32"""
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [ROOT, os.path.join(ROOT, "perf")]

import operators  # noqa: E402
from pacednegatives_amd import kernels as K  # noqa: E402


def main(name, passes):
    operators.own = True
    if "," in name:
        R, V, d, *f32 = name.split(",")
        s = operators.prepare(dict(op="lm", rows=int(R), vocab=int(V), d=int(d), train=True, scale=1.0, ignored=0.0), 3)
        h, w = s["h"], s["w"]
        loss, lse, dh = torch.empty(h.shape[0], device="cuda"), torch.empty(h.shape[0], device="cuda"), torch.empty_like(h)
        dw = torch.zeros(w.shape, device="cuda") if f32 else torch.empty_like(w)

        def run():
            K.linear_ce_fwd(h, w, s["labels"], loss, lse)
            K.linear_ce_bwd(h, w, s["labels"], lse, s["weights"], dh, dw, loss=loss)
    else:
        s = operators.prepare(next(c for c in operators.listed() if c["name"] == name), 3)

        def run():
            operators.run(s)
    for _ in range(passes):
        run()
    torch.cuda.synchronize()
    print(name, passes, flush=True)


if __name__ == "__main__":
    main(sys.argv[1], int(sys.argv[2]) if len(sys.argv) > 2 else 30)
