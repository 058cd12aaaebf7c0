#!/usr/bin/env python3
"""Times of the operators of svae_cf_amd.ops: each listed case of perf/operators.py through the kernels and in its plain form, in
turn, on three sets of inputs in rotation; linear_cross_entropy with its backward pass and its reduction alone; and any sizes of
linear_nll and linear_nll_grad.

    python tools/time_operators.py                                      # the cases, then linear_cross_entropy
    python tools/time_operators.py 64x1000000x256xbfloat16 ...          # rows x vocabulary x width x type: loss | loss and gradients
"""
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import perf.operators as cases
from svae_cf_amd import _lib, ops


def timed(calls, seconds=0.25):
    """us a call: the best of five runs of the calls in turn, each of about `seconds` / 5."""
    for f in calls:
        f()
    torch.cuda.synchronize()
    n, best = 1, float("inf")
    for k in range(6):
        at = time.perf_counter()
        for _ in range(n):
            for f in calls:
                f()
        torch.cuda.synchronize()
        took = (time.perf_counter() - at) / (n * len(calls))
        if k == 0:
            n = max(1, int(seconds / 5 / (took * len(calls))))
        else:
            best = min(best, took)
    return best * 1e6


def listed():
    for case in cases.listed():
        states = [cases.prepare(case, s) for s in (1, 2, 3)]
        us = {}
        for own in (True, False, True, False):
            cases.own = own
            us[own] = min(us.get(own, float("inf")), timed([lambda s=s: cases.run(s) for s in states]))
        print("%-24s plain %9.1f us   kernels %8.1f us" % (case["name"], us[False], us[True]), flush=True)
        del states
        torch.cuda.empty_cache()


def under_autograd():
    """A training step's loss as a user's program calls it, beside the gradients in one call; the reduction alone."""
    for rows, vocab, dim, dtype in ((21800, 20000, 200, torch.bfloat16), (8192, 131072, 1024, torch.bfloat16), (2049, 17770, 150, torch.float32), (16, 20000, 200, torch.bfloat16)):
        g = torch.Generator(device="cuda").manual_seed(1)
        h = torch.randn(rows, dim, generator=g, device="cuda").to(dtype).requires_grad_()
        w = (torch.randn(vocab, dim, generator=g, device="cuda") * 2 / dim ** 0.5).to(dtype).requires_grad_()
        t = torch.randint(-1, vocab, (rows,), generator=g, device="cuda")
        wt = torch.full((rows,), 1.0 / rows, device="cuda")

        def step():
            h.grad = w.grad = None
            ops.linear_cross_entropy(h, w, t).backward()

        a, b = timed([step]), timed([lambda: ops.linear_nll_grad(h.detach(), w.detach(), t, wt)])
        print("linear_cross_entropy + backward %d x %d x %d %s %9.1f us   linear_nll_grad %9.1f us" % (rows, vocab, dim, str(dtype)[6:], a, b), flush=True)
    for rows in (256, 21800, 131072, 1 << 20, 1 << 24):
        nll, t, out = torch.rand(rows, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.empty(2, device="cuda")
        st = torch.cuda.current_stream().cuda_stream
        us = timed([lambda: _lib.call("svae_xent_reduce", nll.data_ptr(), t.data_ptr(), 0, rows, 10, 1, out.data_ptr(), st)])
        print("svae_xent_reduce %d rows %.1f us" % (rows, us), flush=True)


def sizes(args):
    for arg in args:
        rows, vocab, dim, dtype = arg.split("x")
        case = dict(op="nll", rows=int(rows), vocab=int(vocab), dim=int(dim), dtype=dtype, bias=False, pad=0.0)
        cases.own, us = True, []
        for train in (False, True):
            states = [cases.prepare(dict(case, train=train), s) for s in (1, 2, 3)]
            us.append(timed([lambda s=s: cases.run(s) for s in states]))
            del states
        print("%-36s loss %9.1f us   loss and gradients %9.1f us" % (arg, us[0], us[1]), flush=True)


if __name__ == "__main__":
    print(torch.cuda.get_device_name(0), flush=True)
    if len(sys.argv) > 1:
        sizes(sys.argv[1:])
    else:
        listed()
        under_autograd()
