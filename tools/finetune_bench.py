#!/usr/bin/env python3
"""Device time of the fine-tuning objectives: calls of the package's public entry points, forward and backward, captured
into a HIP graph over three sets of inputs and replayed.

    python tools/finetune_bench.py [--only NAME,NAME] [--forms] [--replays 8]
    python tools/finetune_bench.py --trace CASE_kernel_trace.csv      # a rocprofv3 trace of one case: durations by launch

Cases are those of perf/operators.py; --forms: the forms that these leave out instead (forward only, wide float32 rows,
rows beyond the registers, an upstream gradient other than 1, strided logits, long masks).  Under rocprofv3 one case at a
time tells its kernels apart (tools/collect_profiles.sh finetune).
"""
import argparse
import collections
import csv
import math
import os
import re
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
import d3pm_amd  # noqa: E402
from perf import operators  # noqa: E402

DTYPES = operators.DTYPES


def replayed(calls, reps, replays):
    """us a call, the best of `replays` replays of a graph of `reps` calls."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for call in calls:
            call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(reps):
            calls[i % len(calls)]()
    best = float("inf")
    for _ in range(replays + 2):
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        graph.replay()
        e1.record()
        torch.cuda.synchronize()
        best = min(best, e0.elapsed_time(e1) * 1e3 / reps)
    return best


def report(name, us, nbytes):
    print(f"{name:72s} {us:9.1f} us  {nbytes / us / 1e3:6.0f} GB/s", flush=True)


def listed_case(case, replays):
    states = [operators.prepare(case, seed) for seed in range(3)]
    nbytes = operators.work(case)["bytes"]
    us = replayed([lambda s=s: operators.run(s) for s in states], 30 if nbytes < 5e8 else 6, replays)
    report(case["name"], us, nbytes)


def form(op, B, L, V, dtype, replays, kind="plain", grad=True, k=32, up=1.0, masked=False):
    size = torch.finfo(DTYPES[dtype]).bits // 8
    calls = []
    for seed in range(3):
        g = torch.Generator(device="cuda").manual_seed(seed)
        shape, cut = {"plain": ((B, L, V), lambda t: t), "shift": ((B, L + 1, V), lambda t: t[:, :-1]),
                      "padded": ((B, L, V + 1), lambda t: t[..., 1:]),
                      "apart": ((B, V, L), lambda t: t.transpose(1, 2))}[kind]
        z = cut(torch.empty(shape, dtype=DTYPES[dtype], device="cuda").normal_(generator=g))
        y = torch.randint(0, V, (B, L), generator=g, device="cuda")
        lp = torch.full((B, L), -math.log(V), device="cuda")
        idx = torch.randint(0, V, (B, L, k), generator=g, device="cuda")
        tl = torch.randn(B, L, k, generator=g, device="cuda")
        mask = torch.ones(B, L, dtype=torch.bool, device="cuda") if masked else None
        upstream = torch.full((B, L) if op == "logprobs" else (), up, device="cuda")

        def call(z=z, y=y, lp=lp, idx=idx, tl=tl, mask=mask, upstream=upstream):
            q = z.detach().requires_grad_(grad)
            if op == "logprobs":
                out = d3pm_amd.token_logprobs(q, y, mask=mask)
            elif op == "distill":
                out = d3pm_amd.TopKDistillLoss(temperature=2.0)(q, tl, idx, mask=mask)
            elif op == "preference":
                out = d3pm_amd.PreferenceLoss()(q, y, lp, mask=mask)
            else:
                out = d3pm_amd.PolicyLoss(kl_coeff=0.05)(q, y, lp, lp, lp, mask=mask)
            return torch.autograd.grad(out, q, upstream) if grad else out

        calls.append(call)
    nbytes = B * L * V * size * (2 if grad else 1)
    us = replayed(calls, 12 if nbytes < 5e8 else 6, replays)
    words = [f"{op} {B} x {L} x {V} {dtype}", kind if kind != "plain" else "", "" if grad else "forward only",
             f"k {k}" if op == "distill" else "", f"upstream {up}" if up != 1.0 else "", "masked" if masked else ""]
    report(" ".join(w for w in words if w), us, nbytes)
    torch.cuda.empty_cache()


def forms(replays):
    for dtype, L, V in (("f32", 263, 24), ("bf16", 263, 24), ("f32", 512, 32)):
        form("logprobs", 256, L, V, dtype, replays)
    for op in ("distill", "policy", "preference"):
        form(op, 256, 263, 24, "f32", replays, grad=False, k=8)
        form(op, 8, 1024, 131072, "bf16", replays, grad=False, k=64)
    for op in ("logprobs", "distill", "preference", "policy"):
        for V, dtype in ((32000, "f32"), (65528, "f32"), (128256, "f32"), (151936, "bf16"), (256000, "bf16")):
            form(op, 4, 1024, V, dtype, replays, k=64)
    for op in ("distill", "preference", "policy"):
        for up in (1.0, 0.5):
            form(op, 256, 263, 24, "f32", replays, k=8, up=up)
            form(op, 8, 1024, 65536, "bf16", replays, k=64, up=up)
    for op in ("logprobs", "distill", "preference", "policy"):
        for kind in ("plain", "shift", "padded", "apart"):
            form(op, 4, 1000, 32003, "bf16", replays, kind=kind)
    for N in (16384, 65536, 1 << 18, 1 << 21):
        for masked in (False, True):
            form("policy", 1, N, 24, "f32", replays, masked=masked)


def trace(path):
    """Durations of a trace's kernels.  A kernel that is launched twice to a call runs for the loss and again for the
    backward, where it finds an upstream gradient of 1 and returns: told apart by their order."""
    launches = collections.defaultdict(list)
    for r in sorted(csv.DictReader(open(path)), key=lambda r: int(r["Start_Timestamp"])):
        if "d3pm" in r["Kernel_Name"]:
            launches[r["Kernel_Name"]].append((int(r["End_Timestamp"]) - int(r["Start_Timestamp"])) / 1e3)
    calls = min(len(v) for v in launches.values())
    for name, us in launches.items():
        short = re.sub(r"^void |d3pm::|ft::|\(.*$", "", name)
        for part, what in ((us, ""),) if len(us) == calls else ((us[0::2], ""), (us[1::2], ", nothing to do")):
            print(f"  {short + what:60s} launches {len(part):4d}  average {sum(part) / len(part):8.2f}  minimum {min(part):8.2f}")


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--only", default="")
    ap.add_argument("--forms", action="store_true")
    ap.add_argument("--replays", type=int, default=8)
    ap.add_argument("--trace", default="")
    args = ap.parse_args()
    if args.trace:
        return trace(args.trace)
    operators.own = True
    if args.forms:
        return forms(args.replays)
    only = set(filter(None, args.only.split(",")))
    for case in operators.listed():
        if not only or case["name"] in only:
            listed_case(case, args.replays)
            torch.cuda.empty_cache()


if __name__ == "__main__":
    main()
