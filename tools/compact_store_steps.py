#!/usr/bin/env python3
"""Train steps of the EP engine on fp32, bf16 and 4-bit tokens (and 4-bit tokens with a teacher), and what the 4 bits cost a probe.

    python3 tools/compact_store_steps.py            # us per step: device time by events, the host's own time beside it
    python3 tools/compact_store_steps.py --accuracy # held-out accuracy of probes trained on each form of the same synthetic tokens

Batches are read in place from a resident store through an index; LARS, 1000 classes, 64 listed teacher classes and their tail."""
import argparse
import os
import sys
import time
from argparse import Namespace

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from efficient_probing_amd import distill, engine_finetune, mx4, probe_heads, token_store as TS   # noqa: E402
from efficient_probing_amd.engine import ProbeHeadEngine                                          # noqa: E402
from efficient_probing_amd.util.lars import LARS                                                  # noqa: E402

DEV = torch.device("cuda:0")
SHAPES = [(1024, 256, 768, 8), (1024, 256, 768, 32), (512, 256, 1152, 16), (256, 196, 768, 12)]
FORMS = ("fp32", "bf16", "4-bit", "4-bit + teacher")


def head(D, C, Q):
    class Enc(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.head = torch.nn.Linear(D, C)

        def forward(self, x):
            return self.head(x)
    torch.manual_seed(0)
    m = Enc()
    probe_heads.build_probe_head(m, Namespace(cls_features="ep", ep_queries=Q, d_out=1, nb_classes=C))
    return m.to(DEV)


def steps(B, N, D, Q, C=1000, n=200):
    x = torch.randn(2 * B, N, D, device=DEV)
    labels = torch.randint(0, C, (2 * B,), device=DEV)
    values, index, tail = distill.teacher_topk(3 * torch.randn(2 * B, C, device=DEV), 64, 2.0)
    crit = distill.TopKDistillation(values, index, tail, temperature=2.0, alpha=0.5)
    out = []
    for form in FORMS:
        tokens = x if form == "fp32" else x.bfloat16() if form == "bf16" else mx4.quantize_tokens(x)
        kw = {"criterion": crit} if "teacher" in form else {}
        eng = ProbeHeadEngine(head(D, C, Q).head.train(), optimizer="lars", lr=0.1)
        batches = [torch.randperm(2 * B, device=DEV)[:B].to(torch.int32) for _ in range(4)]
        targets = [labels[b.long()] for b in batches]
        run = lambda k: eng.train_step(tokens, targets[k % 4], image_index=batches[k % 4], **kw)
        best = host = 1e9
        for rep in range(4):
            for k in range(20):
                run(k)
            torch.cuda.synchronize()
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            t0 = time.perf_counter()
            a.record()
            for k in range(n):
                run(k)
            b.record()
            t1 = time.perf_counter()
            torch.cuda.synchronize()
            best, host = min(best, a.elapsed_time(b) / n * 1e3), min(host, (t1 - t0) / n * 1e6)
        out.append((best, host))
        del tokens
    return out


def accuracy(n=16384, held=8192, N=64, D=384, Q=8, C=100, epochs=12, seed=0):
    """A tenth of the tokens carry their class among noise; channels of log-normal size, as encoder features have."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    size, means = torch.exp(0.7 * torch.randn(D, device=DEV, generator=g)), torch.randn(C, D, device=DEV, generator=g)
    labels = torch.randint(0, C, (n + held,), device=DEV, generator=g)
    x = torch.randn(n + held, N, D, device=DEV, generator=g)
    x += (torch.rand(n + held, N, 1, device=DEV, generator=g) < 0.1) * 0.55 * means[labels][:, None]
    x *= size
    out = []
    for form in FORMS[:3]:
        store = lambda lo, hi: TS.ResidentTokenStore.from_tensors(x[lo:hi] if form == "fp32" else x[lo:hi].bfloat16() if form == "bf16" else mx4.quantize_tokens(x[lo:hi]), labels[lo:hi])
        train, test, m = store(0, n), store(n, n + held), head(D, C, Q)
        opt = LARS(m.head.parameters(), lr=1.0, weight_decay=0.0)
        args = Namespace(lr=1.0, min_lr=0.0, warmup_epochs=1, epochs=epochs, accum_iter=1, amp="none")
        for e in range(epochs):
            engine_finetune.train_one_epoch(m, None, train.loader(256, epoch=e), opt, DEV, e, None, args=args)
        out.append(engine_finetune.evaluate(test.loader(512, shuffle=False, drop_last=False), m, DEV, precision="fp32")["acc1"])
    return out


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--accuracy", action="store_true")
    a = ap.parse_args()
    if a.accuracy:
        for seed in range(3):
            print(f"seed {seed}: " + ", ".join(f"{f} {v:.2f} %" for f, v in zip(FORMS, accuracy(seed=seed))), flush=True)
    else:
        for s in SHAPES:
            print("%d x %d x %d, %d queries: " % s + ";  ".join(f"{f} {d:.0f} (host {h:.0f})" for f, (d, h) in zip(FORMS, steps(*s))), flush=True)
