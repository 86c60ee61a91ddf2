"""Time and stored activations of a micro-step in each mode of ``activation_checkpoint``, and of scoring with 8-bit projections.

    python -m templar_b200.bench.activation_modes --model 1B --batch 8 --seq-len 2048                       (one GPU)

A micro-step is ``WindowEngine.micro_step``: forward, backward, gradients added into the engine's buffer.  Modes are timed in turn,
``--rounds`` times ``--iters`` steps each, by CUDA events behind three warm-up steps; the median round counts.  ``activations_gib`` is the
most that the device held above the state (weights, gradients, optimizer).  Scoring is a forward pass to logits of the batch and of one token,
in bf16 and by ``Int8Llama``, also in turn.  Inputs are larger than L2 at the default sizes.  One JSON line per case."""

from __future__ import annotations

import argparse
import json
import statistics

import torch

MODES = ("none", "int8", "selective", "full")


def _milliseconds(fn, iters: int, warmup: int = 3) -> float:
    for _ in range(warmup):
        fn()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    torch.cuda.synchronize()
    a.record()
    for _ in range(iters):
        fn()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) / iters


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--model", default="1B")
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--seq-len", type=int, default=2048)
    ap.add_argument("--iters", type=int, default=10)
    ap.add_argument("--rounds", type=int, default=3)
    a = ap.parse_args()

    from ..models.llama import PRESETS, build_model
    from ..models.llama_int8 import Int8Llama
    from ..parallel.window_engine import EngineConfig, WindowEngine

    dev = torch.device("cuda", 0)
    args = PRESETS[a.model]
    model = build_model(args, device=dev, seed=1)              # fp32 initial values, which the engine rounds to bf16
    eng = WindowEngine(model, EngineConfig(max_peers=1), device=dev)
    g = torch.Generator().manual_seed(5)
    tok = torch.randint(0, args.vocab_size, (a.batch, a.seq_len + 1), generator=g).to(dev)
    x, y = tok[:, :-1], tok[:, 1:]
    config = {"model": a.model, "batch": a.batch, "seq_len": a.seq_len, "data": "synthetic"}

    times, held, loss = {m: [] for m in MODES}, {}, {}
    for _ in range(a.rounds):
        for mode in MODES:
            model.activation_checkpointing, model.ac_option = mode, "op"
            loss[mode] = float(eng.micro_step(x, y, 1.0))
            torch.cuda.synchronize()
            torch.cuda.reset_peak_memory_stats()
            base = torch.cuda.memory_allocated()
            times[mode].append(_milliseconds(lambda: eng.micro_step(x, y, 1.0), a.iters))
            held[mode] = (torch.cuda.max_memory_allocated() - base) / 2 ** 30
    for mode in MODES:
        print(json.dumps({"case": "micro_step", "mode": mode, "ms": round(statistics.median(times[mode]), 2),
                          "activations_gib": round(held[mode], 2), "loss": round(loss[mode], 4), **config}), flush=True)

    model.activation_checkpointing = "none"
    q = Int8Llama(model)
    forms = (("bf16", model), ("int8", q))
    with torch.no_grad():
        want, got = model(x).float(), q(x).float()
        off = float((got - want).norm() / want.norm())
        del want, got
        for t in (x, x[:1, :1]):
            times = {n: [] for n, _ in forms}
            for _ in range(a.rounds):
                for n, f in forms:
                    times[n].append(_milliseconds(lambda: f(t), a.iters))
            for n, _ in forms:
                print(json.dumps({"case": "scoring", "form": n, "tokens": t.numel(), "ms": round(statistics.median(times[n]), 3),
                                  **({"logits_off": round(off, 4)} if n == "int8" else {}), **config}), flush=True)


if __name__ == "__main__":
    main()
