"""GPU times of the low-bit dense layers (gp_vae_amd/ops.py) without the host: calls captured into a graph and replayed.

  python3 tools/lowbit_times.py                        the cases of perf/operators.py: us a call, TB/s, TFLOP/s
  python3 tools/lowbit_times.py --only "vjp 1x"        those whose name contains this
  python3 tools/lowbit_times.py --only fwd:bf16:24:4096:32768   cases of their own, any number: op:dtype:M:K:N for fwd, vjp and grads,
                                                       op:dtype:rows:columns for store, quant_w4, load_w4, store_q8 and load_q8
  python3 tools/lowbit_times.py --sets 12              the calls go round 12 sets of operands (default 3): with few sets, operands up
                                                       to some 80 MB stay in the 256 MB last-level cache from one round to the next
  python3 tools/lowbit_times.py --eager                also the wall time of eager calls on the same operands
  python3 tools/lowbit_times.py --potential            one potential and gradient of VAEInference, weights="float" and "w4"
Under `rocprofv3 --kernel-trace --stats --output-format csv -- python3 tools/lowbit_times.py --only NAME` the launches' own times."""
import argparse
import importlib.util
import os
import sys
import time

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from gp_vae_amd import ops  # noqa: E402
from gp_vae_amd.inference import VAEInference  # noqa: E402


def warm(fn, seconds=0.15):
    """Load until the clock, which an idle chip lowers, is up again (tens of milliseconds)."""
    end = time.perf_counter() + seconds
    while time.perf_counter() < end:
        for _ in range(20):
            fn()
        torch.cuda.synchronize()


def graph_us(fn, calls, reps=7, replays=4):
    """Median time of one of `calls` calls fn(0), fn(1), ... of a replayed graph."""
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for i in range(calls):
            fn(i)
    warm(g.replay)
    a, b, t = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True), []
    for _ in range(reps):
        a.record()
        for _ in range(replays):
            g.replay()
        b.record()
        b.synchronize()
        t.append(a.elapsed_time(b) / replays / calls * 1e3)
    return sorted(t)[reps // 2]


def eager_us(fn, calls=300, reps=7):
    warm(lambda: fn(0))
    t = []
    for _ in range(reps):
        a = time.perf_counter()
        for i in range(calls):
            fn(i)
        torch.cuda.synchronize()
        t.append((time.perf_counter() - a) / calls * 1e6)
    return sorted(t)[reps // 2]


class Format:
    """One of the format's readers or writers as a case: prepare, run, work."""

    def prepare(self, c, seed):
        x = torch.randn(c["m"], c["k"], generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
        dt = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[c["dtype"]]
        return {"quant_w4": lambda: (ops.quant_w4, x.to(dt)), "store_q8": lambda: (ops.store_q8, x.to(dt)),
                "load_w4": lambda: (ops.load_w4, ops.quant_w4(x), dt), "load_q8": lambda: (ops.load_q8, ops.store_q8(x), dt)}[c["op"]]()

    def run(self, s):
        return s[0](*s[1:])

    def work(self, c):
        return {"bytes": c["m"] * c["k"] * ((4 if c["dtype"] == "f32" else 2) + (33 / 64 if "w4" in c["op"] else 65 / 64)), "flops": 0}


def cases(only):
    spec = importlib.util.spec_from_file_location("operator_cases", os.path.join(ROOT, "perf", "operators.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    mod.own = True
    for text in only or [""]:
        if ":" not in text:
            yield from ((mod, c) for c in mod.listed() if text in c["name"])
            continue
        op, dt, m, k, *n = text.split(":")
        c = dict(name=text, op=op, dtype=dt, m=int(m), k=int(k), relu=True)
        yield (Format(), c) if op.endswith(("w4", "q8")) else (mod, dict(c, n=int(n[0])) if n else c)


def potential():
    print("%-20s %8s %7s %10s %8s" % ("decoder z-h1-h0-n", "observed", "chains", "float us", "w4 us"))
    for z, h1, h0, n in ((30, 50, 50, 4096), (30, 256, 256, 4096), (30, 1024, 1024, 4096), (30, 1024, 1024, 32768)):
        gen = torch.Generator().manual_seed(0)
        mat = lambda a, b: (torch.randn(a, b, generator=gen) * a ** -0.5).numpy()
        vec = lambda a: (0.1 * torch.randn(a, generator=gen)).numpy()
        dec = [(mat(z, h1), vec(h1)), (), (mat(h1, h0), vec(h0)), (), (mat(h0, n), vec(n))]
        x = torch.arange(n).numpy() / n
        for n_obs in (10, 256):
            obs = list(range(0, n, n // n_obs))[:n_obs]
            for chains in (1, 16, 100):
                q, u = torch.randn(chains, z, generator=gen).cuda(), torch.full((chains,), -2.0).cuda()
                out = []
                for weights in ("float", "w4"):
                    inf = VAEInference(None, dec, z, 1, x, x, obs, {}, weights=weights)
                    out.append(eager_us(lambda i: inf.potential_and_grad(q, u), calls=40, reps=5))
                print("%-20s %8d %7d %10.1f %8.1f" % ("%d-%d-%d-%d" % (z, h1, h0, n), n_obs, chains, *out), flush=True)


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--only", nargs="*")
    ap.add_argument("--sets", type=int, default=3)
    ap.add_argument("--eager", action="store_true")
    ap.add_argument("--potential", action="store_true")
    a = ap.parse_args()
    if a.potential:
        return potential()
    for mod, c in cases(a.only):
        sets = [mod.prepare(c, s) for s in range(1, a.sets + 1)]
        fn = lambda i: mod.run(sets[i % a.sets])
        for i in range(a.sets):
            fn(i)
        t, w = graph_us(fn, max(12, a.sets)), mod.work(c)
        print("%-28s graph %9.2f us  %6.2f TB/s  %7.1f TFLOP/s%s" % (
            c["name"], t, w["bytes"] / t * 1e-6, w["flops"] / t * 1e-6,
            "  eager %9.2f us" % eager_us(fn) if a.eager else ""), flush=True)


if __name__ == "__main__":
    main()
