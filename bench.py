"""Benchmark of the denoiser self-attention path (Sage attention ms/call and TOPS at 16.8k / 47k
tokens, % of the int8 tensor peak, 1/2/4/8 GPUs).

One step = one h3s_attention call of the 47,232-token case (c3: 32 heads x 128, fp16 q/k/v as the strided parts of a
qkv buffer, fp16 out), with a fresh seeded input per denoiser block (50 blocks, each > L2). With N GPUs (torchrun), the
32 heads are split over the ranks (32/N heads each, no exchange: heads are independent), so the total work is fixed
(strong scaling). Also reported: c2 (16,848 tokens, Sage), c1 (2,159 tokens, fp16 SDPA), each leg's parity against
float64 on sampled rows, the neighbouring kernels, and for N > 1 the Ulysses variant c4 (token-sharded activations,
exchanged to head shards and back over peer memory, NCCL's all-to-all timed beside it) with its exposed exchange time.

--impl reference times the reference's attention restated on the CPU (oracle/, the reference itself cannot be built
here) on the host cores, rank 0 only, on a bounded sample of the same workload.
"""
from __future__ import annotations

import argparse
import json
import os
import statistics
import subprocess
import sys
import threading
import time

ROOT = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, ROOT)

METRIC = "Sage attn ms/call & TOPS at 16.8k/47k tokens, % int8 TC peak, 1/2/4/8 GPU"
UNIT = "TOPS"
DATA = ("synthetic: seeded N(0,1) q and v, k = N(0,1) + a per-channel N(0,4) offset, fresh per block "
        "(no dataset; stands in for the denoiser's activations)")


def ops_per_call(S: int, H: int, D: int = 128) -> float:
    """Algorithmic work of one attention call: Q.K^T and P.V, 2*S*S*D*H each."""
    return 4.0 * S * S * D * H


def measured_peaks() -> dict:
    p = os.path.join(ROOT, "MEASURED_PEAKS.json")
    if os.path.exists(p):
        with open(p) as f:
            d = json.load(f)
        return {"hbm_gbs": d["hbm_gbs"], "bf16_tflops": d["bf16_tflops"],
                "bf16_tflops_sustained": d.get("bf16_tflops_sustained", d["bf16_tflops"]), "source": "measured"}
    return {"hbm_gbs": 6650.0, "bf16_tflops": 1590.0, "bf16_tflops_sustained": 1400.0, "source": "fallback"}


class Clocks:
    """nvidia-smi samples of the SM clock and throttle reasons while the timed region runs."""

    FIELDS = ("clocks.sm,clocks.max.sm,clocks_event_reasons.hw_slowdown,clocks_event_reasons.hw_thermal_slowdown,"
              "clocks_event_reasons.sw_thermal_slowdown,clocks_event_reasons.sw_power_cap")

    def __init__(self, index: int):
        self.index = index
        self.rows: list[list[str]] = []
        self.proc = None
        self.thread = None

    def __enter__(self):
        try:
            self.proc = subprocess.Popen(["nvidia-smi", "-i", str(self.index), f"--query-gpu={self.FIELDS}",
                                          "--format=csv,noheader,nounits", "-lms", "100"], stdout=subprocess.PIPE,
                                         stderr=subprocess.DEVNULL, text=True)
            self.thread = threading.Thread(target=self._read, daemon=True)
            self.thread.start()
            time.sleep(0.3)
        except OSError:
            self.proc = None
        return self

    def _read(self):
        for line in self.proc.stdout:
            self.rows.append([x.strip() for x in line.split(",")])

    def __exit__(self, *exc):
        if self.proc:
            self.proc.terminate()
            try:
                self.proc.wait(timeout=5)
            except subprocess.TimeoutExpired:
                self.proc.kill()
            self.thread.join(timeout=2)

    def summary(self) -> dict:
        sm = [float(r[0]) for r in self.rows if len(r) >= 6 and r[0].replace(".", "").isdigit()]
        mx = [float(r[1]) for r in self.rows if len(r) >= 6 and r[1].replace(".", "").isdigit()]
        names = ["hw_slowdown", "hw_thermal_slowdown", "sw_thermal_slowdown", "sw_power_cap"]
        reasons = sorted({names[i] for r in self.rows if len(r) >= 6 for i in range(4) if r[2 + i].lower() == "active"})
        return {"sm_mhz": statistics.median(sm) if sm else None, "sm_max_mhz": max(mx) if mx else None,
                "reasons": reasons, "samples": len(sm)}


def bench_config(S: int, H: int, D: int, world: int, blocks: int) -> dict:
    """The workload both arms name (the same keys and values, so that the lines compare)."""
    return {"workload": (f"c3: {H} heads x {S:,} tokens x {D} per call" if (S, H) == (47232, 32) else
                         f"profiling case: {H} heads x {S:,} tokens x {D} per call") +
                        ", Sage path, fp16 q/k/v inside a qkv buffer (row stride 3*H*D), fp16 out; fresh blocks",
            "S": S, "H": H, "D": D, "blocks": blocks,
            "parallelism": f"heads/{world}" if world > 1 else "1 GPU",
            "l2": "inputs larger than L2 (1.16 GB per block), a different block every step"}


# ---------------------------------------------------------------------------------------------------------------------
# CPU side: the oracle (the reference's attention restated; oracle/sage_ref.cpp)
# ---------------------------------------------------------------------------------------------------------------------
class CpuSage:
    """The oracle's Sage path (oracle/sage_ref.cpp: the reference's attention restated) on this host's cores, on one
    seeded block of the workload: the whole pre-pass once (timed), then samples of query rows spread over heads and
    positions through the int8 attention. A call's time is the pre-pass plus the rows' time scaled by the exact work
    ratio (every row costs 4*S*D ops), so a sample gives the throughput of a whole call."""

    def __init__(self, S: int, H: int, D: int, seed: int = 1):
        import numpy as np

        sys.path.insert(0, os.path.join(ROOT, "oracle"))
        import oracle
        from sycl_minimax_h3_b200.workloads import bits, make_qkv

        oracle.build()
        self.o, self.np = oracle, np
        self.S, self.H, self.D = S, H, D
        host = bits(make_qkv(S, H, D, seed=seed))
        t0 = time.perf_counter()
        self.pre = oracle.sage_prepass(host, (host, H * D), (host, 2 * H * D), oracle.F16, S, H, D, 3 * H * D)
        self.t_pre = time.perf_counter() - t0
        self.rng = np.random.default_rng(seed)

    def sample(self, budget_s: float) -> dict:
        iq, ik, qs, ks, km, hv = self.pre
        S, H, D = self.S, self.H, self.D
        n, t_rows, done = max(8, self.o.threads()), 0.0, 0
        while True:
            rh = self.rng.integers(0, H, n)
            rs = self.rng.integers(0, S, n)
            t0 = time.perf_counter()
            self.o.sage_rows(iq, ik, hv, qs, ks, S, H, D, rh, rs)
            t_rows += time.perf_counter() - t0
            done += n
            if t_rows >= budget_s or done >= H * S:
                break
            n = min(H * S - done, max(n, int(n * (budget_s - t_rows) / max(t_rows, 1e-3))))
        t_call = self.t_pre + t_rows * (H * S) / done
        return {"value": ops_per_call(S, H, D) / t_call / 1e12, "unit": UNIT, "cores": self.o.threads(), "kind": "port",
                "sample": f"S={S}, H={H}: whole pre-pass ({self.t_pre:.2f} s) + {done} of {H * S} query rows "
                          f"({t_rows:.2f} s), scaled to a whole call = {t_call:.1f} s",
                "s_per_call": t_call, "measured": {"prepass_s": self.t_pre, "rows": done, "rows_s": t_rows,
                                                   "rows_total": H * S, "ops_per_row": 4.0 * S * D}}


def run_reference(args) -> None:
    rank = int(os.environ.get("RANK", "0"))
    if rank != 0:
        return
    S, H, D = 47232, 32, 128
    cpu = CpuSage(S, H, D, seed=100)
    per_step_budget = max(0.5, float(os.environ.get("H3_REF_TOTAL_S", "120")) / max(1, args.steps + args.warmup))
    per_step = []
    for i in range(args.warmup + args.steps):
        r = cpu.sample(per_step_budget)
        if i >= args.warmup:
            per_step.append(r)
    tops = statistics.median(r["value"] for r in per_step)
    world = int(os.environ.get("WORLD_SIZE", "1"))
    rows = sum(r["measured"]["rows"] for r in per_step)
    rows_s = sum(r["measured"]["rows_s"] for r in per_step)
    line = {
        "impl": "reference", "metric": METRIC, "value": tops, "unit": UNIT, "n_gpus": args.gpus, "steps": args.steps,
        "warmup": args.warmup, "ms_per_step": 1e3 * statistics.median(r["s_per_call"] for r in per_step),
        "higher_is_better": True, "scaling": "strong", "vs_baseline": None, "dtype": "int8+fp16", "data": DATA,
        "config": bench_config(S, H, D, world, min(50, args.warmup + args.steps)),
        "cpu_baseline": {k: per_step[-1][k] for k in ("value", "unit", "cores", "kind", "sample")},
        "e2e": {"value": tops, "unit": UNIT, "h2d_bytes_per_step": 0, "d2h_bytes_per_step": 0},
        # what was timed, so that the value can be recomputed from this line: per step, a sample of query rows of one
        # call (rows_s seconds for `rows` rows, each 4*S*D ops) plus the whole pre-pass once (prepass_s)
        "measured": {"prepass_s": cpu.t_pre, "rows_timed": rows, "rows_s": rows_s, "rows_per_call": H * S,
                     "ops_per_row": 4.0 * S * D, "steps_timed": len(per_step),
                     "call_s": cpu.t_pre + rows_s / rows * H * S,
                     "recompute": "value = 4*S^2*D*H / (prepass_s + rows_s / rows_timed * rows_per_call) / 1e12 (the "
                                  "median over steps differs from this pooled form by the steps' spread)"},
        "note": "the reference's own attention (SYCL + oneDNN + un-vendored ARK) cannot be built or run here; this is "
                "its algorithm restated in C++ (oracle/sage_ref.cpp; its pre-pass is bit-exact with the reference's "
                "own source) on the host cores, every step a sample of query rows of one 47,232-token call "
                "extrapolated by the exact per-row work; ms_per_step is that extrapolated call time, not wall time",
    }
    line["cpu_baseline"]["value"] = tops
    print(json.dumps(line), flush=True)


# ---------------------------------------------------------------------------------------------------------------------
# GPU side
# ---------------------------------------------------------------------------------------------------------------------
def main() -> None:
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--warmup", type=int, default=5)
    ap.add_argument("--impl", default="ours", choices=["ours", "reference"])
    ap.add_argument("--no-cpu", action="store_true", help="skip the CPU baseline leg")
    ap.add_argument("--quick", action="store_true", help="main workload only (no c1/c2/c4 side numbers)")
    ap.add_argument("--S", type=int, default=47232, help="tokens of the main workload (profiling runs use a smaller case)")
    ap.add_argument("--H", type=int, default=32, help="heads of the main workload")
    ap.add_argument("--only", choices=["c1", "c2", "rms_rope", "rope_prepass", "causal", "int8_linear", "vae"],
                    help="run one side leg alone and print its numbers (for profiling that kernel); no bench line")
    args = ap.parse_args()
    if args.impl == "reference":
        run_reference(args)
        return

    import torch
    import torch.distributed as dist

    from sycl_minimax_h3_b200 import native, ops
    from sycl_minimax_h3_b200.workloads import make_qkv

    world = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    local = int(os.environ.get("LOCAL_RANK", "0"))
    torch.cuda.set_device(local)
    dev = torch.device("cuda", local)
    if world > 1:
        import datetime

        dist.init_process_group("nccl", timeout=datetime.timedelta(seconds=300), device_id=dev)

    def barrier():
        if world > 1:
            dist.barrier()

    def max_over_ranks(x: float) -> float:
        if world == 1:
            return x
        t = torch.tensor([x], device=dev, dtype=torch.float64)
        dist.all_reduce(t, op=dist.ReduceOp.MAX)
        return float(t.item())

    peaks = measured_peaks()
    D = 128
    S, H = args.S, args.H
    if H % world:
        raise SystemExit(f"{H} heads do not split over {world} GPUs")
    h = H // world
    if args.only:
        if args.only == "causal":
            res = causal_leg(dev, max_over_ranks, barrier)
        elif args.only == "int8_linear":
            res = int8_linear_leg(dev, S, peaks, max_over_ranks, barrier)
        elif args.only == "vae":
            res = vae_leg(dev, max_over_ranks, barrier)
        elif args.only in ("rms_rope", "rope_prepass"):
            g = torch.Generator(device=dev)
            g.manual_seed(1000)
            qkv = torch.randn(S, 3 * h * D, generator=g, device=dev, dtype=torch.float16)
            leg = rms_rope_leg if args.only == "rms_rope" else rope_prepass_leg
            res = leg(dev, qkv, S, h, D, peaks, max_over_ranks, barrier)
        else:
            res = side_leg(args.only, dev, h, H, D, max_over_ranks, barrier)
        if rank == 0:
            print(json.dumps({"only": args.only, **res}), flush=True)
        if world > 1:
            dist.barrier()
            dist.destroy_process_group()
        return
    nblocks = 50
    stream = torch.cuda.current_stream()
    ctx = ops.context(dev)

    # ---- inputs: a fresh seeded qkv per denoiser block, this rank's heads ----
    pool = []
    for b in range(min(nblocks, args.warmup + args.steps)):
        g = torch.Generator(device=dev)
        g.manual_seed(1000 + b)
        qkv = torch.randn(S, 3 * H * D, generator=g, device=dev, dtype=torch.float16)
        off = torch.randn(H * D, generator=g, device=dev, dtype=torch.float32) * 2.0
        qkv[:, H * D:2 * H * D] += off.to(torch.float16)
        pool.append(qkv.view(S, 3, H, D)[:, :, rank * h:(rank + 1) * h, :].reshape(S, 3 * h * D).contiguous())
        del qkv
    out = torch.empty(S, h * D, dtype=torch.float16, device=dev)
    torch.cuda.synchronize()

    def call(qkv):
        q, k, v = ops.Rows.qkv(qkv, h, D)
        ops.attention(q, k, v, out)

    # ---- timed region: K calls, one per block ----
    for i in range(args.warmup):
        call(pool[i % len(pool)])
    ctx.wait()
    barrier()
    torch.cuda.synchronize()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    with Clocks(local) as clk:
        e0.record(stream)
        for i in range(args.steps):
            call(pool[(args.warmup + i) % len(pool)])
        e1.record(stream)
        torch.cuda.synchronize()
    ctx.wait()
    if not bool(torch.isfinite(out).all()):
        raise SystemExit("bench: the timed attention produced non-finite values; no number is reported")
    parity = parity_rows(pool[(args.warmup + args.steps - 1) % len(pool)], out, S, h, D, seed=rank)
    barrier()
    ms_total = max_over_ranks(e0.elapsed_time(e1))
    ms_call = ms_total / args.steps
    value = ops_per_call(S, H, D) * args.steps / (ms_total / 1e3) / 1e12
    launches_per_call = 4  # K mean, Q quantiser, K quantiser, attention

    # ---- the dominant kernel alone: attention on quantised inputs, through the plugin's C ABI ----
    nb = (S + 63) // 64
    iq = torch.empty(h, S, D, dtype=torch.int8, device=dev)
    ik = torch.empty_like(iq)
    sc = torch.empty(2 * h * nb + h * D, dtype=torch.float32, device=dev)
    ctx.sage_prepass(pool[0].data_ptr(), pool[0].data_ptr() + h * D * 2, native.F16, S, h, D, 3 * h * D, iq.data_ptr(),
                     ik.data_ptr(), sc.data_ptr())
    ctx.wait()
    sage = native.sage_lib()
    import ctypes

    raw = ctypes.c_void_p(stream.cuda_stream)
    vptr = pool[0].data_ptr() + 2 * h * D * 2

    def kernel_only():
        rc = sage.h3sage_attention_strided(ctypes.byref(raw), iq.data_ptr(), ik.data_ptr(), vptr, 3 * h * D, D,
                                           out.data_ptr(), native.F16, h * D, D, sc.data_ptr(),
                                           sc.data_ptr() + h * nb * 4, 64, S, h, D, 1.0 / D ** 0.5, None, 0)
        if rc != 0:
            raise native.H3Error(sage.h3sage_error().decode())

    for _ in range(3):
        kernel_only()
    torch.cuda.synchronize()
    nk = max(5, min(20, args.steps))
    k0, k1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    k0.record(stream)
    for _ in range(nk):
        kernel_only()
    k1.record(stream)
    torch.cuda.synchronize()
    if sage.h3sage_check(ctypes.byref(raw)) != 0:
        raise native.H3Error(sage.h3sage_error().decode())
    ms_kernel = k0.elapsed_time(k1) / nk
    mixed_peak = 4.0 / 3.0 * peaks["bf16_tflops"]          # half the ops int8 at 2x the bf16 rate, half fp16
    achieved = ops_per_call(S, h, D) / (ms_kernel / 1e3) / 1e12
    # DRAM bytes per launch (dram__bytes_read.sum + dram__bytes_write.sum) of one ncu capture of this kernel at
    # S = 16,384, H = 32: 377.26 MB (268.81 read + 108.45 written); q, k, v and out all scale with S*H, so a launch of
    # this workload moves that times S*H / (16,384 * 32).
    traffic = 377.26e6 * (S * h) / (16384 * 32)
    roofline = {"bound": "tensor", "achieved": achieved, "peak": mixed_peak, "unit": "TFLOP/s",
                "frac": achieved / mixed_peak, "traffic": traffic,
                "traffic_basis": "ncu DRAM bytes of one launch at S=16384, H=32, scaled by S*H",
                "kernel": "attn_sage3 (Sage int8 QK^T + fp16 PV, tcgen05, 2 query tiles per CTA)",
                "peak_basis": f"4/3 x {peaks['source']} bf16 {peaks['bf16_tflops']} TFLOP/s: int8 QK^T at 2x, fp16 PV at 1x",
                "ms_per_launch": ms_kernel,
                "pct_int8_peak_measured_x2": achieved / (2 * peaks["bf16_tflops"]),
                "pct_int8_peak_nominal_4500": achieved / 4500.0,
                # the kernel-only loop runs right after the timed region, with the card at its power cap: the same
                # fraction against the sustained (seconds-long, power-capped) measurement of the bf16 peak
                "peak_sustained": 4.0 / 3.0 * peaks["bf16_tflops_sustained"],
                "frac_vs_sustained": achieved / (4.0 / 3.0 * peaks["bf16_tflops_sustained"])}

    # ---- pre-pass alone: HBM-bound ----
    for _ in range(2):
        ctx.sage_prepass(pool[1 % len(pool)].data_ptr(), pool[1 % len(pool)].data_ptr() + h * D * 2, native.F16, S, h, D,
                         3 * h * D, iq.data_ptr(), ik.data_ptr(), sc.data_ptr())
    torch.cuda.synchronize()
    p0, p1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    p0.record(stream)
    npre = 5
    for i in range(npre):
        blk = pool[(2 + i) % len(pool)]
        ctx.sage_prepass(blk.data_ptr(), blk.data_ptr() + h * D * 2, native.F16, S, h, D, 3 * h * D, iq.data_ptr(),
                         ik.data_ptr(), sc.data_ptr())
    p1.record(stream)
    torch.cuda.synchronize()
    ctx.wait()
    ms_pre = p0.elapsed_time(p1) / npre
    pre_bytes = 6.0 * S * h * D + 4 * h * D + 8 * h * nb     # read q, k (fp16), write int8 q, k, scales and means
    prepass = {"ms": ms_pre, "algorithmic_GBs": pre_bytes / (ms_pre / 1e3) / 1e9,
               "with_mean_reread_GBs": (pre_bytes + 2.0 * S * h * D) / (ms_pre / 1e3) / 1e9,
               "peak_hbm_GBs": peaks["hbm_gbs"]}

    # ---- end to end: host buffers through the public call. Every step uploads its inputs from pinned host memory and
    # reads its output back, as a serving loop would run it: step i+1's upload (one copy stream) and step i-1's
    # read-back (another) overlap step i's attention, with double-buffered device inputs and outputs. The timed region
    # runs from before the first upload to after the last read-back. The same loop without overlap (one stream) is
    # reported beside it.
    ne = min(max(args.steps, 10), 50)   # the pipeline's fill (first upload) and drain (last read-back) over ne steps
    host_in = [pool[i % len(pool)].cpu().pin_memory() for i in range(2)]
    host_out = [torch.empty(S, h * D, dtype=torch.float16).pin_memory() for _ in range(2)]
    dev_in = [torch.empty_like(pool[0]) for _ in range(2)]
    dev_out = [torch.empty(S, h * D, dtype=torch.float16, device=dev) for _ in range(2)]
    s_in, s_out = torch.cuda.Stream(dev), torch.cuda.Stream(dev)

    def attend(qkv, o):
        q, k, v = ops.Rows.qkv(qkv, h, D)
        ops.attention(q, k, v, o)

    def e2e_loop(n, pipelined):
        t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        ev_in = [torch.cuda.Event() for _ in range(2)]
        ev_done = [torch.cuda.Event() for _ in range(2)]
        ev_read = [torch.cuda.Event() for _ in range(2)]
        t0.record(stream)
        s_in.wait_stream(stream)
        s_out.wait_stream(stream)
        for i in range(n):
            b = i % 2 if pipelined else 0
            if pipelined:
                with torch.cuda.stream(s_in):
                    if i >= 2:
                        s_in.wait_event(ev_done[b])          # step i-2's attention has read dev_in[b]
                    dev_in[b].copy_(host_in[i % 2], non_blocking=True)
                    ev_in[b].record(s_in)
                stream.wait_event(ev_in[b])
                if i >= 2:
                    stream.wait_event(ev_read[b])            # step i-2's output has been read back
            else:
                dev_in[b].copy_(host_in[i % 2], non_blocking=True)
            attend(dev_in[b], dev_out[b])
            if pipelined:
                ev_done[b].record(stream)
                with torch.cuda.stream(s_out):
                    s_out.wait_event(ev_done[b])
                    host_out[b].copy_(dev_out[b], non_blocking=True)
                    ev_read[b].record(s_out)
            else:
                host_out[b].copy_(dev_out[b], non_blocking=True)
        stream.wait_stream(s_out)
        t1.record(stream)
        torch.cuda.synchronize()
        ctx.wait()
        return t0.elapsed_time(t1) / n

    e2e_loop(2, True)
    e2e_loop(1, False)
    barrier()
    ms_e2e = max_over_ranks(e2e_loop(ne, True))
    barrier()
    ms_seq = max_over_ranks(e2e_loop(ne, False))
    barrier()
    e2e = {"value": ops_per_call(S, H, D) / (ms_e2e / 1e3) / 1e12, "unit": UNIT,
           "h2d_bytes_per_step": int(dev_in[0].numel() * 2) * world, "d2h_bytes_per_step": int(dev_out[0].numel() * 2) * world,
           "ms_per_step": ms_e2e,
           "pipelined": f"upload of step i+1 and read-back of step i-1 overlap step i; {ne} steps, the first upload "
                        "and the last read-back included",
           "ms_per_step_unpipelined": ms_seq}
    del host_in, host_out, dev_in, dev_out

    extra = {}
    if not args.quick:
        # c2: 16,848 tokens, Sage; c1: 2,159 tokens, fp16 SDPA (heads split the same way)
        for name in ("c2", "c1"):
            extra[name] = side_leg(name, dev, h, H, D, max_over_ranks, barrier)
        extra["rms_rope"] = rms_rope_leg(dev, pool[0], S, h, D, peaks, max_over_ranks, barrier)
        extra["rope_prepass"] = rope_prepass_leg(dev, pool[0], S, h, D, peaks, max_over_ranks, barrier)
        extra["causal"] = causal_leg(dev, max_over_ranks, barrier)
        extra["int8_linear"] = int8_linear_leg(dev, S, peaks, max_over_ranks, barrier)
        extra["vae"] = vae_leg(dev, max_over_ranks, barrier)
        if world > 1:
            extra["c4_ulysses"] = ulysses_leg(dev, world, rank, S, H, D, max_over_ranks, barrier)

    cpu = None
    if rank == 0 and world == 1 and not args.no_cpu:
        cpu = CpuSage(S, H, D, seed=1).sample(float(os.environ.get("H3_CPU_BUDGET_S", "15")))
        cpu.pop("s_per_call", None)

    if rank == 0:
        line = {
            "metric": METRIC, "value": value, "unit": UNIT, "n_gpus": world, "steps": args.steps, "warmup": args.warmup,
            "ms_per_step": ms_call, "higher_is_better": True, "scaling": "strong", "vs_baseline": None,
            "dtype": "int8+fp16", "data": DATA,
            "config": bench_config(S, H, D, world, min(nblocks, args.warmup + args.steps)),
            "ms_per_call": ms_call, "pct_int8_peak_measured_x2": value / world / (2 * peaks["bf16_tflops"]),
            "roofline": roofline, "prepass": prepass, "e2e": e2e, "gpu_launches": launches_per_call * args.steps,
            "parity": parity,
            "clocks": clk.summary(), "extra": extra,
        }
        if cpu is not None:
            line["cpu_baseline"] = cpu
        print(json.dumps(line), flush=True)
    if world > 1:
        dist.barrier()
        dist.destroy_process_group()


SIDE = {"c2": (16848, True), "c1": (2159, False)}     # tokens, Sage path (else the fp16 SDPA)


def parity_rows(qkv, out, S: int, H: int, D: int, n: int = 512, seed: int = 0) -> dict:
    """The output's error on n sampled (head, token) rows, every head covered, against float64 softmax attention of the
    same fp16 inputs computed with torch on the GPU: min per-row cosine and max-abs error (the tolerance the north star
    states: cosine >= 0.999, max-abs stated). Not timed."""
    import torch

    g = torch.Generator().manual_seed(seed)
    rh = torch.arange(n) % H
    rs = torch.randint(0, S, (n,), generator=g)
    rs[0], rs[-1] = 0, S - 1
    x = qkv.view(S, 3, H, D)
    cos_min, abs_max = 1.0, 0.0
    for h in range(H):
        sel = rs[rh == h].to(qkv.device)
        if sel.numel() == 0:
            continue
        q = x[sel, 0, h].double()
        k = x[:, 1, h].double()
        v = x[:, 2, h].double()
        p = torch.softmax((q @ k.T) / D ** 0.5, dim=-1)
        want = p @ v
        got = out.view(S, H, D)[sel, h].double()
        cos = torch.nn.functional.cosine_similarity(got, want, dim=-1)
        cos_min = min(cos_min, float(cos.min()))
        abs_max = max(abs_max, float((got - want).abs().max()))
    return {"rows": n, "min_cos_vs_float64": cos_min, "max_abs_vs_float64": abs_max,
            "reference": "float64 softmax attention of the same inputs (torch, on the GPU), sampled rows of every head"}


def side_leg(name, dev, h, H, D, max_over_ranks, barrier) -> dict:
    """c2 (16,848 tokens, Sage) or c1 (2,159 tokens, fp16 SDPA) on this rank's heads: 20 timed calls."""
    import torch

    from sycl_minimax_h3_b200 import ops
    from sycl_minimax_h3_b200.workloads import make_qkv

    S2, sage_path = SIDE[name]
    qkv2 = make_qkv(S2, h, D, seed=77, device=dev)
    out2 = torch.empty(S2, h * D, dtype=torch.float16, device=dev)
    if not sage_path:
        os.environ["H3S_SAGE_MIN_S"] = str(1 << 30)
        ops._ctx.clear()
    try:
        q2, k2, v2 = ops.Rows.qkv(qkv2, h, D)
        for _ in range(3):
            ops.attention(q2, k2, v2, out2)
        torch.cuda.synchronize()
        barrier()
        a0, a1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        nrep = 20
        a0.record(torch.cuda.current_stream())
        for _ in range(nrep):
            ops.attention(q2, k2, v2, out2)
        a1.record(torch.cuda.current_stream())
        torch.cuda.synchronize()
        ops.context(dev).wait()
        barrier()
        ms2 = max_over_ranks(a0.elapsed_time(a1)) / nrep
    finally:
        if not sage_path:
            os.environ.pop("H3S_SAGE_MIN_S", None)
            ops._ctx.clear()
    parity = parity_rows(qkv2, out2, S2, h, D, seed=S2)
    return {"S": S2, "H": H, "ms_per_call": ms2, "tops": ops_per_call(S2, H, D) / (ms2 / 1e3) / 1e12,
            "path": "sage" if sage_path else "fp16 sdpa", "parity": parity}


def rms_rope_leg(dev, qkv, S, h, D, peaks, max_over_ranks, barrier, rot=96) -> dict:
    """The step before the attention: h3s_rms_rope on q and on k of one c3 block, in place (dit.rs:347-348). HBM-bound:
    each call reads and writes its S x h x D values once and reads the token's rotation table. The model's rot_dim is
    6 x its checkpoint's inverse frequencies (dit.rs:71), which the synthetic setup does not have; 96 stands in."""
    import torch

    from sycl_minimax_h3_b200 import ops

    g = torch.Generator(device=dev)
    g.manual_seed(4242)
    w = (1 + 0.1 * torch.randn(D, generator=g, device=dev)).float()
    ang = torch.rand(S, rot // 2, generator=g, device=dev) * 6.28
    cs = torch.stack([torch.cos(ang), torch.sin(ang)], -1).float().contiguous()
    q, k, _ = ops.Rows.qkv(qkv, h, D)

    def both():
        ops.rms_rope(q, w, 1e-5, cs, rot)
        ops.rms_rope(k, w, 1e-5, cs, rot)

    for _ in range(3):
        both()
    torch.cuda.synchronize()
    barrier()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    n = 20
    e0.record(torch.cuda.current_stream())
    for _ in range(n):
        both()
    e1.record(torch.cuda.current_stream())
    torch.cuda.synchronize()
    ops.context(dev).wait()
    barrier()
    ms = max_over_ranks(e0.elapsed_time(e1)) / n
    nbytes = 2 * (2 * S * h * D * qkv.element_size() + S * rot * 4)      # q and k: read + write, and the table
    return {"kernel": "rms_rope_staged<f16> (q and k, two launches)", "S": S, "heads": h, "rot_dim": rot,
            "ms_q_and_k": ms, "algorithmic_GBs": nbytes / (ms / 1e3) / 1e9, "peak_hbm_GBs": peaks["hbm_gbs"],
            "frac": nbytes / (ms / 1e3) / 1e9 / peaks["hbm_gbs"]}


def rope_prepass_leg(dev, qkv, S, h, D, peaks, max_over_ranks, barrier, rot=96) -> dict:
    """The block's step before the attention and the Sage pre-pass (dit.rs:347-350): h3s_rms_rope on q and on k then
    h3s_sage_prepass, against the fused h3s_sage_prepass_rope (q normalised inside its quantiser's pass). The rows are
    rotated again on every call (values stay finite: the RMS norm rescales them), the same work each time."""
    import torch

    from sycl_minimax_h3_b200 import native, ops

    g = torch.Generator(device=dev)
    g.manual_seed(4243)
    wq = (1 + 0.1 * torch.randn(D, generator=g, device=dev)).float()
    wk = (1 + 0.1 * torch.randn(D, generator=g, device=dev)).float()
    ang = torch.rand(S, rot // 2, generator=g, device=dev) * 6.28
    cs = torch.stack([torch.cos(ang), torch.sin(ang)], -1).float().contiguous()
    nb = (S + 63) // 64
    iq = torch.empty(h, S, D, dtype=torch.int8, device=dev)
    ik = torch.empty_like(iq)
    sc = torch.empty(2 * h * nb + h * D, dtype=torch.float32, device=dev)
    ctx = ops.context(dev)
    st, qp, kp = 3 * h * D, qkv.data_ptr(), qkv.data_ptr() + h * D * 2

    def separate():
        ctx.rms_rope(qp, native.F16, S, h, D, st, wq.data_ptr(), 1e-5, cs.data_ptr(), rot)
        ctx.rms_rope(kp, native.F16, S, h, D, st, wk.data_ptr(), 1e-5, cs.data_ptr(), rot)
        ctx.sage_prepass(qp, kp, native.F16, S, h, D, st, iq.data_ptr(), ik.data_ptr(), sc.data_ptr())

    def fused():
        ctx.sage_prepass_rope(qp, kp, native.F16, S, h, D, st, wq.data_ptr(), wk.data_ptr(), 1e-5, cs.data_ptr(), rot,
                              iq.data_ptr(), ik.data_ptr(), sc.data_ptr())

    def timed(fn):
        for _ in range(3):
            fn()
        torch.cuda.synchronize()
        barrier()
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        n = 10
        e0.record(torch.cuda.current_stream())
        for _ in range(n):
            fn()
        e1.record(torch.cuda.current_stream())
        torch.cuda.synchronize()
        ctx.wait()
        barrier()
        return max_over_ranks(e0.elapsed_time(e1)) / n

    ms_sep, ms_fused = timed(separate), timed(fused)
    return {"kernels": "fused: rms_rope_staged (k), then kmean_tma (priority stream) || rms_rope_staged (q) + quant_rows (q), then quant_rows (k)", "S": S, "heads": h,
            "rot_dim": rot, "ms_rms_rope_then_prepass": ms_sep, "ms_fused": ms_fused}


def causal_leg(dev, max_over_ranks, barrier, L=512, Hq=32, Hkv=8, D=128) -> dict:
    """The text encoder's causal attention with grouped heads (h3s_attention_causal, te.rs:340-346) on one prompt: fp16,
    q [L, Hq*D], k and v [L, Hkv*D], seeded normal values. The encoder's head counts come from its checkpoint, which
    the synthetic setup does not have; 32 query over 8 key/value heads of 128 stand in. Work: 4*D*Hq*L*(L+1)/2 flops."""
    import torch

    from sycl_minimax_h3_b200 import ops

    g = torch.Generator(device=dev)
    g.manual_seed(77)
    q = torch.randn(L, Hq * D, generator=g, device=dev, dtype=torch.float16)
    k = torch.randn(L, Hkv * D, generator=g, device=dev, dtype=torch.float16)
    v = torch.randn(L, Hkv * D, generator=g, device=dev, dtype=torch.float16)
    out = torch.empty(L, Hq * D, device=dev, dtype=torch.float16)
    rq, rk, rv = ops.Rows.packed(q, Hq, D), ops.Rows.packed(k, Hkv, D), ops.Rows.packed(v, Hkv, D)
    for _ in range(3):
        ops.attention_causal(rq, rk, rv, out)
    torch.cuda.synchronize()
    barrier()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    n = 20
    e0.record(torch.cuda.current_stream())
    for _ in range(n):
        ops.attention_causal(rq, rk, rv, out)
    e1.record(torch.cuda.current_stream())
    torch.cuda.synchronize()
    ops.context(dev).wait()
    barrier()
    ms = max_over_ranks(e0.elapsed_time(e1)) / n
    flops = 4.0 * D * Hq * L * (L + 1) / 2
    return {"kernel": "attn_causal<f16> (CUDA cores, fp32 weights)", "L": L, "Hq": Hq, "Hkv": Hkv, "D": D, "ms": ms,
            "tflops": flops / (ms / 1e3) / 1e12}


def int8_linear_leg(dev, M, peaks, max_over_ranks, barrier, K=4096, N=12288, group=256) -> dict:
    """The qkv projection of one denoiser block (h3s_int8_linear, ops.rs:25-80): M tokens x hidden 4096 -> 3 x 4096,
    int8 weights stored rotated in groups of 256 with one scale per output, no bias, bf16 in and out (dit.rs:130-140).
    Seeded normal activations and random int8 weights stand in for a checkpoint's. Each call runs rotq_rows (HBM-bound:
    reads x, writes its int8 copy) and i8gemm (tensor-bound: 2*M*N*K int8 operations); inputs larger than L2."""
    import torch

    from sycl_minimax_h3_b200 import ops

    g = torch.Generator(device=dev)
    g.manual_seed(31)
    x = torch.randn(M, K, generator=g, device=dev).to(torch.bfloat16)
    w = torch.randint(-127, 128, (N, K), generator=g, device=dev, dtype=torch.int8)
    ws = (torch.rand(N, generator=g, device=dev) * 0.01 + 1e-3).float()
    out = torch.empty(M, N, device=dev, dtype=torch.bfloat16)
    lin = ops.Int8Linear(w, ws, None, group)
    for _ in range(3):
        lin.forward(x, out)
    torch.cuda.synchronize()
    barrier()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    n = 20
    e0.record(torch.cuda.current_stream())
    for _ in range(n):
        lin.forward(x, out)
    e1.record(torch.cuda.current_stream())
    torch.cuda.synchronize()
    ops.context(dev).wait()
    barrier()
    ms = max_over_ranks(e0.elapsed_time(e1)) / n
    tops = 2.0 * M * N * K / (ms / 1e3) / 1e12
    peak = 2 * peaks["bf16_tflops"]
    return {"kernels": "rotq_rows<bf16,256> + i8gemm2 (tcgen05.mma cta_group::2 kind::i8, 256x256 tiles per SM pair)",
            "M": M, "K": K, "N": N,
            "group": group, "ms": ms, "tops": tops, "peak_int8_tops": peak, "peak_source": peaks["source"],
            "frac": tops / peak}


def vae_leg(dev, max_over_ranks, barrier, B=4, S=1797, H=32, D=64) -> dict:
    """The VAE decoder's attention (h3s_attention_batch, vae.rs:309-311): a batch of B = 4 tiles (TILE_BATCH) of
    S = 1,797 tokens (7 x 16 x 16 latent cells + 4 registers + 1), 32 heads of 64 (vae.rs:21-22), fp16 q/k/v read in
    place from the qkv buffer (row stride 3 x 2048) and fp16 out; each tile attends to its own tokens (fp16 SDPA path).
    Seeded normal values stand in for the decoder's activations. Work: 4*S^2*D*H*B flops."""
    import torch

    from sycl_minimax_h3_b200 import ops

    g = torch.Generator(device=dev)
    g.manual_seed(64)
    qkv = torch.randn(B * S, 3 * H * D, generator=g, device=dev, dtype=torch.float16)
    out = torch.empty(B * S, H * D, device=dev, dtype=torch.float16)
    q, k, v = ops.Rows.qkv(qkv, H, D)
    for _ in range(3):
        ops.attention_batch(q, k, v, B, out)
    torch.cuda.synchronize()
    barrier()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    n = 20
    e0.record(torch.cuda.current_stream())
    for _ in range(n):
        ops.attention_batch(q, k, v, B, out)
    e1.record(torch.cuda.current_stream())
    torch.cuda.synchronize()
    ops.context(dev).wait()
    barrier()
    ms = max_over_ranks(e0.elapsed_time(e1)) / n
    flops = 4.0 * S * S * D * H * B
    return {"kernel": "attn_sage3<false, 64> (fp16 SDPA, 64-wide heads, batch in the grid)", "B": B, "S": S, "H": H, "D": D, "ms": ms,
            "tflops": flops / (ms / 1e3) / 1e12}


def ulysses_leg(dev, world, rank, S, H, D, max_over_ranks, barrier) -> dict:
    """c4: token-sharded qkv -> all-to-all -> attention of H/P heads over all S tokens -> inverse all-to-all. The
    exchange is ulysses.PeerExchange: one push kernel per direction that stores each rank's data straight into the
    other ranks' buffers over NVLink (relayout included) for the forward, the inverse inside the attention's epilogue
    (each output row stored into its rank's token shard; H3_C4_FUSED=0: a push kernel after the attention). NCCL's
    all_to_all_single with the relayout copies around it is timed beside it."""
    import torch

    from sycl_minimax_h3_b200 import ops, ulysses

    s = S // world
    g = torch.Generator(device=dev)
    g.manual_seed(5000 + rank)
    shard = torch.randn(s, 3 * H * D, generator=g, device=dev, dtype=torch.float16)
    h = H // world
    out = torch.empty(S, h * D, dtype=torch.float16, device=dev)
    # the inverse exchange inside the attention epilogue (h3s_attention_ulysses); H3_C4_FUSED=0: a push kernel after
    # the attention instead
    fused = os.environ.get("H3_C4_FUSED", "1") != "0"
    try:
        ex = ulysses.PeerExchange(s, H, D, torch.float16)   # every rank gets the same outcome (decided collectively)
    except RuntimeError as e:
        ex = None
        why = str(e)

    def step(peer, times=None, local=False):
        ev = [torch.cuda.Event(enable_timing=True) for _ in range(4)]
        ev[0].record()
        qkv_heads = ex.seq_to_heads(shard) if peer else ulysses.seq_to_heads(shard, H, D)
        ev[1].record()
        if peer and fused:   # the attention stores its output rows straight into every rank's token shard
            # local: the same kernel with every row stored into this rank's own buffer (timing only), so that the
            # difference to the peer form is what the inverse exchange costs inside the attention
            res = ex.attention_to_seq(qkv_heads, [ex.dst_out[rank]] * world if local else None)
            ev[2].record()
        elif peer:
            q, k, v = ops.Rows.qkv(qkv_heads, h, D)
            ops.attention(q, k, v, out)
            ev[2].record()
            res = ex.heads_to_seq(out)
        else:
            q, k, v = ops.Rows.qkv(qkv_heads, h, D)
            ops.attention(q, k, v, out)
            ev[2].record()
            res = ulysses.heads_to_seq(out, H, D)
        ev[3].record()
        if times is not None:
            times.append(ev)
        return res

    def measure(peer, local=False):
        for _ in range(3):
            step(peer, local=local)
        torch.cuda.synchronize()
        barrier()
        times = []
        n = 10
        for _ in range(n):
            step(peer, times, local=local)
        torch.cuda.synchronize()
        if peer:
            ex.check()
        else:
            ops.context(dev).wait()
        a2a = sum(e[0].elapsed_time(e[1]) + e[2].elapsed_time(e[3]) for e in times) / n
        att = sum(e[1].elapsed_time(e[2]) for e in times) / n
        tot = sum(e[0].elapsed_time(e[3]) for e in times) / n
        return max_over_ranks(tot), max_over_ranks(a2a), max_over_ranks(att)

    tot_n, a2a_n, att_n = measure(False)
    if ex is None:
        return {"tokens_per_gpu": s, "heads_per_gpu": h, "exchange": f"NCCL all_to_all_single ({why})",
                "ms_per_call": tot_n, "ms_all_to_all_exposed": a2a_n, "ms_attention": att_n,
                "tops": ops_per_call(S, H, D) / (tot_n / 1e3) / 1e12}
    tot, a2a, att = measure(True)
    res = {"tokens_per_gpu": s, "heads_per_gpu": h,
           "exchange": "peer stores over NVLink (CUDA IPC)" + ("; the inverse in the attention epilogue" if fused else
                                                              "; one push kernel per direction"),
           "ms_per_call": tot, "ms_all_to_all_exposed": a2a, "ms_attention": att,
           "tops": ops_per_call(S, H, D) / (tot / 1e3) / 1e12,
           "nccl_all_to_all": {"ms_per_call": tot_n, "ms_all_to_all_exposed": a2a_n}}
    if fused:
        # the same attention with every output row stored locally: ms_attention minus this is the inverse exchange's
        # own cost inside the epilogue (its NVLink stores and the two meetings around the kernel are in both)
        _, _, att_local = measure(True, local=True)
        res["ms_attention_local_stores"] = att_local
        res["ms_inverse_exchange_in_epilogue"] = att - att_local
        res["ms_exchange_total"] = a2a + att - att_local
    ex.close()
    return res


if __name__ == "__main__":
    main()
