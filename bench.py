"""Benchmark: GPT-2 124M-architecture prefill (and KV-cache decode) tokens/s on B200.

    python bench.py [--gpus N] [--steps K] [--warmup W] [--impl ours|reference]
    torchrun --nproc-per-node N bench.py --gpus N ...   (one process per GPU)

Headline (`value`): BASELINE config 3 — GPT-2 124M architecture, bf16,
seeded random weights, uniform random token ids, batch 32 x seq 512 per
GPU, one prefill forward to logits at every position per step. Weak
scaling: every rank runs its own batch of 32 sequences (batch sharding,
no collective in the data path); value = all ranks' tokens / max-over-ranks
device time. Inputs (weights 249 MB, logits 1.65 GB per step) exceed the
126 MB L2, so no extra flush is done between steps.

Extra keys: `roofline` for the dominant kernel family (the tcgen05 GEMMs:
CUDA events around each of their launches, recorded in extra instrumented
steps right after the timed ones, because an event between two kernels holds
back programmatic dependent launch and would slow the headline loop) plus the
whole-forward fraction; `e2e` (public API: host token ids in, full forward,
last-position logits of the whole batch gathered over NCCL at N > 1 and read
back to the host, every step); `decode` (batch 64 sharded
across the ranks, prompt 128, 128 greedy KV-cache steps, the token gather
inside the timed region; at N = 1 also a CPU sample with the reference's
re-forward decode semantics); `extras` (cfg 3' GELU op, cfg 2, cfg 1 on one
GPU; cfg 5 GPT-2 XL at every N: prefill B64 x T1024, KV-cache decode and the
reference's windowed re-prefill decode); `cpu_baseline`; `clocks`.

`--impl reference` times the reference algorithm's CPU restatement
(oracle/ref_gpt.py, fp32, all host threads) on the same config and metric,
each step a bounded sample (one sequence of 512 tokens); the reference
itself (CuPy + cuTile) cannot run on this image, so its restatement, pinned
to the reference's own forward/generate, stands in for it.
"""
from __future__ import annotations

import argparse
import json
import math
import os
import statistics
import subprocess
import sys
import threading
import time

ROOT = os.path.dirname(os.path.abspath(__file__))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

import torch  # noqa: E402
import torch.distributed as dist  # noqa: E402

METRIC = "GPT-2 124M prefill tokens/s (B32xT512 per GPU, bf16)"
UNIT = "tokens/s"


def model_cfg(name):
    from cutilegpt_b200.models.config import GPTConfig
    return GPTConfig.gpt2_xl() if name == "xl" else GPTConfig.gpt2()


def flops_per_token(cfg, T):
    """Algorithmic FLOPs per prefill token: block GEMMs 24·C²·L, causal attention 2·C·(T+1)·L, lm_head 2·C·V."""
    C, L, V = cfg.n_embd, cfg.n_layer, cfg.vocab_size
    return 24 * C * C * L + 2 * C * (T + 1) * L + 2 * C * V


def sustained_tflops():
    """The measured bf16 GEMM rate held for seconds under the power cap (MEASURED_PEAKS.json), the
    denominator for kernels timed inside a long step; 1400 TF/s (an earlier measurement) if absent."""
    try:
        with open(os.path.join(ROOT, "MEASURED_PEAKS.json")) as f:
            return float(json.load(f)["bf16_tflops_sustained"]), "measured"
    except Exception:
        return 1400.0, "fallback"


def load_peaks():
    try:
        with open(os.path.join(ROOT, "MEASURED_PEAKS.json")) as f:
            p = json.load(f)
        return float(p["bf16_tflops"]), float(p["hbm_gbs"]), "measured"
    except Exception:
        return 1590.0, 6650.0, "fallback"


class ClockSampler:
    """Samples nvidia-smi SM clocks and throttle reasons while the timed region runs."""

    Q = ("index,clocks.sm,clocks.max.sm,power.draw,clocks_event_reasons.active,"
         "clocks_event_reasons.hw_slowdown,clocks_event_reasons.hw_thermal_slowdown,"
         "clocks_event_reasons.sw_thermal_slowdown,clocks_event_reasons.sw_power_cap")

    def __init__(self, index: int):
        self.index = index
        self.proc = None
        self.lines = []

    def start(self):
        try:
            self.proc = subprocess.Popen(
                ["nvidia-smi", f"--id={self.index}", f"--query-gpu={self.Q}", "--format=csv,noheader,nounits",
                 "-lms", "200"], stdout=subprocess.PIPE, stderr=subprocess.DEVNULL, text=True)
            self._t = threading.Thread(target=self._read, daemon=True)
            self._t.start()
            time.sleep(0.3)
        except Exception:
            self.proc = None

    def _read(self):
        for line in self.proc.stdout:
            self.lines.append(line.strip())

    def stop(self):
        if self.proc is None:
            return None
        self.proc.terminate()
        try:
            self.proc.wait(timeout=5)
        except Exception:
            self.proc.kill()
        sm, mx, reasons = [], None, set()
        names = ["hw_slowdown", "hw_thermal_slowdown", "sw_thermal_slowdown", "sw_power_cap"]
        for ln in self.lines:
            f = [x.strip() for x in ln.split(",")]
            if len(f) < 9:
                continue
            try:
                sm.append(float(f[1]))
                mx = float(f[2])
            except ValueError:
                continue
            for n, v in zip(names, f[5:9]):
                if v.lower() == "active":
                    reasons.add(n)
        if not sm:
            return None
        return {"sm_mhz": statistics.median(sm), "sm_max_mhz": mx, "reasons": sorted(reasons),
                "samples": len(sm)}


class GemmTimer:
    """CUDA events around every GEMM launch (recorded on the launching stream) + algorithmic FLOPs."""

    def __init__(self):
        self.pairs = []
        self.flops = 0
        self.enabled = False

    def start(self, flops):
        if not self.enabled:
            return
        e = torch.cuda.Event(enable_timing=True)
        e.record()
        self.pairs.append([e, None])
        self.flops += flops

    def stop(self):
        if not self.enabled:
            return
        e = torch.cuda.Event(enable_timing=True)
        e.record()
        self.pairs[-1][1] = e

    def total_ms(self):
        return sum(a.elapsed_time(b) for a, b in self.pairs)


def max_over_ranks(x: float, world: int) -> float:
    if world == 1:
        return x
    t = torch.tensor([x], dtype=torch.float64, device="cuda")
    dist.all_reduce(t, op=dist.ReduceOp.MAX)
    return float(t.item())


def barrier(world):
    if world > 1:
        dist.barrier()
    torch.cuda.synchronize()


# --------------------------------------------------------------------------- ours
def _event_ms(fn, iters=20, warm=3):
    for _ in range(warm):
        fn()
    torch.cuda.synchronize()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    for _ in range(iters):
        fn()
    e1.record()
    torch.cuda.synchronize()
    return e0.elapsed_time(e1) / iters


def run_extras(dev):
    """The other BASELINE configs on one GPU (seeded synthetic inputs), for the record:
    cfg 3' standalone tanh-GELU on a [32,512,768] bf16 N(0,1) tensor (HBM-bound: 50.3 MB per call),
    cfg 2 (6/6/384) prefill B16xT256 in bf16 and fp32, cfg 1 (nano 3/3/48, ctx 1024) fp32 B8xT256.
    Inputs of the GELU exceed L2 only twice over, so a 256 MB buffer is rewritten between calls."""
    from cutilegpt_b200 import CutileGPT, GPTConfig, cutile_gelu
    _, peak_gbs, src = load_peaks()
    g = torch.Generator(device="cpu").manual_seed(2)
    x = torch.randn(32, 512, 768, generator=g).to(torch.bfloat16).to(dev)
    flush = torch.empty(256 << 20, dtype=torch.uint8, device=dev)

    def gelu_once():
        flush.zero_()
        cutile_gelu(x)
    t_all = _event_ms(gelu_once)
    t_flush = _event_ms(lambda: flush.zero_())
    t = max(t_all - t_flush, 1e-6)
    gb = x.numel() * 2 * 2 / 1e9
    out = {"gelu_op": {"config": "cfg3' tanh-GELU [32,512,768] bf16 N(0,1), L2 flushed between calls",
                       "us": t * 1e3, "GB/s": gb / (t / 1e3), "frac_hbm": gb / (t / 1e3) / peak_gbs,
                       "peak_source": src}}
    for name, cfg, B, T, dt in (("cfg2_small_bf16", GPTConfig(n_layer=6, n_head=6, n_embd=384), 16, 256, torch.bfloat16),
                                ("cfg2_small_fp32", GPTConfig(n_layer=6, n_head=6, n_embd=384), 16, 256, torch.float32),
                                ("cfg1_nano_fp32", GPTConfig(n_layer=3, n_head=3, n_embd=48), 8, 256, torch.float32)):
        m = CutileGPT(cfg, dtype=dt, device=dev, seed=0)
        idx = torch.randint(0, cfg.vocab_size, (B, T), generator=torch.Generator().manual_seed(1)).to(dev)
        ms = _event_ms(lambda: m(idx), iters=10)
        out[name] = {"batch": B, "seq_len": T, "ms_per_forward": ms, "tokens_per_s": B * T / (ms / 1e3),
                     "model_tflops": flops_per_token(cfg, T) * B * T / (ms / 1e3) / 1e12}
        del m
    torch.cuda.empty_cache()
    return out


def run_decode(model, cfg, rank, world, dev, Bg=64, P=128, S=128):
    """batch 64 sharded over the ranks, prompt 128, 128 greedy KV-cache steps.

    Config 5 (GPT-2 XL) calls it with batch 64, prompt 768, 256 steps: the config's own 1024-token
    prompt already fills the context, so every step would re-encode a full window (a prefill per
    step); the shortened prompt is the named deviation that keeps 768 + 256 <= 1024.
    The timed call is ShardedGPT.generate with gather=True: at N > 1 the NCCL all_gather of the
    generated [B, P + S] tokens runs inside the timed region and its device time is reported.
    """
    from cutilegpt_b200.distributed import ShardedGPT
    sharded = ShardedGPT(model)
    lo, hi = sharded.local_rows(Bg)
    g2 = torch.Generator().manual_seed(77)
    prompt = torch.randint(0, cfg.vocab_size, (Bg, P), generator=g2).to(dev)
    sharded.generate(prompt, S, top_k=1)               # warm-up; captures the decode-step graph
    barrier(world)
    p0, p1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    d0, d1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    st = model._decode_state(hi - lo, P + S)          # the state the timed generate uses
    p0.record()
    model.forward_last(prompt[lo:hi], out=st.logits, cache=st.cache)   # the prefill inside generate
    p1.record()
    sharded.time_gather = True
    sharded.gather_ms()
    d0.record()
    out = sharded.generate(prompt, S, top_k=1)         # prefill + S-1 graph-replayed steps (+ gather)
    d1.record()
    barrier(world)
    assert out.shape == (Bg, P + S)
    gather_ms = max_over_ranks(sharded.gather_ms(), world)
    gen_ms = max_over_ranks(d0.elapsed_time(d1), world)
    pre_ms = max_over_ranks(p0.elapsed_time(p1), world)
    dec_steps = S - 1
    dec_ms = max(gen_ms - pre_ms, 1e-6)
    dec_tok_s = Bg * dec_steps / (dec_ms / 1e3)
    # HBM bytes per decode step on one rank: weights once + KV read (mean length) + KV write + logits
    Bl = hi - lo
    wbytes = sum(t.numel() * t.element_size() for k, t in model.weights.items() if k != "lm_head.weight")
    C, Lyr = cfg.n_embd, cfg.n_layer
    mean_len = P + 1 + (dec_steps - 1) / 2
    step_bytes = (wbytes + Bl * Lyr * 2 * C * 2 * mean_len + Bl * Lyr * 2 * C * 2
                  + Bl * cfg.vocab_size * 2)
    _, peak_gbs, src = load_peaks()
    step_s = (dec_ms - gather_ms) / dec_steps / 1e3
    return {"value": dec_tok_s, "unit": "tokens/s", "batch": Bg, "prompt": P, "steps": S,
            "ms_per_step": dec_ms / dec_steps, "prefill_ms": pre_ms,
            "gather": {"collective": "all_gather (NCCL) of the generated tokens" if world > 1 else "none (N=1)",
                       "ms": gather_ms, "share_of_decode": gather_ms / dec_ms},
            "hbm_roofline": {"achieved": step_bytes / step_s / 1e9, "peak": peak_gbs, "unit": "GB/s",
                             "frac": step_bytes / step_s / 1e9 / peak_gbs,
                             "bytes_per_step_per_gpu": step_bytes, "peak_source": src},
            "scaling": "strong", "cuda_graph": True}


def decode_cpu_sample(model_name="gpt2", P=128, budget_s=10.0):
    """The reference's decode semantics on the host cores: every new token re-runs the whole forward
    over the prefix (cutile_gpt/models/gpt.py:204-206, no KV cache), greedy, one sequence of prompt P,
    fp32 oracle with bf16-rounded weights; as many steps as fit in budget_s."""
    from cutilegpt_b200.models.init import init_state
    from oracle import ref_gpt as R
    threads = os.cpu_count() or 1
    torch.set_num_threads(threads)
    cfg = model_cfg(model_name)
    w = R.cast_weights(init_state(cfg, 1234), dtype=torch.float32, round_to=torch.bfloat16)
    idx = torch.randint(0, cfg.vocab_size, (1, P), generator=torch.Generator().manual_seed(77))
    steps = 0
    t0 = time.perf_counter()
    with torch.no_grad():
        while time.perf_counter() - t0 < budget_s:
            idx = R.generate_greedy(w, cfg.n_layer, cfg.n_head, cfg.block_size, idx, 1)
            steps += 1
    dt = time.perf_counter() - t0
    return {"value": steps / dt, "unit": "tokens/s", "cores": threads, "kind": "port",
            "sample": f"1 sequence, prompt {P}, {steps} greedy steps, each a full re-forward of the prefix "
                      f"(reference semantics, no KV cache), fp32 oracle with bf16-rounded weights"}


def prefill_bench(model, cfg, B, T, steps, warmup, world, rank, sample_clocks=None):
    """Timed prefill forwards (logits at every position) of B local sequences of T tokens, then a
    separate instrumented pass with CUDA events around every GEMM launch (events between kernels
    hold back programmatic dependent launch, so they stay out of the timed loop)."""
    from cutilegpt_b200 import _lib
    dev = model.device
    gen = torch.Generator(device="cpu").manual_seed(1000 + rank)
    idx = torch.randint(0, cfg.vocab_size, (B, T), generator=gen).to(dev)
    logits = torch.empty((B * T, cfg.vocab_size), dtype=torch.bfloat16, device=dev)
    ws = model._workspace(B, T)
    timer = GemmTimer()
    model.kernel_timer = timer

    def step():
        model._blocks(idx, ws)
        model._lm_head(ws, logits)

    for _ in range(warmup):
        step()
    barrier(world)
    if sample_clocks is not None:
        sample_clocks.start()
    launches0 = _lib.lib().gpt_launch_count()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    e0.record()
    for _ in range(steps):
        step()
    e1.record()
    barrier(world)
    launches = _lib.lib().gpt_launch_count() - launches0
    clk = sample_clocks.stop() if sample_clocks is not None else None
    ms_max = max_over_ranks(e0.elapsed_time(e1), world)
    rsteps = max(3, min(steps, 10))
    timer.enabled = True
    r0, r1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    r0.record()
    for _ in range(rsteps):
        step()
    r1.record()
    torch.cuda.synchronize()
    timer.enabled = False
    model.kernel_timer = None
    out = dict(ms=ms_max / steps, launches=launches, clk=clk, gemm_ms=timer.total_ms(),
               gemm_launches=len(timer.pairs), gemm_flops=timer.flops, gemm_steps=rsteps,
               gemm_step_ms=r0.elapsed_time(r1))
    del logits
    torch.cuda.empty_cache()
    return out


def run_xl(args, rank, world, dev):
    """BASELINE config 5 on every N: GPT-2 XL architecture, bf16, global batch 64 sharded over the
    ranks (strong scaling): prefill B64 x T1024 (3 timed steps), KV-cache decode (prompt 768, 256
    greedy steps, the named deviation) and the reference's own decode semantics past the context
    (cutile_gpt/models/gpt.py:205: the last 1024 tokens re-encoded every step, 2 timed steps)."""
    from cutilegpt_b200 import CutileGPT
    from cutilegpt_b200.distributed import shard_range
    from cutilegpt_b200.models.init import init_state
    cfg = model_cfg("xl")
    model = CutileGPT.__new__(CutileGPT)
    model._setup(cfg, torch.bfloat16, dev)
    model.load_state(init_state(cfg, 1234, device=dev))    # seeded on the device (fast); same on every rank
    Bg, T = 64, 1024
    lo, hi = shard_range(Bg, rank, world)
    r = prefill_bench(model, cfg, hi - lo, T, steps=3, warmup=3, world=world, rank=rank)
    peak_tf, _, src = load_peaks()
    value = Bg * T / (r["ms"] / 1e3)
    gemm_tf = r["gemm_flops"] / (r["gemm_ms"] / 1e3) / 1e12
    model_tf = flops_per_token(cfg, T) * value / world / 1e12
    out = {"config": "cfg5 gpt2-xl (48/25/1600) bf16, global batch 64 sharded over the ranks",
           "prefill": {"value": value, "unit": UNIT, "batch": Bg, "seq_len": T, "ms_per_step": r["ms"],
                       "steps": 3, "warmup": 3, "scaling": "strong",
                       "whole_forward_tflops_per_gpu": model_tf, "whole_forward_frac": model_tf / peak_tf,
                       "gemm_family_tflops": gemm_tf, "gemm_family_frac": gemm_tf / peak_tf,
                       "peak_source": src}}
    out["decode_kv_cache"] = run_decode(model, cfg, rank, world, dev, Bg=64, P=768, S=256)
    # reference semantics: prompt 1024 fills the context; each new token re-encodes the last 1024
    g = torch.Generator().manual_seed(78)
    full = torch.randint(0, cfg.vocab_size, (Bg, T), generator=g)[lo:hi].to(dev)
    model.generate(full, 1, top_k=1)                   # warm-up (windowed path)
    barrier(world)
    w0, w1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    w0.record()
    seq = model.generate(full, 2, top_k=1)             # 2 steps past the context, re-encoding windows
    w1.record()
    barrier(world)
    assert seq.shape == (hi - lo, T + 2)
    wms = max_over_ranks(w0.elapsed_time(w1), world)
    out["decode_reference_semantics"] = {"value": Bg * 2 / (wms / 1e3), "unit": "tokens/s",
                                         "ms_per_step": wms / 2, "steps": 2, "window": T,
                                         "note": "no KV cache: every step is a 1024-token prefill of the "
                                                 "cropped window, as the reference does past block_size"}
    del model
    torch.cuda.empty_cache()
    return out


def run_ours(args, rank, world, local):
    from cutilegpt_b200 import CutileGPT
    from cutilegpt_b200.distributed import ShardedGPT

    dev = torch.device("cuda", local)
    torch.cuda.set_device(dev)
    cfg = model_cfg("gpt2")
    B, T = args.batch, args.seq                        # config 3: 32 sequences per GPU (weak scaling)
    model = CutileGPT(cfg, dtype=torch.bfloat16, device=dev, seed=1234)   # same weights on every rank
    if args.decode_only:
        return {"dec": run_decode(model, cfg, rank, world, dev)}
    clocks = ClockSampler(local)
    r = prefill_bench(model, cfg, B, T, args.steps, args.warmup, world, rank, sample_clocks=clocks)
    tokens = B * world * T * args.steps
    value = tokens / (r["ms"] * args.steps / 1e3)

    # ---- e2e through the public API: host token ids of the whole batch (pinned); each rank copies its
    # rows in, runs the full forward (logits at every position), the last-position logits of the whole
    # batch are gathered (NCCL all_gather at N > 1) and read back to the host, every step.
    Bg = B * world
    gen = torch.Generator(device="cpu").manual_seed(2000)
    idx_host = torch.randint(0, cfg.vocab_size, (Bg, T), generator=gen).pin_memory()
    out_host = torch.empty((Bg, cfg.vocab_size), dtype=torch.bfloat16).pin_memory()
    sharded = ShardedGPT(model)
    lo, hi = sharded.local_rows(Bg)

    def e2e_step():
        d_idx = torch.empty((Bg, T), dtype=torch.int64, device=dev)
        d_idx[lo:hi].copy_(idx_host[lo:hi], non_blocking=True)   # only this rank's rows cross PCIe
        _, last = sharded.forward_gather_last(d_idx)
        out_host.copy_(last, non_blocking=True)

    for _ in range(args.warmup):
        e2e_step()
    barrier(world)
    sharded.time_gather = True
    sharded.gather_ms()
    f0, f1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    f0.record()
    for _ in range(args.steps):
        e2e_step()
    f1.record()
    barrier(world)
    e2e_ms = max_over_ranks(f0.elapsed_time(f1), world)
    e2e_gather = max_over_ranks(sharded.gather_ms(), world)
    e2e_value = tokens / (e2e_ms / 1e3)
    torch.cuda.empty_cache()
    dec = None if args.no_decode else run_decode(model, cfg, rank, world, dev)
    if dec is not None and rank == 0 and world == 1 and not args.no_cpu:
        dec["cpu_baseline"] = decode_cpu_sample("gpt2")
    extras = run_extras(dev) if (world == 1 and not args.no_decode) else None
    del model
    torch.cuda.empty_cache()
    xl = None if args.no_xl else run_xl(args, rank, world, dev)
    return dict(value=value, ms=r["ms"], tokens=tokens, launches=r["launches"], clk=r["clk"],
                gemm_ms=r["gemm_ms"], gemm_launches=r["gemm_launches"], gemm_flops=r["gemm_flops"],
                gemm_steps=r["gemm_steps"], gemm_step_ms=r["gemm_step_ms"], e2e_value=e2e_value,
                e2e_gather_ms=e2e_gather / args.steps,
                e2e_h2d=(hi - lo) * T * 8, e2e_d2h=Bg * cfg.vocab_size * 2, dec=dec, cfg=cfg, extras=extras, xl=xl)


# --------------------------------------------------------------------------- CPU
def _cpu_oracle(seq, model="gpt2"):
    from cutilegpt_b200.models.init import init_state
    from oracle import ref_gpt as R
    cfg = model_cfg(model)
    w = R.cast_weights(init_state(cfg, 1234), dtype=torch.float32, round_to=torch.bfloat16)
    idx = torch.randint(0, cfg.vocab_size, (1, seq), generator=torch.Generator().manual_seed(5))
    return lambda: R.gpt_forward(w, cfg.n_layer, cfg.n_head, idx)


def cpu_sample(seq=512, budget_s=20.0, model="gpt2"):
    """Tokens/s of the fp32 CPU oracle (bf16-rounded weights) on one sequence, all host threads."""
    threads = os.cpu_count() or 1
    torch.set_num_threads(threads)
    fwd = _cpu_oracle(seq, model)
    times = []
    t_start = time.perf_counter()
    with torch.no_grad():
        while True:
            t0 = time.perf_counter()
            fwd()
            times.append(time.perf_counter() - t0)
            if time.perf_counter() - t_start > budget_s or len(times) >= 5:
                break
    return seq / statistics.median(times), threads, len(times)


def run_reference(args, rank):
    if rank != 0:
        return
    threads = os.cpu_count() or 1
    torch.set_num_threads(threads)
    seq = args.seq
    fwd = _cpu_oracle(seq)
    with torch.no_grad():
        fwd()
        t0 = time.perf_counter()
        for _ in range(args.steps):
            fwd()
        dt = time.perf_counter() - t0
    value = seq * args.steps / dt
    sample = f"one sequence of {seq} tokens per step, fp32 oracle with bf16-rounded weights"
    line = {"impl": "reference", "metric": METRIC, "value": value, "unit": UNIT,
            "n_gpus": args.gpus, "steps": args.steps, "warmup": args.warmup, "ms_per_step": dt / args.steps * 1e3,
            "higher_is_better": True, "scaling": "weak", "vs_baseline": None, "dtype": "f32",
            "data": "synthetic (seeded random weights, uniform random token ids)",
            "config": {"workload": f"cfg3 gpt2-124M prefill (CPU sample: 1x{seq} tokens per step)",
                       "model": "gpt2-124M", "seq_len": seq},
            "cpu_baseline": {"value": value, "unit": UNIT, "cores": threads, "kind": "port", "sample": sample},
            "e2e": {"value": value, "unit": UNIT, "h2d_bytes_per_step": 0, "d2h_bytes_per_step": 0},
            "note": "the reference (CuPy + cuTile) cannot run on this image: cupy is not installed and "
                    "cuda.tile finds no tileiras compiler; the CPU restatement of its algorithm "
                    "(oracle/ref_gpt.py, pinned to the reference's own forward/generate) is timed instead"}
    print(json.dumps(line), flush=True)


def run_decode_parts(local):
    """Config-4 decode step (GPT-2 124M, B64, cached length 193) taken apart: each part is the same kernel
    sequence the folded step launches (one launch per layer), captured in a CUDA graph 4 times over and
    replayed 20 times, timed with CUDA events; us = per replay of one part sequence. Prints one JSON line."""
    from cutilegpt_b200 import CutileGPT, GPTConfig
    from cutilegpt_b200 import _lib as L
    from cutilegpt_b200.kernels import ops
    dev = torch.device("cuda", local)
    torch.cuda.set_device(dev)
    cfg = GPTConfig(n_layer=12, n_head=12, n_embd=768, vocab_size=50257, block_size=1024)
    m = CutileGPT(cfg, dtype=torch.bfloat16, device=dev, seed=0)
    B, P, S = 64, 128, 128
    prompt = torch.randint(0, cfg.vocab_size, (B, P), generator=torch.Generator().manual_seed(1)).to(dev)
    m.generate(prompt, 16, top_k=1)
    st = m._decode_state(B, P + S)
    F = m._fold_weights()
    C, H, eps = cfg.n_embd, cfg.n_head, 1e-5
    scale = 1.0 / math.sqrt(C // H)
    q = st.qkv[:, :C]

    def qkv(i):
        wf, u, v = F[f"h.{i}.attn"]
        ops.gemm_fused(st.x, wf, st.qkv, epilogue=L.EPI_BIAS, ln=(st.sums[2 * i], eps, u, v),
                       kv=(st.cache[i, 0], st.cache[i, 1], st.pos, 0))

    def att(i):
        ops.attention_decode(q, st.cache[i, 0], st.cache[i, 1], st.att, 1, st.dec_ws, scale, len_dev=st.pos)

    def cproj(i):   # writes a scratch output (st.h) so the residual stream stays as it is
        p = f"h.{i}."
        ops.gemm_fused(st.att, m._w(p + "attn.c_proj.weight"), st.h, bias=m._w(p + "attn.c_proj.bias"),
                       resid=st.x, row_stats=st.sums[2 * i + 1])

    def fc(i):
        wf, u, v = F[f"h.{i}.fc"]
        ops.gemm_fused(st.x, wf, st.f, epilogue=L.EPI_BIAS_GELU, ln=(st.sums[2 * i + 1], eps, u, v))

    def mproj(i):
        p = f"h.{i}."
        ops.gemm_fused(st.f, m._w(p + "mlp.c_proj.weight"), st.h, bias=m._w(p + "mlp.c_proj.bias"),
                       resid=st.x, row_stats=st.sums[2 * i + 2])

    def lm():
        wf, u, v = F["lm"]
        ops.gemm_fused(st.x, wf, st.logits, epilogue=L.EPI_NONE, ln=(st.sums[2 * cfg.n_layer], eps, u, v))
        ops.argmax(st.logits, st.tok)

    parts = {
        "full_step": lambda: m._decode_step(st),
        "qkv_x12": lambda: [qkv(i) for i in range(12)],
        "attention_x12": lambda: [att(i) for i in range(12)],
        "attn_c_proj_x12": lambda: [cproj(i) for i in range(12)],
        "c_fc_x12": lambda: [fc(i) for i in range(12)],
        "mlp_c_proj_x12": lambda: [mproj(i) for i in range(12)],
        "lm_head_argmax": lm,
        "row_sums_x12 (launch floor)": lambda: [ops.row_sums(st.x, st.sums[0]) for _ in range(12)],
    }
    out = {}
    for name, fn in parts.items():
        st.pos.fill_(192)
        fn()
        torch.cuda.synchronize()
        g = m._capture_fn(lambda: [fn() for _ in range(4)])
        for _ in range(3):
            g.replay()
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        for _ in range(20):
            g.replay()
        e1.record()
        torch.cuda.synchronize()
        out[name] = round(e0.elapsed_time(e1) / 20 / 4 * 1e3, 2)
    print(json.dumps({"probe": "decode_parts", "unit": "us per part sequence", "parts": out}), flush=True)


def run_prefill_parts(local):
    """Config-3 prefill forward (GPT-2 124M, B32xT512) taken apart: each part is the kernel sequence the
    forward launches for it (one launch per layer), captured in a CUDA graph twice over and replayed 10
    times, timed with CUDA events; us = per replay of one part sequence, TF/s from its algorithmic FLOPs
    (attention: the causal half). Prints one JSON line."""
    from cutilegpt_b200 import CutileGPT, GPTConfig
    from cutilegpt_b200.kernels import ops
    dev = torch.device("cuda", local)
    torch.cuda.set_device(dev)
    cfg = GPTConfig(n_layer=12, n_head=12, n_embd=768, vocab_size=50257, block_size=1024)
    m = CutileGPT(cfg, dtype=torch.bfloat16, device=dev, seed=0)
    B, T = 32, 512
    C, H, D, V, n = cfg.n_embd, cfg.n_head, cfg.n_embd // cfg.n_head, cfg.vocab_size, cfg.n_layer
    M = B * T
    idx = torch.randint(0, V, (B, T), generator=torch.Generator().manual_seed(1)).to(dev)
    logits = torch.empty(M, V, dtype=torch.bfloat16, device=dev)
    ws = m._workspace(B, T)
    m._blocks(idx, ws)
    m._lm_head(ws, logits)
    qkv4 = ws.qkv.view(B, T, 3, H, D)
    q, k, v = (qkv4[:, :, j].transpose(1, 2) for j in range(3))
    att4 = ws.att.view(B, T, H, D).transpose(1, 2)
    scratch = torch.empty_like(ws.x)

    def w(i, s):
        return m._w(f"h.{i}.{s}")
    from cutilegpt_b200 import _lib as Lb
    parts = {
        "full_forward": (lambda: (m._blocks(idx, ws), m._lm_head(ws, logits)), 4.2028e12),
        "layernorm_x25": (lambda: [ops.layernorm(ws.x, w(0, "ln_1.weight"), w(0, "ln_1.bias"), ws.h)
                                   for _ in range(2 * n + 1)], 0.0),
        "qkv_x12": (lambda: [m._gemm(ws.h, w(i, "attn.c_attn.weight"), ws.qkv, bias=w(i, "attn.c_attn.bias"))
                             for i in range(n)], n * 2.0 * M * C * 3 * C),
        "attention_x12": (lambda: [ops.attention_prefill(q, k, v, att4, 1.0 / math.sqrt(D)) for _ in range(n)],
                          n * 2.0 * B * H * T * (T + 1) * D),
        "attn_c_proj_x12": (lambda: [m._gemm(ws.att, w(i, "attn.c_proj.weight"), scratch,
                                             bias=w(i, "attn.c_proj.bias"), resid=ws.x) for i in range(n)],
                            n * 2.0 * M * C * C),
        "c_fc_x12": (lambda: [m._gemm(ws.h, w(i, "mlp.c_fc.weight"), ws.f, bias=w(i, "mlp.c_fc.bias"),
                                      epilogue=Lb.EPI_BIAS_GELU) for i in range(n)], n * 2.0 * M * C * 4 * C),
        "mlp_c_proj_x12": (lambda: [m._gemm(ws.f, w(i, "mlp.c_proj.weight"), scratch,
                                            bias=w(i, "mlp.c_proj.bias"), resid=ws.x) for i in range(n)],
                           n * 2.0 * M * 4 * C * C),
        "lm_head": (lambda: m._lm_head(ws, logits), 2.0 * M * C * V),
    }
    out = {}
    for name, (fn, flop) in parts.items():
        fn()
        torch.cuda.synchronize()
        g = m._capture_fn(lambda: [fn() for _ in range(2)])
        for _ in range(2):
            g.replay()
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record()
        for _ in range(10):
            g.replay()
        e1.record()
        torch.cuda.synchronize()
        us = e0.elapsed_time(e1) / 10 / 2 * 1e3
        out[name] = {"us": round(us, 1)}
        if flop:
            out[name]["TF/s"] = round(flop / us / 1e6, 1)
    print(json.dumps({"probe": "prefill_parts", "unit": "us per part sequence", "parts": out}), flush=True)


def run_samples_probe(local):
    """generate_samples (prompt pages shared) beside generate on the repeated prompt: one prompt of 768 tokens, 64 samples
    of 256 tokens, top-k 50, bf16; best of three calls each (wall time, synchronised) and the memory they hold beside
    the weights. Prints one JSON line."""
    from cutilegpt_b200 import CutileGPT, GPTConfig
    dev = torch.device("cuda", local)
    torch.cuda.set_device(dev)
    idx = torch.randint(0, 50257, (1, 768), generator=torch.Generator().manual_seed(1)).to(dev)
    rows = idx.repeat_interleave(64, 0)
    out = {}
    for name, cfg in (("gpt2", GPTConfig.gpt2()), ("gpt2-xl", GPTConfig.gpt2_xl())):
        m = CutileGPT(cfg, dtype=torch.bfloat16, device=dev, seed=0)
        m._fold_weights()            # both use them: not counted
        out[name] = {}
        for what, fn in (("generate_samples", lambda: m.generate_samples(idx, 64, 256, top_k=50)),
                         ("generate", lambda: m.generate(rows, 256, top_k=50))):
            torch.cuda.empty_cache()
            base = torch.cuda.memory_allocated()
            torch.cuda.reset_peak_memory_stats()
            fn()
            best = math.inf
            for _ in range(3):
                torch.cuda.synchronize()
                t0 = time.perf_counter()
                fn()
                torch.cuda.synchronize()
                best = min(best, time.perf_counter() - t0)
            out[name][what] = {"ms": round(best * 1e3, 1), "GB": round((torch.cuda.max_memory_allocated() - base) / 1e9, 2)}
            for cache in (m._samples, m._dec, m._ws):
                cache.clear()
        del m
    print(json.dumps({"probe": "samples", "prompt": 768, "samples": 64, "new": 256, "models": out}), flush=True)


def run_probe(name, local):
    """One HBM-bound kernel alone, at a size whose inputs exceed the 126 MB L2, timed with CUDA events
    (3 warm-up + 10 timed launches); the profiling command runs the same probe under ncu.
      layernorm    x [262144, 768] bf16 -> y (403 MB read + 403 MB written per launch)
      gelu         [512, 512, 768] bf16 -> same (403 MB + 403 MB per launch)
      decode_attn  cfg 4 decode attention: B64, 12 heads, head_dim 64, 192 cached positions, the 12 layers'
                   caches rotated so every launch reads a cache last touched 11 launches earlier
                   (37.7 MB of K/V per launch, 600 MB in all)"""
    from cutilegpt_b200.kernels import ops
    dev = torch.device("cuda", local)
    torch.cuda.set_device(dev)
    _, peak_gbs, src = load_peaks()
    g = torch.Generator(device="cpu").manual_seed(3)
    if name == "layernorm":
        x = torch.randn(262144, 768, generator=g).to(torch.bfloat16).to(dev)
        w = torch.randn(768, generator=g).to(torch.bfloat16).to(dev)
        b = torch.randn(768, generator=g).to(torch.bfloat16).to(dev)
        y = torch.empty_like(x)
        fns = [lambda: ops.layernorm(x, w, b, y)]
        nbytes = 2 * x.numel() * 2
    elif name == "gelu":
        x = torch.randn(512, 512, 768, generator=g).to(torch.bfloat16).to(dev)
        y = torch.empty_like(x)
        fns = [lambda: ops.gelu(x, y)]
        nbytes = 2 * x.numel() * 2
    elif name == "decode_attn":
        B, H, D, Tmax, Lq = 64, 12, 64, 256, 192
        caches = [(torch.randn(B, H, Tmax, D, generator=g).to(torch.bfloat16).to(dev),
                   torch.randn(B, H, Tmax, D, generator=g).to(torch.bfloat16).to(dev)) for _ in range(12)]
        q = torch.randn(B, 3 * H * D, generator=g).to(torch.bfloat16).to(dev)
        out = torch.empty(B, H * D, dtype=torch.bfloat16, device=dev)
        ws = torch.empty(max(ops.decode_workspace_bytes(B, H, D, Lq), 16), dtype=torch.uint8, device=dev)
        fns = [(lambda kc=kc, vc=vc: ops.attention_decode(q, kc, vc, out, Lq, ws)) for kc, vc in caches]
        nbytes = 2 * B * H * Lq * D * 2 + q.numel() // 3 * 2 + out.numel() * 2
    else:
        raise SystemExit(f"unknown probe {name}")
    i = 0
    for _ in range(3):
        fns[i % len(fns)]()
        i += 1
    torch.cuda.synchronize()
    e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    n = 10
    e0.record()
    for _ in range(n):
        fns[i % len(fns)]()
        i += 1
    e1.record()
    torch.cuda.synchronize()
    us = e0.elapsed_time(e1) / n * 1e3
    gbs = nbytes / (us / 1e6) / 1e9
    print(json.dumps({"probe": name, "us_per_launch": us, "algorithmic_bytes": nbytes, "GB/s": gbs,
                      "frac_hbm": gbs / peak_gbs, "peak_gbs": peak_gbs, "peak_source": src}), flush=True)


# Per-launch DRAM traffic of the GEMM family in one cfg-3 step, from one ncu capture of the full-size
# bench step (dram__bytes_read.sum + dram__bytes_write.sum over the gemm_tc_kernel launches of one
# step, divided by their count: 5723 MB over 49 launches). The block GEMMs read less than their
# algorithmic bytes because their activations are still in L2; the lm_head writes its logits once.
GEMM_TRAFFIC_BYTES_PER_LAUNCH = 116.8e6


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--warmup", type=int, default=5)
    ap.add_argument("--impl", choices=["ours", "reference"], default="ours")
    ap.add_argument("--batch", type=int, default=32, help="sequences per GPU (config 3: 32)")
    ap.add_argument("--seq", type=int, default=512)
    ap.add_argument("--no-decode", action="store_true")
    ap.add_argument("--no-cpu", action="store_true")
    ap.add_argument("--no-xl", action="store_true", help="skip the config-5 (GPT-2 XL) extras")
    ap.add_argument("--decode-only", action="store_true", help="only the config-4 decode run (profiling)")
    ap.add_argument("--probe", choices=["layernorm", "gelu", "decode_attn", "decode_parts", "prefill_parts", "samples"],
                    default=None, help="time one HBM-bound kernel alone at a size larger than L2 (profiling), the parts "
                                       "of a step, or samples of a prompt beside generate")
    args = ap.parse_args()
    args.warmup = max(args.warmup, 3)

    world_env = int(os.environ.get("WORLD_SIZE", "1"))
    if args.probe == "prefill_parts":
        run_prefill_parts(int(os.environ.get("LOCAL_RANK", "0")))
        return
    if args.probe == "samples":
        run_samples_probe(int(os.environ.get("LOCAL_RANK", "0")))
        return
    if args.probe == "decode_parts":
        run_decode_parts(int(os.environ.get("LOCAL_RANK", "0")))
        return
    if args.probe:
        run_probe(args.probe, int(os.environ.get("LOCAL_RANK", "0")))
        return
    if args.impl == "reference":
        run_reference(args, int(os.environ.get("RANK", "0")))
        return
    from cutilegpt_b200.distributed import init_from_env
    rank, world, local = init_from_env("nccl" if world_env > 1 else None)
    r = run_ours(args, rank, world, local)
    if args.decode_only:
        if rank == 0:
            print(json.dumps({"decode": r["dec"]}), flush=True)
        if world > 1:
            dist.destroy_process_group()
        return

    cpu = None
    if rank == 0 and world == 1 and not args.no_cpu:
        v, cores, n = cpu_sample(args.seq)
        cpu = {"value": v, "unit": UNIT, "cores": cores, "kind": "port",
               "sample": f"GPT-2 124M fp32 CPU oracle (bf16-rounded weights), "
                         f"1 sequence x {args.seq} tokens, median of {n} forwards"}
    if rank == 0:
        peak_tf, _, src = load_peaks()
        achieved = r["gemm_flops"] / (r["gemm_ms"] / 1e3) / 1e12
        model_tf = flops_per_token(r["cfg"], args.seq) * r["value"] / world / 1e12
        line = {
            "metric": METRIC, "value": r["value"], "unit": UNIT, "n_gpus": world,
            "steps": args.steps, "warmup": args.warmup, "ms_per_step": r["ms"], "higher_is_better": True,
            "scaling": "weak", "vs_baseline": None, "dtype": "bf16",
            "data": "synthetic (seeded random-init weights, uniform random token ids)",
            "config": {"workload": "cfg3 gpt2-124M prefill, logits at all positions",
                       "model": "gpt2-124M", "global_batch": args.batch * world, "seq_len": args.seq,
                       "parallelism": f"dp{world} (batch-sharded replicas)",
                       "l2": "inputs larger than L2 (weights 249 MB, logits 1.65 GB per step); no flush"},
            "roofline": {"kernel": "gemm_tc_kernel (tcgen05 GEMM, all launches)", "bound": "tensor",
                         "achieved": achieved, "peak": peak_tf, "unit": "TFLOP/s", "frac": achieved / peak_tf,
                         "traffic": GEMM_TRAFFIC_BYTES_PER_LAUNCH, "peak_source": src,
                         "launches_per_step": r["gemm_launches"] // r["gemm_steps"],
                         "share_of_step": r["gemm_ms"] / r["gemm_step_ms"],
                         "measured_in": f"{r['gemm_steps']} extra steps with CUDA events around every GEMM",
                         "peak_sustained": sustained_tflops()[0],
                         "frac_sustained": achieved / sustained_tflops()[0],
                         "peak_note": "peak = burst cuBLAS bf16 rate; the GEMMs run inside a multi-second "
                                      "loop under the 1 kW power cap, for which peak_sustained is the measured rate",
                         "whole_forward": {"tflops": model_tf, "frac": model_tf / peak_tf,
                                           "frac_sustained": model_tf / sustained_tflops()[0],
                                           "flop_per_forward": flops_per_token(r["cfg"], args.seq)
                                           * args.batch * args.seq,
                                           "note": "all algorithmic FLOPs of the forward / step time"}},
            "model_tflops": model_tf,
            "e2e": {"value": r["e2e_value"], "unit": UNIT, "h2d_bytes_per_step": r["e2e_h2d"],
                    "d2h_bytes_per_step": r["e2e_d2h"], "gather_ms_per_step": r["e2e_gather_ms"],
                    "path": "host ids -> ShardedGPT.forward_gather_last (full forward, last-position logits "
                            "all-gathered over NCCL at N>1) -> host"},
            "gpu_launches": r["launches"],
            "cpu_baseline": cpu,
            "decode": r["dec"],
            "extras": dict(r["extras"] or {}, **({"cfg5_xl": r["xl"]} if r["xl"] else {})),
            "clocks": r["clk"],
        }
        print(json.dumps(line), flush=True)
    if world > 1:
        dist.barrier()
        dist.destroy_process_group()


if __name__ == "__main__":
    main()
