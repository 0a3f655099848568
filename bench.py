#!/usr/bin/env python
"""KV-cache block save/load throughput on B200 (one process per GPU).

Workload (default, BASELINE config 3 at TP=N): Llama-3-70B-shaped paged KV,
80 layers of KV-first [2, 4096, 16, 8/N, 128] bf16 ~N(0,1) per rank, each of
the N ranks holding its own slice of the 8 KV heads on its own GPU; 2,048
blocks (one 32,768-token prefix) saved from seeded-shuffled ids into the
rank's pinned pool region and restored into 2,048 other ids. At N=1 this is
TP1 of the same config. Seeded synthetic data; no collective on the data path.
`--workload llama8b` runs BASELINE config 1 (32 layers x 640 blocks) instead.

One step = save of the blocks x layers + load of them back.
  value : payload GB/s of all ranks (save + load bytes / time) of the transfer
          executor, device-timed with CUDA events on the calling stream, the
          slowest rank's time.
  e2e   : the same through the engine API (PegaEngine.batch_save_kv_blocks +
          batch_load_kv_blocks + LoadState completion), host wall clock.
  verified : every restored block equals its source bit for bit, on every rank
          (destinations are zeroed before each timed region).
Also reported: save/load split, p50 load ms, host-link peaks (each GPU alone
and all at once) and fractions, the pack/unpack kernel HBM roofline, the other
block order, configs[1] in both orders (N=1), a P/D NVLink handoff check
(N>=2), the reference's own copy strategy timed on the same GPU, and a CPU
gather/scatter baseline.

--impl reference: the reference's CPU implementation of the path (the oracle
port of its copies, multi-threaded) on this host's cores over the whole job
(all N head shards); rank 0 only.
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
from pathlib import Path

import numpy as np

ROOT = Path(__file__).resolve().parent
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))

METRIC = "KV save/load GB/s per GPU at 1/2/4/8 B200 vs host-link roofline; p50 load ms"

WORKLOADS = {
    # BASELINE config 1
    "llama8b": dict(layers=32, num_blocks=8192, heads=8, head_dim=128, block_size=16, blocks=640,
                    desc="Llama-3.1-8B layer-wise offload: 32 layers, KV-first [2,8192,16,8,128] bf16, 640 blocks"),
    # BASELINE config 3 at TP=t (t = world size): each rank holds 8/t heads
    "llama70b_tp": dict(layers=80, num_blocks=4096, heads=8, head_dim=128, block_size=16, blocks=2048, tp=True,
                        desc="Llama-3-70B TP sharding: 80 layers, [2,4096,16,8/t,128] bf16, 2048 blocks per rank"),
    # BASELINE config 0 (separate K and V tensors, segments=1)
    "gpt2": dict(layers=24, num_blocks=256, heads=12, head_dim=64, block_size=16, blocks=64, separate=True,
                 desc="GPT-2-small: 12 layers x separate K,V [256,16,12,64] fp16, 64 blocks"),
}


def log(*a):
    print(*a, file=sys.stderr, flush=True)


# ----------------------------------------------------------------------------- clocks


class ClockSampler:
    """nvidia-smi clock / throttle sampling during the timed region."""

    QUERY = ("index,clocks.sm,clocks.max.sm,power.draw,clocks_event_reasons.active,"
             "clocks_event_reasons.hw_slowdown,clocks_event_reasons.hw_thermal_slowdown,"
             "clocks_event_reasons.sw_thermal_slowdown,clocks_event_reasons.sw_power_cap")

    def __init__(self, index: int):
        self.index = index
        self.proc = None
        self.lines: list[str] = []

    def start(self):
        try:
            self.proc = subprocess.Popen(
                ["nvidia-smi", "-i", str(self.index), f"--query-gpu={self.QUERY}", "--format=csv,noheader,nounits",
                 "-lms", "100"], stdout=subprocess.PIPE, stderr=subprocess.DEVNULL, text=True)
            self._t = threading.Thread(target=self._read, daemon=True)
            self._t.start()
        except OSError:
            self.proc = None

    def _read(self):
        for line in self.proc.stdout:
            self.lines.append(line.strip())

    def stop(self) -> dict:
        if self.proc is None:
            return {"sm_mhz": None, "sm_max_mhz": None, "reasons": ["nvidia-smi unavailable"]}
        time.sleep(0.25)
        self.proc.terminate()
        try:
            self.proc.wait(timeout=5)
        except subprocess.TimeoutExpired:
            self.proc.kill()
        sm, smax, reasons = [], None, set()
        names = ["hw_slowdown", "hw_thermal_slowdown", "sw_thermal_slowdown", "sw_power_cap"]
        for line in self.lines:
            f = [x.strip() for x in line.split(",")]
            if len(f) < 9:
                continue
            try:
                sm.append(float(f[1]))
                smax = float(f[2])
            except ValueError:
                continue
            for n, v in zip(names, f[5:9]):
                if v.lower() == "active":
                    reasons.add(n)
        return {"sm_mhz": statistics.median(sm) if sm else None, "sm_max_mhz": smax, "reasons": sorted(reasons),
                "samples": len(sm)}


# ----------------------------------------------------------------------------- helpers


def measured_peaks() -> dict:
    p = ROOT / "MEASURED_PEAKS.json"
    if p.exists():
        d = json.loads(p.read_text())
        return {"hbm_gbs": d["hbm_gbs"], "source": "measured"}
    return {"hbm_gbs": 6650.0, "source": "fallback"}


# DRAM traffic of one pack or unpack launch, from one ncu capture of
# dram__bytes_read.sum / dram__bytes_write.sum of the bulk kernel on 128 MiB
# (pack) and 160 MiB (unpack) chunks, larger than L2; not a per-run
# measurement. Reads equal the payload (no re-reads). Writes still in the
# 126 MB L2 when a launch ends (about 50 MB, whatever the chunk size) reach
# DRAM after it, so a launch's write traffic is its payload less that.
TRAFFIC_READ_PER_BYTE = (134_253_056 + 167_813_120) / (134_217_728 + 167_772_160)
TRAFFIC_WRITE_RESIDUE = ((134_217_728 - 81_046_272) + (167_772_160 - 118_041_088)) / 2


def traffic_per_launch(kernel_bytes_per_launch: float) -> int:
    """ncu-measured DRAM traffic model applied to the average launch
    (payload = half the algorithmic bytes: each payload byte is read once and
    written once)."""
    payload = kernel_bytes_per_launch / 2
    return round(payload * TRAFFIC_READ_PER_BYTE + max(0.0, payload - TRAFFIC_WRITE_RESIDUE))


def link_peaks(torch, device: int, barrier=None) -> dict:
    """Pinned host<->device copy-engine bandwidth with 1 GiB buffers (best of
    3). With `barrier` (one process per GPU), every rank copies at the same
    time, so the figure is this GPU's share of the host link while all GPUs
    use it: the denominator the transfers of a multi-GPU run compete for."""
    n = 1 << 30
    host = torch.empty(n, dtype=torch.uint8, pin_memory=True)
    dev = torch.empty(n, dtype=torch.uint8, device=device)
    out = {}
    s = torch.cuda.Stream(device)
    for name, fn in (("h2d", lambda: dev.copy_(host, non_blocking=True)),
                     ("d2h", lambda: host.copy_(dev, non_blocking=True))):
        best = 0.0
        with torch.cuda.stream(s):
            fn()
            for _ in range(3):
                s.synchronize()
                if barrier:
                    barrier()
                a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
                a.record(s)
                fn()
                b.record(s)
                b.synchronize()
                best = max(best, n / (a.elapsed_time(b) / 1e3) / 1e9)
        out[name] = round(best, 2)
    del host, dev
    return out


def duplex_peak(torch, device: int) -> float:
    """Pinned copies in both directions at once: 1 GiB D2H and 1 GiB H2D on
    two streams from one start event to both ends (best of 3), total GB/s."""
    n = 1 << 30
    h_out = torch.empty(n, dtype=torch.uint8, pin_memory=True)
    h_in = torch.empty(n, dtype=torch.uint8, pin_memory=True)
    d_out = torch.empty(n, dtype=torch.uint8, device=device)
    d_in = torch.empty(n, dtype=torch.uint8, device=device)
    s1, s2 = torch.cuda.Stream(device), torch.cuda.Stream(device)
    best = 0.0
    for _ in range(4):
        torch.cuda.synchronize(device)
        start, end, other = (torch.cuda.Event(enable_timing=True) for _ in range(3))
        start.record(s1)
        s2.wait_event(start)
        with torch.cuda.stream(s1):
            h_out.copy_(d_out, non_blocking=True)
        with torch.cuda.stream(s2):
            d_in.copy_(h_in, non_blocking=True)
        other.record(s2)
        s1.wait_event(other)
        end.record(s1)
        end.synchronize()
        best = max(best, 2 * n / (start.elapsed_time(end) / 1e3) / 1e9)
    del h_out, h_in, d_out, d_in
    return round(best, 2)


def aligned_rates(torch, stream, fn, nbytes: int, barrier, reps: int = 3) -> float:
    """GB/s of `fn` (work enqueued on `stream`) started on every rank at once;
    median of `reps`, device-timed on the stream."""
    vals = []
    for _ in range(reps):
        stream.synchronize()
        barrier()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record(stream)
        fn()
        b.record(stream)
        b.synchronize()
        vals.append(nbytes / (a.elapsed_time(b) / 1e3) / 1e9)
    return statistics.median(vals)


def make_workload(torch, wl: dict, device: int, rank: int, world: int, order: str):
    """KV tensors on the GPU plus seeded src/dst block lists. For the TP
    workload each rank holds its own slice of the KV heads."""
    from pegaflow_b200.ranks import block_lists, tp_heads

    if wl.get("tp"):
        lo, hi = tp_heads(wl["heads"], rank, world)
        heads = hi - lo
    else:
        heads = wl["heads"]
    nb, bs, hd = wl["num_blocks"], wl["block_size"], wl["head_dim"]
    gen = torch.Generator(device=f"cuda:{device}").manual_seed(1000 + rank)
    tensors = []
    for _ in range(wl["layers"]):
        shape = (nb, bs, heads, hd) if wl.get("separate") else (2, nb, bs, heads, hd)
        dt = torch.float16 if wl.get("separate") else torch.bfloat16
        tensors.append(torch.randn(shape, generator=gen, device=f"cuda:{device}", dtype=torch.float32).to(dt))
    src, dst = block_lists(nb, wl["blocks"], rank, order)
    return tensors, src, dst


def executor_specs(tensors, src, dst, pool_ptr):
    from pegaflow_b200 import Layout, LoadSpec, SaveSpec

    saves, loads = [], []
    off = 0
    n = len(src)
    for t in tensors:
        lay = Layout.from_tensor(t)
        if lay.split:
            k, v = pool_ptr + off, pool_ptr + off + n * lay.bytes_per_block
            unit = lay.bytes_per_block
            off += 2 * n * unit
            ks = np.arange(n, dtype=np.uint64) * unit + k
            saves.append(SaveSpec(lay, src, k, v))
            loads.append(LoadSpec(lay, dst, ks, ks + (v - k)))
        else:
            unit = lay.block_size_bytes
            k = pool_ptr + off
            off += n * unit
            ks = np.arange(n, dtype=np.uint64) * unit + k
            saves.append(SaveSpec(lay, src, k, None))
            loads.append(LoadSpec(lay, dst, ks, None))
        off = (off + 4095) // 4096 * 4096
    return saves, loads, off


def duplex_block(torch, ex, tensors, src, dst, payload: int, steps: int, device: int, serial_gbps: float) -> dict:
    """Save and load at once on one GPU, same tensors and executor as the
    serial step: the source blocks are saved into pool region A on one stream
    (the executor's save lane) while blocks saved earlier are restored from
    region B on another (its load lane), as when a prefill's offload overlaps
    another request's restore. Source and destination ids are disjoint. The
    destination blocks are zeroed and region A cleared after the warm-up, so
    the checks see only what the timed steps moved."""
    from pegaflow_b200 import PinnedBuffer

    peak = duplex_peak(torch, device)
    half = (payload + len(tensors) * 8192 + (1 << 20) + 4095) // 4096 * 4096
    pool2 = PinnedBuffer(2 * half, write_combined=True)
    saves_a, _, _ = executor_specs(tensors, src, dst, pool2.ptr)
    saves_b, loads_b, _ = executor_specs(tensors, src, dst, pool2.ptr + half)
    a, b = torch.cuda.Stream(device), torch.cuda.Stream(device)
    ex.save(saves_b, stream=a.cuda_stream)  # region B now holds the source blocks
    a.synchronize()

    def one():
        e0, e1, eb = (torch.cuda.Event(enable_timing=True) for _ in range(3))
        e0.record(a)
        b.wait_event(e0)
        ex.save(saves_a, stream=a.cuda_stream)
        ex.load(loads_b, stream=b.cuda_stream)
        eb.record(b)
        a.wait_event(eb)
        e1.record(a)
        return e0, e1

    for _ in range(2):
        one()
    torch.cuda.synchronize(device)
    scribble(torch, tensors, dst)
    pool2.numpy()[:half] = 0
    torch.cuda.synchronize(device)
    evs = [one() for _ in range(steps)]
    torch.cuda.synchronize(device)
    ms = statistics.median(x.elapsed_time(y) for x, y in evs)
    gbps = 2 * payload / (ms / 1e3) / 1e9
    verified = restored(torch, tensors, src, dst) and pool_matches(torch, tensors, saves_a, pool2, src)
    pool2.close()
    return {"GBps": round(gbps, 3), "ms_per_step": round(ms, 3), "steps": steps,
            "vs_serial": round(gbps / serial_gbps, 3) if serial_gbps else None,
            "peak_duplex_GBps": peak, "frac_of_duplex_peak": round(gbps / peak, 3) if peak else None,
            "verified": verified,
            "how": "the same save and load as the serial step, on two streams at once (save lane: source "
                   "blocks into pool region A; load lane: region B into the destination blocks); median "
                   "device time per step; peak_duplex: a 1 GiB pinned D2H and a 1 GiB H2D at once"}


def payload_bytes(tensors, n) -> int:
    from pegaflow_b200 import Layout

    total = 0
    for t in tensors:
        lay = Layout.from_tensor(t)
        total += n * (2 * lay.bytes_per_block if lay.split else lay.block_size_bytes)
    return total


# ----------------------------------------------------------------------------- CPU arms


class CpuWorkload:
    """Oracle port of the reference's copies (multi-threaded memcpy gather and
    scatter) on host-resident buffers with the workload's layout: a bounded
    sample of `max_layers` layers of every TP shard (`world` shards of
    heads/world KV heads each, with each rank's own block lists).

    `pool` picks the memory the pool regions live in: "malloc" (cacheable
    pages), "pinned" (page-locked, cacheable) or "pinned_wc" (page-locked and
    write-combined, the reference's pool memory, pinned_mem.rs:159, which the
    CPU reads uncached)."""

    def __init__(self, wl: dict, threads: int, max_layers: int = 8, pool: str = "malloc", world: int = 1,
                 order: str = "shuffled"):
        from oracle import oracle
        from pegaflow_b200.ranks import block_lists

        self.oracle = oracle
        oracle.build()
        self.threads = threads
        self._keep = []
        L = min(wl["layers"], max_layers)
        nb, bs, hd = wl["num_blocks"], wl["block_size"], wl["head_dim"]
        shards = world if wl.get("tp") else 1
        heads = wl["heads"] // shards
        seg = bs * heads * hd * 2
        n = wl["blocks"]

        def region(nbytes):
            if pool == "malloc":
                return np.zeros(nbytes, np.uint8)
            from pegaflow_b200 import PinnedBuffer

            buf = PinnedBuffer(nbytes, write_combined=pool == "pinned_wc")
            self._keep.append(buf)
            arr = buf.numpy()
            arr[::4096] = 0
            return arr

        self.saves, self.loads = [], []
        for r in range(shards):
            src, dst = block_lists(nb, n, r, order)
            for i in range(L):
                lay = oracle.Layout(nb * seg, nb, seg, 0, 1) if wl.get("separate") else \
                    oracle.Layout(2 * nb * seg, nb, seg, nb * seg, 2)
                cache = np.empty(lay.size_bytes, np.uint8)
                cache[::4096] = i  # fault every page in before timing
                kp = region(n * seg)
                vp = region(n * seg) if lay.split else None
                self.saves.append((lay, cache, src, kp, vp))
                self.loads.append((lay, cache, dst, kp, vp))
        shard_txt = f"{shards} TP shards x " if shards > 1 else ""
        self.sample = (f"{shard_txt}{L} of {wl['layers']} layers x {n} blocks ({order} ids; save + load), "
                       f"host-resident buffers, pool: {pool}")

    def close(self) -> None:
        for b in self._keep:
            b.close()
        self._keep.clear()

    def step(self) -> int:
        moved = self.oracle.mt_transfer(self.saves, True, self.threads)
        moved += self.oracle.mt_transfer(self.loads, False, self.threads)
        return moved

    def rate(self, seconds: float) -> dict:
        self.step()
        moved, reps = 0, 0
        t0 = time.perf_counter()
        while True:
            moved += self.step()
            reps += 1
            el = time.perf_counter() - t0
            if el >= seconds:
                break
        return {"value": round(moved / el / 1e9, 3), "unit": "GB/s", "cores": self.threads, "kind": "port",
                "sample": f"{self.sample}, {reps} reps in {el:.1f} s"}


def run_reference_arm(args, wl) -> None:
    """The reference's CPU implementation of the path (the oracle port of its
    copies) on every host core, over the whole job: at N GPUs of the TP
    workload, all N head shards, so its GB/s compares with the b200 arm's
    whole-job value. Rank 0 alone runs; the other ranks exit at once."""
    rank = int(os.environ.get("RANK", "0"))
    if rank != 0:
        return
    threads = os.cpu_count() or 1
    cw = CpuWorkload(wl, threads, world=args.gpus, order=args.order)
    for _ in range(args.warmup):
        cw.step()
    times, vals = [], []
    for _ in range(args.steps):
        t0 = time.perf_counter()
        moved = cw.step()
        el = time.perf_counter() - t0
        times.append(el * 1e3)
        vals.append(moved / el / 1e9)
    value = round(statistics.median(vals), 3)
    line = {
        "impl": "reference", "metric": METRIC, "value": value, "unit": "GB/s", "n_gpus": args.gpus,
        "steps": args.steps, "warmup": args.warmup, "ms_per_step": round(statistics.median(times), 3),
        "higher_is_better": True, "scaling": "weak", "vs_baseline": None, "dtype": "u8",
        "data": "synthetic (host-resident, seeded block lists)", "config": config_block(args, wl, args.gpus),
        "cpu_baseline": {"value": value, "unit": "GB/s", "cores": threads, "kind": "port", "sample": cw.sample},
        "e2e": {"value": value, "unit": "GB/s", "h2d_bytes_per_step": 0, "d2h_bytes_per_step": 0},
        "note": "the reference path is Rust over cudarc copies with no CPU implementation and cannot be built "
                "here (no Rust toolchain); this arm times the oracle port of its copy algorithm on host cores",
    }
    print(json.dumps(line), flush=True)


def run_pd(args) -> None:
    """Qwen3-8B-shaped prefill -> decode handoff in one
    process over two GPUs. 36 layers of KV-first [2, 2048, 16, 8, 128] bf16 on
    each GPU; 200 requests x 313 blocks, each moved from seeded block ids on
    GPU0 into seeded free ids on GPU1. Three ways: NVLink P2P pull (kernel on
    GPU1 reads GPU0), P2P push (kernel on GPU0 writes GPU1), and the host-pool
    bounce (save on GPU0 + load on GPU1). Device-timed per request."""
    import torch

    from pegaflow_b200 import Executor, Layout, LoadSpec, P2PSpec, PinnedBuffer, SaveSpec

    if torch.cuda.device_count() < 2:
        print(json.dumps({"metric": METRIC, "workload": "qwen3_pd", "unavailable": "needs 2 GPUs in one process"}))
        return
    layers, nb, n, requests = 36, 2048, 313, args.pd_requests
    g0 = torch.Generator(device="cuda:0").manual_seed(7)
    g1 = torch.Generator(device="cuda:1").manual_seed(8)
    src = [torch.randn((2, nb, 16, 8, 128), generator=g0, device="cuda:0").to(torch.bfloat16) for _ in range(layers)]
    dst = [torch.randn((2, nb, 16, 8, 128), generator=g1, device="cuda:1").to(torch.bfloat16) for _ in range(layers)]
    reqs = [(np.random.default_rng(4 + r).permutation(nb)[:n], np.random.default_rng(10_000 + r).permutation(nb)[:n])
            for r in range(requests)]
    payload = n * layers * 2 * 32768
    ex0, ex1 = Executor(0), Executor(1)
    s0, s1 = torch.cuda.Stream("cuda:0"), torch.cuda.Stream("cuda:1")
    sl, dl = [Layout.from_tensor(t) for t in src], [Layout.from_tensor(t) for t in dst]

    # Peer copy peak (1 GiB, best of 3) for the NVLink roofline.
    a = torch.empty(1 << 30, dtype=torch.uint8, device="cuda:0")
    b = torch.empty(1 << 30, dtype=torch.uint8, device="cuda:1")
    peak = 0.0
    for _ in range(4):
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        with torch.cuda.stream(s1):
            e0.record(s1)
            b.copy_(a, non_blocking=True)
            e1.record(s1)
        e1.synchronize()
        peak = max(peak, (1 << 30) / (e0.elapsed_time(e1) / 1e3) / 1e9)
    del a, b

    def timed(fn, stream, reps):
        ms = []
        for r in range(reps):
            e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            e0.record(stream)
            fn(r, stream)
            e1.record(stream)
            ms.append((e0, e1))
        torch.cuda.synchronize(0)
        torch.cuda.synchronize(1)
        return [x.elapsed_time(y) for x, y in ms]

    def pull(r, stream):
        si, di = reqs[r]
        ex1.p2p([P2PSpec(x, y, si, di) for x, y in zip(sl, dl)], 0, push=False, stream=stream.cuda_stream)

    def push(r, stream):
        si, di = reqs[r]
        ex0.p2p([P2PSpec(x, y, si, di) for x, y in zip(sl, dl)], 1, push=True, stream=stream.cuda_stream)

    # Two pool regions: the pipelined bounce saves request r+1 on GPU0 while
    # GPU1 still loads request r.
    region = payload + layers * 4096
    pool = PinnedBuffer(2 * region, write_combined=True)
    saves, loads = [[], []], [[], []]
    for half in (0, 1):
        off = half * region
        for x, y in zip(sl, dl):
            k, v = pool.ptr + off, pool.ptr + off + n * 32768
            ks = np.arange(n, dtype=np.uint64) * 32768 + k
            saves[half].append((x, k, v))
            loads[half].append((y, ks, ks + n * 32768))
            off += 2 * n * 32768 + 4096

    def bounce(r, stream):
        si, di = reqs[r]
        go = torch.cuda.Event()
        go.record(stream)  # the save starts after the request's start event
        s0.wait_event(go)
        ex0.save([SaveSpec(x, si, k, v) for x, k, v in saves[0]], stream=s0.cuda_stream)
        ev = torch.cuda.Event()
        ev.record(s0)
        stream.wait_event(ev)
        ex1.load([LoadSpec(y, di, ks, vs) for y, ks, vs in loads[0]], stream=stream.cuda_stream)

    def bounce_pipelined(reps):
        """Saves run ahead on GPU0 (one region ahead); each load on GPU1 waits
        for its own save. Returns ms from the first save to the last load."""
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record(s1)
        s0.wait_event(start)
        saved, loaded = [], []
        for r in range(reps):
            si, di = reqs[r]
            if r >= 2:
                s0.wait_event(loaded[r - 2])  # its pool region is free again
            ex0.save([SaveSpec(x, si, k, v) for x, k, v in saves[r % 2]], stream=s0.cuda_stream)
            saved.append(torch.cuda.Event())
            saved[-1].record(s0)
            s1.wait_event(saved[-1])
            ex1.load([LoadSpec(y, di, ks, vs) for y, ks, vs in loads[r % 2]], stream=s1.cuda_stream)
            loaded.append(torch.cuda.Event())
            loaded[-1].record(s1)
        end.record(s1)
        end.synchronize()
        return start.elapsed_time(end)

    for fn in (pull, push, bounce):
        timed(fn, s1 if fn is not push else s0, min(3, requests))
    res = {}
    for name, fn, st in (("p2p_pull", pull, s1), ("p2p_push", push, s0), ("host_pool", bounce, s1)):
        reps = requests if name != "host_pool" else min(requests, args.pd_bounce_requests)
        ms = timed(fn, st, reps)
        res[name] = {"GBps": round(payload * reps / (sum(ms) / 1e3) / 1e9, 2),
                     "p50_request_ms": round(statistics.median(ms), 3), "requests": reps}
    reps = min(requests, args.pd_bounce_requests)
    bounce_pipelined(2)
    res["host_pool"]["pipelined_GBps"] = round(payload * reps / (bounce_pipelined(reps) / 1e3) / 1e9, 2)
    res["host_pool"]["how"] = ("GBps and p50: one request at a time (save on GPU0, then load on GPU1); "
                               "pipelined_GBps: saves run one request ahead of loads, two pool regions")
    best = max(("p2p_pull", "p2p_push"), key=lambda k: res[k]["GBps"])
    line = {
        "metric": METRIC, "value": res[best]["GBps"], "unit": "GB/s", "n_gpus": 2, "steps": requests,
        "warmup": 3, "ms_per_step": res[best]["p50_request_ms"], "higher_is_better": True, "scaling": "none",
        "vs_baseline": None, "dtype": "u8", "data": "synthetic (seeded ~N(0,1) bf16 KV)",
        "config": {"workload": "qwen3_pd", "desc": "Qwen3-8B P/D handoff: 36 layers, [2,2048,16,8,128] bf16 per GPU, "
                   f"{requests} requests x 313 blocks, GPU0 -> GPU1", "payload_bytes_per_request": payload},
        "best": best, "p2p_pull": res["p2p_pull"], "p2p_push": res["p2p_push"], "host_pool_bounce": res["host_pool"],
        "nvlink": {"peer_copy_peak_GBps": round(peak, 1), "frac": round(res[best]["GBps"] / peak, 3),
                   "how": "1 GiB cudaMemcpyPeer GPU0->GPU1, best of 4"},
        "gpu_launches": ex0.stats()["kernel_launches"] + ex1.stats()["kernel_launches"],
    }
    print(json.dumps(line), flush=True)


def run_fp8_evict(args) -> None:
    print(json.dumps(fp8_evict_result(args)), flush=True)


def fp8_evict_result(args) -> dict:
    """mixed warm/cold restore under eviction, through the
    engine API. Llama-3.1-8B shape with fp8 (e4m3 bit patterns) KV, 32 layers
    [2, 2048, 16, 8, 128] uint8 plus one fp32 scale per block per layer (32
    more layers [2048] fp32, 4-byte units); 64 requests with prefixes of
    U[1K, 16K] tokens (seed 6), the first half of each request's blocks saved
    beforehand; 30 GB pool with LRU eviction (admission off). Per request: the
    warm prefix is restored layer by layer while a dummy per-layer compute
    kernel (0.5 ms) runs on a second stream as soon as its layer is in place,
    then the cold half is saved. Compared with waiting for the whole load
    before computing.

    With ``--fp8-compute attention`` the compute of a layer is what a model does
    there: the request's new tokens (up to 2,048) are quantised into their blocks
    and attend, 32 query heads on 8, over the restored prefix and themselves."""
    import torch

    from pegaflow_b200 import Layout, PegaEngine, PyLoadState

    torch.cuda.set_device(0)
    layers, nb, n_req = 32, 2048, args.fp8_requests
    rng = np.random.default_rng(6)
    lens = rng.integers(1024, 16385, size=n_req)
    blocks_per_req = [int(x) // 16 for x in lens]
    g = torch.Generator(device="cuda:0").manual_seed(0)
    kv = [torch.randint(0, 256, (2, nb, 16, 8, 128), generator=g, device="cuda:0", dtype=torch.uint8)
          for _ in range(layers)]
    sc = [torch.rand((nb,), generator=g, device="cuda:0", dtype=torch.float32) for _ in range(layers)]
    attend = args.fp8_compute == "attention"
    if attend:
        from pegaflow_b200 import KVCache, chunk_attention, kv_write

        # Codes of normal values (random bit patterns hold NaNs) at scales that make them about 1.
        for t, s in zip(kv, sc):
            t.copy_((torch.randn((nb, 16, 8, 128), generator=g, device="cuda:0") * 100).to(torch.float8_e4m3fn)
                    .view(torch.uint8))
            s.mul_(0.01).add_(0.005)
        caches = [KVCache.from_tensor(t, s) for t, s in zip(kv, sc)]
        new_kv = torch.randn((2, 2048, 8, 128), generator=g, device="cuda:0").to(torch.bfloat16)
        query = torch.randn((2048, 32, 128), generator=g, device="cuda:0").to(torch.bfloat16)
    # Forward order, each layer's KV next to its scales: a load restores its
    # layers in the order the request lists them, so layer i is usable once
    # entries 2i and 2i+1 are in place.
    names, tensors = [], []
    for i in range(layers):
        names += [f"model.layers.{i}.attn", f"model.layers.{i}.attn.scale"]
        tensors += [kv[i], sc[i]]
    pool = args.fp8_pool_gb << 30
    per_block = layers * (2 * 16 * 8 * 128 + 4)

    def hashes(r, lo, hi):
        return [f"req{r}-blk{i}".encode() for i in range(lo, hi)]

    def ids_for(r, count):
        return np.random.default_rng(1000 + r).permutation(nb)[:count].tolist()

    def fresh_engine():
        e = PegaEngine(pool, enable_lfu_admission=False)
        for nm, t in zip(names, tensors):
            lay = Layout.from_tensor(t)
            e.register_context_layer("fp8", "ns", 0, nm, lay.data_ptr, lay.size_bytes, lay.num_blocks,
                                     lay.bytes_per_block, lay.kv_stride_bytes, lay.segments, 0, 1, len(names))
        # Warm half of every request, saved beforehand (the pool overflows later).
        for r in range(n_req):
            half = blocks_per_req[r] // 2
            e.batch_save_kv_blocks("fp8", 0, 0, [(nm, ids_for(r, half), hashes(r, 0, half)) for nm in names])
        return e

    compute = torch.cuda.Stream("cuda:0")
    cycles = int(args.fp8_compute_ms * 1e-3 * 1.9e9)

    def wait_ready(state, timeout=120.0):
        deadline = time.perf_counter() + timeout
        while not state.is_ready():
            if time.perf_counter() > deadline:
                raise TimeoutError("load did not complete")

    def chunk_of(hit, dst):
        """The request's new tokens: their slots, and what attention needs to know (made once, for all layers)."""
        n = min((len(dst) - hit) * 16, 2048)
        pos = torch.arange(hit * 16, hit * 16 + n)
        ids = torch.tensor(dst)
        with torch.cuda.stream(compute):
            return (n, hit * 16 + n, (ids[pos // 16] * 16 + pos % 16).cuda(), ids.to(torch.int32).view(1, -1).cuda(),
                    torch.tensor([0, n], dtype=torch.int32).cuda(),
                    torch.tensor([hit * 16 + n], dtype=torch.int32).cuda())

    def compute_layer(li, chunk):
        if not attend:
            torch.cuda._sleep(cycles)
            return
        n, total, slots, table, q_start, kv_len = chunk
        kv_write(caches[li], new_kv[0, :n], new_kv[1, :n], slots, given_scales=True)
        chunk_attention(query[:n], caches[li], table, q_start, kv_len, max_q=n, max_kv=total)

    def serve(r, overlap):
        nblk = blocks_per_req[r]
        hs_all = hashes(r, 0, nblk)
        hit = eng.count_prefix_hit_blocks("fp8", hs_all)
        dst = ids_for(50_000 + r, nblk)
        chunk = chunk_of(hit, dst) if attend else None
        t0 = time.perf_counter()
        state = PyLoadState(len(names))
        if hit:
            eng.batch_load_kv_blocks("fp8", 0, 0, state.shm_name(), names, dst[:hit], hs_all[:hit])
        else:
            state.set_completed()
        for li in range(layers):
            if hit and overlap:
                if not (state.wait_layer(2 * li, 60) and state.wait_layer(2 * li + 1, 60)):
                    raise RuntimeError("layer load failed")
            elif hit and li == 0:
                wait_ready(state)
            with torch.cuda.stream(compute):
                compute_layer(li, chunk)
        t_issue = time.perf_counter()
        wait_ready(state)
        load_done = time.perf_counter()
        compute.synchronize()
        t_end = time.perf_counter()
        if state.get_state() != 1:
            raise RuntimeError("load failed")
        cold = hashes(r, hit, nblk)
        if cold:
            eng.batch_save_kv_blocks("fp8", 0, 0, [(nm, dst[hit:], cold) for nm in names])
        return hit, (load_done - t0) * 1e3, (t_end - t0) * 1e3, (t_issue - t0) * 1e3

    out = {}
    for mode in ("overlap", "serial"):
        eng = fresh_engine()  # the same starting cache for both modes
        with torch.cuda.stream(compute):
            torch.cuda._sleep(cycles)  # warm the compute stream
        compute.synchronize()
        rows = [serve(r, mode == "overlap") for r in range(n_req)]
        if mode == "overlap":
            m = eng.metrics()
        eng.close()
        hit_blocks = sum(x[0] for x in rows)
        load_ms = [x[1] for x in rows if x[0]]
        total = sum(x[2] for x in rows)
        out[mode] = {"requests": n_req, "hit_blocks": hit_blocks, "p50_load_ms": round(statistics.median(load_ms), 3),
                     "load_GBps": round(hit_blocks * per_block / (sum(load_ms) / 1e3) / 1e9, 2),
                     "request_ms_p50": round(statistics.median(x[2] for x in rows), 3),
                     "total_s": round(total / 1e3, 3)}
    line = {
        "metric": METRIC, "value": out["overlap"]["load_GBps"], "unit": "GB/s", "n_gpus": 1, "steps": n_req,
        "warmup": 0, "ms_per_step": out["overlap"]["request_ms_p50"], "higher_is_better": True, "scaling": "none",
        "vs_baseline": None, "dtype": "u8", "data": "synthetic (seeded e4m3 bit patterns + fp32 scales)",
        "config": {"workload": "llama8b_fp8_evict", "layers": "32 KV + 32 scale", "pool_gb": args.fp8_pool_gb,
                   "requests": n_req, "prefix_tokens": "U[1024,16384] seed 6", "warm_fraction": 0.5,
                   "compute_ms_per_layer": args.fp8_compute_ms if not attend else
                   "attention of up to 2048 new tokens, 32 heads on 8"},
        "layerwise_overlap": out["overlap"], "load_then_compute": out["serial"],
        "overlap_speedup": round(out["serial"]["total_s"] / out["overlap"]["total_s"], 3),
        "engine": {k: m[k] for k in ("cache_block_evictions", "cache_block_hits", "cache_block_misses",
                                     "pool_alloc_failures", "load_failures", "cached_blocks")},
    }
    return line


def run_duplex(args) -> None:
    """Save and load at once on one GPU (a prefill saving its KV while another
    request's prefix is restored). Llama-3.1-8B shape (32 layers of KV-first
    [2, 8192, 16, 8, 128] bf16); one seeded permutation gives 640 block ids to
    save and 640 other ids to restore into, so the two transfers touch
    disjoint blocks. Executor: the save on one stream and the load on another
    (the executor's save and load lanes), against the same two back to back on
    one stream. Engine: a queued batch_load_kv_blocks of the previous step's
    hashes while batch_save_kv_blocks stores this step's."""
    import torch

    from pegaflow_b200 import Executor, Layout, PegaEngine, PinnedBuffer, PyLoadState

    torch.cuda.set_device(0)
    wl = dict(WORKLOADS["llama8b"])
    if args.layers:
        wl["layers"] = args.layers
    nb, n = wl["num_blocks"], wl["blocks"]
    gen = torch.Generator(device="cuda:0").manual_seed(1000)
    tensors = [torch.randn((2, nb, 16, 8, 128), generator=gen, device="cuda:0", dtype=torch.float32)
               .to(torch.bfloat16) for _ in range(wl["layers"])]
    perm = np.random.default_rng(5).permutation(nb)
    save_ids, load_ids = perm[:n].astype(np.int64), perm[n:2 * n].astype(np.int64)
    payload = payload_bytes(tensors, n)
    link = link_peaks(torch, 0)
    link["duplex"] = duplex_peak(torch, 0)
    pool = PinnedBuffer(2 * payload + (4 << 20), write_combined=True)
    saves, _, off = executor_specs(tensors, save_ids, save_ids, pool.ptr)
    _, loads, _ = executor_specs(tensors, load_ids, load_ids, pool.ptr + off)
    ex = Executor(0, save_mode=args.save_mode, load_mode=args.load_mode, staging_chunk_bytes=args.chunk_mib << 20,
                  staging_slots=args.slots, copy_streams=args.copy_streams, first_chunk_bytes=args.first_chunk_mib << 20,
                  copy_kernel=args.copy_kernel)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()

    def timed(duplex):
        e0, e1, ea, eb = (torch.cuda.Event(enable_timing=True) for _ in range(4))
        e0.record(a)
        if duplex:
            b.wait_event(e0)
            ex.save(saves, stream=a.cuda_stream)
            ea.record(a)
            ex.load(loads, stream=b.cuda_stream)
            eb.record(b)
            a.wait_event(eb)
        else:
            ex.save(saves, stream=a.cuda_stream)
            ea.record(a)
            ex.load(loads, stream=a.cuda_stream)
            eb.record(a)
        e1.record(a)
        return e0, e1, ea, eb

    for _ in range(args.warmup):
        timed(True)
        timed(False)
    torch.cuda.synchronize()
    sampler = ClockSampler(0)
    sampler.start()
    res = {}
    for mode in ("serial", "duplex"):
        evs = [timed(mode == "duplex") for _ in range(args.steps)]
        torch.cuda.synchronize()
        ms = [x.elapsed_time(y) for x, y, _, _ in evs]
        # Each lane's end from the step's start (serial: the load ends after the save).
        save_end = [x.elapsed_time(s) for x, _, s, _ in evs]
        load_end = [x.elapsed_time(l) for x, _, _, l in evs]
        res[mode] = {"ms_per_step": round(statistics.median(ms), 3),
                     "GBps": round(2 * payload / (statistics.median(ms) / 1e3) / 1e9, 2),
                     "save_end_ms": round(statistics.median(save_end), 3),
                     "load_end_ms": round(statistics.median(load_end), 3)}
    clocks = sampler.stop()

    # Engine: this step's save runs while the previous step's blocks load.
    eng = PegaEngine(3 * payload + (512 << 20), enable_lfu_admission=False,
                     executor=dict(save_mode=args.save_mode, load_mode=args.load_mode,
                                   staging_chunk_bytes=args.chunk_mib << 20, staging_slots=args.slots,
                                   copy_streams=args.copy_streams, first_chunk_bytes=args.first_chunk_mib << 20,
                                   copy_kernel=args.copy_kernel))
    names = [f"model.layers.{i}.self_attn" for i in range(len(tensors))]
    for nm, t in zip(names, tensors):
        lay = Layout.from_tensor(t)
        eng.register_context_layer("dup", "bench", 0, nm, lay.data_ptr, lay.size_bytes, lay.num_blocks,
                                   lay.bytes_per_block, lay.kv_stride_bytes, lay.segments, 0, 1, len(names))
    sl, ll = save_ids.tolist(), load_ids.tolist()

    def hashes(k):
        return [f"dup-s{k}-b{i}".encode() for i in range(n)]

    def wait(state):
        deadline = time.perf_counter() + 120.0
        while not state.is_ready():
            if time.perf_counter() > deadline:
                raise TimeoutError("engine load did not complete within 120 s")
        if state.get_state() != 1:
            raise RuntimeError("engine load failed")

    def e2e_step(k, duplex):
        new, old = hashes(k), hashes(k - 1)  # one list per request, shared by its layers
        t0 = time.perf_counter()
        s = PyLoadState(len(names))
        if duplex:
            eng.batch_load_kv_blocks("dup", 0, 0, s.shm_name(), names, ll, old)
            eng.batch_save_kv_blocks("dup", 0, 0, [(nm, sl, new) for nm in names])
            wait(s)
        else:
            eng.batch_save_kv_blocks("dup", 0, 0, [(nm, sl, new) for nm in names])
            eng.batch_load_kv_blocks("dup", 0, 0, s.shm_name(), names, ll, old)
            wait(s)
        s.close()
        return time.perf_counter() - t0

    first = hashes(0)
    eng.batch_save_kv_blocks("dup", 0, 0, [(nm, sl, first) for nm in names])
    k = 1
    e2e = {}
    for mode in ("serial", "duplex"):
        for _ in range(args.warmup):
            e2e_step(k, mode == "duplex")
            k += 1
        times = []
        for _ in range(args.steps):
            times.append(e2e_step(k, mode == "duplex"))
            k += 1
        e2e[mode] = {"ms_per_step": round(statistics.median(times) * 1e3, 3),
                     "GBps": round(2 * payload * len(times) / sum(times) / 1e9, 2)}
    m = eng.metrics()
    eng.close()
    line = {
        "metric": METRIC, "value": res["duplex"]["GBps"], "unit": "GB/s", "n_gpus": 1, "steps": args.steps,
        "warmup": args.warmup, "ms_per_step": res["duplex"]["ms_per_step"], "higher_is_better": True,
        "scaling": "none", "vs_baseline": None, "dtype": "u8", "data": "synthetic (seeded ~N(0,1) bf16 KV)",
        "config": {"workload": "llama8b_duplex", "layers": wl["layers"], "num_blocks": nb, "blocks_saved": n,
                   "blocks_loaded": n, "block_ids": "one seeded permutation, disjoint save and load ids",
                   "l2": "inputs larger than L2"},
        "executor": res, "duplex_speedup": round(res["serial"]["ms_per_step"] / res["duplex"]["ms_per_step"], 3),
        "e2e": {"value": e2e["duplex"]["GBps"], "unit": "GB/s", "h2d_bytes_per_step": payload,
                "d2h_bytes_per_step": payload, "serial": e2e["serial"], "duplex": e2e["duplex"],
                "api": "batch_load_kv_blocks (queued) + batch_save_kv_blocks, then LoadState"},
        "host_link": {"peak_h2d_GBps": link["h2d"], "peak_d2h_GBps": link["d2h"],
                      "duplex_frac_of_sum": round(res["duplex"]["GBps"] / (link["h2d"] + link["d2h"]), 3),
                      "peak_duplex_GBps": link["duplex"],
                      "duplex_frac": round(res["duplex"]["GBps"] / link["duplex"], 3),
                      "how": "pinned 1 GiB copies, best of 3; peak_duplex: one D2H and one H2D at once"},
        "engine": {k2: (round(m[k2], 2) if isinstance(m[k2], float) else m[k2])
                   for k2 in ("load_failures", "cache_block_evictions", "pool_alloc_failures", "save_plan_ms",
                              "save_transfer_ms", "save_insert_ms", "save_ms", "load_ms")},
        "engine_calls": {"saves": 1 + 2 * (args.warmup + args.steps), "loads": 2 * (args.warmup + args.steps)},
        "clocks": clocks,
    }
    print(json.dumps(line), flush=True)


def run_one_engine(args) -> None:
    """The reference's deployment shape for BASELINE config 3: ONE engine
    (one server process) drives N GPUs into one shared pinned pool, as
    pegaflow-server does with its per-device workers (gpu_worker.rs:61-93).
    Each TP rank r registers its head shard on GPU r as tp_rank r of tp_size N
    (slot = layer * N + r, lib.rs:204-218), so a block becomes loadable only
    when every rank has saved it (storage.rs:161-193). One thread per rank
    calls the engine, as the server's RPC threads do; all ranks use the same
    block ids and hashes, as vLLM's TP workers share one block table. Per
    step: every rank saves at once, then every rank loads at once; wall clock
    per phase. Run as one process: python bench.py --workload
    llama70b_tp_one_engine --gpus N [--numa-pools node|device]."""
    import torch

    from pegaflow_b200 import Layout, PegaEngine, PyLoadState
    from pegaflow_b200.ranks import block_lists

    world = args.gpus
    if torch.cuda.device_count() < world:
        print(json.dumps({"metric": METRIC, "workload": "llama70b_tp_one_engine",
                          "unavailable": f"needs {world} GPUs in one process"}))
        return
    wl = dict(WORKLOADS["llama70b_tp"])
    if args.layers:
        wl["layers"] = args.layers
    src, dst = block_lists(wl["num_blocks"], wl["blocks"], 0, args.order)
    shards = [make_workload(torch, wl, d, d, world, args.order)[0] for d in range(world)]
    n = len(src)
    payload = payload_bytes(shards[0], n)  # per rank, per direction
    torch.cuda.synchronize()
    eng = PegaEngine(2 * world * payload + (512 << 20), enable_lfu_admission=False, numa_pools=args.numa_pools)
    names = [f"model.layers.{i}.self_attn" for i in range(wl["layers"])]
    for d in range(world):
        for nm, t in zip(names, shards[d]):
            lay = Layout.from_tensor(t)
            eng.register_context_layer("tp", "bench", d, nm, lay.data_ptr, lay.size_bytes, lay.num_blocks,
                                       lay.bytes_per_block, lay.kv_stride_bytes, lay.segments, d, world, len(names))
    src_l, dst_l = src.tolist(), dst.tolist()

    def phase(fn) -> float:
        errs = []

        def run(r):
            try:
                fn(r)
            except Exception as e:  # reported after the join
                errs.append(e)

        ths = [threading.Thread(target=run, args=(r,)) for r in range(world)]
        t0 = time.perf_counter()
        for th in ths:
            th.start()
        for th in ths:
            th.join()
        el = time.perf_counter() - t0
        if errs:
            raise errs[0]
        return el

    def one_step(k):
        hashes = [f"s{k}-b{i}".encode() for i in range(n)]
        t_save = phase(lambda r: eng.batch_save_kv_blocks("tp", r, r, [(nm, src_l, hashes) for nm in names]))
        assert eng.count_prefix_hit_blocks("tp", hashes) == n  # sealed: every rank's slots are filled

        def load(r):
            s = PyLoadState(len(names))
            eng.batch_load_kv_blocks("tp", r, r, s.shm_name(), names, dst_l, hashes)
            # Each rank's vLLM worker polls its LoadState in its own process;
            # here the ranks share one interpreter, so the wait blocks in the
            # library (GIL released) instead of spinning against the others.
            eng.wait_loads(r, 120.0)
            ok = s.get_state() == 1
            s.close()
            if not ok:
                raise RuntimeError(f"load of rank {r} failed")

        return t_save, phase(load)

    for k in range(args.warmup):
        one_step(-1 - k)
    for sh in shards:
        scribble(torch, sh, dst)
    torch.cuda.synchronize()
    m0 = eng.metrics()
    times = [one_step(k) for k in range(args.steps)]
    verified = all(restored(torch, sh, src, dst) for sh in shards)
    m = eng.metrics()
    # Per timed step, summed over the ranks' calls.
    phases = {k: round((m[k] - m0[k]) / len(times), 3)
              for k in ("save_plan_ms", "save_transfer_ms", "save_insert_ms", "load_lookup_ms", "load_queue_ms",
                        "load_setup_ms", "load_transfer_ms", "load_first_layer_ms")}
    eng.close()
    save_s = statistics.median(t for t, _ in times)
    load_s = statistics.median(t for _, t in times)
    total = sum(a + b for a, b in times)
    value = world * 2 * payload * len(times) / total / 1e9
    line = {
        "metric": METRIC, "value": round(value, 3), "unit": "GB/s", "n_gpus": world, "steps": args.steps,
        "warmup": args.warmup, "ms_per_step": round(total / len(times) * 1e3, 3), "higher_is_better": True,
        "scaling": "weak", "vs_baseline": None, "dtype": "u8", "data": "synthetic (seeded ~N(0,1) bf16 KV)",
        "config": dict(config_block(args, wl, world), workload="llama70b_tp_one_engine",
                       parallelism=f"tp{world} in one engine process (one thread per rank), one pool"
                                   + ("" if args.numa_pools == "off" else f" per NUMA {args.numa_pools}")),
        "verified": verified, "per_gpu_GBps": round(value / world, 3),
        "save_GBps": round(world * payload / save_s / 1e9, 3), "load_GBps": round(world * payload / load_s / 1e9, 3),
        "p50_save_ms": round(save_s * 1e3, 3), "p50_load_ms": round(load_s * 1e3, 3),
        "payload_bytes_per_direction_per_rank": payload, "numa_pools": args.numa_pools,
        "engine": {k: (round(m[k], 2) if isinstance(m[k], float) else m[k])
                   for k in ("load_failures", "cache_block_evictions", "pool_alloc_failures", "save_calls",
                             "save_plan_ms", "save_transfer_ms", "save_insert_ms", "save_ms", "load_ms")},
        "engine_phases_ms_per_step": phases,
        "how": "host wall clock per phase (all ranks save at once, then all load at once); value = all ranks' "
               "save + load bytes / summed phase times; engine *_ms are summed over every call of every rank "
               "(engine_phases_ms_per_step: over the timed steps, divided by the steps)",
    }
    print(json.dumps(line), flush=True)


def run_server_e2e(args) -> None:
    """The deployment path end to end: this process holds the KV cache (as a
    vLLM worker does), `python -m pegaflow_b200.server` runs as its own
    process and maps the cache over CUDA IPC, and every step is a Save RPC
    (all layers, one hash list) followed by a Load RPC and its LoadState
    completion, through EngineRpcClient over gRPC. BASELINE config 3 at TP1
    (80 layers x 2,048 blocks, 10 GiB per direction) by default, or config 1
    with --server-shape llama8b. Host wall clock; bytes checked after the
    timed steps."""
    import pickle
    import socket

    import torch

    from pegaflow_b200 import CudaIPCWrapper, EngineRpcClient, Layout, PyLoadState
    from pegaflow_b200.ranks import block_lists

    torch.cuda.set_device(0)
    if args.server_bind:
        # The server inherits this process's CPU affinity, so its pool pages
        # are first touched on the NUMA node next to GPU 0.
        from pegaflow_b200.ranks import bind_to_gpu_cpus

        bind_to_gpu_cpus(0)
    wl = dict(WORKLOADS[args.server_shape])
    if args.layers:
        wl["layers"] = args.layers
    tensors, _, _ = make_workload(torch, wl, 0, 0, 1, args.order)
    src, dst = block_lists(wl["num_blocks"], wl["blocks"], 0, args.order)
    n = len(src)
    payload = payload_bytes(tensors, n)
    torch.cuda.synchronize()
    with socket.socket() as sk:
        sk.bind(("127.0.0.1", 0))
        port = sk.getsockname()[1]
    pool_mib = (2 * payload + (512 << 20)) >> 20
    proc = subprocess.Popen([sys.executable, "-m", "pegaflow_b200.server", "--addr", f"127.0.0.1:{port}",
                             "--pool-size", f"{pool_mib}mb", "--disable-lfu-admission", "--log-level", "warning"],
                            cwd=str(ROOT), stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    client, deadline = None, time.time() + 300
    while client is None:
        try:
            client = EngineRpcClient(f"http://127.0.0.1:{port}", connect_timeout_s=1.0)
        except RuntimeError:
            if proc.poll() is not None or time.time() > deadline:
                out = proc.stdout.read().decode(errors="replace") if proc.stdout else ""
                proc.kill()
                raise RuntimeError(f"server did not start: {out[-2000:]}")
    names = [f"model.layers.{i}.self_attn" for i in range(len(tensors))]
    try:
        for nm, t in zip(names, tensors):
            lay = Layout.from_tensor(t)
            ok, msg = client.register_context("srv", "bench", 0, 1, 0, len(names), nm, pickle.dumps(CudaIPCWrapper(t)),
                                              lay.num_blocks, lay.bytes_per_block, lay.kv_stride_bytes, lay.segments)
            if not ok:
                raise RuntimeError(msg)
        src_l, dst_l = src.tolist(), dst.tolist()

        def step(k):
            hashes = [f"s{k}-b{i}".encode() for i in range(n)]
            t0 = time.perf_counter()
            ok, msg = client.save("srv", 0, 0, [(nm, src_l, hashes) for nm in names])
            if not ok:
                raise RuntimeError(msg)
            t1 = time.perf_counter()
            st = PyLoadState(len(names))
            ok, msg = client.load("srv", 0, 0, st.shm_name(), names, dst_l, hashes)
            if not ok:
                raise RuntimeError(msg)
            limit = time.perf_counter() + 120.0
            while not st.is_ready():
                if time.perf_counter() > limit:
                    raise TimeoutError("load did not complete within 120 s")
            t2 = time.perf_counter()
            good = st.get_state() == 1
            st.close()
            if not good:
                raise RuntimeError("load failed")
            return t1 - t0, t2 - t1

        for k in range(args.warmup):
            step(-1 - k)
        from pegaflow_b200.client import encode_save_request

        enc = []
        for k in range(5):
            hs = [f"e{k}-b{i}".encode() for i in range(n)]
            t0 = time.perf_counter()
            encode_save_request("srv", 0, 0, [(nm, src_l, hs) for nm in names])
            enc.append(time.perf_counter() - t0)
        scribble(torch, tensors, dst)
        torch.cuda.synchronize()
        times = [step(k) for k in range(args.steps)]
        torch.cuda.synchronize()
        verified = restored(torch, tensors, src, dst)
    finally:
        try:
            client.shutdown()
        except RuntimeError:
            pass
        try:
            proc.wait(timeout=60)
        except subprocess.TimeoutExpired:
            proc.kill()
    total = sum(a + b for a, b in times)
    value = 2 * payload * len(times) / total / 1e9
    line = {
        "metric": METRIC, "value": round(value, 3), "unit": "GB/s", "n_gpus": 1, "steps": args.steps,
        "warmup": args.warmup, "ms_per_step": round(total / len(times) * 1e3, 3), "higher_is_better": True,
        "scaling": "none", "vs_baseline": None, "dtype": "u8", "data": "synthetic (seeded ~N(0,1) bf16 KV)",
        "config": dict(config_block(args, wl, 1), workload="server_e2e", shape=args.server_shape,
                       parallelism="one vLLM-like client process and the engine server process on one GPU"),
        "verified": verified,
        "save_GBps": round(payload / statistics.median(a for a, _ in times) / 1e9, 3),
        "load_GBps": round(payload / statistics.median(b for _, b in times) / 1e9, 3),
        "p50_save_ms": round(statistics.median(a for a, _ in times) * 1e3, 3),
        "p50_load_ms": round(statistics.median(b for _, b in times) * 1e3, 3),
        "payload_bytes_per_direction": payload,
        "client_encode_ms_p50": round(statistics.median(enc) * 1e3, 3),
        "server_bound_to_gpu_cpus": bool(args.server_bind),
        "e2e": {"value": round(value, 3), "unit": "GB/s", "h2d_bytes_per_step": payload, "d2h_bytes_per_step": payload,
                "api": "EngineRpcClient.save / load over gRPC to python -m pegaflow_b200.server (CUDA IPC), "
                       "PyLoadState completion"},
        "how": "host wall clock per RPC: Save returns once the bytes are in the pool; Load is timed from the RPC "
               "to the LoadState's success",
    }
    print(json.dumps(line), flush=True)


def config_block(args, wl, world: int) -> dict:
    cfg = {"workload": args.workload, "desc": wl["desc"], "layers": wl["layers"], "num_blocks": wl["num_blocks"],
           "blocks_moved": wl["blocks"], "block_ids": args.order,
           "kv_dtype": "fp16" if wl.get("separate") else "bf16",
           "save_mode": args.save_mode, "load_mode": args.load_mode, "copy_kernel": args.copy_kernel,
           "pool": "pinned, write-combined" if args.pool_wc else "pinned, cacheable",
           "staging": {"slot_MiB": args.chunk_mib or 1024, "slots": args.slots or 2, "lanes": "save, load",
                       "first_chunk_MiB": args.first_chunk_mib or 256, "growth": "x2 per chunk",
                       "save_first_chunk": "max(first chunk, half a slot)",
                       "load_first_chunk": "a whole slot; with per-layer flags (the e2e engine loads) "
                                           "the first layer, at most the first chunk"},
           "l2": "inputs larger than L2 (payload >= 36 MiB per layer set; KV cache >> 126 MB)"}
    if wl.get("tp"):
        cfg["tp"] = world
        cfg["heads_per_rank"] = wl["heads"] // world
        cfg["parallelism"] = (f"tp{world} (one process per GPU; each rank saves and restores its own KV head "
                              "shard in its own pool region; no collective on the data path)")
    else:
        cfg["parallelism"] = f"dp{world} (independent ranks, weak scaling)"
    return cfg


# ----------------------------------------------------------------------------- byte checks


def _block_dim(t) -> int:
    """Dimension of the block index: 1 for KV-first [2, nb, ...], else 0."""
    return 1 if (t.dim() == 5 and t.shape[0] == 2) else 0


def scribble(torch, tensors, ids) -> None:
    """Zero the destination blocks, so a later check sees only bytes that the
    transfers after this call restored."""
    idx = torch.as_tensor(np.asarray(ids), device=tensors[0].device)
    for t in tensors:
        t.index_fill_(_block_dim(t), idx, 0)


def restored(torch, tensors, src, dst) -> bool:
    """Every destination block equals its source block, bit for bit (sources
    and destinations are disjoint, so sources are never overwritten)."""
    si = torch.as_tensor(np.asarray(src), device=tensors[0].device)
    di = torch.as_tensor(np.asarray(dst), device=tensors[0].device)
    return all(torch.equal(t.index_select(_block_dim(t), di), t.index_select(_block_dim(t), si)) for t in tensors)


def pool_matches(torch, tensors, saves, pool, src) -> bool:
    """The pinned pool holds each layer's K region, then its V region, in the
    order of the block list (lib.rs:639-679): checked on the first and last
    layer against the source blocks."""
    si = torch.as_tensor(np.asarray(src), device=tensors[0].device)
    host = pool.numpy()
    for li in sorted({0, len(tensors) - 1}):
        t, sp = tensors[li], saves[li]
        parts = [(t[0], sp.k_dst), (t[1], sp.v_dst)] if sp.layout.split else [(t, sp.k_dst)]
        for kv, base in parts:
            want = kv.index_select(0, si).contiguous().view(-1).view(torch.uint8)
            off = base - pool.ptr
            got = torch.from_numpy(host[off:off + want.numel()].copy()).to(t.device)
            if not torch.equal(got, want):
                return False
    return True


def executor_rates(torch, ex, stream, saves, loads, payload: int, steps: int, warmup: int, barrier) -> dict:
    """Save then load, `steps` times on one stream, device-timed per step."""
    sp = stream.cuda_stream
    for _ in range(warmup):
        ex.save(saves, stream=sp)
        ex.load(loads, stream=sp)
    stream.synchronize()
    barrier()
    evs = []
    for _ in range(steps):
        e = [torch.cuda.Event(enable_timing=True) for _ in range(3)]
        e[0].record(stream)
        ex.save(saves, stream=sp)
        e[1].record(stream)
        ex.load(loads, stream=sp)
        e[2].record(stream)
        evs.append(e)
    stream.synchronize()
    save_ms = [e[0].elapsed_time(e[1]) for e in evs]
    load_ms = [e[1].elapsed_time(e[2]) for e in evs]
    total = sum(e[0].elapsed_time(e[2]) for e in evs)
    return {"total_ms": total, "save_GBps": payload / (statistics.median(save_ms) / 1e3) / 1e9,
            "load_GBps": payload / (statistics.median(load_ms) / 1e3) / 1e9,
            "p50_load_ms": statistics.median(load_ms)}


# ----------------------------------------------------------------------------- extra blocks


def config_rates_block(torch, args, ex, local: int, workload: str) -> dict:
    """Another BASELINE config on this GPU through the same executor, once
    with seeded-shuffled and once with sorted-contiguous block ids; bytes
    checked after each: configs[1] (Llama-3.1-8B, 32 layers x 640 blocks) or
    configs[0] (GPT-2-small, separate K and V tensors, 24 segments=1 layers x
    64 blocks)."""
    from pegaflow_b200 import PinnedBuffer
    from pegaflow_b200.ranks import block_lists

    wl = WORKLOADS[workload]
    tensors, _, _ = make_workload(torch, wl, local, 0, 1, "shuffled")
    n = wl["blocks"]
    payload = payload_bytes(tensors, n)
    pool = PinnedBuffer(payload + wl["layers"] * 8192 + (1 << 20), write_combined=True)
    stream = torch.cuda.Stream(local)
    steps = max(3, min(args.steps, 10)) if workload == "llama8b" else max(3, args.steps)
    out = {"desc": wl["desc"], "payload_bytes_per_direction": payload, "steps": steps}
    for order in ("shuffled", "sorted"):
        src, dst = block_lists(wl["num_blocks"], n, 0, order)
        saves, loads, _ = executor_specs(tensors, src, dst, pool.ptr)
        scribble(torch, tensors, dst)
        r = executor_rates(torch, ex, stream, saves, loads, payload, steps, 2, lambda: None)
        out[order] = {"GBps": round(2 * payload * steps / (r["total_ms"] / 1e3) / 1e9, 3),
                      "save_GBps": round(r["save_GBps"], 3), "load_GBps": round(r["load_GBps"], 3),
                      "p50_load_ms": round(r["p50_load_ms"], 3),
                      "verified": restored(torch, tensors, src, dst) and pool_matches(torch, tensors, saves, pool, src)}
    pool.close()
    del tensors
    torch.cuda.empty_cache()
    return out


def pd_check(torch, ex0, reps: int = 10) -> dict:
    """BASELINE config 2's handoff for one request, inside the multi-GPU run:
    Qwen3-8B-shaped KV (36 layers of [2, 1024, 16, 8, 128] bf16) on GPU0 and
    GPU1, 313 seeded blocks moved GPU0 -> GPU1 by the decode-side pull kernel
    (plain 16-byte peer loads over NVLink), bytes checked, timed against the
    1 GiB peer-copy peak and against one host-pool bounce (save on GPU0, load
    on GPU1). Runs in rank 0's process; the other ranks wait on the host."""
    from pegaflow_b200 import Executor, Layout, LoadSpec, P2PSpec, PinnedBuffer, SaveSpec

    layers, nb, n = 36, 1024, 313
    g0 = torch.Generator(device="cuda:0").manual_seed(7)
    g1 = torch.Generator(device="cuda:1").manual_seed(8)
    shape = (2, nb, 16, 8, 128)
    src = [torch.randn(shape, generator=g0, device="cuda:0").to(torch.bfloat16) for _ in range(layers)]
    dst = [torch.randn(shape, generator=g1, device="cuda:1").to(torch.bfloat16) for _ in range(layers)]
    si = np.random.default_rng(4).permutation(nb)[:n]
    di = np.random.default_rng(10_000).permutation(nb)[:n]
    si0 = torch.as_tensor(si, device="cuda:0")
    payload = n * layers * 2 * 32768
    dev_before = torch.cuda.current_device()
    ex1 = Executor(1)
    s0, s1 = torch.cuda.Stream("cuda:0"), torch.cuda.Stream("cuda:1")
    specs = [P2PSpec(Layout.from_tensor(x), Layout.from_tensor(y), si, di) for x, y in zip(src, dst)]

    def expected_ok() -> bool:
        return all(torch.equal(y.index_select(1, torch.as_tensor(di, device="cuda:1")),
                               x.index_select(1, si0).to("cuda:1")) for x, y in zip(src, dst))

    ex1.p2p(specs, 0, push=False, stream=s1.cuda_stream)  # warm-up (enables peer access)
    s1.synchronize()
    scribble(torch, dst, di)
    torch.cuda.synchronize(1)
    ms = []
    for _ in range(reps):
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record(s1)
        ex1.p2p(specs, 0, push=False, stream=s1.cuda_stream)
        e1.record(s1)
        ms.append((e0, e1))
    s1.synchronize()
    pull_ms = [a.elapsed_time(b) for a, b in ms]
    pull_ok = expected_ok()

    # Peer copy peak: 1 GiB cudaMemcpyPeer GPU0 -> GPU1, best of 4.
    a = torch.empty(1 << 30, dtype=torch.uint8, device="cuda:0")
    b = torch.empty(1 << 30, dtype=torch.uint8, device="cuda:1")
    peak = 0.0
    for _ in range(4):
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        with torch.cuda.stream(s1):
            e0.record(s1)
            b.copy_(a, non_blocking=True)
            e1.record(s1)
        e1.synchronize()
        peak = max(peak, (1 << 30) / (e0.elapsed_time(e1) / 1e3) / 1e9)
    del a, b

    # One request through the host pool: the reference's handoff (docs/pd.md).
    pool = PinnedBuffer(payload + layers * 4096, write_combined=True)
    saves, loads, off = [], [], 0
    for x, y in zip(specs, dst):
        k, v = pool.ptr + off, pool.ptr + off + n * 32768
        ks = np.arange(n, dtype=np.uint64) * 32768 + k
        saves.append(SaveSpec(x.src, si, k, v))
        loads.append(LoadSpec(Layout.from_tensor(y), di, ks, ks + n * 32768))
        off += 2 * n * 32768 + 4096
    scribble(torch, dst, di)
    torch.cuda.synchronize(1)
    bounce_ms = []
    for _ in range(3):
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record(s1)
        s0.wait_event(e0)
        ex0.save(saves, stream=s0.cuda_stream)
        ev = torch.cuda.Event()
        ev.record(s0)
        s1.wait_event(ev)
        ex1.load(loads, stream=s1.cuda_stream)
        e1.record(s1)
        e1.synchronize()
        bounce_ms.append(e0.elapsed_time(e1))
    bounce_ok = expected_ok()
    launches = ex1.stats()["kernel_launches"]
    pool.close()
    ex1.close()
    dev_after = torch.cuda.current_device()
    del src, dst
    torch.cuda.synchronize(1)
    torch.cuda.empty_cache()
    pull_gbps = payload / (statistics.median(pull_ms) / 1e3) / 1e9
    bounce_gbps = payload / (statistics.median(bounce_ms) / 1e3) / 1e9
    return {"workload": "qwen3_pd, one request: 36 layers x 313 blocks GPU0 -> GPU1",
            "payload_bytes": payload, "p2p_pull_GBps": round(pull_gbps, 2),
            "p2p_pull_p50_ms": round(statistics.median(pull_ms), 3),
            "peer_copy_peak_GBps": round(peak, 1), "frac_of_peer_peak": round(pull_gbps / peak, 3),
            "host_pool_bounce_GBps": round(bounce_gbps, 2), "p2p_over_bounce": round(pull_gbps / bounce_gbps, 2),
            "verified": bool(pull_ok and bounce_ok), "device_restored": dev_after == dev_before,
            "gpu1_launches": launches,
            "how": "pull: kernel on GPU1 reads GPU0's paged KV with plain 16-byte peer loads (no TMA, no multicast); "
                   "median of 10 device-timed requests; bounce: executor save on GPU0 then load on GPU1, median of 3"}


# ----------------------------------------------------------------------------- main arm


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=10)
    ap.add_argument("--warmup", type=int, default=3)
    ap.add_argument("--impl", choices=["b200", "reference"], default="b200")
    ap.add_argument("--workload", choices=sorted(WORKLOADS) + ["qwen3_pd", "llama8b_fp8_evict", "llama8b_duplex",
                                                               "llama70b_tp_one_engine", "server_e2e"],
                    default="llama70b_tp")
    ap.add_argument("--server-shape", default="llama70b_tp", choices=["llama70b_tp", "llama8b"],
                    help="server_e2e: the KV shape moved through the gRPC server")
    ap.add_argument("--server-bind", action="store_true",
                    help="server_e2e: start the server on the CPUs local to GPU 0")
    ap.add_argument("--numa-pools", default="off", choices=["off", "node", "device"],
                    help="llama70b_tp_one_engine: one pool, or one per NUMA node / per GPU")
    ap.add_argument("--fp8-requests", type=int, default=64)
    ap.add_argument("--fp8-pool-gb", type=int, default=30)
    ap.add_argument("--fp8-compute-ms", type=float, default=0.5)
    ap.add_argument("--fp8-compute", choices=["sleep", "attention"], default="sleep",
                    help="llama8b_fp8_evict: a layer's compute is a wait of --fp8-compute-ms, or the request's new "
                         "tokens written into the cache and attending over it")
    ap.add_argument("--pd-requests", type=int, default=200)
    ap.add_argument("--pd-bounce-requests", type=int, default=20)
    ap.add_argument("--order", choices=["shuffled", "sorted"], default="shuffled")
    ap.add_argument("--save-mode", default="auto", choices=["auto", "staged", "direct"])
    ap.add_argument("--load-mode", default="auto", choices=["auto", "staged", "direct"])
    ap.add_argument("--chunk-mib", type=int, default=0)
    ap.add_argument("--first-chunk-mib", type=int, default=0)
    ap.add_argument("--slots", type=int, default=0)
    ap.add_argument("--copy-streams", type=int, default=0)
    ap.add_argument("--ctas-per-sm", type=int, default=0)
    ap.add_argument("--cache-streaming", action="store_true", help="evict-first loads/stores in the kernels")
    ap.add_argument("--pool-wc", type=int, default=1, choices=[0, 1],
                    help="pinned pool memory write-combined (1, the reference's pool kind) or cacheable (0)")
    ap.add_argument("--copy-kernel", default="auto", choices=["auto", "registers", "bulk"],
                    help="how staged tiles move: registers, or TMA bulk copies through shared memory")
    ap.add_argument("--e2e-steps", type=int, default=0, help="engine-API steps (default: --steps)")
    ap.add_argument("--no-refcopy", action="store_true")
    ap.add_argument("--no-cpu", action="store_true")
    ap.add_argument("--no-extra", action="store_true",
                    help="skip the other-order, configs[1] and P/D blocks (short profiling runs)")
    ap.add_argument("--cpu-seconds", type=float, default=8.0)
    ap.add_argument("--layers", type=int, default=0, help="override the layer count (small profiling runs)")
    args = ap.parse_args()
    if args.workload == "qwen3_pd":
        if args.impl == "reference":
            print(json.dumps({"impl": "reference", "workload": "qwen3_pd",
                              "unavailable": "the reference hands P/D blocks over through its host pool; "
                                             "see host_pool_bounce in the b200 line"}))
            return 0
        run_pd(args)
        return 0
    if args.workload == "llama8b_fp8_evict":
        if args.impl == "reference":
            print(json.dumps({"impl": "reference", "workload": "llama8b_fp8_evict",
                              "unavailable": "engine-level scenario; the reference engine cannot be built here"}))
            return 0
        run_fp8_evict(args)
        return 0
    if args.workload == "llama8b_duplex":
        if args.impl == "reference":
            print(json.dumps({"impl": "reference", "workload": "llama8b_duplex",
                              "unavailable": "engine-level scenario; the reference engine cannot be built here"}))
            return 0
        if int(os.environ.get("RANK", "0")) == 0:
            run_duplex(args)
        return 0
    if args.workload == "server_e2e":
        if args.impl == "reference":
            print(json.dumps({"impl": "reference", "workload": "server_e2e",
                              "unavailable": "the reference server is Rust and cannot be built here"}))
            return 0
        if int(os.environ.get("RANK", "0")) == 0:
            run_server_e2e(args)
        return 0
    if args.workload == "llama70b_tp_one_engine":
        if args.impl == "reference":
            print(json.dumps({"impl": "reference", "workload": "llama70b_tp_one_engine",
                              "unavailable": "engine-level scenario; the reference engine cannot be built here"}))
            return 0
        run_one_engine(args)
        return 0
    wl = dict(WORKLOADS[args.workload])
    if args.layers:
        wl["layers"] = args.layers
    args.warmup = max(args.warmup, 0)

    if args.impl == "reference":
        run_reference_arm(args, wl)
        return 0

    import torch

    from pegaflow_b200.ranks import Ranks

    local = int(os.environ.get("LOCAL_RANK", "0"))
    torch.cuda.set_device(local)
    ranks = Ranks.from_env("nccl", timeout_s=600)
    rank, world, local = ranks.rank, ranks.world, ranks.local
    barrier, max_over_ranks, min_over_ranks = ranks.barrier, ranks.max, ranks.min

    from pegaflow_b200 import Executor, Layout, PegaEngine, PinnedBuffer, PyLoadState, refcopy_load, refcopy_save
    from pegaflow_b200.ranks import bind_to_gpu_cpus, block_lists

    cpus = bind_to_gpu_cpus(local)
    peaks = measured_peaks()
    # Host-link peaks: each rank alone (the others wait on the host), then
    # every rank at once (its share of the link while all GPUs copy).
    link_alone = None
    for r in range(world):
        ranks.host_barrier()
        if r == rank:
            link_alone = link_peaks(torch, local)
    ranks.host_barrier()
    link = link_peaks(torch, local, barrier) if world > 1 else dict(link_alone)
    alone_d2h_all, alone_h2d_all = ranks.gather(link_alone["d2h"]), ranks.gather(link_alone["h2d"])
    link_d2h_all, link_h2d_all = ranks.gather(link["d2h"]), ranks.gather(link["h2d"])
    tensors, src, dst = make_workload(torch, wl, local, rank, world, args.order)
    n = len(src)
    payload = payload_bytes(tensors, n)
    torch.cuda.synchronize()

    ex = Executor(local, save_mode=args.save_mode, load_mode=args.load_mode,
                  staging_chunk_bytes=args.chunk_mib << 20, staging_slots=args.slots,
                  copy_streams=args.copy_streams, ctas_per_sm=args.ctas_per_sm,
                  cache_streaming=args.cache_streaming, first_chunk_bytes=args.first_chunk_mib << 20,
                  copy_kernel=args.copy_kernel)
    pool = PinnedBuffer(payload + wl["layers"] * 8192 + (1 << 20), write_combined=args.pool_wc == 1)
    saves, loads, _ = executor_specs(tensors, src, dst, pool.ptr)
    stream = torch.cuda.Stream(local)
    sp = stream.cuda_stream

    def step(evs=None):
        if evs:
            evs[0].record(stream)
        ex.save(saves, stream=sp)
        if evs:
            evs[1].record(stream)
        ex.load(loads, stream=sp)
        if evs:
            evs[2].record(stream)

    for _ in range(args.warmup):
        step()
    stream.synchronize()
    scribble(torch, tensors, dst)  # the check below then sees only what the timed steps restored
    torch.cuda.synchronize()

    ex.reset_stats()
    ex.set_timing(True)
    sampler = ClockSampler(local)
    sampler.start()
    barrier()
    torch.cuda.synchronize()
    per = [[torch.cuda.Event(enable_timing=True) for _ in range(3)] for _ in range(args.steps)]
    t_start, t_end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    t_start.record(stream)
    for k in range(args.steps):
        step(per[k])
    t_end.record(stream)
    t_end.synchronize()
    barrier()
    torch.cuda.synchronize()
    clocks = sampler.stop()
    ex.set_timing(False)
    st = ex.stats()
    ms = t_start.elapsed_time(t_end)
    save_ms = [e[0].elapsed_time(e[1]) for e in per]
    load_ms = [e[1].elapsed_time(e[2]) for e in per]
    ms_max = max_over_ranks(ms)
    steps = args.steps
    value = world * 2 * payload * steps / (ms_max / 1e3) / 1e9
    my_save = payload / (statistics.median(save_ms) / 1e3) / 1e9
    my_load = payload / (statistics.median(load_ms) / 1e3) / 1e9
    save_gbps, load_gbps = min_over_ranks(my_save), min_over_ranks(my_load)
    # Each rank against its own peaks: measured alone, and measured while every rank copies.
    save_frac_alone = min_over_ranks(my_save / link_alone["d2h"])
    load_frac_alone = min_over_ranks(my_load / link_alone["h2d"])
    save_frac = min_over_ranks(my_save / link["d2h"])
    load_frac = min_over_ranks(my_load / link["h2d"])
    p50_load = max_over_ranks(statistics.median(load_ms))
    kernel_gbps = st["kernel_bytes"] / (st["kernel_ms"] / 1e3) / 1e9 if st["kernel_ms"] > 0 else 0.0
    kernel_all = ranks.gather(kernel_gbps)
    launch_us_all = ranks.gather(st["kernel_ms"] * 1e3 / max(1, st["timed_launches"]))
    # The same launches timed inside the kernels (%globaltimer, first CTA start
    # to last CTA end): the body alone, without the launch's own latency.
    body_bytes = st["kernel_bytes"] * st["body_launches"] / max(1, st["timed_launches"])
    body_gbps = body_bytes / (st["kernel_body_ms"] / 1e3) / 1e9 if st["kernel_body_ms"] > 0 else 0.0
    body_all = ranks.gather(body_gbps)
    body_us_all = ranks.gather(st["kernel_body_ms"] * 1e3 / max(1, st["body_launches"]))
    verified_main = ranks.all_true(restored(torch, tensors, src, dst)
                                   and pool_matches(torch, tensors, saves, pool, src))

    # Saves alone and loads alone, started on every rank at once: the same
    # traffic pattern as the concurrent link peaks, so the fractions compare like
    # with like (inside a step, ranks drift apart and one rank's saves meet
    # another's loads).
    al_save = aligned_rates(torch, stream, lambda: ex.save(saves, stream=sp), payload, barrier)
    al_load = aligned_rates(torch, stream, lambda: ex.load(loads, stream=sp), payload, barrier)
    al_save_all, al_load_all = ranks.gather(al_save), ranks.gather(al_load)

    # The other block order, same tensors and executor (sorted-contiguous runs
    # are where the reference's run merging differs from shuffled ids).
    other = None
    if not args.no_extra:
        o_order = "sorted" if args.order == "shuffled" else "shuffled"
        o_src, o_dst = block_lists(wl["num_blocks"], n, rank, o_order)
        o_saves, o_loads, _ = executor_specs(tensors, o_src, o_dst, pool.ptr)
        scribble(torch, tensors, o_dst)
        o_steps = max(3, min(steps, 10))
        r = executor_rates(torch, ex, stream, o_saves, o_loads, payload, o_steps, 2, barrier)
        o_ms = max_over_ranks(r["total_ms"])
        other = {"block_ids": o_order, "steps": o_steps,
                 "GBps": round(world * 2 * payload * o_steps / (o_ms / 1e3) / 1e9, 3),
                 "save_GBps": round(min_over_ranks(r["save_GBps"]), 3),
                 "load_GBps": round(min_over_ranks(r["load_GBps"]), 3),
                 "p50_load_ms": round(max_over_ranks(r["p50_load_ms"]), 3),
                 "verified": ranks.all_true(restored(torch, tensors, o_src, o_dst)
                                            and pool_matches(torch, tensors, o_saves, pool, o_src))}

    # ---- e2e through the engine API (host wall clock) ------------------------
    e2e_steps = args.e2e_steps or args.steps
    eng = PegaEngine(2 * payload + (256 << 20), enable_lfu_admission=False, write_combined=args.pool_wc == 1,
                     executor=dict(save_mode=args.save_mode, load_mode=args.load_mode,
                                   staging_chunk_bytes=args.chunk_mib << 20, staging_slots=args.slots,
                                   copy_streams=args.copy_streams, ctas_per_sm=args.ctas_per_sm,
                                   cache_streaming=1 if args.cache_streaming else 0,
                                   first_chunk_bytes=args.first_chunk_mib << 20, copy_kernel=args.copy_kernel))
    names = [f"model.layers.{i}.self_attn" for i in range(len(tensors))]
    for nm, t in zip(names, tensors):
        lay = Layout.from_tensor(t)
        eng.register_context_layer(f"bench{rank}", "bench", local, nm, lay.data_ptr, lay.size_bytes, lay.num_blocks,
                                   lay.bytes_per_block, lay.kv_stride_bytes, lay.segments, 0, 1, len(tensors))
    src_l, dst_l = src.tolist(), dst.tolist()

    def e2e_step(k):
        hashes = [f"r{rank}-s{k}-b{i}".encode() for i in range(n)]
        t0 = time.perf_counter()
        eng.batch_save_kv_blocks(f"bench{rank}", 0, local, [(nm, src_l, hashes) for nm in names])
        t1 = time.perf_counter()
        s = PyLoadState(len(names))  # with per-layer completion words
        eng.batch_load_kv_blocks(f"bench{rank}", 0, local, s.shm_name(), names, dst_l, hashes)
        deadline = time.perf_counter() + 120.0
        t_first = None
        while not s.is_ready():
            if t_first is None and s.layer_ready(0):
                t_first = time.perf_counter()
            if time.perf_counter() > deadline:
                raise TimeoutError("engine load did not complete within 120 s")
        t2 = time.perf_counter()
        assert s.get_state() == 1, "engine load failed"
        s.close()
        return t1 - t0, t2 - t1, (t_first or t2) - t1

    for k in range(args.warmup):
        e2e_step(-1 - k)
    eng.executor(local).reset_stats()  # host time of the timed calls only (no first-call allocations)
    eng_before = eng.metrics()
    scribble(torch, tensors, dst)
    barrier()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    e2e_times = [e2e_step(k) for k in range(e2e_steps)]
    e2e_wall = time.perf_counter() - t0
    barrier()
    e2e_wall = max_over_ranks(e2e_wall)
    e2e_value = world * 2 * payload * e2e_steps / e2e_wall / 1e9
    e2e_load_p50 = max_over_ranks(statistics.median([b for _, b, _ in e2e_times]) * 1e3)
    e2e_first_layer_p50 = max_over_ranks(statistics.median([f for _, _, f in e2e_times]) * 1e3)
    verified_e2e = ranks.all_true(restored(torch, tensors, src, dst))
    eng_metrics = eng.metrics()
    eng_ex = eng.executor(local).stats()
    eng_metrics["executor_host_ms_per_call"] = eng_ex["host_ms"] / max(1, 2 * e2e_steps)
    # Per timed step (the warm-up's first-call costs left out).
    eng_metrics["phases_ms_per_step"] = {
        k: round((eng_metrics[k] - eng_before[k]) / e2e_steps, 3)
        for k in ("save_plan_ms", "save_transfer_ms", "save_insert_ms", "load_lookup_ms", "load_queue_ms",
                  "load_setup_ms", "load_transfer_ms", "load_first_layer_ms")}
    eng.close()

    # ---- save and load at once (one GPU) --------------------------------------
    duplex = None
    if world == 1 and not args.no_extra:
        duplex = duplex_block(torch, ex, tensors, src, dst, payload, max(3, min(steps, 8)), local, value)

    # ---- the reference's copy strategy on the same GPU ------------------------
    ref = None
    if not args.no_refcopy:
        scribble(torch, tensors, dst)
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        refcopy_save(local, saves)
        t1 = time.perf_counter()
        runs = refcopy_load(local, loads)
        t2 = time.perf_counter()
        ref = {"save_GBps": round(payload / (t1 - t0) / 1e9, 3), "load_GBps": round(payload / (t2 - t1) / 1e9, 3),
               "value": round(2 * payload / (t2 - t0) / 1e9, 3), "load_ms": round((t2 - t1) * 1e3, 3),
               "h2d_runs": runs, "d2h_copies": sum(len(s.block_idx) * (2 if s.layout.split else 1) for s in saves),
               "verified": restored(torch, tensors, src, dst),
               "how": "per-segment synchronous D2H (gpu_worker.rs:343-360) + merged-run async H2D "
                      "(transfer.rs:116-198), restated in C++, same GPU and pool; rank 0's figures"}

    cpu = None
    if rank == 0 and world == 1 and not args.no_cpu:
        cpu = CpuWorkload(wl, os.cpu_count() or 1, order=args.order).rate(args.cpu_seconds)
        # The same copies with the pool in page-locked memory, cacheable and
        # write-combined (shorter samples; reported beside the baseline).
        cpu["pool_variants_GBps"] = {}
        for kind in ("pinned", "pinned_wc"):
            cw = CpuWorkload(wl, os.cpu_count() or 1, pool=kind, order=args.order)
            cpu["pool_variants_GBps"][kind] = cw.rate(args.cpu_seconds / 4)["value"]
            cw.close()

    pool.close()
    cfg1 = cfg0 = cfg4 = None
    if world == 1 and args.workload == "llama70b_tp" and not args.no_extra:
        del tensors, saves, loads
        torch.cuda.empty_cache()
        cfg1 = config_rates_block(torch, args, ex, local, "llama8b")
        cfg0 = config_rates_block(torch, args, ex, local, "gpt2")
        r4 = fp8_evict_result(args)
        cfg4 = {"desc": "Llama-3.1-8B fp8 e4m3 KV + fp32 per-block scales, 64 requests of U[1K,16K] tokens, "
                        f"half of each prefix warm, {args.fp8_pool_gb} GB pool with LRU eviction, layer-wise "
                        "restore overlapped with 0.5 ms of compute per layer (engine API)",
                "layerwise_overlap": r4["layerwise_overlap"], "load_then_compute": r4["load_then_compute"],
                "overlap_speedup": r4["overlap_speedup"], "engine": r4["engine"],
                "verified": "not byte-checked here (requests reuse one cache); the fp8 + scale layout is "
                            "checked at full size by the GPU tests"}

    # P/D handoff check: rank 0 alone, GPU0 -> GPU1; the others wait on the
    # host so no collective kernel of theirs sits on GPU1 meanwhile.
    pd = None
    if world >= 2 and not args.no_extra:
        ranks.host_barrier()
        if rank == 0:
            if torch.cuda.device_count() >= 2:
                pd = pd_check(torch, ex)
            else:
                pd = {"unavailable": "rank 0 sees one GPU (the P/D check needs GPU 0 and GPU 1 in one process)"}
        ranks.host_barrier()

    if rank == 0:
        verified = bool(verified_main and verified_e2e and (other is None or other["verified"])
                        and all(c is None or all(c[o]["verified"] for o in ("shuffled", "sorted"))
                                for c in (cfg1, cfg0))
                        and (pd is None or "unavailable" in pd or pd["verified"])
                        and (ref is None or ref["verified"]))
        achieved = min(kernel_all)
        line = {
            "metric": METRIC, "value": round(value, 3), "unit": "GB/s", "n_gpus": world, "steps": steps,
            "warmup": args.warmup, "ms_per_step": round(ms_max / steps, 4), "higher_is_better": True,
            "scaling": "weak", "vs_baseline": None, "dtype": "u8", "data": "synthetic (seeded ~N(0,1) bf16 KV)",
            "config": config_block(args, wl, world),
            "verified": verified,
            "verified_how": "destination blocks zeroed before each timed region, then every restored block "
                            "compared bit for bit with its source on the GPU (torch.equal), every rank; pool "
                            "K/V regions of the first and last layer compared with the source blocks",
            "per_gpu_GBps": round(value / world, 3),
            "save_GBps": round(save_gbps, 3), "load_GBps": round(load_gbps, 3), "p50_load_ms": round(p50_load, 3),
            "payload_bytes_per_direction": payload,
            "host_link": {"peak_h2d_GBps": link["h2d"], "peak_d2h_GBps": link["d2h"],
                          "save_frac": round(save_frac, 3), "load_frac": round(load_frac, 3),
                          "save_frac_alone": round(save_frac_alone, 3), "load_frac_alone": round(load_frac_alone, 3),
                          "per_rank_alone_d2h_GBps": [round(x, 2) for x in alone_d2h_all],
                          "per_rank_alone_h2d_GBps": [round(x, 2) for x in alone_h2d_all],
                          "per_rank_peak_d2h_GBps": [round(x, 2) for x in link_d2h_all],
                          "per_rank_peak_h2d_GBps": [round(x, 2) for x in link_h2d_all],
                          "aligned": {
                              "save_GBps_per_rank": [round(x, 2) for x in al_save_all],
                              "load_GBps_per_rank": [round(x, 2) for x in al_load_all],
                              "save_frac_min": round(min(a / p for a, p in zip(al_save_all, link_d2h_all)), 3),
                              "load_frac_min": round(min(a / p for a, p in zip(al_load_all, link_h2d_all)), 3),
                              "how": "saves alone, then loads alone, started on every rank at once (median "
                                     "of 3); each rank against its own concurrent peak"},
                          "how": "pinned 1 GiB cudaMemcpyAsync, best of 3; *_alone: each rank measured while "
                                 "the others wait; peak_* / per_rank_peak_*: every rank copying at once; "
                                 "*_frac = min over ranks of the step's save (load) rate over that rank's own "
                                 "concurrent peak, *_frac_alone over its own single-GPU peak"},
            "roofline": {"bound": "hbm", "achieved": round(achieved, 1),
                         "peak": peaks["hbm_gbs"], "unit": "GB/s", "frac": round(achieved / peaks["hbm_gbs"], 3),
                         "traffic": traffic_per_launch(st["kernel_bytes"] / max(1, st["timed_launches"])),
                         "traffic_how": "not measured per run: from one ncu capture of dram__bytes_read.sum + "
                                        "dram__bytes_write.sum (128 and 160 MiB chunks): reads = payload, writes = "
                                        "payload less the ~50 MB still in L2 at kernel end; applied to this run's "
                                        "average launch",
                         "peak_source": peaks["source"],
                         "kernel": "kv_copy_kernel (pack+unpack)",
                         "bytes_per_launch": round(st["kernel_bytes"] / max(1, st["timed_launches"])),
                         "avg_launch_us": round(max(launch_us_all), 2),
                         "achieved_per_rank": [round(x, 1) for x in kernel_all],
                         "how": "algorithmic bytes (payload read + written per launch) / CUDA-event launch "
                                "duration over the timed region; the slowest rank's figure",
                         "body": {"achieved": round(min(body_all), 1),
                                  "frac": round(min(body_all) / peaks["hbm_gbs"], 3),
                                  "avg_us": round(max(body_us_all), 2), "launches": st["body_launches"],
                                  "how": "the same launches timed inside the kernel (%globaltimer: first CTA "
                                         "start to last CTA end); the CUDA-event figure above adds each "
                                         "launch's own latency, which grows while the copy engines stream"}},
            "e2e": {"value": round(e2e_value, 3), "unit": "GB/s", "h2d_bytes_per_step": payload * world,
                    "d2h_bytes_per_step": payload * world, "p50_load_ms": round(e2e_load_p50, 3),
                    "p50_first_layer_ms": round(e2e_first_layer_p50, 3), "steps": e2e_steps,
                    "verified": verified_e2e,
                    "api": "PegaEngine.batch_save_kv_blocks + batch_load_kv_blocks + PyLoadState, one engine "
                           "per rank"},
            "gpu_launches": st["kernel_launches"],
            "host_cpus": (f"{len(cpus)} CPUs local to the GPU (NVML affinity)" if cpus else "unbound"),
            "copy_calls": st["copy_calls"],
            "other_order": other,
            "duplex": duplex,
            "configs1": cfg1,
            "configs0": cfg0,
            "configs4": cfg4,
            "pd": pd,
            "reference_copy_path": ref,
            "cpu_baseline": cpu,
            "clocks": clocks,
            "engine_metrics": {k: (round(eng_metrics[k], 2) if isinstance(eng_metrics[k], float) else eng_metrics[k])
                               for k in ("save_bytes", "load_bytes", "load_failures", "cache_block_evictions",
                                         "save_plan_ms", "save_transfer_ms", "save_insert_ms", "save_ms",
                                         "load_ms", "executor_host_ms_per_call", "phases_ms_per_step")},
        }
        print(json.dumps(line), flush=True)
    ranks.close()
    return 0


if __name__ == "__main__":
    sys.exit(main())
