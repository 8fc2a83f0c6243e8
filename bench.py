#!/usr/bin/env python
"""Benchmark driver: achieved HBM GB/s (and GPoints/s) of the 7x7 stencil /
depthwise hot path on 1..8 B200s, with the reference's CPU path beside it.

    python bench.py [--gpus N] [--steps K] [--warmup W] [--impl ours|reference]
                    [--workload NAME]

N > 1 is launched one process per GPU by torch.distributed.run.  Rank 0 prints
one JSON line.  Workloads (the benchmark configurations; synthetic seeded inputs):

  iterate_cfg5   (default) one Jacobi step of the 32768^2 fp32 iterated stencil
                 (seed 4), row bands over the GPUs with a 3-row halo exchange
                 fused into the step kernel (strong scaling); e2e = the whole
                 100-step job with the band copied in and out; after timing,
                 rows of every band are checked bit for bit against the CPU
                 oracle ("parity" in the line; exit 3 on a mismatch)
  stencil_cfg2   single-step 7x7 stencil, fp32 1x1x4096x4096, seed 1;
                 one grid per GPU (weak scaling, no collective)
  dw_cfg1        depthwise fp32 1x96x56x56 + bias, seed 0
  dw_cfg3_nchw   depthwise bf16 128x384x14x14 + bias, NCHW, seed 2
  dw_cfg3_nhwc   same, channels_last
  dw_cfg4        depthwise bf16 ConvNeXt-T stages at N=256, batch sharded
                 over the GPUs (weak in the sense of fixed total work: strong)
  dw_k3          3x3 depthwise fp32 1x32x1024x1024, no bias: the operator and
                 input recipe of the reference's MetaSchedule benchmark
                 (benchmark/MetaSchedule/depthwise_conv.py, common.py)
  dwln_cfg4      the dw_cfg4 stages in channels_last with the next ConvNeXt
                 layer, LayerNorm over C, fused into the depthwise launch
                 (no reference counterpart; the unfused pair is timed beside it)

A "step" is one pass of the hot path over one batch of input already resident
in HBM; consecutive steps rotate over enough buffer sets that every step's
inputs are out of L2 (footprint > 2 x 126 MB; the iterated stencil's 4 GiB
grid is far larger).  The K timed steps of the single-launch workloads are
captured as one CUDA graph and replayed once (stream launches with --no-graph;
always for the iterated stencil); the line also gives the stream-launch time
of the same K steps (`stream_ms_per_step`).  `value` is whole-job
compulsory bytes (input + output + weights + bias) / device time (CUDA events,
max over ranks).  `e2e` repeats the measurement through the public API with
pinned host buffers, host<->device copies inside the timed region.
"""
from __future__ import annotations

import argparse
import json
import math
import os
import statistics
import sys
import threading
import time

# The reference arm times a CPU path with every host core.  torch.distributed.run
# exports OMP_NUM_THREADS=1 to each rank, and the OpenMP runtime keeps the
# value it read when torch loaded even after torch.set_num_threads(): the
# convolution then ran 1.6x (one process) to 4x (under the launcher) slower.
# Rank 0 of that arm is the only process that works, so it takes the cores
# before torch is imported.
if "--impl" in sys.argv and "reference" in sys.argv and os.environ.get("RANK", "0") == "0":
    os.environ["OMP_NUM_THREADS"] = str(os.cpu_count() or 1)

import numpy as np
import torch
import torch.distributed as dist

ROOT = os.path.dirname(os.path.abspath(__file__))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

METRIC = "achieved HBM GB/s (% of roofline) and GPoints/s at 1/2/4/8 B200 vs CPU ref"
L2_BYTES = 126 * 1024 * 1024
NOMINAL_HBM_GBS = 8000.0
FALLBACK_HBM_GBS = 6650.0
FMA_PER_SM_PER_CLK = 128  # B200 FP32 lanes per SM (a microbenchmark reads 124-127 FFMA/clk/SM)
TAPS = 49


# ---------------------------------------------------------------------------
# helpers
# ---------------------------------------------------------------------------
def profiled_traffic(workload: str):
    """DRAM bytes of one launch of the workload's dominant kernel, from profiles/traffic.json (ncu)."""
    try:
        with open(os.path.join(ROOT, "profiles", "traffic.json")) as f:
            d = json.load(f)[workload]
        return d["dram_read_bytes"] + d["dram_write_bytes"], d["source"]
    except Exception:
        return None, None


def measured_peaks():
    path = os.path.join(ROOT, "MEASURED_PEAKS.json")
    try:
        with open(path) as f:
            d = json.load(f)
        return float(d["hbm_gbs"]), "measured"
    except Exception:
        return FALLBACK_HBM_GBS, "fallback"


class ClockSampler:
    """NVML samples of SM clock and clock-event reasons on one GPU, in a thread."""

    REASONS = {0x1: "gpu_idle", 0x2: "applications_clocks_setting", 0x4: "sw_power_cap", 0x8: "hw_slowdown",
               0x10: "sync_boost", 0x20: "sw_thermal_slowdown", 0x40: "hw_thermal_slowdown",
               0x80: "hw_power_brake_slowdown", 0x100: "display_clock_setting"}

    def __init__(self, device: torch.device, period_s: float = 0.01):
        self.period = period_s
        self.samples = []
        self.reasons = 0
        self.max_mhz = None
        self._stop = threading.Event()
        self._thread = None
        self.handle = None
        try:
            import pynvml

            pynvml.nvmlInit()
            self.nv = pynvml
            props = torch.cuda.get_device_properties(device)
            uuid = str(getattr(props, "uuid", ""))
            h = None
            if uuid:
                for cand in (uuid, "GPU-" + uuid):
                    try:
                        h = pynvml.nvmlDeviceGetHandleByUUID(cand.encode() if isinstance(cand, str) else cand)
                        break
                    except Exception:
                        h = None
            if h is None:
                vis = os.environ.get("CUDA_VISIBLE_DEVICES", "")
                idx = device.index or 0
                if vis and vis.split(",")[idx].strip().isdigit():
                    idx = int(vis.split(",")[idx])
                h = pynvml.nvmlDeviceGetHandleByIndex(idx)
            self.handle = h
            self.max_mhz = pynvml.nvmlDeviceGetMaxClockInfo(h, pynvml.NVML_CLOCK_SM)
        except Exception:
            self.handle = None

    def _sample(self):
        nv = self.nv
        try:
            self.samples.append(nv.nvmlDeviceGetClockInfo(self.handle, nv.NVML_CLOCK_SM))
            try:
                r = nv.nvmlDeviceGetCurrentClocksEventReasons(self.handle)
            except Exception:
                r = nv.nvmlDeviceGetCurrentClocksThrottleReasons(self.handle)
            self.reasons |= int(r) & ~0x1
        except Exception:
            pass

    def _run(self):
        while not self._stop.is_set():
            self._sample()
            self._stop.wait(self.period)

    def __enter__(self):
        if self.handle is not None:
            self._thread = threading.Thread(target=self._run, daemon=True)
            self._thread.start()
        return self

    def __exit__(self, *exc):
        if self._thread is not None:
            self._stop.set()
            self._thread.join()
            self._sample()

    def summary(self):
        if self.handle is None or not self.samples:
            return {"sm_mhz": None, "sm_max_mhz": self.max_mhz, "reasons": ["unavailable"], "samples": 0}
        names = [n for bit, n in self.REASONS.items() if self.reasons & bit]
        return {"sm_mhz": statistics.median(self.samples), "sm_max_mhz": self.max_mhz, "reasons": names,
                "samples": len(self.samples)}


def compulsory_bytes(points_in: int, points_out: int, elem: int, weights: int, bias: int, welem: int) -> int:
    return (points_in + points_out) * elem + (weights + bias) * welem


def rotate_sets(bytes_per_set: int, cap: int = 12) -> int:
    return max(2, min(cap, math.ceil(2 * L2_BYTES / max(1, bytes_per_set)) + 1))


# ---------------------------------------------------------------------------
# workloads
# ---------------------------------------------------------------------------
class StencilCfg2:
    """single-step 7x7 stencil fp32 4096x4096, x~U(-1,1), w~U(-1,1)/49, seed 1."""

    name = "stencil7x7_cfg2_4096x4096_f32"
    dtype = "f32"
    scaling = "weak"
    H = W = 4096

    def __init__(self, rank, world, dev):
        self.dev = dev
        g = torch.Generator().manual_seed(1)
        self.x_cpu = (torch.rand(1, 1, self.H, self.W, generator=g) * 2 - 1)
        self.w_cpu = (torch.rand(1, 1, 7, 7, generator=g) * 2 - 1) / 49
        self.b_cpu = (torch.rand(1, generator=g) * 2 - 1) / 49
        self.points = self.H * self.W
        self.bytes = compulsory_bytes(self.points, self.points, 4, TAPS, 1, 4)
        self.nsets = rotate_sets(2 * self.points * 4)
        self.launches_per_step = 1
        if dev is None:  # CPU reference arm only
            return
        from pla_b200.stencil import ModelNew

        self.model = ModelNew().to(dev)
        with torch.no_grad():
            self.model.conv1.weight.copy_(self.w_cpu)
            self.model.conv1.bias.copy_(self.b_cpu)
        x = self.x_cpu.to(dev)
        self.xs = [x] + [x.clone() for _ in range(self.nsets - 1)]
        self.ys = [torch.empty_like(x) for _ in range(self.nsets)]
        # Device-timed loop: the C-ABI call the module's default path makes
        # (pla_stencil7x7_forward: filter read from device memory by the
        # kernel), with its arguments bound once so the host keeps ahead of
        # the GPU.
        from pla_b200 import _lib

        L = _lib.lib()
        w, b = self.model.conv1.weight.detach(), self.model.conv1.bias.detach()
        stream = torch.cuda.current_stream(dev).cuda_stream
        self._call = L.pla_stencil7x7_forward
        self._args = [(self.xs[k].data_ptr(), w.data_ptr(), b.data_ptr(), self.ys[k].data_ptr(), 1, self.H,
                       self.W, self.H * self.W, self.W, 1, _lib.PLA_F32, stream) for k in range(self.nsets)]

    def config(self):
        return {"workload": self.name, "shape": [1, 1, self.H, self.W], "seed": 1, "bias": True,
                "x": "U(-1,1)", "w": "U(-1,1)/49",
                "l2": f"inputs rotate over {self.nsets} buffer sets "
                      f"({self.nsets * 2 * self.points * 4 >> 20} MiB > 126 MB L2)",
                "parallelism": "one grid per GPU (replicas, no collective)"}

    def step(self, i):
        st = self._call(*self._args[i % self.nsets])
        if st:
            raise RuntimeError(f"pla_stencil7x7_forward failed: {st}")

    graph_ok = True  # a step is one plain launch on the bound stream

    def rebind(self, stream_ptr):
        """Launch the bound calls on another stream (the CUDA-graph capture stream)."""
        self._args = [a[:-1] + (stream_ptr,) for a in self._args]

    # end-to-end through the public module API, pinned host buffers
    def e2e_setup(self):
        self.hx = [self.x_cpu.clone().pin_memory() for _ in range(2)]
        self.hy = [torch.empty_like(self.x_cpu).pin_memory() for _ in range(2)]
        self.dx = [torch.empty_like(self.xs[0]) for _ in range(2)]
        self.h2d_bytes = self.points * 4
        self.d2h_bytes = self.points * 4

    def e2e_step(self, i, s_in, s_cmp, s_out, ev):
        k = i % 2
        with torch.cuda.stream(s_in):
            s_in.wait_event(ev["cmp_done"][k]) if ev["cmp_done"][k] is not None else None
            self.dx[k].copy_(self.hx[k], non_blocking=True)
            ev["in_done"][k] = torch.cuda.Event()
            ev["in_done"][k].record(s_in)
        with torch.cuda.stream(s_cmp):
            s_cmp.wait_event(ev["in_done"][k])
            if ev["out_done"][k] is not None:
                s_cmp.wait_event(ev["out_done"][k])
            y = self.model(self.dx[k])
            ev["cmp_done"][k] = torch.cuda.Event()
            ev["cmp_done"][k].record(s_cmp)
        with torch.cuda.stream(s_out):
            s_out.wait_event(ev["cmp_done"][k])
            self.hy[k].copy_(y, non_blocking=True)
            y.record_stream(s_out)
            ev["out_done"][k] = torch.cuda.Event()
            ev["out_done"][k].record(s_out)

    # the reference's CPU path: data/stencil_7x7.py's Model (torch.nn.Conv2d)
    def cpu_reference(self):
        from oracle.reference_modules import StencilModel

        m = StencilModel()
        with torch.no_grad():
            m.conv1.weight.copy_(self.w_cpu)
            m.conv1.bias.copy_(self.b_cpu)
        x = self.x_cpu

        def run_rows(r0, r1):
            a0, a1 = max(0, r0 - 3), min(self.H, r1 + 3)
            with torch.no_grad():
                out = m(x[:, :, a0:a1])
            return out[:, :, r0 - a0:r1 - a0]

        def bytes_rows(nrows):
            return compulsory_bytes(nrows * self.W, nrows * self.W, 4, TAPS, 1, 4)

        return run_rows, bytes_rows, self.H, "torch.nn.Conv2d(1,1,7,padding=3) CPU forward " \
                                            "(data/stencil_7x7.py Model)"


class DepthwiseBase:
    scaling = "weak"
    stages: list = []  # (N, C, H, W)
    layout = "nchw"
    bias = True
    seed = 0
    torch_dtype = torch.float32
    k = 7               # filter side
    recipe = "normal"   # x ~ N(0,1), w ~ N(0,1/49), b ~ N(0,0.01), torch generator
    cpu_kind = "reference"

    def __init__(self, rank, world, dev):
        self.dev = dev
        self.taps = self.k * self.k
        if dev is not None:  # (the reference arm's process loads nothing of the package)
            from pla_b200.depthwise import depthwise7x7, depthwise_kxk

            self._fn = depthwise7x7 if self.k == 7 else depthwise_kxk
        es = torch.tensor([], dtype=self.torch_dtype).element_size()
        self.items = []
        self.bytes = 0
        self.points = 0
        per_set = 0
        for (N, C, H, W) in self.stages:
            n_local = self.local_batch(N, world, rank)
            if self.recipe == "uniform":
                # benchmark/MetaSchedule/common.py:176-177: numpy default_rng(seed), x then w ~ U(-1, 1)
                rng = np.random.default_rng(self.seed)
                x = torch.from_numpy(rng.uniform(-1, 1, (N, C, H, W)).astype(np.float32))
                x = x[self.batch_slice(N, world, rank)]
                w = torch.from_numpy(rng.uniform(-1, 1, (C, 1, self.k, self.k)).astype(np.float32))
                b = None
            else:
                g = torch.Generator().manual_seed(self.seed)
                x = torch.randn(N, C, H, W, generator=g)[self.batch_slice(N, world, rank)]
                w = torch.randn(C, 1, 7, 7, generator=g) / 7
                b = torch.randn(C, generator=g) * 0.1 if self.bias else None
            x, w = x.to(self.torch_dtype), w.to(self.torch_dtype)
            b = None if b is None else b.to(self.torch_dtype)
            pts = n_local * C * H * W
            self.points += pts
            self.bytes += compulsory_bytes(pts, pts, es, C * self.taps, C if self.bias else 0, es)
            per_set += 2 * pts * es
            self.items.append((x, w, b))
        self.nsets = rotate_sets(per_set)
        self.launches_per_step = len(self.stages)
        if dev is None:  # CPU reference arm only
            return
        fmt = torch.channels_last if self.layout == "nhwc" else torch.contiguous_format
        self.dev_items = []
        for (x, w, b) in self.items:
            xd = x.to(dev).contiguous(memory_format=fmt)
            xs = [xd] + [xd.clone() for _ in range(self.nsets - 1)]
            ys = [torch.empty_like(xd) for _ in range(self.nsets)]
            self.dev_items.append((xs, ys, w.to(dev), None if b is None else b.to(dev)))
        # Device-timed loop: pla_depthwise7x7_forward with arguments bound once.
        from pla_b200 import _lib

        L = _lib.lib()
        self._call = L.pla_depthwise7x7_forward if self.k == 7 else L.pla_depthwise_forward
        stream = torch.cuda.current_stream(dev).cuda_stream
        code = _lib.DTYPE_CODE[self.torch_dtype]
        lay = _lib.PLA_NHWC if self.layout == "nhwc" else _lib.PLA_NCHW
        self._args = []
        for k in range(self.nsets):
            per = []
            for (xs, ys, w, b) in self.dev_items:
                N, C, H, W = xs[k].shape
                shape = (N, C, H, W) if self.k == 7 else (N, C, H, W, self.k)
                per.append((xs[k].data_ptr(), w.data_ptr(), None if b is None else b.data_ptr(), ys[k].data_ptr(),
                            *shape, code, lay, stream))
            self._args.append(per)

    @staticmethod
    def local_batch(N, world, rank):
        return N

    @staticmethod
    def batch_slice(N, world, rank):
        return slice(0, N)

    graph_ok = True  # a step is one plain launch per stage on the bound stream

    def rebind(self, stream_ptr):
        """Launch the bound calls on another stream (the CUDA-graph capture stream)."""
        self._args = [[a[:-1] + (stream_ptr,) for a in per] for per in self._args]
        if self.concurrent:
            self._bind_many(stream_ptr)

    _stage_events = None

    def dominant_stage(self):
        """Index of the stage with the most compulsory bytes (the roofline kernel)."""
        sizes = [x.numel() for (x, _, _) in self.items]
        return sizes.index(max(sizes))

    def arm_stage_timing(self, steps):
        """Bracket the dominant stage's launch of the next `steps` steps with CUDA events."""
        self._stage_events = [(torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True))
                              for _ in range(steps)]
        self._stage_n = 0
        self._dom = self.dominant_stage()

    def stage_ms(self):
        """Mean device time of the dominant stage's launch over the armed steps (ms)."""
        evs, self._stage_events = self._stage_events, None
        return sum(a.elapsed_time(b) for a, b in evs) / len(evs)

    concurrent = False  # True: a step is one pla_depthwise7x7_forward_many call over all stages

    def _bind_many(self, stream_ptr):
        from pla_b200 import _lib

        code = _lib.DTYPE_CODE[self.torch_dtype]
        lay = _lib.PLA_NHWC if self.layout == "nhwc" else _lib.PLA_NCHW
        self._many = []
        for per in self._args:
            arr = (_lib.DwProblem * len(per))()
            for j, a in enumerate(per):
                arr[j] = _lib.DwProblem(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7])
            self._many.append((arr, len(per), code, lay, stream_ptr))
        self._many_call = _lib.lib().pla_depthwise7x7_forward_many

    def step(self, i):
        evs = self._stage_events
        if self.concurrent and evs is None:
            st = self._many_call(*self._many[i % self.nsets])
            if st:
                raise RuntimeError(f"pla_depthwise7x7_forward_many failed: {st}")
            return
        for j, args in enumerate(self._args[i % self.nsets]):
            if evs is not None and j == self._dom:
                evs[self._stage_n][0].record()
            st = self._call(*args)
            if st:
                raise RuntimeError(f"pla_depthwise7x7_forward failed: {st}")
            if evs is not None and j == self._dom:
                evs[self._stage_n][1].record()
                self._stage_n += 1

    def config(self):
        c = {"workload": self.name, "stages": [list(s) for s in self.stages], "layout": self.layout,
             "bias": self.bias, "seed": self.seed, "x": "N(0,1)", "w": "N(0,1/49)",
             "l2": f"inputs rotate over {self.nsets} buffer sets", "parallelism": self.parallelism}
        if self.concurrent:
            c["stream_pass"] = "stages one after another on one stream, the largest bracketed by CUDA events " \
                               "(roofline of that kernel)"
        return c

    parallelism = "one batch per GPU (replicas, no collective)"

    def e2e_setup(self):
        fmt = torch.channels_last if self.layout == "nhwc" else torch.contiguous_format
        self.hx = [[x.contiguous(memory_format=fmt).pin_memory() for (x, _, _) in self.items] for _ in range(2)]
        self.hy = [[torch.empty_like(h).pin_memory() for h in hs] for hs in self.hx]
        self.dx = [[torch.empty_like(xs[0]) for (xs, _, _, _) in self.dev_items] for _ in range(2)]
        es = torch.tensor([], dtype=self.torch_dtype).element_size()
        self.h2d_bytes = self.points * es
        self.d2h_bytes = self.points * es

    def e2e_step(self, i, s_in, s_cmp, s_out, ev):
        k = i % 2
        with torch.cuda.stream(s_in):
            if ev["cmp_done"][k] is not None:
                s_in.wait_event(ev["cmp_done"][k])
            for d, h in zip(self.dx[k], self.hx[k]):
                d.copy_(h, non_blocking=True)
            ev["in_done"][k] = torch.cuda.Event()
            ev["in_done"][k].record(s_in)
        with torch.cuda.stream(s_cmp):
            s_cmp.wait_event(ev["in_done"][k])
            if ev["out_done"][k] is not None:
                s_cmp.wait_event(ev["out_done"][k])
            if self.concurrent:
                from pla_b200.depthwise import depthwise7x7_many

                ys = depthwise7x7_many([(d, w, b) for d, (_, _, w, b) in zip(self.dx[k], self.dev_items)])
            else:
                ys = [self._fn(d, w, b) for d, (_, _, w, b) in zip(self.dx[k], self.dev_items)]
            ev["cmp_done"][k] = torch.cuda.Event()
            ev["cmp_done"][k].record(s_cmp)
        with torch.cuda.stream(s_out):
            s_out.wait_event(ev["cmp_done"][k])
            for hy, y in zip(self.hy[k], ys):
                hy.copy_(y, non_blocking=True)
                y.record_stream(s_out)
            ev["out_done"][k] = torch.cuda.Event()
            ev["out_done"][k].record(s_out)

    def cpu_reference(self):
        from oracle.reference_modules import DepthwiseModel

        mods = []
        for (x, w, b) in self.items:
            C = x.shape[1]
            m = DepthwiseModel(C, self.k, 1, self.k // 2, bias=b is not None).to(self.torch_dtype)
            with torch.no_grad():
                m.conv2d.weight.copy_(w)
                if b is not None:
                    m.conv2d.bias.copy_(b)
            xx = x.contiguous(memory_format=torch.channels_last) if self.layout == "nhwc" else x
            mods.append((m, xx))
        nb = self.items[0][0].shape[0]
        es = torch.tensor([], dtype=self.torch_dtype).element_size()

        def run_rows(r0, r1):  # "rows" = images of the batch here
            with torch.no_grad():
                for m, xx in mods:
                    m(xx[r0:r1])

        def bytes_rows(nimg):
            tot = 0
            for (x, w, b) in self.items:
                _, C, H, W = x.shape
                pts = nimg * C * H * W
                tot += compulsory_bytes(pts, pts, es, C * self.taps, C if b is not None else 0, es)
            return tot

        if self.k != 7:
            return run_rows, bytes_rows, nb, \
                f"torch.nn.Conv2d(C,C,{self.k},padding={self.k // 2},groups=C) CPU forward, the operator of " \
                f"benchmark/MetaSchedule/depthwise_conv.py (its own CPU check is numpy inside the reference " \
                f"tree, its GPU path TVM; neither is on this host), {self.layout}"
        return run_rows, bytes_rows, nb, f"torch.nn.Conv2d(C,C,7,padding=3,groups=C) CPU forward " \
                                         f"(data/depthwise_conv_7x7.py Model), {self.layout}"


class DwK3(DepthwiseBase):
    """3x3 depthwise of the reference's MetaSchedule benchmark at its logged 1x32x1024x1024 shape."""

    name = "depthwise3x3_metaschedule_1x32x1024x1024_f32"
    dtype = "f32"
    stages = [(1, 32, 1024, 1024)]
    k = 3
    bias = False
    seed = 0
    recipe = "uniform"
    cpu_kind = "port"


class DwCfg1(DepthwiseBase):
    name = "depthwise7x7_cfg1_1x96x56x56_f32"
    dtype = "f32"
    stages = [(1, 96, 56, 56)]
    seed = 0


class DwCfg3Nchw(DepthwiseBase):
    name = "depthwise7x7_cfg3_128x384x14x14_bf16_nchw"
    dtype = "bf16"
    torch_dtype = torch.bfloat16
    stages = [(128, 384, 14, 14)]
    seed = 2


class DwCfg3Nhwc(DwCfg3Nchw):
    name = "depthwise7x7_cfg3_128x384x14x14_bf16_nhwc"
    layout = "nhwc"


class DwCfg4(DepthwiseBase):
    name = "depthwise7x7_cfg4_convnext_t_N256_bf16"
    dtype = "bf16"
    torch_dtype = torch.bfloat16
    stages = [(256, 96, 56, 56), (256, 192, 28, 28), (256, 384, 14, 14), (256, 768, 7, 7)]
    bias = False
    seed = 3
    scaling = "strong"
    parallelism = "batch sharded over GPUs (N/world images per GPU), no collective; the four stages of a step " \
                  "run concurrently in one pla_depthwise7x7_forward_many call"
    concurrent = True

    def __init__(self, rank, world, dev):
        super().__init__(rank, world, dev)
        if dev is not None and self.concurrent:
            self._bind_many(torch.cuda.current_stream(dev).cuda_stream)

    @staticmethod
    def local_batch(N, world, rank):
        s = DwCfg4.batch_slice(N, world, rank)
        return s.stop - s.start

    @staticmethod
    def batch_slice(N, world, rank):
        base, extra = divmod(N, world)
        a = rank * base + min(rank, extra)
        return slice(a, a + base + (1 if rank < extra else 0))


class DwLnCfg4(DwCfg4):
    """dw_cfg4's ConvNeXt-T stages (seed 3) in channels_last, each followed by
    LayerNorm over C fused into the same launch (pla_depthwise7x7_layernorm_nhwc).

    LayerNorm scale / shift: 1 + 0.1 N(0,1) and 0.1 N(0,1) from a second
    generator seeded 3.  Compulsory bytes add the scale and shift.
    """

    name = "depthwise7x7_layernorm_cfg4_convnext_t_N256_bf16_nhwc"
    layout = "nhwc"
    ln_params = 2  # scale and shift: C elements each
    concurrent = False
    parallelism = "batch sharded over GPUs (N/world images per GPU), no collective"

    def __init__(self, rank, world, dev):
        super().__init__(rank, world, dev)
        g = torch.Generator().manual_seed(3)
        es = torch.tensor([], dtype=self.torch_dtype).element_size()
        self.norm = []
        for (x, _, _) in self.items:
            C = x.shape[1]
            gamma = (1 + 0.1 * torch.randn(C, generator=g)).to(self.torch_dtype)
            beta = (0.1 * torch.randn(C, generator=g)).to(self.torch_dtype)
            self.norm.append((gamma, beta))
            self.bytes += 2 * C * es
        self._fn = None
        if dev is None:
            return
        from pla_b200 import _lib
        from pla_b200.depthwise import depthwise7x7_layernorm

        self.dev_norm = [(g_.to(dev), b_.to(dev)) for (g_, b_) in self.norm]
        self._ln_fn = depthwise7x7_layernorm
        self._call = _lib.lib().pla_depthwise7x7_layernorm_nhwc
        stream = torch.cuda.current_stream(dev).cuda_stream
        code = _lib.DTYPE_CODE[self.torch_dtype]
        self._args = []
        for k in range(self.nsets):
            per = []
            for (xs, ys, w, b), (gd, bd) in zip(self.dev_items, self.dev_norm):
                N, C, H, W = xs[k].shape
                per.append((xs[k].data_ptr(), w.data_ptr(), None if b is None else b.data_ptr(), gd.data_ptr(),
                            bd.data_ptr(), 1e-6, ys[k].data_ptr(), N, C, H, W, code, stream))
            self._args.append(per)

    def config(self):
        c = super().config()
        c.update({"layernorm": "over C per pixel, eps 1e-6, scale 1+0.1N(0,1), shift 0.1N(0,1), fp32 math on "
                               "the bf16-rounded depthwise outputs"})
        return c

    def e2e_step(self, i, s_in, s_cmp, s_out, ev):
        self._fn = lambda d, w, b: self._ln_fn(d, w, b, *self.dev_norm[self._stage_of_input(d)], eps=1e-6)
        return super().e2e_step(i, s_in, s_cmp, s_out, ev)

    def _stage_of_input(self, d):
        return [xs[0].shape for (xs, _, _, _) in self.dev_items].index(d.shape)

    def unfused_ms(self, steps):
        """Device time per step of the unfused pair on the same inputs: this
        library's NHWC depthwise, then torch's LayerNorm on the NHWC view."""
        from pla_b200.depthwise import depthwise7x7

        def one(i):
            k = i % self.nsets
            for (xs, ys, w, b), (gd, bd) in zip(self.dev_items, self.dev_norm):
                y = depthwise7x7(xs[k], w, b, out=ys[k])
                torch.nn.functional.layer_norm(y.permute(0, 2, 3, 1), (y.shape[1],), gd, bd, 1e-6)

        for i in range(3):
            one(i)
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        e0.record()
        for i in range(steps):
            one(i)
        e1.record()
        torch.cuda.synchronize()
        return e0.elapsed_time(e1) / steps

    def cpu_reference(self):
        from oracle.reference_modules import DepthwiseModel

        mods = []
        for (x, w, b), (gamma, beta) in zip(self.items, self.norm):
            C = x.shape[1]
            m = DepthwiseModel(C, 7, 1, 3, bias=b is not None).to(self.torch_dtype)
            with torch.no_grad():
                m.conv2d.weight.copy_(w)
            mods.append((m, x.contiguous(memory_format=torch.channels_last), gamma, beta))
        nb = self.items[0][0].shape[0]
        es = torch.tensor([], dtype=self.torch_dtype).element_size()

        def run_rows(r0, r1):
            with torch.no_grad():
                for m, xx, gamma, beta in mods:
                    y = m(xx[r0:r1])
                    torch.nn.functional.layer_norm(y.permute(0, 2, 3, 1), (y.shape[1],), gamma, beta, 1e-6)

        def bytes_rows(nimg):
            tot = 0
            for (x, w, b) in self.items:
                _, C, H, W = x.shape
                pts = nimg * C * H * W
                tot += compulsory_bytes(pts, pts, es, C * TAPS, 2 * C, es)
            return tot

        return run_rows, bytes_rows, nb, "torch.nn.Conv2d(C,C,7,padding=3,groups=C) (data/depthwise_conv_7x7.py " \
                                         "Model) then torch.nn.functional.layer_norm over C, CPU, channels_last"


class IterateCfg5:
    """the 32768^2 fp32 iterated stencil (seed 4), row-band partitioned.

    A step is one Jacobi step of the whole grid: every rank advances its band
    (BandedStencil; at N > 1 one fused kernel per step that also stores the
    band's edge rows into the neighbours' halos over NVLink).  The e2e job is
    the configuration's whole job through the same public API: the band from
    pinned host memory, 100 steps, the band back to pinned host memory.
    """

    name = "iterate7x7_cfg5_32768x32768_f32_step"
    dtype = "f32"
    scaling = "strong"
    job_steps = 100    # the configuration's time steps
    parity_steps = 2

    def __init__(self, rank, world, dev, H=32768):
        self.H = self.W = H
        self.name = f"iterate7x7_cfg5_{H}x{H}_f32_step"
        self.rank, self.world, self.dev = rank, world, dev
        g = torch.Generator().manual_seed(4)
        self.r0, self.r1 = 0, H
        if world > 1:  # (the reference arm's process loads nothing of the package)
            from pla_b200.iterate import band_rows

            self.r0, self.r1 = band_rows(H, world, rank)
        self.rows = self.r1 - self.r0
        # Grid rows [s0, s1) on the host: the band, its 3 halo rows and 3 more
        # on each side (a two-step parity check of an edge row reads 6 rows
        # past it).  Pinned: the e2e job copies the band from here.
        self.s0, self.s1 = max(0, self.r0 - 6), min(H, self.r1 + 6)
        self.slab = self._rows(g, self.s0, self.s1, pin=dev is not None)
        w = torch.rand(7, 7, generator=g) * 2 - 1
        self.w_cpu = w / w.sum()
        self.points = self.rows * self.W
        self.bytes = compulsory_bytes(self.points, self.points, 4, TAPS, 0, 4)
        self.nsets = 1
        self.launches_per_step = 1
        if dev is None:  # CPU reference arm only
            return
        from pla_b200.iterate import BandedStencil

        self.bs = BandedStencil(H, self.W, self.w_cpu.to(dev), group=None, device=dev)
        if world > 1 and self.bs.mode != "p2p":
            self.launches_per_step = 3  # edge rows, interior, edge rows (NCCL exchange on a side stream)
        self.bs.load(self.slab, row0=self.s0)

    def _rows(self, g, a0, a1, pin=False):
        # Rows a0..a1 of the seeded U(-1,1) grid, drawn in grid order (row blocks).
        # Every rank draws the same full sequence but keeps only its rows, in
        # chunks, so no rank holds the 4 GiB grid.
        out = torch.empty(a1 - a0, self.W, pin_memory=pin)
        chunk = 1024
        for r in range(0, self.H, chunk):
            blk = torch.rand(min(chunk, self.H - r), self.W, generator=g) * 2 - 1
            lo, hi = max(r, a0), min(r + blk.shape[0], a1)
            if lo < hi:
                out[lo - a0:hi - a0].copy_(blk[lo - r:hi - r])
        return out

    def step(self, i):
        self.bs.step()

    def close(self):
        self.bs.check_faults()
        self.bs.close()

    def config(self):
        if self.world == 1:
            par = "one band (the whole grid) on one GPU, zero halos (Dirichlet boundary)"
        elif self.bs.mode == "p2p":
            par = ("row bands, 3-row halo exchange per step fused into the step kernel (edge tiles first, "
                   "rows stored into the neighbours' halos over NVLink via CUDA IPC, flag handshake; no "
                   "collective call)")
        else:
            par = "row bands, 3-row halo exchange per step (NCCL send/recv on a side stream, overlapped with " \
                  "interior rows)"
        return {"workload": self.name, "shape": [self.H, self.W], "seed": 4, "x": "U(-1,1)",
                "w": "U(-1,1) normalised to sum 1", "bias": False, "steps_per_job": self.job_steps,
                "l2": f"{self.H * self.W * 4 >> 20} MiB grid per buffer (> 126 MB L2 from 6144^2 up)",
                "parallelism": par}

    # -- end to end: the configuration's whole job through the public API --
    def e2e_setup(self):
        a0, a1 = self.bs.halo_span()
        self.host_out = torch.empty(self.rows, self.W, pin_memory=True)
        self.h2d_job = (a1 - a0) * self.W * 4
        self.d2h_job = self.host_out.numel() * 4

    def e2e_job(self):
        """Band + halo rows pinned host -> device, job_steps steps, band -> pinned host
        (BandedStencil.run_job: on one GPU the copies overlap the first and last steps)."""
        self.bs.run_job(self.slab, self.s0, self.job_steps, self.host_out)

    # -- parity: the CPU oracle is the checker here, after all timing -------
    def parity_segments(self):
        """Band rows checked: the 3 edge rows at each end, the 3 rows inside
        each of them (the rows next to the halo exchange) and 4 seeded interior
        rows, as [c0, c1) segments."""
        R = self.rows
        segs = [(0, min(6, R)), (max(0, R - 6), R)]
        inner = list(range(6, R - 6))
        pick = np.random.default_rng(4 + self.rank).choice(len(inner), size=min(4, len(inner)), replace=False) \
            if inner else []
        segs += [(inner[k], inner[k] + 1) for k in sorted(pick)]
        return segs

    def parity(self):
        """Reload the seeded grid, run parity_steps steps and compare rows of
        this rank's band bit for bit with the CPU oracle (oracle/pla_oracle.c)
        run on the grid rows they depend on."""
        from oracle import oracle

        self.bs.load(self.slab, row0=self.s0)
        self.bs.run(self.parity_steps)
        if self.bs.device.type == "cuda":
            torch.cuda.synchronize(self.bs.device)
            self.bs.check_faults()
        n, bad = 0, []
        reach = 3 * self.parity_steps
        for c0, c1 in self.parity_segments():
            g0, g1 = self.r0 + c0, self.r0 + c1
            i0, i1 = max(0, g0 - reach), min(self.H, g1 + reach)
            sub = self.slab[i0 - self.s0:i1 - self.s0].contiguous()
            ref = oracle.stencil7x7_iterate(sub, self.w_cpu, self.parity_steps)[g0 - i0:g1 - i0]
            got = self.bs.band()[c0:c1].cpu()
            n += c1 - c0
            if not torch.equal(got, ref):
                bad.append(f"rank {self.rank} grid rows [{g0}, {g1}): "
                           f"{int((got != ref).sum())} of {got.numel()} points differ")
        return {"rows_checked": n, "mismatches": bad}

    def cpu_reference(self):
        from oracle.reference_modules import StencilModel

        m = StencilModel()
        with torch.no_grad():
            m.conv1.weight.copy_(self.w_cpu.view(1, 1, 7, 7))
            m.conv1.bias = None
        slab, rows, off = self.slab, self.rows, self.r0 - self.s0

        def run_rows(r0, r1):
            # band rows [r0, r1) from grid rows r0 - 3 .. r1 + 3 (zero rows
            # outside the grid, as the Dirichlet boundary)
            a0, a1 = off + r0 - 3, off + r1 + 3
            x = slab[max(0, a0):min(slab.shape[0], a1)]
            if a0 < 0 or a1 > slab.shape[0]:
                x = torch.nn.functional.pad(x, (0, 0, max(0, -a0), max(0, a1 - slab.shape[0])))
            with torch.no_grad():
                return m(x.reshape(1, 1, r1 - r0 + 6, self.W))

        def bytes_rows(n):
            return compulsory_bytes(n * self.W, n * self.W, 4, TAPS, 0, 4)

        return run_rows, bytes_rows, rows, "torch.nn.Conv2d(1,1,7,padding=3) CPU forward " \
                                           "(data/stencil_7x7.py Model), row bands"


WORKLOADS = {"stencil_cfg2": StencilCfg2, "dw_cfg1": DwCfg1, "dw_cfg3_nchw": DwCfg3Nchw,
             "dw_cfg3_nhwc": DwCfg3Nhwc, "dw_cfg4": DwCfg4, "iterate_cfg5": IterateCfg5, "dw_k3": DwK3,
             "dwln_cfg4": DwLnCfg4}


# ---------------------------------------------------------------------------
# CPU timing of the reference path (bounded sample)
# ---------------------------------------------------------------------------
def time_cpu_reference(wl, budget_s: float, steps: int | None = None, warmup: int = 0):
    """Time the reference's CPU path on a bounded sample; returns (GB/s, detail dict)."""
    run_rows, bytes_rows, nrows, what = wl.cpu_reference()
    threads = os.cpu_count() or 1
    torch.set_num_threads(threads)
    # probe: size one sample so the whole measurement fits the budget
    probe = max(1, min(nrows, 64))
    t0 = time.perf_counter()
    run_rows(0, probe)
    t_probe = max(1e-6, time.perf_counter() - t0)
    per_row = t_probe / probe
    if steps is None:
        target = min(2.0, budget_s / 5)
        n_calls = None
    else:
        target = max(0.002, budget_s / max(1, steps + warmup))
        n_calls = steps
    rows = int(max(1, min(nrows, target / per_row)))
    times = []
    for _ in range(warmup):
        run_rows(0, rows)
    t_start = time.perf_counter()
    i = 0
    while True:
        r0 = (i * rows) % max(1, nrows - rows + 1)
        t0 = time.perf_counter()
        run_rows(r0, r0 + rows)
        times.append(time.perf_counter() - t0)
        i += 1
        if n_calls is not None:
            if i >= n_calls:
                break
        elif (time.perf_counter() - t_start > budget_s and i >= 3) or i >= 50:
            break
    total = sum(times)
    gbs = bytes_rows(rows) * len(times) / total / 1e9
    sample = f"{what}; {len(times)} calls of {rows} of {nrows} rows/images each, " \
             f"{total:.2f} s, {threads} threads (OMP_NUM_THREADS={os.environ.get('OMP_NUM_THREADS', 'unset')})"
    return gbs, {"value": gbs, "unit": "GB/s", "cores": torch.get_num_threads(),
                 "kind": getattr(wl, "cpu_kind", "reference"),
                 "sample": sample, "s_per_call": total / len(times)}


# ---------------------------------------------------------------------------
# main
# ---------------------------------------------------------------------------
def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--gpus", type=int, default=1)
    ap.add_argument("--steps", type=int, default=400)
    ap.add_argument("--warmup", type=int, default=10)
    ap.add_argument("--impl", choices=["ours", "reference"], default="ours")
    ap.add_argument("--workload", choices=sorted(WORKLOADS), default="iterate_cfg5")
    ap.add_argument("--e2e-steps", type=int, default=20)
    ap.add_argument("--grid", type=int, default=32768,
                    help="iterate_cfg5 grid side (32768 is the configuration; smaller for profiling captures)")
    ap.add_argument("--cpu-budget", type=float, default=15.0, help="seconds of CPU work for cpu_baseline")
    ap.add_argument("--no-cpu-baseline", action="store_true")
    ap.add_argument("--no-graph", action="store_true", help="time the K steps as stream launches, no CUDA graph")
    args = ap.parse_args()
    if args.warmup < 3:
        args.warmup = 3

    world = int(os.environ.get("WORLD_SIZE", "1"))
    rank = int(os.environ.get("RANK", "0"))
    local_rank = int(os.environ.get("LOCAL_RANK", "0"))
    Wl = WORKLOADS[args.workload]

    if args.impl == "reference":
        return run_reference(args, Wl, rank, world)

    dev = torch.device("cuda", local_rank)
    torch.cuda.set_device(dev)
    if world > 1:
        import datetime

        dist.init_process_group("nccl", device_id=dev, timeout=datetime.timedelta(seconds=120))

    wl = Wl(rank, world, dev, H=args.grid) if Wl is IterateCfg5 else Wl(rank, world, dev)
    # Workloads whose step is one plain launch per stage run their K timed
    # steps as one CUDA graph (captured once, replayed once): the graph holds
    # exactly those K steps' launches with the same bound arguments, and the
    # host's per-launch submission drops out of the device timeline.
    # --no-graph times the K steps as stream launches instead.  The multi-GPU
    # iterated stencil (halo exchange) always runs as stream launches.
    use_graph = getattr(wl, "graph_ok", False) and not args.no_graph
    if use_graph:
        stream = torch.cuda.Stream(dev)
        wl.rebind(stream.cuda_stream)
        torch.cuda.set_stream(stream)
    else:
        stream = torch.cuda.current_stream(dev)

    def barrier():
        if world > 1:
            dist.barrier()
        torch.cuda.synchronize(dev)

    def run_steps(first, n):
        for i in range(n):
            wl.step(first + i)

    run_steps(0, args.warmup)
    barrier()

    K = args.steps
    # One event pair around the K steps: events between steps would add
    # their own gaps to the kernels they bracket.  Steps of several launches
    # (the ConvNeXt sweep) also bracket their dominant launch, for the
    # roofline of that kernel (in stream mode: in the timed loop; in graph
    # mode: in the stream-mode pass after it).
    multi = getattr(wl, "launches_per_step", 1) > 1 and hasattr(wl, "arm_stage_timing")
    graph = None
    if use_graph:
        graph = torch.cuda.CUDAGraph()
        # thread_local: the process group's watchdog thread may query its
        # (completed) events while this thread captures.
        with torch.cuda.graph(graph, stream=stream, capture_error_mode="thread_local"):
            run_steps(args.warmup, K)
        # One untimed replay: the GPU idled through the capture.
        graph.replay()
        barrier()
    elif multi:
        wl.arm_stage_timing(K)
    e_start, e_end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    with ClockSampler(dev) as clk:
        barrier()
        t_wall = time.perf_counter()
        e_start.record(stream)
        if graph is not None:
            graph.replay()
        else:
            run_steps(args.warmup, K)
        e_end.record(stream)
        barrier()
        t_wall = time.perf_counter() - t_wall
    total_ms = e_start.elapsed_time(e_end)
    mean_step_ms = total_ms / K
    stream_ms_per_step = None
    if graph is not None:
        del graph
        # The same K steps as stream launches, for comparison (this rank).
        if multi:
            wl.arm_stage_timing(K)
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        barrier()
        e0.record(stream)
        run_steps(args.warmup, K)
        e1.record(stream)
        barrier()
        stream_ms_per_step = e0.elapsed_time(e1) / K
    dom_ms = wl.stage_ms() if multi else None
    t = torch.tensor([total_ms, float(wl.bytes), float(wl.points)], dtype=torch.float64, device=dev)
    if world > 1:
        tmax = t[:1].clone()
        dist.all_reduce(tmax, op=dist.ReduceOp.MAX)
        sums = t[1:].clone()
        dist.all_reduce(sums, op=dist.ReduceOp.SUM)
        total_ms_max = tmax.item()
        job_bytes, job_points = sums[0].item(), sums[1].item()
    else:
        total_ms_max, job_bytes, job_points = total_ms, float(wl.bytes), float(wl.points)
    ms_per_step = total_ms_max / K
    value = job_bytes / (ms_per_step * 1e-3) / 1e9
    gpoints = job_points / (ms_per_step * 1e-3) / 1e9

    # ---- end to end through the public API, pinned host buffers ----------
    e2e = None
    if hasattr(wl, "e2e_job"):
        # The configuration's whole job (H2D of the inputs, all its steps, D2H
        # of the result) per timed region; the copies are amortised over the
        # job's steps.
        wl.e2e_setup()
        barrier()
        wl.e2e_job()  # untimed
        barrier()
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        e0.record(stream)
        wl.e2e_job()
        e1.record(stream)
        barrier()
        e_ms = torch.tensor([e0.elapsed_time(e1)], dtype=torch.float64, device=dev)
        if world > 1:
            dist.all_reduce(e_ms, op=dist.ReduceOp.MAX)
        J = wl.job_steps
        e_step = e_ms.item() / J
        e2e = {"value": job_bytes / (e_step * 1e-3) / 1e9, "unit": "GB/s", "gpoints_per_s":
               job_points / (e_step * 1e-3) / 1e9, "ms_per_step": e_step, "steps": J, "ms_per_job": e_ms.item(),
               "h2d_bytes_per_step": int(wl.h2d_job // J), "d2h_bytes_per_step": int(wl.d2h_job // J),
               "h2d_bytes_per_job": int(wl.h2d_job), "d2h_bytes_per_job": int(wl.d2h_job),
               "path": f"per rank: band + halo rows pinned host -> device, {J} Jacobi steps, band -> pinned "
                       f"host, through BandedStencil.run_job, all in one timed region (max over ranks; one "
                       f"band: the copies run in 16 row chunks on a side stream, overlapped with the first "
                       f"and last steps); bytes per step = bytes per job / {J}"}
    else:
        wl.e2e_setup()
        s_in, s_cmp, s_out = torch.cuda.Stream(dev), torch.cuda.Stream(dev), torch.cuda.Stream(dev)
        evs = {"in_done": [None, None], "cmp_done": [None, None], "out_done": [None, None]}
        for i in range(2):
            wl.e2e_step(i, s_in, s_cmp, s_out, evs)
        barrier()
        E = max(1, args.e2e_steps)
        e0, e1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        barrier()
        e0.record(stream)
        s_in.wait_stream(stream)
        for i in range(E):
            wl.e2e_step(i, s_in, s_cmp, s_out, evs)
        stream.wait_stream(s_out)
        e1.record(stream)
        barrier()
        e_ms = torch.tensor([e0.elapsed_time(e1)], dtype=torch.float64, device=dev)
        if world > 1:
            dist.all_reduce(e_ms, op=dist.ReduceOp.MAX)
        e_step = e_ms.item() / E
        e2e = {"value": job_bytes / (e_step * 1e-3) / 1e9, "unit": "GB/s", "gpoints_per_s":
               job_points / (e_step * 1e-3) / 1e9, "ms_per_step": e_step, "steps": E,
               "h2d_bytes_per_step": int(wl.h2d_bytes), "d2h_bytes_per_step": int(wl.d2h_bytes),
               "path": "pinned host -> H2D (stream A) -> public API call (stream B) -> D2H (stream C), "
                       "double-buffered"}

    # ---- parity: after all timing, the CPU oracle checks rows of the result
    parity = None
    if hasattr(wl, "parity"):
        res = wl.parity()
        bad = torch.tensor([len(res["mismatches"])], dtype=torch.float64, device=dev)
        if world > 1:
            dist.all_reduce(bad, op=dist.ReduceOp.SUM)
            lists = [None] * world
            dist.all_gather_object(lists, res["mismatches"])
            mism = [m for lst in lists for m in lst]
        else:
            mism = res["mismatches"]
        parity = {"status": "ok" if bad.item() == 0 else "MISMATCH", "mismatches": mism[:8],
                  "rows_checked_per_rank": res["rows_checked"],
                  "what": f"after the timed region: the seeded grid reloaded, {wl.parity_steps} steps, then "
                          "every rank's 3 edge rows at each end, the 3 rows inside them and 4 seeded interior "
                          "rows compared bit for bit with the CPU oracle (oracle/pla_oracle.c) run on the grid "
                          "rows they depend on"}

    clocks = clk.summary()
    peak, peak_kind = measured_peaks()
    # per-rank compulsory bytes of one step over that step's event-timed
    # duration (this rank's launches back to back, gaps included)
    achieved = wl.bytes / (mean_step_ms * 1e-3) / 1e9
    kernel_bytes, kernel_ms, kernel_what = wl.bytes // max(1, wl.launches_per_step), \
        mean_step_ms / max(1, wl.launches_per_step), "every launch of the step"
    if dom_ms is not None:
        d = wl.dominant_stage()
        dx = wl.items[d][0]
        es = dx.element_size()
        kernel_bytes = compulsory_bytes(dx.numel(), dx.numel(), es, dx.shape[1] * TAPS,
                                        dx.shape[1] * ((wl.items[d][2] is not None) + getattr(wl, "ln_params", 0)),
                                        es)
        kernel_ms = dom_ms
        kernel_what = f"launch of stage {list(dx.shape)} (the step's largest), CUDA events in the timed region"
    sm_mhz = clocks.get("sm_mhz") or 1965
    fma_gpts = torch.cuda.get_device_properties(dev).multi_processor_count * FMA_PER_SM_PER_CLK * sm_mhz * 1e6 \
        / getattr(wl, "taps", TAPS) / 1e9

    unfused = None
    if hasattr(wl, "unfused_ms"):
        u_ms = wl.unfused_ms(max(3, min(K, 50)))
        unfused = {"ms_per_step": u_ms, "value": wl.bytes / (u_ms * 1e-3) / 1e9, "unit": "GB/s",
                   "what": "same inputs, unfused: pla_b200 NHWC depthwise, then torch.nn.functional.layer_norm "
                           "on the NHWC view (a second pass over HBM)"}
    traffic, traffic_src = profiled_traffic(wl.name)
    cpu_baseline = None
    if rank == 0 and world == 1 and not args.no_cpu_baseline:
        _, cpu_baseline = time_cpu_reference(wl, args.cpu_budget)

    if rank == 0:
        line = {
            "metric": METRIC, "value": value, "unit": "GB/s", "n_gpus": world, "steps": K,
            "warmup": args.warmup, "ms_per_step": ms_per_step, "higher_is_better": True,
            "scaling": wl.scaling, "vs_baseline": None, "dtype": wl.dtype,
            "data": "synthetic (seeded generator draws of the benchmark recipe)", "config": wl.config(),
            "gpoints_per_s": gpoints, "frac_of_8tbs": value / world / NOMINAL_HBM_GBS,
            "roofline": {"bound": "hbm", "achieved": kernel_bytes / (kernel_ms * 1e-3) / 1e9, "peak": peak,
                         "unit": "GB/s", "frac": kernel_bytes / (kernel_ms * 1e-3) / 1e9 / peak,
                         "peak_source": f"{peak_kind} (MEASURED_PEAKS.json hbm_gbs)"
                         if peak_kind == "measured" else "fallback 6.65 TB/s",
                         "traffic": traffic, "traffic_source": traffic_src,
                         "kernel": kernel_what,
                         "algorithmic_bytes_per_launch": kernel_bytes,
                         "per_launch_ms": kernel_ms,
                         "step_achieved": achieved, "step_frac": achieved / peak,
                         "fma_ceiling_gpoints_per_s": fma_gpts,
                         "fma_frac": (job_points / world) / (mean_step_ms * 1e-3) / 1e9 / fma_gpts},
            "cpu_baseline": cpu_baseline, "e2e": e2e, **({"unfused_pair": unfused} if unfused else {}),
            **({"parity": parity} if parity else {}),
            "gpu_launches": K * wl.launches_per_step, "clocks": clocks,
            "launch_mode": "one CUDA graph of the K steps, replayed once" if use_graph else "stream launches",
            **({"stream_ms_per_step": stream_ms_per_step} if stream_ms_per_step is not None else {}),
            "wall_s_timed_region": t_wall,
        }
        print(json.dumps(line), flush=True)
    if hasattr(wl, "close"):
        wl.close()
    if world > 1:
        dist.barrier()
        dist.destroy_process_group()
    if parity and parity["status"] != "ok":
        return 3


def run_reference(args, Wl, rank, world):
    """--impl reference: the reference's CPU path (torch.nn.Conv2d modules of
    data/stencil_7x7.py / data/depthwise_conv_7x7.py) on the host cores."""
    if rank != 0:
        return 0
    wl = Wl(0, 1, None, H=args.grid) if Wl is IterateCfg5 else Wl(0, 1, None)
    budget = 120.0
    gbs, cpu = time_cpu_reference(wl, budget, steps=args.steps, warmup=args.warmup)
    s_per = cpu["s_per_call"]
    line = {
        "metric": METRIC, "value": gbs, "unit": "GB/s", "n_gpus": world, "steps": args.steps,
        "warmup": args.warmup, "ms_per_step": s_per * 1e3, "higher_is_better": True, "scaling": wl.scaling,
        "vs_baseline": None, "dtype": wl.dtype, "data": "synthetic (seeded generator draws of the benchmark recipe)",
        "config": wl.config(), "impl": "reference", "cpu_baseline": cpu,
        "e2e": {"value": gbs, "unit": "GB/s", "h2d_bytes_per_step": 0, "d2h_bytes_per_step": 0},
    }
    print(json.dumps(line), flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main() or 0)
