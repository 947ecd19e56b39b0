"""
Benchmark of the attorch layer-kernel hot path on one MI355X.

    python bench.py [--gpus 1] [--steps K] [--warmup W] [--configs c1,c2,c2x8,c3,c5] [--no-cpu]
                    [--detail-file PATH]

A "step" is one forward + backward pass of the headline workload over one batch of synthetic
input that is already resident in HBM: attorch_amd.Linear with fused GELU(tanh), bf16,
X[16384, 4096] x W[4096, 16384] (the configuration the 70 %-of-MFMA-peak
target is quoted on).  stdout ends with ONE compact JSON line (a few KB); besides the contract
fields it carries
  roofline      the dominant kernel (the forward MFMA GEMM with its fused epilogue) against
                the MI355X dense bf16 MFMA peak, timed with HIP events on the launch stream
  cpu_baseline  the CPU oracle of the same workload on a bounded sample of rows, timed on
                this host's cores (a reported baseline, not a target)
  amp           the same step with float32 tensors under torch.autocast(float16) against the
                step on float16 tensors
  configs       the other BASELINE configs (c1 Linear fp32, c2 LayerNorm / RMSNorm / Softmax
                / LogSoftmax, c2x8 the same layers on eight times the rows, c3 CrossEntropy,
                c5 Conv2d + BatchNorm2d), each as tag, absolute throughput, fraction of its
                roofline, measured HBM traffic and CPU baseline.
The full record (module-level and torch-native timings, CPU functional baselines, notes) is
written to --detail-file (bench_detail.json in the run-output folder beside this script by
default).
Buffers of the bandwidth-bound configs are rotated over several sets so the 256 MB Infinity
Cache cannot serve them.  Secondary configs are timed with 10 warm-up and 60 timed calls (median
of 6 groups of 10) whatever --steps says.
"""

import argparse
import json
import os
import sys
import time
from typing import Callable, Dict, List, Optional, Tuple

import torch

PEAK_HBM_GBS = 8000.0          # MI355X HBM3E, GB/s
PEAK_MFMA_16BIT_TFLOPS = 2500.0  # dense bf16 / fp16 MFMA
PEAK_MFMA_FP32_TFLOPS = 157.3    # dense fp32 MFMA

# Bytes that cross between L2 and the memory fabric per launch (per forward + backward for the
# multi-kernel workloads), from the rocprofv3 FETCH_SIZE / WRITE_SIZE passes summarised in
# profiles/bench_all_configs.hbm_traffic.txt (scaled there by a copy of known size).  Counters are
# taken in separate profiling runs, so these are recorded measurements, not live ones; reads that
# the 256 MB Infinity Cache serves are included.  They belong to the kernel sources whose digest is
# TRAFFIC_SOURCE_DIGEST: when the sources of the loaded library differ, `traffic` is reported as
# null and the recorded figure moves to `traffic_recorded` (stale until the profile is redone).
TRAFFIC_SOURCE_DIGEST = 'adaa724635842b9f'
MEASURED_TRAFFIC_BYTES = {
    'c4_linear_fwd': 4705493680,      # gemm_mfma16_kernel<bf16, ..., GELU-tanh>: 3.7 GiB read, 1.0 GiB written
    'c2_layer_norm': 362246782,       # norm_fwd + norm_bwd + reduce_partials
    'c2_rms_norm': 361809038,
    'c2_softmax': 335901896,          # softmax_fwd + softmax_bwd (same kernels for log-softmax)
    'c2_act_dropout': 335771228,      # act_dropout forward + backward
    'c2_glu': 268579817,              # glu forward + backward
    'c2_mse': 335723406,              # p_loss forward + backward
    'c3_cross_entropy': 1683527018,   # ce_row_kernel (ignored rows are not read)
    'c3_cross_entropy_autocast': 2436782254,
    'c3_nll_loss': 826899934,         # nll forward (a gather) + the single-pass gradient write
    'c5_conv_channels_last': 397515918,     # the two ring kernels + weight gradient + weight reorders, no copies
    'c5_conv': 595354072,             # the same + 2 layout copies
    'c5_batch_norm_channels_last': 567988040,
    'c5_batch_norm': 565877886,       # stats + apply + backward reduce + backward apply
}


def kernel_source_digest() -> str:
    """
    Digest of the sources (csrc/*.hip, csrc/*.h, include/*.h) of the kernels measured here, which the
    files of the attention and rotary kernels are not among.
    """
    import hashlib
    root = os.path.dirname(os.path.abspath(__file__))
    h = hashlib.sha256()
    files = []
    for sub in ('attorch_amd/csrc', 'include'):
        d = os.path.join(root, sub)
        files += [os.path.join(d, f) for f in os.listdir(d)
                  if f.endswith(('.hip', '.h')) and not f.startswith(('attention', 'rotary'))]
    for f in sorted(files):
        h.update(os.path.basename(f).encode())
        with open(f, 'rb') as fh:
            h.update(fh.read())
    return h.hexdigest()[:16]


_DIGEST_MATCHES = None
MODULE_TIMINGS = True


def traffic_fields(key: str) -> Dict:
    """
    {'traffic': bytes or None} for a roofline object, plus provenance when a figure is recorded.
    """
    global _DIGEST_MATCHES
    if _DIGEST_MATCHES is None:
        _DIGEST_MATCHES = kernel_source_digest() == TRAFFIC_SOURCE_DIGEST
    recorded = MEASURED_TRAFFIC_BYTES.get(key)
    if recorded is None:
        return {'traffic': None}
    if _DIGEST_MATCHES:
        return {'traffic': recorded, 'traffic_source': 'profiles/bench_all_configs.hbm_traffic.txt'}
    return {'traffic': None, 'traffic_recorded': recorded,
            'traffic_note': 'recorded for other kernel sources than the ones loaded; see profiles/'}


def parse_args() -> argparse.Namespace:
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawTextHelpFormatter)
    parser.add_argument('--gpus', type=int, default=1)
    parser.add_argument('--steps', type=int, default=20)
    parser.add_argument('--warmup', type=int, default=5)
    parser.add_argument('--configs', type=str, default='c1,c2,c2x8,c3,c5',
                        help='secondary configs to measure besides the headline (c4); "none" skips them')
    parser.add_argument('--no-cpu', action='store_true', help='skip the CPU baselines')
    parser.add_argument('--no-modules', action='store_true',
                        help='skip the module-level (nn.Module + autograd, eager and HIP graph) timings; '
                             'hardware-counter runs use this to profile the C-ABI launches only')
    parser.add_argument('--calibrate-copy', action='store_true',
                        help='also run a plain 256 MiB -> 256 MiB device copy, the known-size kernel that '
                             'hardware byte counters of a profiling run are scaled by')
    parser.add_argument('--detail-file', type=str,
                        default=os.path.join(os.path.dirname(os.path.abspath(__file__)), 'gpurun_out',
                                             'bench_detail.json'),
                        help='where the full per-config record (module-level, torch-native, CPU figures) goes')
    return parser.parse_args()


def gpu_time_ms(fn: Callable[[], None], iters: int, warmup: int = 2, batches: int = 1) -> float:
    """
    Duration of fn's GPU work in ms, from HIP events recorded on the stream the kernels are
    launched on (PyTorch's current stream).  `batches` event-bracketed groups of `iters` calls
    are timed back to back and the median of the groups' means is returned (one group: its mean).
    """
    for _ in range(warmup):
        fn()
    torch.cuda.synchronize()
    events = [torch.cuda.Event(enable_timing=True) for _ in range(batches + 1)]
    events[0].record()
    for b in range(batches):
        for _ in range(iters):
            fn()
        events[b + 1].record()
    torch.cuda.synchronize()
    times = sorted(events[b].elapsed_time(events[b + 1]) / iters for b in range(batches))
    return times[len(times) // 2]


def kernel_time_ms(fn: Callable[[], None]) -> float:
    """
    The protocol of the secondary configs, whatever --steps says: 10 warm-up calls, then 60 timed
    calls in 6 event-bracketed groups of 10, median of the groups.
    """
    return gpu_time_ms(fn, 10, 10, 6)


def wall_time_ms(fn: Callable[[], None], steps: int, warmup: int) -> float:
    """
    Wall-clock ms per step: warm-up, then exactly `steps` calls bracketed by device syncs.
    """
    for _ in range(warmup):
        fn()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(steps):
        fn()
    torch.cuda.synchronize()
    return (time.perf_counter() - t0) * 1e3 / steps


def module_times_ms(forward: Callable[[int], torch.Tensor], backward: Callable[[torch.Tensor, int], None],
                    iters: int, warmup: int, sets: int = 1) -> Dict:
    """
    Timings of a layer called the way a user calls it (nn.Module + autograd, allocations and
    host work included): forward alone, forward + backward, and their difference.
    forward(i) runs the layer on input set i and returns its output; backward(out, i)
    back-propagates from it.  Wall-clock over `iters` calls bracketed by device syncs, the least of
    three such passes.
    """
    if not MODULE_TIMINGS:
        return {}
    count = [0]

    def fwd_only():
        count[0] += 1
        forward(count[0] % sets)

    def fwd_bwd():
        count[0] += 1
        i = count[0] % sets
        backward(forward(i), i)
    # the least of three passes: a pass that meets an allocator growth or a collection of garbage
    # says nothing about the layer
    ms_f = min(wall_time_ms(fwd_only, iters, warmup if rep == 0 else 1) for rep in range(3))
    ms_fb = min(wall_time_ms(fwd_bwd, iters, warmup if rep == 0 else 1) for rep in range(3))

    # The same forward + backward calls captured once into a HIP graph (one pass over every input
    # set) and replayed: what the module path costs on the GPU with the host out of the way.
    def all_sets():
        for i in range(sets):
            backward(forward(i), i)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            all_sets()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        all_sets()
    ms_graph = gpu_time_ms(graph.replay, max(2, iters // sets), 2) / sets
    del graph
    return {'ms_fwd': ms_f, 'ms_bwd': ms_fb - ms_f, 'ms_fwd_bwd': ms_fb, 'ms_fwd_bwd_hip_graph': ms_graph,
            'note': 'nn.Module + autograd calls with their allocations and casts: wall clock per eager call '
                    '(host-bound below about 0.1 ms), and per replay of the same calls captured in a HIP graph'}


def functional_cpu_entry(fn: Callable[[], None], units: float, unit: str, sample: str, dtype) -> Dict:
    """
    torch's own CPU kernels (torch.nn.functional, forward + backward through autograd) in the
    workload's dtype on all host threads torch uses: `units` of work per call of fn.
    """
    sec = cpu_time_s(fn)
    return {'value': units / sec, 'unit': unit, 'cores': torch.get_num_threads(),
            'kind': 'torch.nn.functional on the CPU', 'dtype': str(dtype).replace('torch.', ''), 'sample': sample}


def cpu_time_s(fn: Callable[[], None], reps: int = 3) -> float:
    fn()
    times = []
    for _ in range(reps):
        t0 = time.perf_counter()
        fn()
        times.append(time.perf_counter() - t0)
    return sorted(times)[len(times) // 2]


def gen(shape, seed, dtype, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return (shift + scale * torch.randn(shape, generator=g)).to(dtype)


class Raw:
    """
    Direct calls into the C ABI with preallocated tensors (kernel-level timing).
    """
    def __init__(self):
        from attorch_amd import _lib
        self.lib = _lib.load()
        self._lib = _lib

    def stream(self):
        return torch.cuda.current_stream().cuda_stream

    def check(self, rc, what):
        self._lib.check(rc, what)


# ------------------------------------------------------------------------------------------
# c4 / c1: Linear
# ------------------------------------------------------------------------------------------
def linear_workload(cfg: str):
    if cfg == 'c4':
        m, k, n, dtype, act = 16384, 4096, 16384, torch.bfloat16, 'geluapprox'
        x = gen((m, k), 4001, dtype)
        w = gen((k, n), 4002, dtype, 0.02)
        b = torch.zeros(n, dtype=dtype)
    else:
        m, k, n, dtype, act = 512, 784, 256, torch.float32, 'relu'
        x = gen((m, k), 1001, dtype)
        torch.manual_seed(1002)
        lin = torch.nn.Linear(k, n)
        w = lin.weight.detach().T.contiguous()
        b = lin.bias.detach().clone()
    dy = gen((m, n), 1000 * int(cfg[1]) + 3, dtype)
    return m, k, n, dtype, act, x, w, b, dy


def bench_linear(cfg: str, steps: int, warmup: int, with_cpu: bool) -> Dict:
    import attorch_amd
    from attorch_amd.act import act_id, parse_act_func
    raw = Raw()
    lib = raw.lib
    m, k, n, dtype, act, x, w, b, dy = linear_workload(cfg)
    dt = raw._lib.dtype_id(dtype)
    xd, dyd = x.cuda(), dy.cuda()
    layer = attorch_amd.Linear(k, n, bias=True, act_func=act, dtype=dtype)
    with torch.no_grad():
        layer.weight.copy_(w.cuda())
        layer.bias.copy_(b.cuda())
    xin = xd.clone().requires_grad_(True)

    def step():
        xin.grad = None
        layer.weight.grad = None
        layer.bias.grad = None
        layer(xin).backward(dyd)

    ms_step = wall_time_ms(step, steps, warmup)
    flop = 6.0 * m * k * n
    peak = PEAK_MFMA_16BIT_TFLOPS if dtype is not torch.float32 else PEAK_MFMA_FP32_TFLOPS

    # kernel-level timing through the C ABI
    wd, bd = layer.weight.detach(), layer.bias.detach()
    y = torch.empty((m, n), dtype=dtype, device='cuda')
    pre = torch.empty_like(y)
    dz = torch.empty_like(y)
    dx = torch.empty((m, k), dtype=dtype, device='cuda')
    dw = torch.empty((k, n), dtype=dtype, device='cuda')
    db = torch.empty(n, dtype=dtype, device='cuda')
    wsb = lib.at_colsum_workspace_bytes(m, n)
    ws = torch.empty(wsb, dtype=torch.uint8, device='cuda')
    name, param = parse_act_func(act)
    aid = act_id(name, param)
    st = raw.stream

    def k_fwd():
        raw.check(lib.at_linear_fwd(xd.data_ptr(), wd.data_ptr(), bd.data_ptr(), pre.data_ptr(), y.data_ptr(),
                                    m, k, n, k, n, n, n, aid, 0.0, dt, dt, dt, st()), 'fwd')

    awsb = lib.at_act_bwd_workspace_bytes(m, n)
    aws = torch.empty(awsb, dtype=torch.uint8, device='cuda')

    def k_act():
        raw.check(lib.at_act_bwd(dyd.data_ptr(), pre.data_ptr(), dz.data_ptr(), db.data_ptr(), aws.data_ptr(), awsb,
                                 m, n, n, n, n, aid, 0.0, dt, dt, dt, st()), 'act_bwd')

    def k_dx():
        raw.check(lib.at_linear_bwd_input(dz.data_ptr(), wd.data_ptr(), dx.data_ptr(), m, k, n, n, n, k, dt, dt,
                                          st()), 'dx')

    dwsb = lib.at_linear_bwd_weight_workspace_bytes(m, k, n, dt)
    dws = torch.empty(max(dwsb, 1), dtype=torch.uint8, device='cuda')

    def k_dw():
        raw.check(lib.at_linear_bwd_weight(xd.data_ptr(), dz.data_ptr(), dw.data_ptr(), dws.data_ptr(), dwsb,
                                           m, k, n, k, n, n, dt, dt, st()), 'dw')

    def k_db():
        raw.check(lib.at_colsum(dz.data_ptr(), db.data_ptr(), ws.data_ptr(), wsb, m, n, n, dt, dt, st()), 'colsum')

    iters = max(3, min(steps, 10))
    kernels = {}
    for kname, fn in (('linear_fwd', k_fwd), ('act_bwd_with_bias_grad', k_act), ('linear_bwd_input', k_dx),
                      ('linear_bwd_weight', k_dw), ('colsum_unfused', k_db)):
        kernels[kname] = kernel_time_ms(fn) if cfg == 'c1' else gpu_time_ms(fn, iters, 2, 3)
    gemm_flop = 2.0 * m * k * n
    fwd_tflops = gemm_flop / kernels['linear_fwd'] / 1e9
    out = {
        'tag': f'{cfg} linear {str(dtype)[6:]} {act}',
        'workload': f'{cfg}: Linear {str(dtype)[6:]} fwd+bwd X[{m},{k}] W[{k},{n}] act={act}',
        'metric': 'Linear fwd+bwd TFLOP/s', 'value': flop / ms_step / 1e9, 'unit': 'TFLOP/s',
        'ms_per_step': ms_step,
        'kernel_ms': kernels,
        'kernel_tflops': {kk: gemm_flop / kernels[kk] / 1e9
                          for kk in ('linear_fwd', 'linear_bwd_input', 'linear_bwd_weight')},
        'roofline': {'bound': 'mfma', 'kernel': 'linear_fwd (GEMM + bias + activation epilogue)',
                     'achieved': fwd_tflops, 'peak': peak, 'unit': 'TFLOP/s', 'frac': fwd_tflops / peak,
                     **(traffic_fields('c4_linear_fwd') if cfg == 'c4' else {'traffic': None})},
        'frac_of_peak_step': flop / ms_step / 1e9 / peak,
    }
    def mod_bwd(result, _):
        xin.grad = None
        layer.weight.grad = None
        layer.bias.grad = None
        result.backward(dyd)
    out['module_level'] = module_times_ms(lambda _: layer(xin), mod_bwd, max(3, min(steps, 20)), warmup)
    if cfg == 'c4' and MODULE_TIMINGS:
        out['amp'] = bench_linear_autocast(m, k, n, act, x, w, b, dy, max(3, min(steps, 10)), warmup)
    # torch's own GPU path for the same step (vendor BLAS + separate bias/activation kernels)
    ref_layer = torch.nn.Linear(k, n, bias=True, device='cuda', dtype=dtype)
    ref_act = torch.nn.GELU(approximate='tanh') if act == 'geluapprox' else torch.nn.ReLU()
    xref = xd.clone().requires_grad_(True)

    def ref_bwd(result, _):
        xref.grad = None
        ref_layer.weight.grad = None
        ref_layer.bias.grad = None
        result.backward(dyd)
    out['torch_native'] = module_times_ms(lambda _: ref_act(ref_layer(xref)), ref_bwd, max(3, min(steps, 20)), warmup)
    del ref_layer, xref
    if with_cpu:
        import oracle
        rows = min(m, 2048)
        xs, dys = x[:rows], dy[:rows]
        name, param = parse_act_func(act)
        torch.set_num_threads(os.cpu_count())

        def cpu_step():
            yy, pre_act = oracle.linear_forward(xs, w, b, name, param, dtype)
            oracle.linear_backward(dys, xs, w, pre_act, name, param, dtype)

        sec = cpu_time_s(cpu_step)
        out['cpu_baseline'] = {'value': 6.0 * rows * k * n / sec / 1e12, 'unit': 'TFLOP/s',
                               'cores': torch.get_num_threads(), 'kind': 'port',
                               'sample': f'first {rows} of {m} rows, full K and N, oracle fwd+bwd in fp32 compute'}
        F = torch.nn.functional
        xg = xs.clone().requires_grad_(True)
        wg, bg = w.T.contiguous().requires_grad_(True), b.clone().requires_grad_(True)
        act_fn = (lambda t: F.gelu(t, approximate='tanh')) if name == 'geluapprox' else F.relu

        def cpu_functional():
            xg.grad = wg.grad = bg.grad = None
            act_fn(F.linear(xg, wg, bg)).backward(dys)
        out['cpu_functional'] = functional_cpu_entry(
            cpu_functional, 6.0 * rows * k * n / 1e12, 'TFLOP/s', f'first {rows} of {m} rows, full K and N', dtype)
    return out


def bench_linear_autocast(m, k, n, act, x, w, b, dy, steps: int, warmup: int) -> Dict:
    """
    The c4 layer as the reference's examples run it (examples/utils.py:13-36, amp=True): float32
    input and parameters, forward under torch.autocast(float16), float16 output, float32 gradients
    on the leaves; beside it the same layer with float16 tensors throughout.
    """
    import attorch_amd
    f16 = torch.float16
    result = {}
    for label, store in (('fp16_tensors', f16), ('autocast_fp16_over_fp32_tensors', torch.float32)):
        layer = attorch_amd.Linear(k, n, bias=True, act_func=act, dtype=store)
        with torch.no_grad():
            layer.weight.copy_(w.cuda())
            layer.bias.copy_(b.cuda())
        xin = x.to(store).cuda().requires_grad_(True)
        dyd = dy.to(f16).cuda()

        def step():
            xin.grad = None
            layer.weight.grad = None
            layer.bias.grad = None
            with torch.autocast('cuda', dtype=f16, enabled=store is torch.float32):
                y = layer(xin)
            y.backward(dyd)
        result['ms_per_step_' + label] = _r(wall_time_ms(step, steps, warmup), 5)
        del layer, xin, dyd
        torch.cuda.empty_cache()
    result['autocast_over_fp16'] = _r(result['ms_per_step_autocast_fp16_over_fp32_tensors'] /
                                      result['ms_per_step_fp16_tensors'], 4)
    return result


# ------------------------------------------------------------------------------------------
# c2: LayerNorm / RMSNorm / Softmax / LogSoftmax, bf16 [8192, 4096]
# ------------------------------------------------------------------------------------------
def bench_rows(steps: int, warmup: int, with_cpu: bool) -> List[Dict]:
    raw = Raw()
    lib = raw.lib
    rows_, feat, dtype = 8192, 4096, torch.bfloat16
    dt = raw._lib.dtype_id(dtype)
    nsets = 6
    xs = [gen((rows_, feat), 2001 + i, dtype).cuda() for i in range(nsets)]
    dys = [gen((rows_, feat), 2101 + i, dtype).cuda() for i in range(nsets)]
    ys = [torch.empty_like(xs[0]) for _ in range(nsets)]
    dxs = [torch.empty_like(xs[0]) for _ in range(nsets)]
    w = gen((feat,), 2201, dtype, 0.1, 1.0).cuda()
    b = gen((feat,), 2202, dtype, 0.1).cuda()
    mean = torch.empty(rows_, device='cuda')
    rstd = torch.empty(rows_, device='cuda')
    dwg = torch.empty(feat, device='cuda')
    dbg = torch.empty(feat, device='cuda')
    wsb = lib.at_norm_bwd_workspace_bytes(rows_, feat, 2)
    ws = torch.empty(wsb, dtype=torch.uint8, device='cuda')
    tbytes = rows_ * feat * 2
    st = raw.stream
    counter = [0]

    def nxt():
        counter[0] = (counter[0] + 1) % nsets
        return counter[0]

    def ln_f():
        i = nxt()
        raw.check(lib.at_layer_norm_fwd(xs[i].data_ptr(), w.data_ptr(), b.data_ptr(), mean.data_ptr(),
                                        rstd.data_ptr(), ys[i].data_ptr(), rows_, feat, feat, feat, 1e-5, dt, dt,
                                        dt, st()), 'ln_fwd')

    def ln_b():
        i = nxt()
        raw.check(lib.at_layer_norm_bwd(dys[i].data_ptr(), xs[i].data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                        w.data_ptr(), dxs[i].data_ptr(), dwg.data_ptr(), dbg.data_ptr(),
                                        ws.data_ptr(), wsb, rows_, feat, feat, feat, feat, dt, dt, dt, dt, st()),
                  'ln_bwd')

    def rms_f():
        i = nxt()
        raw.check(lib.at_rms_norm_fwd(xs[i].data_ptr(), w.data_ptr(), rstd.data_ptr(), ys[i].data_ptr(), rows_,
                                      feat, feat, feat, 1e-5, dt, dt, dt, st()), 'rms_fwd')

    def rms_b():
        i = nxt()
        raw.check(lib.at_rms_norm_bwd(dys[i].data_ptr(), xs[i].data_ptr(), rstd.data_ptr(), w.data_ptr(),
                                      dxs[i].data_ptr(), dwg.data_ptr(), ws.data_ptr(), wsb, rows_, feat, feat,
                                      feat, feat, dt, dt, dt, dt, st()), 'rms_bwd')

    def sm(log):
        def f():
            i = nxt()
            raw.check(lib.at_softmax_fwd(xs[i].data_ptr(), ys[i].data_ptr(), rows_, feat, feat, feat, 0, log, dt,
                                         dt, st()), 'softmax_fwd')

        def bwd():
            i = nxt()
            raw.check(lib.at_softmax_bwd(dys[i].data_ptr(), ys[i].data_ptr(), dxs[i].data_ptr(), rows_, feat,
                                         feat, feat, feat, 0, log, dt, dt, dt, st()), 'softmax_bwd')
        return f, bwd

    import oracle
    results = []
    iters = max(10, steps)
    sm_f, sm_b = sm(0)
    lsm_f, lsm_b = sm(1)
    xc, dyc, wc, bc = xs[0].cpu(), dys[0].cpu(), w.cpu(), b.cpu()
    crow = 2048  # CPU sample rows

    def cpu_ln():
        y, m_, r_ = oracle.layer_norm_forward(xc[:crow], wc, bc, 1e-5, dtype)
        oracle.layer_norm_backward(dyc[:crow], xc[:crow], m_, r_, wc, dtype)

    def cpu_rms():
        y, r_ = oracle.rms_norm_forward(xc[:crow], wc, 1e-5)
        oracle.rms_norm_backward(dyc[:crow], xc[:crow], r_, wc)

    def cpu_sm(log):
        def f():
            y = oracle.softmax_forward(xc[:crow], False, log, dtype)
            oracle.softmax_backward(dyc[:crow], y, False, log)
        return f

    # What a plain elementwise pass reaches on the same buffers, for scale: one read + one write of
    # a tensor (torch.mul) and two reads + one write (torch.add), timed the same way.
    def ew2():
        i = nxt()
        torch.mul(xs[i], 2.0, out=ys[i])

    def ew3():
        i = nxt()
        torch.add(xs[i], dys[i], out=dxs[i])
    stream_ref = {'read1_write1_gbs': 2 * tbytes / kernel_time_ms(ew2) / 1e6,
                  'read2_write1_gbs': 3 * tbytes / kernel_time_ms(ew3) / 1e6}
    # standalone activation layer with fused dropout on the same buffers (GELU-tanh, p = 0.1)
    def act_f():
        i = nxt()
        raw.check(lib.at_act_dropout_fwd(xs[i].data_ptr(), ys[i].data_ptr(), rows_ * feat, 6, 0.0, 0.1, 4711, dt,
                                         st()), 'act_fwd')

    def act_b():
        i = nxt()
        raw.check(lib.at_act_dropout_bwd(dys[i].data_ptr(), xs[i].data_ptr(), dxs[i].data_ptr(), rows_ * feat, 6,
                                         0.0, 0.1, 4711, dt, st()), 'act_bwd')

    def cpu_act():
        dropped = torch.rand(crow, feat) < 0.1
        oracle.act_dropout_forward(xc[:crow], 'geluapprox', None, dropped, 0.1)
        oracle.act_dropout_backward(dyc[:crow], xc[:crow], 'geluapprox', None, dropped, 0.1)

    # the same layers as a user calls them: nn.Module + autograd on the rotating inputs
    import attorch_amd
    F = torch.nn.functional
    xins = [x.clone().requires_grad_(True) for x in xs]
    ln_mod = attorch_amd.LayerNorm(feat, dtype=dtype, device='cuda')
    rms_mod = attorch_amd.RMSNorm(feat, eps=1e-5, dtype=dtype, device='cuda')
    act_mod = attorch_amd.GELU(approximate='tanh', drop_p=0.1)
    with torch.no_grad():
        ln_mod.weight.copy_(w), ln_mod.bias.copy_(b), rms_mod.weight.copy_(w)
    modules = {'LayerNorm': ln_mod, 'RMSNorm': rms_mod, 'Softmax': attorch_amd.Softmax(dim=-1),
               'LogSoftmax': attorch_amd.LogSoftmax(dim=-1), 'GELU(tanh)+Dropout(0.1) layer': act_mod}

    ln_ref = torch.nn.LayerNorm(feat, dtype=dtype, device='cuda')
    rms_ref = torch.nn.RMSNorm(feat, eps=1e-5, dtype=dtype, device='cuda')
    natives = {'LayerNorm': ln_ref, 'RMSNorm': rms_ref, 'Softmax': torch.nn.Softmax(dim=-1),
               'LogSoftmax': torch.nn.LogSoftmax(dim=-1),
               'GELU(tanh)+Dropout(0.1) layer': torch.nn.Sequential(torch.nn.GELU(approximate='tanh'),
                                                                    torch.nn.Dropout(0.1))}

    def module_level(mod):
        def fwd(i):
            return mod(xins[i])

        def bwd(out, i):
            xins[i].grad = None
            for prm in mod.parameters():
                prm.grad = None
            out.backward(dys[i])
        return module_times_ms(fwd, bwd, iters, warmup, nsets)

    xg = xc[:crow].clone().requires_grad_(True)
    wg, bg = wc.clone().requires_grad_(True), bc.clone().requires_grad_(True)
    functional = {
        'LayerNorm': lambda: F.layer_norm(xg, (feat,), wg, bg, 1e-5),
        'RMSNorm': lambda: F.rms_norm(xg, (feat,), wg, 1e-5),
        'Softmax': lambda: F.softmax(xg, dim=-1),
        'LogSoftmax': lambda: F.log_softmax(xg, dim=-1),
        'GELU(tanh)+Dropout(0.1) layer': lambda: F.dropout(F.gelu(xg, approximate='tanh'), 0.1),
    }

    def cpu_functional(name):
        def f():
            xg.grad = wg.grad = bg.grad = None
            functional[name]().backward(dyc[:crow])
        return f

    traffic_key = {'LayerNorm': 'c2_layer_norm', 'RMSNorm': 'c2_rms_norm', 'Softmax': 'c2_softmax',
                   'LogSoftmax': 'c2_softmax', 'GELU(tanh)+Dropout(0.1) layer': 'c2_act_dropout'}
    for name, f, bwd, cpu in (('LayerNorm', ln_f, ln_b, cpu_ln), ('RMSNorm', rms_f, rms_b, cpu_rms),
                              ('Softmax', sm_f, sm_b, cpu_sm(False)), ('LogSoftmax', lsm_f, lsm_b, cpu_sm(True)),
                              ('GELU(tanh)+Dropout(0.1) layer', act_f, act_b, cpu_act)):
        ms_f = kernel_time_ms(f)
        ms_b = kernel_time_ms(bwd)
        gbs = 5 * tbytes / (ms_f + ms_b) / 1e6
        entry = {
            'tag': f'c2 {name}',
            'workload': f'c2: {name} bf16 fwd+bwd X[{rows_},{feat}]', 'metric': 'HBM GB/s', 'value': gbs,
            'unit': 'GB/s', 'ms_fwd': ms_f, 'ms_bwd': ms_b,
            'fwd_gbs': 2 * tbytes / ms_f / 1e6, 'bwd_gbs': 3 * tbytes / ms_b / 1e6,
            'roofline': {'bound': 'hbm', 'achieved': gbs, 'peak': PEAK_HBM_GBS, 'unit': 'GB/s',
                         'frac': gbs / PEAK_HBM_GBS, **traffic_fields(traffic_key[name])},
            'buffer_rotation': f'{nsets} sets of X/dY/Y/dX (64 MiB each)',
            'elementwise_reference': stream_ref,
            'module_level': module_level(modules[name]),
            'torch_native': module_level(natives[name]),
        }
        if with_cpu:
            sec = cpu_time_s(cpu)
            entry['cpu_baseline'] = {'value': 5 * crow * feat * 2 / sec / 1e9, 'unit': 'GB/s',
                                     'cores': torch.get_num_threads(), 'kind': 'port',
                                     'sample': f'first {crow} of {rows_} rows, oracle fwd+bwd'}
            entry['cpu_functional'] = functional_cpu_entry(
                cpu_functional(name), 5 * crow * feat * 2 / 1e9, 'GB/s', f'first {crow} of {rows_} rows', dtype)
        results.append(entry)

    # Elementwise layers outside the headline configs, on the same buffers: GLU (sigmoid) gated
    # along the feature dimension, and the mean squared error with the gradient of the input.
    half = feat // 2
    glu_out = [torch.empty((rows_, half), dtype=dtype, device='cuda') for _ in range(nsets)]
    glu_dy = [gen((rows_, half), 2301 + i, dtype).cuda() for i in range(nsets)]

    def glu_f():
        i = nxt()
        raw.check(lib.at_glu_fwd(xs[i].data_ptr(), glu_out[i].data_ptr(), rows_, half, 1, 0.0, dt, st()), 'glu_fwd')

    def glu_b():
        i = nxt()
        raw.check(lib.at_glu_bwd(glu_dy[i].data_ptr(), xs[i].data_ptr(), dxs[i].data_ptr(), rows_, half, 1, 0.0, dt,
                                 st()), 'glu_bwd')
    loss = torch.empty((), dtype=dtype, device='cuda')
    one = torch.ones((), dtype=dtype, device='cuda')
    lwsb = lib.at_p_loss_workspace_bytes(rows_ * feat)
    lws = torch.empty(lwsb, dtype=torch.uint8, device='cuda')

    def mse_f():
        i = nxt()
        raw.check(lib.at_p_loss_fwd(xs[i].data_ptr(), dys[i].data_ptr(), loss.data_ptr(), lws.data_ptr(), lwsb,
                                    rows_ * feat, 2, 1, 1.0, dt, dt, st()), 'mse_fwd')

    def mse_b():
        i = nxt()
        raw.check(lib.at_p_loss_bwd(one.data_ptr(), xs[i].data_ptr(), dys[i].data_ptr(), dxs[i].data_ptr(), None,
                                    rows_ * feat, 2, 1, 1.0, dt, dt, dt, st()), 'mse_bwd')
    for name, f, bwd, fwd_units, bwd_units in (('GLU(sigmoid) over the features', glu_f, glu_b, 1.5, 2.5),
                                               ('MSELoss(mean), input gradient', mse_f, mse_b, 2.0, 3.0)):
        ms_f = kernel_time_ms(f)
        ms_b = kernel_time_ms(bwd)
        gbs = (fwd_units + bwd_units) * tbytes / (ms_f + ms_b) / 1e6
        results.append({
            'tag': f'c2-shaped {name.split("(")[0]}',
            'workload': f'c2-shaped: {name} bf16 fwd+bwd X[{rows_},{feat}]', 'metric': 'HBM GB/s', 'value': gbs,
            'unit': 'GB/s', 'ms_fwd': ms_f, 'ms_bwd': ms_b,
            'fwd_gbs': fwd_units * tbytes / ms_f / 1e6, 'bwd_gbs': bwd_units * tbytes / ms_b / 1e6,
            'roofline': {'bound': 'hbm', 'achieved': gbs, 'peak': PEAK_HBM_GBS, 'unit': 'GB/s',
                         'frac': gbs / PEAK_HBM_GBS,
                         **traffic_fields('c2_glu' if name.startswith('GLU') else 'c2_mse')},
            'elementwise_reference': stream_ref,
        })
    return results


def bench_rows_tall() -> List[Dict]:
    """
    The c2 layers on eight times the rows ([65536, 4096] bf16, 512 MiB per tensor): the kernels
    run for a quarter of a millisecond, so what they reach here is their bandwidth without the
    launch and ramp-up cost that weighs on the 25-50 us launches of c2 itself.
    """
    raw = Raw()
    lib = raw.lib
    rows_, feat, dtype = 65536, 4096, torch.bfloat16
    dt = raw._lib.dtype_id(dtype)
    nsets = 2
    xs = [gen((rows_, feat), 2401 + i, dtype).cuda() for i in range(nsets)]
    dys = [gen((rows_, feat), 2411 + i, dtype).cuda() for i in range(nsets)]
    ys = [torch.empty_like(xs[0]) for _ in range(nsets)]
    dxs = [torch.empty_like(xs[0]) for _ in range(nsets)]
    w = gen((feat,), 2201, dtype, 0.1, 1.0).cuda()
    b = gen((feat,), 2202, dtype, 0.1).cuda()
    mean, rstd = torch.empty(rows_, device='cuda'), torch.empty(rows_, device='cuda')
    dwg, dbg = torch.empty(feat, device='cuda'), torch.empty(feat, device='cuda')
    wsb = lib.at_norm_bwd_workspace_bytes(rows_, feat, 2)
    ws = torch.empty(wsb, dtype=torch.uint8, device='cuda')
    tbytes = rows_ * feat * 2
    st = raw.stream
    counter = [0]

    def nxt():
        counter[0] = (counter[0] + 1) % nsets
        return counter[0]

    def ln_f():
        i = nxt()
        raw.check(lib.at_layer_norm_fwd(xs[i].data_ptr(), w.data_ptr(), b.data_ptr(), mean.data_ptr(),
                                        rstd.data_ptr(), ys[i].data_ptr(), rows_, feat, feat, feat, 1e-5, dt, dt,
                                        dt, st()), 'ln_fwd')

    def ln_b():
        i = nxt()
        raw.check(lib.at_layer_norm_bwd(dys[i].data_ptr(), xs[i].data_ptr(), mean.data_ptr(), rstd.data_ptr(),
                                        w.data_ptr(), dxs[i].data_ptr(), dwg.data_ptr(), dbg.data_ptr(),
                                        ws.data_ptr(), wsb, rows_, feat, feat, feat, feat, dt, dt, dt, dt, st()),
                  'ln_bwd')

    def rms_f():
        i = nxt()
        raw.check(lib.at_rms_norm_fwd(xs[i].data_ptr(), w.data_ptr(), rstd.data_ptr(), ys[i].data_ptr(), rows_,
                                      feat, feat, feat, 1e-5, dt, dt, dt, st()), 'rms_fwd')

    def rms_b():
        i = nxt()
        raw.check(lib.at_rms_norm_bwd(dys[i].data_ptr(), xs[i].data_ptr(), rstd.data_ptr(), w.data_ptr(),
                                      dxs[i].data_ptr(), dwg.data_ptr(), ws.data_ptr(), wsb, rows_, feat, feat,
                                      feat, feat, dt, dt, dt, dt, st()), 'rms_bwd')

    def sm_f():
        i = nxt()
        raw.check(lib.at_softmax_fwd(xs[i].data_ptr(), ys[i].data_ptr(), rows_, feat, feat, feat, 0, 0, dt, dt,
                                     st()), 'softmax_fwd')

    def sm_b():
        i = nxt()
        raw.check(lib.at_softmax_bwd(dys[i].data_ptr(), ys[i].data_ptr(), dxs[i].data_ptr(), rows_, feat, feat,
                                     feat, feat, 0, 0, dt, dt, dt, st()), 'softmax_bwd')
    results = []
    for name, f, bwd in (('LayerNorm', ln_f, ln_b), ('RMSNorm', rms_f, rms_b), ('Softmax', sm_f, sm_b)):
        ms_f, ms_b = gpu_time_ms(f, 5, 3, 3), gpu_time_ms(bwd, 5, 3, 3)
        gbs = 5 * tbytes / (ms_f + ms_b) / 1e6
        results.append({
            'tag': f'c2x8 {name}',
            'workload': f'c2 shape with eight times the rows: {name} bf16 fwd+bwd X[{rows_},{feat}]',
            'metric': 'HBM GB/s', 'value': gbs, 'unit': 'GB/s', 'ms_fwd': ms_f, 'ms_bwd': ms_b,
            'fwd_gbs': 2 * tbytes / ms_f / 1e6, 'bwd_gbs': 3 * tbytes / ms_b / 1e6,
            'roofline': {'bound': 'hbm', 'achieved': gbs, 'peak': PEAK_HBM_GBS, 'unit': 'GB/s',
                         'frac': gbs / PEAK_HBM_GBS, 'traffic': None},
        })
    return results


# ------------------------------------------------------------------------------------------
# c3: CrossEntropy fp16 [8192, 50257]
# ------------------------------------------------------------------------------------------
def bench_cross_entropy(steps: int, warmup: int, with_cpu: bool) -> List[Dict]:
    raw = Raw()
    lib = raw.lib
    rows_, feat, dtype = 8192, 50257, torch.float16
    dt = raw._lib.dtype_id(dtype)
    logits = gen((rows_, feat), 3001, dtype, 2.0).cuda()
    g = torch.Generator().manual_seed(3002)
    target = torch.randint(0, feat, (rows_,), generator=g)
    target[torch.rand(rows_, generator=g) < 0.05] = -100
    weight = (0.5 + torch.rand(feat, generator=g)).cuda()
    tgt = target.cuda()
    dlogits = torch.empty_like(logits)
    loss = torch.empty((), dtype=dtype, device='cuda')
    wsb = lib.at_cross_entropy_workspace_bytes(rows_)
    ws = torch.empty(wsb, dtype=torch.uint8, device='cuda')
    one = torch.ones((), dtype=dtype, device='cuda')
    tbytes = rows_ * feat * 2
    st = raw.stream
    results = []
    import oracle
    import attorch_amd
    kept = int((target != -100).sum())
    iters = max(5, steps // 2)
    # rows whose target is ignore_index are never read: T * kept / rows read, T written
    read_bytes = tbytes * kept / rows_

    def c_abi_step(wt, gdt, grad, loss_):
        def f():
            raw.check(lib.at_cross_entropy_fwd_bwd(logits.data_ptr(), tgt.data_ptr(),
                                                   None if wt is None else wt.data_ptr(), loss_.data_ptr(),
                                                   grad.data_ptr(), ws.data_ptr(), wsb, rows_, feat, feat, feat,
                                                   -100, dt, 0, gdt, gdt, st()), 'ce')
            # backward with an upstream gradient of one: the kernel reads the upstream value on
            # the device and leaves the gradient the forward pass wrote as it is
            raw.check(lib.at_cross_entropy_bwd(logits.data_ptr(), tgt.data_ptr(),
                                               None if wt is None else wt.data_ptr(), one.data_ptr(),
                                               ws.data_ptr(), grad.data_ptr(), rows_, feat, feat, feat, -100, 1,
                                               dt, 0, dt, gdt, st()), 'ce_bwd')
        return f

    def module_times(wt, autocast, native=False):
        crit = (torch.nn if native else attorch_amd).CrossEntropyLoss(weight=wt)
        xin = logits.clone().requires_grad_(True)

        def fwd(_):
            with torch.autocast('cuda', dtype=dtype, enabled=autocast):
                return crit(xin, tgt)

        def bwd(out, _):
            xin.grad = None
            out.backward()
        return module_times_ms(fwd, bwd, iters, warmup)

    for label, wt in (('unweighted', None), ('class-weighted', weight)):
        ms = kernel_time_ms(c_abi_step(wt, dt, dlogits, loss))
        gbs = (read_bytes + tbytes) / ms / 1e6
        entry = {
            'tag': f'c3 CE {label}',
            'workload': f'c3: CrossEntropyLoss fp16 fwd+bwd logits[{rows_},{feat}], 5% ignore_index, {label}',
            'metric': 'HBM GB/s', 'value': gbs, 'unit': 'GB/s', 'ms_fwd_bwd': ms,
            'algorithmic_bytes': int(read_bytes + tbytes),
            'roofline': {'bound': 'hbm', 'achieved': gbs, 'peak': PEAK_HBM_GBS, 'unit': 'GB/s',
                         'frac': gbs / PEAK_HBM_GBS, **traffic_fields('c3_cross_entropy')},
            'module_level': module_times(wt, False),
            'torch_native': module_times(None if wt is None else wt.to(dtype), False, native=True),
        }
        if with_cpu and wt is None:
            crow = 512
            lc, tc = logits[:crow].cpu(), target[:crow]

            def cpu():
                oracle.cross_entropy_forward(lc, tc, None, -100, dtype)
                oracle.cross_entropy_backward(torch.tensor(1.0), lc, tc, None, -100, dtype)
            sec = cpu_time_s(cpu)
            entry['cpu_baseline'] = {'value': 2 * crow * feat * 2 / sec / 1e9, 'unit': 'GB/s',
                                     'cores': torch.get_num_threads(), 'kind': 'port',
                                     'sample': f'first {crow} of {rows_} rows, oracle loss + gradient'}
            lcg = lc.clone().requires_grad_(True)

            def cpu_functional():
                lcg.grad = None
                torch.nn.functional.cross_entropy(lcg, tc, ignore_index=-100).backward()
            entry['cpu_functional'] = functional_cpu_entry(
                cpu_functional, 2 * crow * feat * 2 / 1e9, 'GB/s', f'first {crow} of {rows_} rows', dtype)
        results.append(entry)

    # Under autocast the loss and the gradient of the fp16 logits are fp32 (the reference's
    # custom_fwd(cast_inputs=float32) semantics): T read, 2T written, still one pass.
    grad32 = torch.empty((rows_, feat), dtype=torch.float32, device='cuda')
    loss32 = torch.empty((), dtype=torch.float32, device='cuda')
    ms = kernel_time_ms(c_abi_step(None, raw._lib.dtype_id(torch.float32), grad32, loss32))
    gbs = (read_bytes + 2 * tbytes) / ms / 1e6
    results.append({
        'tag': 'c3 CE autocast fp32 grad',
        'workload': f'c3 autocast: CrossEntropyLoss fp16 logits[{rows_},{feat}] -> fp32 loss and gradient, '
                    f'5% ignore_index, unweighted',
        'metric': 'HBM GB/s', 'value': gbs, 'unit': 'GB/s', 'ms_fwd_bwd': ms,
        'algorithmic_bytes': int(read_bytes + 2 * tbytes),
        'roofline': {'bound': 'hbm', 'achieved': gbs, 'peak': PEAK_HBM_GBS, 'unit': 'GB/s',
                     'frac': gbs / PEAK_HBM_GBS, **traffic_fields('c3_cross_entropy_autocast')},
        'module_level': module_times(None, True),
        'torch_native': module_times(None, True, native=True),
    })
    del grad32

    # The reference's alternative to the fused loss: LogSoftmax followed by NLLLoss
    # (weighted mean).  The NLL kernels gather one element per row forward and write the whole
    # gradient once backward, so their algorithmic traffic is one write of the gradient.
    logp = torch.log_softmax(logits.float(), dim=1).to(dtype)
    tgt_valid = torch.where(tgt < 0, torch.zeros_like(tgt), tgt)
    dlogp = torch.empty_like(logp)
    sum_weights = torch.empty(1, dtype=torch.float32, device='cuda')
    nwsb = lib.at_nll_loss_workspace_bytes(rows_, 1)
    nws = torch.empty(nwsb, dtype=torch.uint8, device='cuda')

    def nll_fwd():
        raw.check(lib.at_nll_loss_fwd(logp.data_ptr(), tgt_valid.data_ptr(), weight.data_ptr(), loss.data_ptr(),
                                      sum_weights.data_ptr(), nws.data_ptr(), nwsb, rows_, feat, 1, 1, dt, 0, dt,
                                      st()), 'nll_fwd')

    def nll_bwd():
        raw.check(lib.at_nll_loss_bwd(one.data_ptr(), tgt_valid.data_ptr(), weight.data_ptr(),
                                      sum_weights.data_ptr(), dlogp.data_ptr(), rows_, feat, 1, 1, dt, 0, dt,
                                      st()), 'nll_bwd')
    ms_f = kernel_time_ms(nll_fwd)
    ms_b = kernel_time_ms(nll_bwd)
    gbs = tbytes / (ms_f + ms_b) / 1e6
    results.append({
        'tag': 'c3 NLL weighted',
        'workload': f'c3: NLLLoss fp16 fwd+bwd log-probabilities[{rows_},{feat}], class-weighted mean',
        'metric': 'HBM GB/s', 'value': gbs, 'unit': 'GB/s', 'ms_fwd': ms_f, 'ms_bwd': ms_b,
        'bwd_gbs': tbytes / ms_b / 1e6,
        'roofline': {'bound': 'hbm', 'achieved': gbs, 'peak': PEAK_HBM_GBS, 'unit': 'GB/s',
                     'frac': gbs / PEAK_HBM_GBS, **traffic_fields('c3_nll_loss')},
    })
    return results


# ------------------------------------------------------------------------------------------
# c5: Conv2d 3x3 + BatchNorm2d(train) + residual + ReLU, bf16 [128, 64, 56, 56]
# ------------------------------------------------------------------------------------------
def bench_conv_bn(steps: int, warmup: int, with_cpu: bool) -> List[Dict]:
    import attorch_amd
    raw = Raw()
    lib = raw.lib
    n, c, h, w_ = 128, 64, 56, 56
    dtype = torch.bfloat16
    dt = raw._lib.dtype_id(dtype)
    nsets = 3
    xs = [gen((n, c, h, w_), 5001 + i, dtype).cuda() for i in range(nsets)]
    ress = [gen((n, c, h, w_), 5011 + i, dtype).cuda() for i in range(nsets)]
    dys = [gen((n, c, h, w_), 5021 + i, dtype).cuda() for i in range(nsets)]
    torch.manual_seed(5031)
    wt = torch.nn.init.kaiming_normal_(torch.empty(c, c, 3, 3)).to(dtype).cuda()
    ys = [torch.empty_like(xs[0]) for _ in range(nsets)]
    bn_ys = [torch.empty_like(xs[0]) for _ in range(nsets)]
    dzs = [torch.empty_like(xs[0]) for _ in range(nsets)]
    dxs = [torch.empty_like(xs[0]) for _ in range(nsets)]
    dwt = torch.empty_like(wt)
    bn_w = torch.ones(c, dtype=dtype, device='cuda')
    bn_b = torch.zeros(c, dtype=dtype, device='cuda')
    rm, rv = torch.zeros(c, device='cuda'), torch.ones(c, device='cuda')
    mean, rstd = torch.empty(c, device='cuda'), torch.empty(c, device='cuda')
    wg, bg = torch.empty(c, device='cuda'), torch.empty(c, device='cuda')
    bn_wsb = lib.at_batch_norm_workspace_bytes(c)
    bn_ws = torch.empty(bn_wsb, dtype=torch.uint8, device='cuda')
    dims = (n, c, h, w_, c, h, w_, 3, 3, 1, 1, 1, 1, 1)
    cf_wsb = lib.at_conv2d_fwd_workspace_bytes(*dims, dt, dt)
    cx_wsb = lib.at_conv2d_bwd_input_workspace_bytes(*dims, dt)
    cw_wsb = lib.at_conv2d_bwd_weight_workspace_bytes(*dims, dt)
    conv_wsb = max(cf_wsb, cx_wsb, cw_wsb, 16)
    conv_ws = torch.empty(conv_wsb, dtype=torch.uint8, device='cuda')
    # as attorch_amd.Conv2d does it: the forward workspace (channels-last input at its start) is
    # kept for the weight gradient, and one channels-last copy of dY serves both gradients
    fwd_wss = [torch.empty(max(cf_wsb, 16), dtype=torch.uint8, device='cuda') for _ in range(nsets)]
    dyhs = [torch.empty_like(dys[0]) for _ in range(nsets)]
    share = cf_wsb > 0 and cx_wsb > 0
    st = raw.stream
    counter = [0]

    def nxt():
        counter[0] = (counter[0] + 1) % nsets
        return counter[0]

    def conv_f():
        i = nxt()
        raw.check(lib.at_conv2d_fwd(xs[i].data_ptr(), wt.data_ptr(), None, ys[i].data_ptr(), fwd_wss[i].data_ptr(),
                                    cf_wsb, *dims, dt, dt, dt, st()), 'conv_fwd')

    def conv_dyh():
        i = nxt()
        if share:
            raw.check(lib.at_nchw_to_nhwc(dys[i].data_ptr(), dyhs[i].data_ptr(), n, c, h * w_, dt, st()), 'nhwc')

    def conv_dx():
        i = nxt()
        raw.check(lib.at_conv2d_bwd_input(dys[i].data_ptr(), dyhs[i].data_ptr() if share else None, wt.data_ptr(),
                                          dxs[i].data_ptr(), conv_ws.data_ptr(),
                                          conv_wsb, *dims, dt, st()), 'conv_dx')

    def conv_dw():
        i = nxt()
        raw.check(lib.at_conv2d_bwd_weight(dys[i].data_ptr(), dyhs[i].data_ptr() if share else None,
                                           xs[i].data_ptr(), fwd_wss[i].data_ptr() if share else None,
                                           dwt.data_ptr(), conv_ws.data_ptr(),
                                           conv_wsb, *dims, dt, st()), 'conv_dw')

    def bn_f():
        i = nxt()
        # as attorch_amd.BatchNorm2d does it for relu: no pre-activation is written, the output
        # stands in for it in the backward pass (same derivative)
        raw.check(lib.at_batch_norm_fwd(xs[i].data_ptr(), bn_w.data_ptr(), bn_b.data_ptr(), mean.data_ptr(),
                                        rstd.data_ptr(), ress[i].data_ptr(), None, bn_ys[i].data_ptr(),
                                        rm.data_ptr(), rv.data_ptr(), bn_ws.data_ptr(), bn_wsb, n, c, h * w_, 0.1,
                                        1e-5, 4, 0.0, 1, 1, dt, dt, 0, st()), 'bn_fwd')

    def bn_b_():
        i = nxt()
        raw.check(lib.at_batch_norm_bwd(dys[i].data_ptr(), bn_ys[i].data_ptr(), xs[i].data_ptr(), mean.data_ptr(),
                                        rstd.data_ptr(), bn_w.data_ptr(), dxs[i].data_ptr(), dzs[i].data_ptr(),
                                        wg.data_ptr(), bg.data_ptr(), bn_ws.data_ptr(), bn_wsb, n, c, h * w_, 4, 0.0,
                                        dt, dt, st()), 'bn_bwd')

    iters = max(5, steps // 2)
    for i in range(nsets):   # pre-activations and channels-last copies must exist before the backward timing
        counter[0] = i - 1
        bn_f()
        counter[0] = i - 1
        conv_f()
        counter[0] = i - 1
        conv_dyh()
    t = {k_: kernel_time_ms(f) for k_, f in (('conv_fwd', conv_f), ('conv_grad_to_channels_last', conv_dyh),
                                                        ('conv_bwd_input', conv_dx),
                                                        ('conv_bwd_weight', conv_dw), ('bn_fwd', bn_f),
                                                        ('bn_bwd', bn_b_))}
    gflop = 2.0 * n * c * h * w_ * c * 9 / 1e9
    conv_ms = t['conv_fwd'] + t['conv_grad_to_channels_last'] + t['conv_bwd_input'] + t['conv_bwd_weight']
    conv_tf = 3 * gflop / conv_ms
    tbytes = n * c * h * w_ * 2
    # forward reads x and the residual and writes y; backward reads dy, y and x and writes dx and the
    # residual gradient: 8 tensors
    bn_gbs = 8 * tbytes / (t['bn_fwd'] + t['bn_bwd']) / 1e6
    conv_entry = {
        'tag': 'c5 conv NCHW',
        'workload': f'c5: Conv2d 3x3 s1 p1 bf16 fwd+bwd X[{n},{c},{h},{w_}] W[{c},{c},3,3]',
        'metric': 'conv TFLOP/s', 'value': conv_tf, 'unit': 'TFLOP/s', 'kernel_ms': {k_: t[k_] for k_ in t if 'conv' in k_},
        'roofline': {'bound': 'mfma', 'achieved': conv_tf, 'peak': PEAK_MFMA_16BIT_TFLOPS, 'unit': 'TFLOP/s',
                     'frac': conv_tf / PEAK_MFMA_16BIT_TFLOPS, **traffic_fields('c5_conv')},
    }
    bn_entry = {
        'tag': 'c5 BN NCHW',
        'workload': f'c5: BatchNorm2d(train)+residual+ReLU bf16 fwd+bwd X[{n},{c},{h},{w_}]',
        'metric': 'HBM GB/s', 'value': bn_gbs, 'unit': 'GB/s', 'ms_fwd': t['bn_fwd'], 'ms_bwd': t['bn_bwd'],
        'roofline': {'bound': 'hbm', 'achieved': bn_gbs, 'peak': PEAK_HBM_GBS, 'unit': 'GB/s',
                     'frac': bn_gbs / PEAK_HBM_GBS, **traffic_fields('c5_batch_norm')},
        'buffer_rotation': f'{nsets} sets of 6 tensors (49 MiB each)',
    }
    # The same three products on tensors that are channels-last in memory (torch.channels_last): the
    # layout the kernels work in, so the two layout copies disappear.
    last = torch.channels_last
    xl = [x.contiguous(memory_format=last) for x in xs]
    dyl = [d.contiguous(memory_format=last) for d in dys]
    yl = [torch.empty_like(xl[0]) for _ in range(nsets)]
    dxl = [torch.empty_like(xl[0]) for _ in range(nsets)]
    lws = [lib.at_conv2d_nhwc_workspace_bytes(k_, *dims, dt) for k_ in range(3)]
    lwork = torch.empty(max(*lws, 16), dtype=torch.uint8, device='cuda')

    def last_f():
        i = nxt()
        raw.check(lib.at_conv2d_fwd_nhwc(xl[i].data_ptr(), wt.data_ptr(), None, yl[i].data_ptr(), lwork.data_ptr(),
                                         lws[0], *dims, dt, dt, st()), 'conv_fwd_nhwc')

    def last_dx():
        i = nxt()
        raw.check(lib.at_conv2d_bwd_input_nhwc(dyl[i].data_ptr(), wt.data_ptr(), dxl[i].data_ptr(), lwork.data_ptr(),
                                               lws[1], *dims, dt, st()), 'conv_dx_nhwc')

    def last_dw():
        i = nxt()
        raw.check(lib.at_conv2d_bwd_weight_nhwc(dyl[i].data_ptr(), xl[i].data_ptr(), dwt.data_ptr(),
                                                lwork.data_ptr(), lws[2], *dims, dt, st()), 'conv_dw_nhwc')
    tl = {k_: kernel_time_ms(f) for k_, f in (('conv_fwd', last_f), ('conv_bwd_input', last_dx),
                                                         ('conv_bwd_weight', last_dw))}
    last_ms = sum(tl.values())
    last_tf = 3 * gflop / last_ms
    conv_last_entry = {
        'tag': 'c5 conv NHWC',
        'workload': f'c5 with channels-last tensors: Conv2d 3x3 s1 p1 bf16 fwd+bwd X[{n},{c},{h},{w_}] '
                    f'W[{c},{c},3,3], memory format torch.channels_last',
        'metric': 'conv TFLOP/s', 'value': last_tf, 'unit': 'TFLOP/s', 'kernel_ms': tl,
        'roofline': {'bound': 'mfma', 'achieved': last_tf, 'peak': PEAK_MFMA_16BIT_TFLOPS, 'unit': 'TFLOP/s',
                     'frac': last_tf / PEAK_MFMA_16BIT_TFLOPS, **traffic_fields('c5_conv_channels_last')},
    }

    # BatchNorm on the same channels-last tensors
    rl = [r.contiguous(memory_format=last) for r in ress]
    bn_yl = [torch.empty_like(xl[0]) for _ in range(nsets)]
    dzl = [torch.empty_like(xl[0]) for _ in range(nsets)]

    def bn_last_f():
        i = nxt()
        raw.check(lib.at_batch_norm_fwd_nhwc(xl[i].data_ptr(), bn_w.data_ptr(), bn_b.data_ptr(), mean.data_ptr(),
                                             rstd.data_ptr(), rl[i].data_ptr(), None, bn_yl[i].data_ptr(),
                                             rm.data_ptr(), rv.data_ptr(), bn_ws.data_ptr(), bn_wsb, n, c, h * w_,
                                             0.1, 1e-5, 4, 0.0, 1, 1, dt, dt, 0, st()), 'bn_fwd_nhwc')

    def bn_last_b():
        i = nxt()
        raw.check(lib.at_batch_norm_bwd_nhwc(dyl[i].data_ptr(), bn_yl[i].data_ptr(), xl[i].data_ptr(),
                                             mean.data_ptr(), rstd.data_ptr(), bn_w.data_ptr(), dxl[i].data_ptr(),
                                             dzl[i].data_ptr(), wg.data_ptr(), bg.data_ptr(), bn_ws.data_ptr(),
                                             bn_wsb, n, c, h * w_, 4, 0.0, dt, dt, st()), 'bn_bwd_nhwc')
    for i in range(nsets):
        counter[0] = i - 1
        bn_last_f()
    tbl = {k_: kernel_time_ms(f) for k_, f in (('bn_fwd', bn_last_f), ('bn_bwd', bn_last_b))}
    bn_last_gbs = 8 * n * c * h * w_ * 2 / (tbl['bn_fwd'] + tbl['bn_bwd']) / 1e6
    bn_last_entry = {
        'tag': 'c5 BN NHWC',
        'workload': f'c5 with channels-last tensors: BatchNorm2d(train)+residual+ReLU bf16 fwd+bwd X[{n},{c},{h},{w_}]',
        'metric': 'HBM GB/s', 'value': bn_last_gbs, 'unit': 'GB/s', 'ms_fwd': tbl['bn_fwd'], 'ms_bwd': tbl['bn_bwd'],
        'roofline': {'bound': 'hbm', 'achieved': bn_last_gbs, 'peak': PEAK_HBM_GBS, 'unit': 'GB/s',
                     'frac': bn_last_gbs / PEAK_HBM_GBS, **traffic_fields('c5_batch_norm_channels_last')},
    }

    # the block end to end through the modules (conv -> bn + residual + relu, fwd + bwd)
    conv = attorch_amd.Conv2d(c, c, 3, padding=1, bias=False, dtype=dtype)
    bn = attorch_amd.BatchNorm2d(c, act_func='relu', dtype=dtype)
    with torch.no_grad():
        conv.weight.copy_(wt)
    xin = xs[0].clone().requires_grad_(True)
    rin = ress[0].clone().requires_grad_(True)

    def block():
        xin.grad = None
        rin.grad = None
        conv.weight.grad = None
        bn.weight.grad = None
        bn.bias.grad = None
        bn(conv(xin), rin).backward(dys[0])

    conv_entry['block_ms_fwd_bwd_modules'] = wall_time_ms(block, max(3, steps // 4), 2)
    xin_l = xs[0].detach().clone(memory_format=last).requires_grad_(True)
    rin_l = ress[0].detach().clone(memory_format=last).requires_grad_(True)

    def block_last():
        xin_l.grad = None
        rin_l.grad = None
        conv.weight.grad = None
        bn.weight.grad = None
        bn.bias.grad = None
        bn(conv(xin_l), rin_l).backward(dyl[0])
    conv_last_entry['block_ms_fwd_bwd_modules'] = wall_time_ms(block_last, max(3, steps // 4), 2)

    # each layer on its own through its module, inputs rotating as above
    xins = [x.clone().requires_grad_(True) for x in xs]
    rins = [r.clone().requires_grad_(True) for r in ress]

    def bn_fwd_mod(i):
        return bn(xins[i], rins[i])

    def conv_fwd_mod(i):
        return conv(xins[i])

    def mod_bwd(out, i):
        xins[i].grad = None
        rins[i].grad = None
        conv.weight.grad = None
        bn.weight.grad = None
        bn.bias.grad = None
        out.backward(dys[i])
    bn_entry['module_level'] = module_times_ms(bn_fwd_mod, mod_bwd, iters, warmup, nsets)
    conv_entry['module_level'] = module_times_ms(conv_fwd_mod, mod_bwd, iters, warmup, nsets)
    # torch's own GPU path (MIOpen) for the same two layers
    conv_ref = torch.nn.Conv2d(c, c, 3, padding=1, bias=False, device='cuda', dtype=dtype)
    bn_ref = torch.nn.BatchNorm2d(c, device='cuda', dtype=dtype)

    def ref_bwd(out, i):
        xins[i].grad = None
        rins[i].grad = None
        conv_ref.weight.grad = None
        bn_ref.weight.grad = None
        bn_ref.bias.grad = None
        out.backward(dys[i])
    bn_entry['torch_native'] = module_times_ms(lambda i: torch.relu(bn_ref(xins[i]) + rins[i]), ref_bwd, iters,
                                               warmup, nsets)
    conv_entry['torch_native'] = module_times_ms(lambda i: conv_ref(xins[i]), ref_bwd, iters, warmup, nsets)
    xlins = [x.detach().clone(memory_format=last).requires_grad_(True) for x in xs]

    def last_bwd(out, i):
        xlins[i].grad = None
        conv.weight.grad = None
        out.backward(dyl[i])
    conv_last_entry['module_level'] = module_times_ms(lambda i: conv(xlins[i]), last_bwd, iters, warmup, nsets)
    conv_ref_last = conv_ref.to(memory_format=last)

    def ref_last_bwd(out, i):
        xlins[i].grad = None
        conv_ref_last.weight.grad = None
        out.backward(dyl[i])
    conv_last_entry['torch_native'] = module_times_ms(lambda i: conv_ref_last(xlins[i]), ref_last_bwd, iters, warmup,
                                                      nsets)
    if with_cpu:
        import oracle
        cn = 8
        xc, rc, dyc, wc = xs[0][:cn].cpu(), ress[0][:cn].cpu(), dys[0][:cn].cpu(), wt.cpu()

        def cpu_conv():
            oracle.conv2d_forward(xc, wc, None, (1, 1), (1, 1), 1, dtype)
            oracle.conv2d_backward(dyc, xc, wc, (1, 1), (1, 1), 1, dtype)

        def cpu_bn():
            out, pre_act, m_, r_, _, _ = oracle.batch_norm_forward(xc, True, bn_w.cpu(), bn_b.cpu(), rm.cpu(), rv.cpu(),
                                                                   0.1, 1e-5, True, rc, 'relu', None)
            oracle.batch_norm_backward(dyc, xc, m_, r_, bn_w.cpu(), True, pre_act, 'relu', None)
        sec = cpu_time_s(cpu_conv)
        conv_entry['cpu_baseline'] = {'value': 3 * gflop * cn / n / sec / 1e3, 'unit': 'TFLOP/s',
                                      'cores': torch.get_num_threads(), 'kind': 'port',
                                      'sample': f'first {cn} of {n} images, oracle fwd+bwd'}
        sec = cpu_time_s(cpu_bn)
        bn_entry['cpu_baseline'] = {'value': 8 * tbytes * cn / n / sec / 1e9, 'unit': 'GB/s',
                                    'cores': torch.get_num_threads(), 'kind': 'port',
                                    'sample': f'first {cn} of {n} images, oracle fwd+bwd'}
        F = torch.nn.functional
        xg, rg = xc.clone().requires_grad_(True), rc.clone().requires_grad_(True)
        wg_, bw_, bb_ = (wc.clone().requires_grad_(True), bn_w.cpu().requires_grad_(True),
                         bn_b.cpu().requires_grad_(True))
        rm_c, rv_c = rm.cpu().to(dtype), rv.cpu().to(dtype)

        def cpu_conv_functional():
            xg.grad = wg_.grad = None
            F.conv2d(xg, wg_, None, 1, 1).backward(dyc)

        def cpu_bn_functional():
            xg.grad = rg.grad = bw_.grad = bb_.grad = None
            F.relu(F.batch_norm(xg, rm_c, rv_c, bw_, bb_, True, 0.1, 1e-5) + rg).backward(dyc)
        conv_entry['cpu_functional'] = functional_cpu_entry(
            cpu_conv_functional, 3 * gflop * cn / n / 1e3, 'TFLOP/s', f'first {cn} of {n} images', dtype)
        bn_entry['cpu_functional'] = functional_cpu_entry(
            cpu_bn_functional, 8 * tbytes * cn / n / 1e9, 'GB/s', f'first {cn} of {n} images', dtype)
    return [conv_entry, conv_last_entry, bn_entry, bn_last_entry]


def mfma_probe() -> Dict:
    """
    What the matrix cores sustain without any memory traffic (at_mfma_probe: bf16 32x32x16 MFMAs
    back to back on every CU, operands in registers), once with a constant operand pair and once
    with operands that change from MFMA to MFMA as in a real product.  The second figure is the
    ceiling an MFMA-bound kernel on real data can reach on this device (it is power-limited); the
    first reaches the published peak.  Median of 5 launches of about 10 ms each.
    """
    from attorch_amd import _lib
    lib = _lib.load()
    scratch = torch.zeros(4, dtype=torch.uint8, device='cuda')
    stream = torch.cuda.current_stream().cuda_stream
    iters = 4000
    flop = lib.at_mfma_probe_flop(iters)
    out = {}
    for name, rnd in (('constant_operands', 0), ('changing_operands', 1)):
        def launch() -> None:
            _lib.check(lib.at_mfma_probe(iters, rnd, scratch.data_ptr(), stream), 'at_mfma_probe')
        ms = gpu_time_ms(launch, 1, 2, 5)
        out[name] = flop / ms / 1e9
    return {'unit': 'TFLOP/s', 'tflops_constant_operands': out['constant_operands'],
            'tflops_changing_operands': out['changing_operands'],
            'note': 'bf16 MFMA 32x32x16 from registers, no memory traffic; changing operands = ceiling for real data'}


def main() -> int:
    args = parse_args()
    if args.gpus != 1:
        print(f'bench.py: this build targets one GPU; --gpus {args.gpus} is not supported (every BASELINE '
              'config is a single-GPU workload). Run with --gpus 1.', file=sys.stderr)
        return 2
    if not torch.cuda.is_available():
        print('bench.py: no HIP device visible; the kernels have no CPU path.', file=sys.stderr)
        return 2
    sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
    torch.set_num_threads(os.cpu_count())
    with_cpu = not args.no_cpu
    global MODULE_TIMINGS
    MODULE_TIMINGS = not args.no_modules
    if args.calibrate_copy:
        src = torch.empty(256 << 20, dtype=torch.uint8, device='cuda').fill_(1)
        dst = torch.empty_like(src)
        for _ in range(3):
            dst.copy_(src)
        torch.cuda.synchronize()
        del src, dst
    head = bench_linear('c4', args.steps, args.warmup, with_cpu)
    head['mfma_probe'] = mfma_probe()
    head['frac_of_mfma_probe_step'] = head['value'] / head['mfma_probe']['tflops_changing_operands']
    extra: List[Dict] = []
    wanted = [] if args.configs == 'none' else args.configs.split(',')
    if 'c1' in wanted:
        extra.append(bench_linear('c1', max(args.steps, 50), args.warmup, with_cpu))
    if 'c2' in wanted:
        extra.extend(bench_rows(args.steps, args.warmup, with_cpu))
    if 'c2x8' in wanted:
        extra.extend(bench_rows_tall())
    if 'c3' in wanted:
        extra.extend(bench_cross_entropy(args.steps, args.warmup, with_cpu))
    if 'c5' in wanted:
        extra.extend(bench_conv_bn(args.steps, args.warmup, with_cpu))
    detail = {
        'metric': METRIC, 'value': head['value'], 'unit': 'TFLOP/s', 'n_gpus': 1, 'steps': args.steps,
        'warmup': args.warmup, 'ms_per_step': head['ms_per_step'],
        'config': {'workload': head['workload']},
        'roofline': head['roofline'],
        'cpu_baseline': head.get('cpu_baseline'),
        'cpu_functional': head.get('cpu_functional'),
        'module_level': head.get('module_level'),
        'torch_native': head.get('torch_native'),
        'frac_of_peak_step': head['frac_of_peak_step'],
        'kernel_ms': head['kernel_ms'], 'kernel_tflops': head['kernel_tflops'],
        'amp': head.get('amp'),
        'mfma_probe': head.get('mfma_probe'),
        'frac_of_mfma_probe_step': head.get('frac_of_mfma_probe_step'),
        'configs': extra,
    }
    # Everything measured goes to a file (--detail-file); stdout carries only the one compact line.
    try:
        os.makedirs(os.path.dirname(os.path.abspath(args.detail_file)), exist_ok=True)
        with open(args.detail_file, 'w') as fh:
            fh.write(json.dumps(detail) + '\n')
    except OSError as exc:
        print(f'bench.py: detail file not written ({exc})', file=sys.stderr)
    print(json.dumps(compact_line(args, head, extra)))
    return 0


METRIC = 'Linear fwd+bwd TFLOP/s; norm/softmax/CE HBM GB/s; % of MI355X roofline'


def _r(v, digits=4):
    return None if v is None else float(f'{v:.{digits}g}')


def compact_line(args, head: Dict, extra: List[Dict]) -> Dict:
    """
    The one JSON line a harness parses: the contract fields, the headline's roofline and CPU
    baseline, and per secondary config its tag, value, unit, roofline fraction, measured traffic
    and CPU baseline.  Kept well under 4 KB.
    """
    configs = []
    for e in extra:
        item = {'tag': e.get('tag', e['workload'][:40]), 'value': _r(e['value']), 'unit': e['unit'],
                'frac': _r(e['roofline']['frac']), 'traffic': e['roofline'].get('traffic')}
        if e.get('cpu_baseline') is not None:
            item['cpu'] = _r(e['cpu_baseline']['value'])
        if 'ms_per_step' in e:
            item['ms_per_step'] = _r(e['ms_per_step'])
        if 'frac_of_peak_step' in e:
            item['frac_step'] = _r(e['frac_of_peak_step'])
        configs.append(item)
    roof = head['roofline']
    cb = head.get('cpu_baseline')
    line = {
        'metric': METRIC,
        'value': _r(head['value'], 6), 'unit': 'TFLOP/s', 'n_gpus': 1, 'steps': args.steps, 'warmup': args.warmup,
        'ms_per_step': _r(head['ms_per_step'], 6), 'higher_is_better': True, 'scaling': 'weak',
        'vs_baseline': None, 'dtype': 'bf16', 'data': 'synthetic',
        'config': {'workload': head['workload'], 'step': 'attorch_amd.Linear forward + backward (dX, dW, db)',
                   'algorithmic_flop_per_step': 6 * 16384 * 4096 * 16384},
        'roofline': {'bound': roof['bound'], 'achieved': _r(roof['achieved'], 6), 'peak': roof['peak'],
                     'unit': roof['unit'], 'frac': _r(roof['frac']), 'traffic': roof.get('traffic'),
                     'kernel': roof.get('kernel')},
        'cpu_baseline': None if cb is None else {'value': _r(cb['value']), 'unit': cb['unit'], 'cores': cb['cores'],
                                                 'kind': cb['kind'], 'sample': cb['sample']},
        'frac_of_peak_step': _r(head['frac_of_peak_step']),
        'kernel_ms': {k: _r(v) for k, v in head['kernel_ms'].items()},
        'configs_note': 'per secondary config: value in unit, frac of its roofline, traffic = measured HBM bytes '
                        'per fwd+bwd, cpu = oracle on the host cores (cpu_baseline.cores threads) in the same unit',
        'configs': configs,
    }
    if head.get('amp') is not None:
        line['amp'] = head['amp']
    if head.get('mfma_probe') is not None:
        probe = head['mfma_probe']
        line['mfma_probe'] = {'unit': 'TFLOP/s', 'constant_operands': _r(probe['tflops_constant_operands']),
                              'changing_operands': _r(probe['tflops_changing_operands']),
                              'step_over_changing': _r(head['frac_of_mfma_probe_step']),
                              'note': 'register-resident bf16 MFMAs, no memory traffic: the device sustains the '
                                      'published peak only with constant operands'}
    return line


if __name__ == '__main__':
    sys.exit(main())
