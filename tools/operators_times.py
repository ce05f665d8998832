"""Times of the layer norm, distillation and 4-bit kernels.

    python tools/operators_times.py [text ...]            each case (whose name holds one of the texts): twenty calls recorded
                                                          into a graph, median and least of eleven replays, per call
    python tools/operators_times.py --calls N [text ...]  each case called N times from Python and nothing else (for a profiler)
    python tools/operators_times.py --passes [text ...]   the passes of perf/operators.py (a call, or a call and its gradients) made
                                                          from Python in a row: elementary operations and the kernels

A kernel's time is that of a call in a row of the same calls on the same tensors: what fits stays in the caches, and the launch of one call
runs under the end of the one before it.  Rates count what the call cannot do without: each input read, each output written once.
"""
import importlib.util
import os
import sys
import time

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
from dreamer_amd import _native as N  # noqa: E402
from dreamer_amd import mx4  # noqa: E402

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
NAME = {F32: "fp32", BF16: "bf16", F16: "fp16"}


def rand(*shape):
    return torch.randn(*shape, device=DEV)


def weight(rows, K):
    out = N.mx4_quantize(rand(min(rows, 8192), K))
    return tuple(t.repeat(-(-rows // t.shape[0]), 1)[:rows].contiguous() for t in out)


# every builder returns (call, bytes, flops)
def norm_forward(rows, E, dtype, save=True):
    x, w, b = rand(rows, E).to(dtype), torch.ones(E, device=DEV), torch.zeros(E, device=DEV)
    return lambda: N.layer_norm_forward(x, w, b, 1e-5, save), 2 * rows * E * x.element_size(), 0


def norm_backward(rows, E, dtype):
    x, dy, w, b = rand(rows, E).to(dtype), rand(rows, E).to(dtype), torch.ones(E, device=DEV), torch.zeros(E, device=DEV)
    _, stats = N.layer_norm_forward(x, w, b, 1e-5, True)
    return lambda: N.layer_norm_backward(x, dy, w, stats, True, True, True, F32), 3 * rows * E * x.element_size(), 0


def _distill(rows, V, k, dtype, rest):
    values, idx = rand(rows, V).topk(k, 1)
    return rand(rows, V).to(dtype), values, idx, torch.full((rows,), 12.0, device=DEV) if rest else None


def distill_forward(rows, V, k, dtype, rest):
    s, values, idx, lse = _distill(rows, V, k, dtype, rest)
    return lambda: N.distill_topk_forward(s, values, idx, lse, 1.0), rows * (V * s.element_size() + k * 16), 0


def distill_backward(rows, V, k, dtype, rest):
    s, values, idx, lse = _distill(rows, V, k, dtype, rest)
    _, p, row = N.distill_topk_forward(s, values, idx, lse, 1.0)
    g = torch.ones(rows, device=DEV)
    return lambda: N.distill_topk_backward(s, idx, p, row, g, 1.0), rows * (2 * V * s.element_size() + k * 12), 0


def quantise(rows, K, dtype):
    x = rand(rows, K).to(dtype)
    return lambda: N.mx4_quantize(x), rows * K * (x.element_size() + 17 / 32), 0


def dequantise(rows, K, dtype):
    codes, scales = weight(rows, K)
    return lambda: N.mx4_dequantize(codes, scales, K, dtype), rows * K * (torch.finfo(dtype).bits // 8 + 17 / 32), 0


def linear(M, out, K, dtype, pad=0):
    codes, scales = weight(out, K)
    x = rand(M, K + pad).to(dtype)[:, :K]
    return lambda: N.mx4_linear(x, codes, scales), out * K * 17 / 32 + M * (K + out) * x.element_size(), 2 * M * out * K


def gradient(M, out, K, dtype):
    codes, scales = weight(out, K)
    dy = rand(M, out).to(dtype)
    return lambda: N.mx4_linear_dgrad(dy, codes, scales, K), out * K * 17 / 32 + M * (K + out) * dy.element_size(), 2 * M * out * K


def bias_gradient(M, out, dtype):
    dy = rand(M, out).to(dtype)
    return lambda: N.mx4_bias_grad(dy, dtype), M * out * dy.element_size(), 0


def product(M, out, K, dtype=BF16):
    x, w = mx4.quantize(rand(M, K)), weight(out, K)
    return (lambda: N.mx4_product(x.codes, x.scales, *w, K, None, dtype)), (M + out) * K * 17 / 32 + M * out * torch.finfo(dtype).bits // 8, 2 * M * out * K


CASES = [(norm_forward, 16, 512, F32, False), (norm_forward, 1024, 512, F32), (norm_backward, 1024, 512, F32),
         (norm_forward, 16384, 4096, BF16), (norm_backward, 16384, 4096, BF16), (norm_forward, 1048576, 64, BF16), (norm_backward, 1048576, 64, BF16),
         (norm_forward, 65536, 512, F32), (norm_backward, 65536, 512, F32), (norm_forward, 65536, 1024, BF16), (norm_backward, 65536, 1024, BF16),
         (norm_backward, 1024, 1024, F32), (norm_forward, 8192, 8192, BF16), (norm_forward, 4096, 16384, BF16), (norm_backward, 4096, 16384, BF16),
         (norm_forward, 4096, 16384, F32), (norm_backward, 4096, 16384, F32), (norm_forward, 2048, 32768, BF16), (norm_backward, 2048, 32768, BF16),
         (norm_forward, 1024, 32768, F32), (norm_forward, 1024, 65536, BF16), (norm_forward, 2000000, 3, F32), (norm_backward, 2000000, 3, F32),
         (distill_forward, 240, 255, 16, F32, False), (distill_backward, 240, 255, 16, F32, False),
         (distill_forward, 5, 128001, 100, F16, False), (distill_backward, 5, 128001, 100, F16, False),
         (distill_forward, 4096, 32768, 64, BF16, False), (distill_forward, 4096, 32768, 64, BF16, True), (distill_backward, 4096, 32768, 64, BF16, True),
         (distill_forward, 65536, 1024, 16, BF16, False), (distill_forward, 65536, 1024, 16, BF16, True), (distill_forward, 8192, 4096, 64, BF16, False),
         (distill_forward, 256, 8192, 64, BF16, False), (distill_forward, 16, 131072, 64, BF16, True), (distill_backward, 32768, 1024, 16, BF16, False),
         (distill_backward, 1024, 4096, 64, BF16, False), (distill_backward, 16, 32768, 64, BF16, False),
         (quantise, 1024, 4096, F32), (quantise, 12288, 4096, BF16), (quantise, 16384, 8192, F32), (quantise, 257, 4080, F32), (quantise, 8192, 8192, BF16),
         (dequantise, 1024, 4096, F32), (dequantise, 12288, 4096, BF16),
         (linear, 16, 12288, 4096, BF16), (linear, 16, 12288, 4096, F16), (linear, 16, 12288, 4096, F32), (linear, 16, 8192, 8192, BF16),
         (linear, 16, 4096, 4096, BF16), (linear, 16, 4096, 4096, BF16, 1), (linear, 1, 4096, 4096, BF16), (linear, 32, 12288, 4096, BF16),
         (linear, 32, 4096, 4096, F32), (linear, 33, 4096, 4096, BF16), (linear, 64, 4096, 2048, BF16), (linear, 64, 4096, 4096, BF16),
         (linear, 512, 2048, 2048, BF16), (linear, 1024, 4096, 4096, BF16), (linear, 1024, 4096, 4096, F16), (linear, 1024, 4096, 4096, F32),
         (linear, 2048, 8192, 4096, BF16), (gradient, 1, 4096, 4096, BF16), (gradient, 16, 4096, 4096, BF16), (gradient, 64, 4096, 4096, BF16),
         (gradient, 1024, 4096, 4096, BF16), (gradient, 1024, 4096, 4096, F16), (gradient, 1024, 4096, 4096, F32), (gradient, 2048, 8192, 4096, BF16),
         (bias_gradient, 1024, 4096, BF16), (bias_gradient, 2048, 8192, BF16), (product, 16, 4096, 4096), (product, 257, 1000, 4080, F32), (product, 257, 1000, 8192),
         (product, 1024, 4096, 4096), (product, 2048, 6144, 4096), (product, 4096, 4096, 4096), (product, 8192, 8192, 8192)]


def name_of(build, *args):
    sizes = [a for a in args if isinstance(a, int) and not isinstance(a, bool)]
    if build in (distill_forward, distill_backward):
        extra = f", {sizes.pop()} listed" + (", with the rest" if args[-1] else "")
    else:
        extra = ", rows that start anywhere" if build is linear and len(sizes) == 4 and sizes.pop() else ""
    types = [NAME[a] for a in args if isinstance(a, torch.dtype)] or ["bf16"]
    return f"{build.__name__.replace('_', ' ')} {' x '.join(map(str, sizes))} {types[0]}{extra}"


def graph_times(call, calls=20, replays=11):
    for _ in range(3):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(calls):
            call()
    times = []
    for n in range(replays + 3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b) * 1e3 / calls)
    times = sorted(times[3:])
    return times[replays // 2], times[0]


def passes(texts):
    spec = importlib.util.spec_from_file_location("operators", os.path.join(ROOT, "perf", "operators.py"))
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    print(f"{'pass':20s} {'floor us':>9s} {'plain us':>9s} {'here us':>9s}    (medians of 9; floor: bytes at 4.73 TB/s, operations at 1.6 PFLOP/s, in 4 bits 6.2)")
    for case in ops.listed():
        if texts and not any(t in case["name"] for t in texts):
            continue
        shown = []
        for own in (False, True):
            ops.own = own
            state = ops.prepare(case, 1)
            for _ in range(5):
                ops.run(state)
            torch.cuda.synchronize()
            t0 = time.perf_counter()
            ops.run(state)
            torch.cuda.synchronize()
            n = max(3, min(2000, int(0.1 / (time.perf_counter() - t0))))
            times = []
            for _ in range(9):
                t0 = time.perf_counter()
                for _ in range(n):
                    ops.run(state)
                torch.cuda.synchronize()
                times.append((time.perf_counter() - t0) / n * 1e6)
            shown.append(sorted(times)[4])
            del state
        w = ops.work(case)
        print(f"{case['name']:20s} {max(w['bytes'] / 4.73e6, w['flops'] / (6.2e9 if case['op'] == 'product' else 1.6e9)):9.2f} {shown[0]:9.1f} {shown[1]:9.1f}", flush=True)


def main(argv):
    if argv[:1] == ["--passes"]:
        return passes(argv[1:])
    calls = 0
    if argv[:1] == ["--calls"]:
        calls, argv = int(argv[1]), argv[2:]
    torch.manual_seed(0)
    if not calls:
        print(f"{'case':66s} {'median us':>10s} {'least us':>9s} {'TB/s':>6s} {'TFLOP/s':>8s}")
    for build, *args in CASES:
        name = name_of(build, *args)
        if argv and not any(t in name for t in argv):
            continue
        call, nbytes, flops = build(*args)
        if calls:
            for _ in range(calls):
                call()
            torch.cuda.synchronize()
            print(name, flush=True)
        else:
            median, least = graph_times(call)
            print(f"{name:66s} {median:10.2f} {least:9.2f} {nbytes / median / 1e6:6.2f} {flops / median / 1e6:8.0f}", flush=True)
        del call
        torch.cuda.empty_cache()


if __name__ == "__main__":
    main(sys.argv[1:])
