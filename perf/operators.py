"""Cases of the gradient operators: the global norm over many tensors, clipping, and the averaging fold.

A data-parallel training step averages the ranks' gradients, takes one norm over all of them and
scales them down when it is too large.  `run` is one such call (or two of them in a row, as a step
makes them), in plain torch operations or, with `own`, through the library's C-ABI.

Gradients lie in one flat buffer, as bucketed data-parallel training keeps them, each tensor a view
of it; the ragged layouts start tensors at any element and leave gaps of zeros between some of them.
The plain form works on the flat buffer as a whole, gaps included; the library takes the tensors.
"""
import ctypes
import math
import pathlib
import random
import sys

import numpy as np
import torch

own = False

_TYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_CODES = {"f64": 1, "f32": 2, "f16": 3, "bf16": 4}       # PGK_DT_* of include/pgk.h
_WORK_BYTES = 65536                                      # PGK_GRAD_WORK_BYTES
_EPS = 1e-6                                              # the constant beside the norm in the clip coefficient
_MAX_NORM = 1.0


# ---- the cases -----------------------------------------------------------------------------------

def listed():
    return [
        # one bias gradient: a call's latency
        dict(name="norm-one-f32", kind="norm", layout="one", n=4099, dt="f32"),
        # the gradients of one transformer layer, what a pipeline stage of one layer holds
        dict(name="norm-layer-bf16", kind="norm", layout="model", hidden=1280, layers=1, vocab=0, dt="bf16"),
        # a whole decoder's gradients, 147 tensors
        dict(name="norm-model-bf16", kind="norm", layout="model", hidden=2048, layers=12, vocab=32000, dt="bf16"),
        # sharded gradients: hundreds of pieces that start and end anywhere, empty ones among them
        dict(name="norm-ragged-f32", kind="norm", layout="ragged", tensors=701, n=150_000_001, dt="f32"),
        # the norms' and biases' gradients alone: many small tensors, one launch's worth of work
        dict(name="clip-small-bf16", kind="clip", layout="ragged", tensors=37, n=47_360, dt="bf16", out_dt="bf16", scale=1.0),
        # bf16 gradients summed over 8 ranks, averaged, clipped and widened for the optimizer in one pass
        dict(name="clip-widen-bf16", kind="clip", layout="model", hidden=2048, layers=4, vocab=32000, dt="bf16", out_dt="f32", scale=0.125),
        # norm, then clip, of one layer in 32 bits
        dict(name="step-layer-f32", kind="norm_clip", layout="model", hidden=1280, layers=1, vocab=0, dt="f32", out_dt="f32", scale=1.0),
        # norm, then clip, of the whole decoder
        dict(name="step-model-bf16", kind="norm_clip", layout="model", hidden=2048, layers=12, vocab=32000, dt="bf16", out_dt="bf16", scale=1.0),
        # two ranks' copies of a small odd block, the latency of one exchange's fold
        dict(name="fold-2-small-f32", kind="fold", n=4099, nsrc=2, dt="f32", out_dt="f32"),
        # the direct exchange on 8 ranks: 64 MiB of bf16 gradients from each
        dict(name="fold-8-bf16", kind="fold", n=33_554_432, nsrc=8, dt="bf16", out_dt="bf16"),
        # 4 ranks, fp16 copies widened for the optimizer, odd length
        dict(name="fold-4-widen-f16", kind="fold", n=50_000_003, nsrc=4, dt="f16", out_dt="f32"),
        # 3 ranks' f32 shards averaged and then clipped by their own norm
        dict(name="shard-3-f32", kind="fold_clip", n=30_000_001, nsrc=3, dt="f32", out_dt="f32"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["norm", "clip", "norm_clip", "fold", "fold_clip"])
    dt = rng.choice(["f64", "f32", "f16", "bf16", "bf16", "f32"])
    out_dt = "f32" if dt in ("f16", "bf16") and rng.random() < 0.4 else dt
    width = {"f64": 4, "f32": 2, "f16": 1, "bf16": 1}[dt]
    if kind.startswith("fold"):
        nsrc = rng.randint(1, 16)
        n = _log_int(rng, 1, 200_000_000 // (nsrc * width))
        return dict(kind=kind, n=n, nsrc=nsrc, dt=dt, out_dt=out_dt)
    case = dict(kind=kind, dt=dt)
    layout = rng.choice(["one", "ragged", "ragged", "model"])
    if layout == "one":
        case.update(layout="one", n=_log_int(rng, 1, 300_000_000 // width))
    elif layout == "ragged":
        tensors = _log_int(rng, 2, 1200)
        case.update(layout="ragged", tensors=tensors, n=_log_int(rng, 4 * tensors, 200_000_000 // width))
    else:
        case.update(layout="model", hidden=rng.randint(64, 1300), layers=rng.randint(1, 8 // width),
                    vocab=rng.choice([0, 5003, 32000]))
    if kind != "norm":
        case.update(out_dt=out_dt, scale=rng.choice([1.0, 0.5, 0.125, 1 / 3]))
    return case


def _sizes(case):
    """[(first element, elements)] of every tensor in the flat buffer, and the buffer's elements."""
    if case["layout"] == "one":
        return [(0, case["n"])], case["n"]
    if case["layout"] == "model":
        h, v = case["hidden"], case["vocab"]
        layer = [3 * h * h, 3 * h, h * h, h, 4 * h * h, 4 * h, 4 * h * h, h, h, h, h, h]
        numels = layer * case["layers"] + ([v * h, h, h] if v else [])
        gaps = [0] * len(numels)
    else:
        r = random.Random(case["tensors"])
        weights = [math.exp(r.uniform(0.0, 7.0)) for _ in range(case["tensors"])]
        share = case["n"] / sum(weights)
        numels = [0 if i % 29 == 7 else 1 if i % 31 == 9 else max(1, int(w * share)) for i, w in enumerate(weights)]
        gaps = [r.choice([0, 0, 0, 1, 3, 64]) for _ in numels]
    at, spans = 0, []
    for n, gap in zip(numels, gaps):
        spans.append((at, n))
        at += n + gap
    return spans, max(at, 1)


def _pointers(flat, spans):
    base, size = flat.data_ptr(), flat.element_size()
    return (ctypes.c_void_p * len(spans))(*[base + a * size for a, _ in spans])


def prepare(case, seed):
    """Gradients on the GPU, the buffers that results go to, and the lists that the calls take.

    A training program makes the lists once: its gradients keep their places from step to step.
    """
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _TYPES[case["dt"]]
    state = dict(case=case, work=torch.zeros(_WORK_BYTES // 8, dtype=torch.float64, device="cuda"),
                 sumsq=torch.zeros(1, dtype=torch.float64, device="cuda"),
                 norm=torch.zeros(1, dtype=torch.float64, device="cuda"))

    def values(n, sigma):
        # gradients are near normal; the spread differs along the buffer
        return torch.randn(n, generator=gen, device="cuda", dtype=torch.float32).mul_(sigma).to(dt)

    if case["kind"].startswith("fold"):
        state["srcs"] = [values(case["n"], 0.01) for _ in range(case["nsrc"])]
        state["src_list"] = (ctypes.c_void_p * case["nsrc"])(*[s.data_ptr() for s in state["srcs"]])
        state["mean"] = torch.zeros(case["n"], dtype=_TYPES[case["out_dt"]], device="cuda")
        if case["kind"] == "fold_clip":
            spans = [(0, case["n"])]
            state.update(spans=spans, ns=(ctypes.c_size_t * 1)(case["n"]), grad_list=_pointers(state["mean"], spans),
                         out=torch.zeros_like(state["mean"]))
            state["out_list"] = _pointers(state["out"], spans)
        return state
    spans, total = _sizes(case)
    flat = torch.empty(total, dtype=dt, device="cuda")
    piece = 1 << 26
    for k, at in enumerate(range(0, total, piece)):
        flat[at:at + piece] = values(min(piece, total - at), 0.003 * (1 + k % 5))
    for (a, n), (b, _) in zip(spans, spans[1:] + [(total, 0)]):
        if a + n < b:
            flat[a + n:b] = 0
    state.update(spans=spans, flat=flat, ns=(ctypes.c_size_t * len(spans))(*[n for _, n in spans]),
                 grad_list=_pointers(flat, spans))
    if case["kind"] == "clip":
        # the norm of an earlier call, or of all ranks: a number on the GPU
        state["sumsq"] = _plain_sumsq(flat)
    if case["kind"] != "norm":
        state["out"] = torch.zeros(total, dtype=_TYPES[case["out_dt"]], device="cuda")
        state["out_list"] = _pointers(state["out"], spans)
    return state


# ---- plain form ------------------------------------------------------------------------------------

def _plain_sumsq(flat):
    # 64 bits: a sum of up to 1e9 squares, each of which may leave the range of 32 bits
    return flat.double().square().sum().reshape(1)


def _wide(x):
    return x if x.dtype == torch.float64 else x.float()


def _plain_clip(flat, out, sumsq, scale):
    norm = abs(scale) * sumsq.sqrt()
    c = scale * torch.clamp(_MAX_NORM / (norm + _EPS), max=1.0)
    wide = _wide(flat)
    out.copy_(wide * c.to(wide.dtype))
    return norm


def _plain_fold(srcs, out):
    # 64 bits: a mean rounded more than once is off to one side, and the sum of its squares shows it
    total = sum((s.double() for s in srcs[1:]), srcs[0].double())
    out.copy_(total * (1.0 / len(srcs)))
    return _plain_sumsq(out)


# ---- one pass --------------------------------------------------------------------------------------

def _library():
    at = str(pathlib.Path(__file__).resolve().parents[1] / "rdma-ring-collectives_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import pgamd
    return pgamd, pgamd.load()


def _own_sumsq(state):
    pgamd, lib = _library()
    pgamd.check(lib.pgk_grad_sumsq(state["grad_list"], state["ns"], len(state["spans"]), _CODES[state["case"]["dt"]],
                                   state["sumsq"].data_ptr(), state["work"].data_ptr(),
                                   torch.cuda.current_stream().cuda_stream), "pgk_grad_sumsq")
    return state["sumsq"]


def _own_clip(state, dt, scale):
    pgamd, lib = _library()
    pgamd.check(lib.pgk_grad_clip(state["out_list"], _CODES[state["case"]["out_dt"]], state["grad_list"], _CODES[dt],
                                  state["ns"], len(state["spans"]), state["sumsq"].data_ptr(), 1, scale, _MAX_NORM,
                                  state["norm"].data_ptr(), torch.cuda.current_stream().cuda_stream), "pgk_grad_clip")
    return state["norm"]


def _own_fold(state):
    pgamd, lib = _library()
    case = state["case"]
    pgamd.check(lib.pgk_grad_fold(state["mean"].data_ptr(), _CODES[case["out_dt"]], state["src_list"], case["nsrc"],
                                  case["n"], _CODES[case["dt"]], 1.0 / case["nsrc"], state["sumsq"].data_ptr(),
                                  state["work"].data_ptr(), torch.cuda.current_stream().cuda_stream), "pgk_grad_fold")
    return state["sumsq"]


def run(state):
    case = state["case"]
    kind = case["kind"]
    if kind == "norm":
        return dict(sumsq=_own_sumsq(state) if own else _plain_sumsq(state["flat"]))
    if kind == "clip":
        norm = _own_clip(state, case["dt"], case["scale"]) if own else \
            _plain_clip(state["flat"], state["out"], state["sumsq"], case["scale"])
        return dict(norm=norm, out=state["out"])
    if kind == "norm_clip":
        if own:
            sumsq = _own_sumsq(state)
            norm = _own_clip(state, case["dt"], case["scale"])
        else:
            sumsq = _plain_sumsq(state["flat"])
            norm = _plain_clip(state["flat"], state["out"], sumsq, case["scale"])
        return dict(sumsq=sumsq, norm=norm, out=state["out"])
    sumsq = _own_fold(state) if own else _plain_fold(state["srcs"], state["mean"])
    if kind == "fold":
        return dict(sumsq=sumsq, mean=state["mean"])
    norm = _own_clip(state, case["out_dt"], 1.0) if own else \
        _plain_clip(state["mean"], state["out"], sumsq, 1.0)
    return dict(sumsq=sumsq, mean=state["mean"], norm=norm, out=state["out"])


# ---- what a pass cannot do without, and its results in 64 bits ---------------------------------------

def work(case):
    size = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}
    if case["kind"].startswith("fold"):
        n, k = case["n"], case["nsrc"]
        read, wrote = n * k * size[case["dt"]], n * size[case["out_dt"]]
        more = 2 if case["kind"] == "fold_clip" else 1
        return dict(bytes=read + more * wrote + 16, flops=n * (k + 2 + (more - 1)))
    n = sum(m for _, m in _sizes(case)[0])
    read = n * size[case["dt"]]
    wrote = n * size[case["out_dt"]] if case["kind"] != "norm" else 0
    return dict(bytes=read + wrote + 16, flops=n * {"norm": 2, "clip": 1, "norm_clip": 3}[case["kind"]])


def _exact_sumsq(flat):
    step = 1 << 24
    parts = [flat[a:a + step].to(torch.float64) for a in range(0, flat.numel(), step)]
    return math.fsum(float(torch.dot(p, p)) for p in parts)


def exact(case, seed):
    state = prepare(case, seed)

    def number(v):
        return np.array([v], dtype=np.float64)

    if case["kind"].startswith("fold"):
        mean = torch.stack([s.to(torch.float64) for s in state["srcs"]]).sum(0) / case["nsrc"]
        stored = mean.to(_TYPES[case["out_dt"]])
        sumsq = _exact_sumsq(stored)
        found = dict(sumsq=number(sumsq), mean=mean)
        if case["kind"] == "fold_clip":
            norm = math.sqrt(sumsq)
            c = min(1.0, _MAX_NORM / (norm + _EPS))
            found.update(norm=number(norm), out=stored.to(torch.float64) * c)
        return found
    sumsq = math.fsum(_exact_sumsq(state["flat"][a:a + n]) for a, n in state["spans"])
    if case["kind"] == "norm":
        return dict(sumsq=number(sumsq))
    norm = abs(case["scale"]) * math.sqrt(sumsq)
    c = case["scale"] * min(1.0, _MAX_NORM / (norm + _EPS))
    out = torch.zeros(state["flat"].numel(), dtype=torch.float64, device="cuda")
    for a, n in state["spans"]:
        out[a:a + n] = state["flat"][a:a + n].to(torch.float64) * c
    found = dict(norm=number(norm), out=out)
    if case["kind"] == "norm_clip":
        found["sumsq"] = number(sumsq)
    return found
