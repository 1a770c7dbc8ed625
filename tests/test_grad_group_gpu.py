"""pg_grad_clip (include/pg_ext.h): gradients spread over the ranks of a group,
clipped by their global norm.  One rank in this process, and real processes on
the one GPU of the test box over the xgmi and the rccl transport; every rank
checks its tensors against the norm of all ranks' gradients, formed in 64 bits
on the host.  Tolerances as in test_grad_gpu.py, with one more rounding per rank
for the sum over them."""
import ctypes
import math
import os
import pathlib
import socket
import sys

import pytest

import pgamd

pytestmark = pytest.mark.gpu
ROOT = pathlib.Path(__file__).resolve().parents[1]
U = 2.0 ** -53

# type, output type (0: in place), scale, max_norm, sizes of every rank's tensors (rank r takes entry r mod their number)
CASES = [
    ("f32", "f32", 1.0, 1.0, [[1000, 0, 4097], [5], [100_003, 7]]),
    ("bf16", "f32", 0.25, 2.0, [[70_001], [], [513, 513]]),                # a rank without tensors
    ("bf16", None, 0.5, 0.5, [[4099, 1], [300_001], [2]]),                 # in place
    ("f64", "f64", 1.0, 1e9, [[1], [1], [1]]),                             # nothing to clip
    ("f16", None, 1.0, 1.0, [[3] * 400, [17], [9] * 5]),                   # more tensors than one launch holds
]


def _types(torch):
    return {"f64": (pgamd.DT_DOUBLE, torch.float64), "f32": (pgamd.DT_F32, torch.float32),
            "f16": (pgamd.DT_F16, torch.float16), "bf16": (pgamd.DT_BF16, torch.bfloat16)}


def _gradients(torch, case, i, rank):
    g = torch.Generator().manual_seed(1000 * i + rank)
    dt = _types(torch)[case[0]][1]
    sizes = case[4][rank % len(case[4])]
    return [(torch.randn(n, generator=g, dtype=torch.float64) * 0.1 * (1 + rank)).to(dt) for n in sizes]


def _check(torch, lib, h, rank, world):
    """What every rank runs; a list of what went wrong."""
    T, fails = _types(torch), []
    for i, case in enumerate(CASES):
        dt, out_dt, scale, max_norm, _ = case
        every = [_gradients(torch, case, i, r) for r in range(world)]
        n = sum(t.numel() for ts in every for t in ts)
        sq = math.fsum(math.fsum((t.double().numpy() ** 2).tolist()) for ts in every for t in ts)
        want_norm = abs(scale) * math.sqrt(sq)
        c = scale * min(1.0, max_norm / (want_norm + 1e-6))
        ts = [t.cuda() for t in every[rank]]
        outs = ts if out_dt is None else [torch.full((t.numel(),), 7.0, dtype=T[out_dt][1], device="cuda") for t in ts]
        gp, ns, k = pgamd.tensor_list(ts)
        op = pgamd.tensor_list(outs)[0]
        norm = ctypes.c_double(math.nan)
        rc = lib.pg_grad_clip(op, T[out_dt or dt][0], gp, T[dt][0], ns, k, scale, max_norm, ctypes.byref(norm), h)
        if rc != 0:
            return fails + [(i, "rc", pgamd.last_error())]
        near = (n + 3 + world) * U
        if not abs(norm.value - want_norm) <= near * want_norm:
            fails.append((i, "norm", norm.value, want_norm))
        f = torch.finfo(T[out_dt or dt][1])
        step = f.eps / 2 + (2.0 ** -24 if f.bits == 16 else 0.0) + near + 7 * U
        for j, (t, o) in enumerate(zip(every[rank], outs)):
            want = t.double() * c
            off = (o.cpu().double() - want).abs()
            if not (off <= want.abs() * step * (1 + f.eps) + f.smallest_normal * f.eps).all():
                fails.append((i, j, "values", float(off.max())))
    # one rank's arguments are refused: the call fails everywhere, nothing changes, and the next one works
    x = torch.full((100,), 3.0, device="cuda")
    gp, ns, k = pgamd.tensor_list([x])
    bad = rank == world - 1
    rc = lib.pg_grad_clip(gp, pgamd.DT_BF16 if bad else pgamd.DT_F32, gp, pgamd.DT_F32, ns, k, 1.0, 1.0, None, h)
    msg = pgamd.last_error()
    if rc != -1 or ("output type" if bad else "1 of") not in msg or not bool((x == 3.0).all()):
        fails.append(("refused", rc, msg))
    norm = ctypes.c_double()
    rc = lib.pg_grad_clip(gp, pgamd.DT_F32, gp, pgamd.DT_F32, ns, k, 1.0, math.inf, ctypes.byref(norm), h)
    if rc != 0 or abs(norm.value - 30.0 * math.sqrt(world)) > 1e-12 or not bool((x == 3.0).all()):
        fails.append(("after", rc, norm.value))
    return fails


def test_one_rank(gpu, lib):
    h = ctypes.c_void_p()
    pgamd.check(lib.pg_connect_local(0, 1, pgamd.PG_TRANSPORT_SELF, ctypes.byref(h)), "pg_connect_local")
    try:
        assert _check(gpu, lib, h, 0, 1) == []
        assert lib.pg_grad_clip(None, 2, None, 2, None, 0, 1.0, 1.0, None, None) == -1
        assert "NULL handle" in (lib.pg_last_error() or b"").decode()
        norm = ctypes.c_double(5.0)
        assert lib.pg_grad_clip(None, 2, None, 2, None, 0, 1.0, 1.0, ctypes.byref(norm), h) == 0
        assert norm.value == 0.0
    finally:
        lib.pg_close(h)


def test_host_memory_is_refused(gpu, lib):
    h = ctypes.c_void_p()
    pgamd.check(lib.pg_connect_local(0, 1, pgamd.PG_TRANSPORT_SELF, ctypes.byref(h)), "pg_connect_local")
    try:
        dev, host = gpu.ones(8, device="cuda"), gpu.ones(8)
        d, ns, _ = pgamd.tensor_list([dev])
        o = pgamd.tensor_list([host])[0]
        for out, grad, word in ((d, o, "gradient 0"), (o, d, "output 0")):
            assert lib.pg_grad_clip(out, pgamd.DT_F32, grad, pgamd.DT_F32, ns, 1, 1.0, 1.0, None, h) == -1
            assert f"{word} is not device memory" in pgamd.last_error()
        assert bool((dev == 1).all()) and bool((host == 1).all())
    finally:
        lib.pg_close(h)


def test_gradients_produced_on_the_null_stream(gpu, lib):
    """Work on torch's default stream that is still running when the call is entered is waited for."""
    torch = gpu
    h = ctypes.c_void_p()
    pgamd.check(lib.pg_connect_local(0, 1, pgamd.PG_TRANSPORT_SELF, ctypes.byref(h)), "pg_connect_local")
    try:
        x = torch.zeros(50_000_000, device="cuda")
        for _ in range(50):
            x.add_(1.0)
        gp, ns, k = pgamd.tensor_list([x])
        norm = ctypes.c_double()
        assert lib.pg_grad_clip(gp, pgamd.DT_F32, gp, pgamd.DT_F32, ns, k, 1.0, math.inf, ctypes.byref(norm), h) == 0
        assert norm.value == math.sqrt(50_000_000 * 2500.0)
    finally:
        lib.pg_close(h)


def _free_port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


def _worker(rank, world, port, q, transport):
    os.environ.update(PG_TRANSPORT=transport, PG_RANK=str(rank), PG_DEVICE="0", PG_PORT=str(port),
                      PG_CONNECT_TIMEOUT_MS="60000", PG_BARRIER_TIMEOUT_MS="60000", NCCL_SOCKET_IFNAME="lo",
                      NCCL_IB_DISABLE="1", NCCL_HOSTID=f"pg-grad-test-{port}-rank{rank}")
    sys.path[:0] = [str(ROOT), str(ROOT / "rdma-ring-collectives_amd")]
    try:
        import torch
        torch.cuda.set_device(0)
        lib = pgamd.load()
        h = ctypes.c_void_p()
        if lib.connect_process_group(" ".join(["127.0.0.1"] * world).encode(), ctypes.byref(h)) != 0:
            q.put((rank, ["connect: " + pgamd.last_error()]))
            return
        fails = _check(torch, lib, h, rank, world)
        lib.pg_close(h)
    except Exception as e:  # report, never hang the parent
        fails = [("exception", repr(e))]
    q.put((rank, fails))


@pytest.mark.parametrize("transport,world", [("xgmi", 2), ("xgmi", 3), ("rccl", 2), ("rccl", 3)])
def test_ranks_in_processes(gpu, transport, world):
    import torch.multiprocessing as mp
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, world, port, q, transport)) for r in range(world)]
    for p in procs:
        p.start()
    results = []
    try:
        for _ in range(world):
            results.append(q.get(timeout=300))
    finally:
        for p in procs:
            p.join(timeout=60)
            if p.is_alive():
                p.kill()
    for rank, fails in results:
        assert not fails, (rank, fails)
    assert all(p.exitcode == 0 for p in procs)
