"""The gradient operators (include/pgk.h, pgk_grad_*) on dense gradients below and
above the size of the 256 MiB Infinity Cache, behind a producer on a stream of
their own, on sources in another process's memory, and without a sum.

Tolerances: none.  Gradients are small integers, so every square, every partial sum
(below 2^53) and every product with a power of two is exact in any order; the fold
is the same IEEE operations in the same order."""
import ctypes
import math

import pytest
import torch

import pgamd
import test_grad_gpu as base
from test_grad_gpu import PAIRS, TYPES, cell, ptrs, sizes, stream, work

pytestmark = pytest.mark.gpu
MIB = 1 << 20


def whole_numbers(n, dt, seed):
    """Whole numbers from -4 to 4 without 0: an element that is missed or counted twice shows in any sum of squares."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randint(1, 9, (n,), generator=g, device="cuda", dtype=torch.int8)
    return torch.where(x > 4, x - 9, x).to(TYPES[dt][1])


def exact_sum(x):
    """The sum of squares of whole numbers, in 64-bit integers."""
    return sum(int(p.to(torch.int64).square().sum()) for p in x.split(1 << 24))


def ragged(nbytes, tensors, dt):
    """Sizes that sum to nbytes, from one element to some hundred tiles, and gaps between them."""
    es = torch.finfo(TYPES[dt][1]).bits // 8
    total = nbytes // es
    shares = [((i * 7919) % 1009) ** 2 + 1 for i in range(tensors)]
    numels = [1 if i % 17 == 3 else 0 if i % 23 == 5 else 1 + total * s // (sum(shares) + tensors) for i, s in enumerate(shares)]
    numels[0] += total - sum(numels)
    return numels, [1 + i % 5 for i in range(tensors)]


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("nbytes", [256 * MIB - 4096, 256 * MIB, 256 * MIB + 4096])
def test_norm_and_clip_of_dense_gradients_around_the_cache(gpu, lib, nbytes, dt):
    """700 tensors, which two launches share, and some twenty tiles per block: blocks step from tensor to tensor,
    end in ragged tiles, and add to the sums of the first launch.  NaN between the tensors."""
    numels, gaps = ragged(nbytes, 700, dt)
    assert sum(numels) * (torch.finfo(TYPES[dt][1]).bits // 8) == nbytes and min(numels) == 0
    flat = torch.full((sum(numels) + sum(gaps) + 3,), math.nan, dtype=TYPES[dt][1], device="cuda")
    dense = whole_numbers(sum(numels), dt, nbytes % 1000)
    ts, at, off = [], 3, 0
    for n, gap in zip(numels, gaps):
        flat[at:at + n] = dense[off:off + n]
        ts.append(flat[at:at + n])
        at, off = at + n + gap, off + n
    want = exact_sum(dense)
    s = base.sumsq(lib, ts, dt)
    assert float(s) == want
    assert torch.equal(base.sumsq(lib, ts[::-1], dt), s)          # exact sums know no order
    # outputs with addresses of their own: as dense, without gaps
    out = torch.empty(sum(numels), dtype=TYPES[dt][1], device="cuda")
    norm = base.clip(lib, list(out.split(numels)), dt, ts, dt, s, 0.5, math.inf)
    assert abs(float(norm) - 0.5 * math.sqrt(want)) <= 2.0 ** -52 * float(norm)      # a root and a product
    assert torch.equal(out, dense * 0.5)


def test_norm_of_dense_gradients_of_one_tensor(gpu, lib):
    for dt, n in (("f64", 40 * MIB + 1), ("f32", 80 * MIB + 3), ("f16", 160 * MIB + 5), ("bf16", 160 * MIB + 7)):
        x = whole_numbers(n + 1, dt, 9)[1:]
        assert float(base.sumsq(lib, [x], dt)) == exact_sum(x)


# ---- the order on a stream -----------------------------------------------------------------------------

def test_calls_run_on_the_stream_they_are_given(gpu, lib):
    """On a stream that is not the current one, behind a long producer and before a consumer; only that stream is
    waited for.  A launch on any other stream would see the gradients as they were, or be seen too late."""
    n = 50_000_000
    side = torch.cuda.Stream()
    x, y, out, mean = torch.ones(n, device="cuda"), torch.full((n,), 3.0, device="cuda"), *torch.empty(2, n, device="cuda")
    s, norm, f, ws = cell(), cell(), cell(), work()
    seen = [torch.zeros(1, dtype=torch.float64, device="cuda") for _ in range(3)]
    tails = torch.zeros(2, 5, device="cuda")
    lists = [(ptrs([t]), sizes([t])) for t in (x, out)]
    srcs = ptrs([x, y])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(64):                                  # about 4 ms until x is 65
            x.add_(1.0)
    F32, handle = pgamd.DT_F32, side.cuda_stream
    assert stream() != handle
    assert lib.pgk_grad_sumsq(*lists[0], 1, F32, s.data_ptr(), ws.data_ptr(), handle) == 0
    assert lib.pgk_grad_clip(lists[1][0], F32, lists[0][0], F32, lists[0][1], 1, s.data_ptr(), 1, 0.5, math.inf,
                             norm.data_ptr(), handle) == 0
    assert lib.pgk_grad_fold(mean.data_ptr(), F32, srcs, 2, n, F32, 0.5, f.data_ptr(), ws.data_ptr(), handle) == 0
    with torch.cuda.stream(side):
        for a, b in zip(seen, (s, norm, f)):
            a.copy_(b)
        tails[0].copy_(out[-5:])
        tails[1].copy_(mean[-5:])
        got = [a.cpu() for a in seen] + [tails.cpu()]        # waits for the side stream alone
    assert float(got[0]) == n * 65.0 ** 2
    assert float(got[1]) == pytest.approx(0.5 * 65.0 * math.sqrt(n), rel=1e-15)
    assert float(got[2]) == n * 34.0 ** 2
    assert (got[3][0] == 32.5).all() and (got[3][1] == 34.0).all()
    torch.cuda.synchronize()


# ---- without a sum ---------------------------------------------------------------------------------------

@pytest.mark.parametrize("dt,out_dt", PAIRS)
@pytest.mark.parametrize("nsrc", [1, 3, 8, 9])
def test_fold_without_a_sum_in_any_number_of_blocks(gpu, lib, nsrc, dt, out_dt):
    """From one vector to a megabyte in all: with a sum up to 512 KiB are one block's, without one none are."""
    per = nsrc * torch.finfo(TYPES[dt][1]).bits // 8 + torch.finfo(TYPES[out_dt][1]).bits // 8
    for n in (1, 5, 1023, 4097, 8191, (512 << 10) // per, (512 << 10) // per + 1, (1 << 20) // per):
        srcs = [whole_numbers(n + 1, dt, 31 * k + n)[1:] for k in range(nsrc)]
        want = base.large_fold(srcs, 1.0 / nsrc, out_dt)
        out = torch.full((n + 2,), 7.0, dtype=TYPES[out_dt][1], device="cuda")
        base.fold(lib, out[1:n + 1], out_dt, srcs, dt, 1.0 / nsrc, want_sum=False)
        assert torch.equal(out[1:n + 1], want), n
        assert float(out[0]) == 7.0 and float(out[-1]) == 7.0
        again = torch.empty(n, dtype=TYPES[out_dt][1], device="cuda")
        s = base.fold(lib, again, out_dt, srcs, dt, 1.0 / nsrc)
        assert torch.equal(again, want)
        assert abs(float(s) - float(want.double().square().sum())) <= 2 * (n + 3) * 2.0 ** -53 * float(s)


# ---- sources in another process's memory -----------------------------------------------------------------

class _Handle(ctypes.Structure):
    _fields_ = [("reserved", ctypes.c_char * 64)]


def _hip():
    hip = ctypes.CDLL("libamdhip64.so.7")
    hip.hipMalloc.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_size_t]
    hip.hipFree.argtypes = [ctypes.c_void_p]
    hip.hipMemcpy.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int]
    hip.hipIpcGetMemHandle.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    hip.hipIpcOpenMemHandle.argtypes = [ctypes.POINTER(ctypes.c_void_p), _Handle, ctypes.c_uint]
    hip.hipIpcCloseMemHandle.argtypes = [ctypes.c_void_p]
    return hip


# type, output type, sources, elements of each: one block, many blocks, the burst form, more sources than one unrolls
REMOTE = [("f32", "f32", 3, 1001), ("bf16", "f32", 4, 300_001), ("bf16", "bf16", 5, 17 * MIB), ("f32", "f32", 9, 70_003)]


def _remote_sources(i):
    dt, _, nsrc, n = REMOTE[i]
    return whole_numbers(nsrc * n, dt, 900 + i)


def _owner(to_parent, from_parent):
    try:
        torch.cuda.set_device(0)
        hip, held = _hip(), []
        for i in range(len(REMOTE)):
            x = _remote_sources(i)
            p, h = ctypes.c_void_p(), _Handle()
            nbytes = x.numel() * x.element_size()
            torch.cuda.synchronize()
            rc = hip.hipMalloc(ctypes.byref(p), nbytes) or hip.hipMemcpy(p, x.data_ptr(), nbytes, 3)
            torch.cuda.synchronize()
            rc = rc or hip.hipIpcGetMemHandle(ctypes.byref(h), p)
            held.append(p)
            to_parent.put((rc, bytes(h)))
        from_parent.get(timeout=100)                         # the parent has closed its mappings
        for p in held:
            hip.hipFree(p)
        to_parent.put("done")
    except Exception as e:  # report, never hang the parent
        to_parent.put(repr(e))


def test_fold_of_another_process_s_memory(gpu, lib):
    """Sources that a peer process allocated, mapped through HIP IPC."""
    import torch.multiprocessing as mp
    ctx = mp.get_context("spawn")
    back, forth = ctx.Queue(), ctx.Queue()
    p = ctx.Process(target=_owner, args=(back, forth))
    p.start()
    hip = _hip()
    try:
        for i, (dt, out_dt, nsrc, n) in enumerate(REMOTE):
            rc, raw = back.get(timeout=100)
            assert rc == 0
            at = ctypes.c_void_p()
            assert hip.hipIpcOpenMemHandle(ctypes.byref(at), _Handle.from_buffer_copy(raw), 1) == 0
            es = torch.finfo(TYPES[dt][1]).bits // 8
            srcs = (ctypes.c_void_p * nsrc)(*[at.value + k * n * es for k in range(nsrc)])
            out = torch.full((n,), 7.0, dtype=TYPES[out_dt][1], device="cuda")
            s, ws = cell(), work()
            assert lib.pgk_grad_fold(out.data_ptr(), TYPES[out_dt][0], srcs, nsrc, n, TYPES[dt][0], 0.25, s.data_ptr(),
                                     ws.data_ptr(), stream()) == 0
            want = base.large_fold(list(_remote_sources(i).split(n)), 0.25, out_dt)
            torch.cuda.synchronize()
            assert hip.hipIpcCloseMemHandle(at) == 0
            assert torch.equal(out, want), i
            assert float(s) == exact_sum(want * 4) / 16      # quarters of whole numbers: exact as well
        forth.put("closed")
        assert back.get(timeout=100) == "done"
    finally:
        forth.put("closed")
        p.join(timeout=60)
        if p.is_alive():
            p.kill()
    assert p.exitcode == 0


def _replayed_us(call):
    """Time of one of 60 calls captured one behind the other, the shortest of nine replays."""
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        for _ in range(60):
            call()
    took = []
    for _ in range(12):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        took.append(a.elapsed_time(b) * 1e3 / 60)
    return min(took[3:])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("want_sum", [False, True])
def test_a_small_fold_takes_no_longer_than_one_of_twice_its_size(gpu, lib, dt, want_sum):
    """The form of one block is for calls that it makes shorter.  Two sources, 480 KiB in all against 960: where one
    block took the smaller one, it was 2 to 4 times as long."""
    took = []
    for n in (480 * 1024, 960 * 1024):
        n //= 3 * torch.finfo(TYPES[dt][1]).bits // 8
        srcs, ws, s = [whole_numbers(n, dt, k) for k in range(2)], work(), cell()
        out, lst, code = torch.empty_like(srcs[0]), ptrs(srcs), TYPES[dt][0]

        def call():
            assert lib.pgk_grad_fold(out.data_ptr(), code, lst, 2, n, code, 0.5, s.data_ptr() if want_sum else None,
                                     ws.data_ptr() if want_sum else None, stream()) == 0

        took.append(_replayed_us(call))
    assert took[0] <= 1.6 * took[1], took
