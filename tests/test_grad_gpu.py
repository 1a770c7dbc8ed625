"""Gradient operators (include/pgk.h: pgk_grad_sumsq, pgk_grad_clip,
pgk_grad_fold) against plain forms in 64 bits on the host.

Tolerances.  h = finfo.eps / 2 is the half step that one rounding may be off by.
  sumsq   every square of an f32, f16 or bf16 value is exact in 64 bits; a sum of n
          positive terms in any order is within (n - 1) 2^-53 of itself, the square
          of an f64 value within one more on either side, and the two sums of the
          reference are rounded once each: (n + 3) 2^-53, relative.
  clip    c takes a sum of nsum terms, a root, two products, a sum and a quotient:
          within (nsum + 6) 2^-53.  The product adds 2^-53, its rounding to f32
          2^-24, that to 16 bits h.  Below the smallest normal number a rounding is
          off by half the smallest subnormal one.
  fold    the same IEEE operations in the same order: equal bits.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

import pgamd

pytestmark = pytest.mark.gpu

TYPES = {"f64": (pgamd.DT_DOUBLE, torch.float64), "f32": (pgamd.DT_F32, torch.float32),
         "f16": (pgamd.DT_F16, torch.float16), "bf16": (pgamd.DT_BF16, torch.bfloat16)}
PAIRS = [("f64", "f64"), ("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f32")]
U = 2.0 ** -53


def stream():
    return torch.cuda.current_stream().cuda_stream


def ptrs(ts):
    return (ctypes.c_void_p * max(len(ts), 1))(*[t.data_ptr() if t.numel() else None for t in ts])


def sizes(ts):
    return (ctypes.c_size_t * max(len(ts), 1))(*[t.numel() for t in ts])


def cell(value=math.nan, n=1):
    return torch.full((n,), value, dtype=torch.float64, device="cuda")


def work():
    """Workspace with contents that must not matter."""
    return torch.full((pgamd.PGK_GRAD_WORK_BYTES // 8,), math.nan, dtype=torch.float64, device="cuda")


def sumsq(lib, ts, dt, out=None, ws=None):
    out = cell() if out is None else out
    ws = work() if ws is None else ws
    rc = lib.pgk_grad_sumsq(ptrs(ts), sizes(ts), len(ts), TYPES[dt][0], out.data_ptr(), ws.data_ptr(), stream())
    assert rc == 0, pgamd.last_error()
    return out


def clip(lib, outs, out_dt, ts, dt, sums, scale=1.0, max_norm=1.0, norm=None):
    norm = cell() if norm is None else norm
    rc = lib.pgk_grad_clip(ptrs(outs), TYPES[out_dt][0], ptrs(ts), TYPES[dt][0], sizes(ts), len(ts), sums.data_ptr(),
                           sums.numel(), scale, max_norm, norm.data_ptr(), stream())
    assert rc == 0, pgamd.last_error()
    return norm


def fold(lib, out, out_dt, srcs, dt, scale, n=None, want_sum=True):
    s, ws = (cell(), work()) if want_sum else (None, None)
    rc = lib.pgk_grad_fold(out.data_ptr(), TYPES[out_dt][0], ptrs(srcs), len(srcs), srcs[0].numel() if n is None else n,
                           TYPES[dt][0], scale, s.data_ptr() if want_sum else None, ws.data_ptr() if want_sum else None,
                           stream())
    assert rc == 0, pgamd.last_error()
    return s


def bucket(numels, dt, seed, gap=0, pad=math.nan):
    """Tensors of these sizes as views of one buffer, `gap` elements of `pad` before, between and behind them."""
    g = torch.Generator().manual_seed(seed)
    total = sum(numels) + gap * (len(numels) + 1)
    flat = torch.full((total,), pad, dtype=torch.float64)
    spans, at = [], gap
    for n in numels:
        flat[at:at + n] = torch.randn(n, generator=g, dtype=torch.float64) * 10 ** float(torch.rand(1, generator=g) * 4 - 3)
        spans.append((at, n))
        at += n + gap
    flat = flat.to(TYPES[dt][1]).cuda()
    return flat, [flat[a:a + n] for a, n in spans]


def exact_sumsq(ts):
    return math.fsum(math.fsum((t.detach().cpu().double().numpy() ** 2).tolist()) for t in ts)


def n_of(ts):
    return sum(t.numel() for t in ts)


def near_sum(got, want, n):
    """A sum of n squares against the exact one; see the head of the file."""
    return abs(float(got) - want) <= (n + 3) * U * want


# sizes around what one thread, one wave, one block and one tile take, in every type
EDGES = [1, 2, 3, 7, 8, 9, 63, 64, 65, 255, 257, 511, 513, 1023, 1024, 1025, 2047, 2048, 2049, 4095, 4096, 4097, 8191,
         8192, 8193, 16385, 32769]
LISTS = {
    "none": [], "empty": [0], "empties": [0, 0, 0], "one": [1], "one-between-empties": [0, 1, 0],
    "edges": EDGES, "edges-backwards": EDGES[::-1], "one-large": [1_000_003],
    "fills-a-launch": [5] * 351, "one-more": [5] * 352, "fills-with-outputs": [5] * 218, "one-more-with-outputs": [5] * 219,
    "many": [(37 * i) % 301 for i in range(1000)],
    "large-behind-many": [3] * 400 + [300_001], "large-before-many": [300_001] + [3] * 400,
}


# ---- sum of squares --------------------------------------------------------------------------------

@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("which", list(LISTS))
def test_sumsq(gpu, lib, which, dt):
    for gap in (0, 1, 5):
        _, ts = bucket(LISTS[which], dt, 17 + gap, gap)      # NaN between the tensors: a stray read shows
        got, want = float(sumsq(lib, ts, dt)), exact_sumsq(ts)
        assert near_sum(got, want, n_of(ts)), (which, dt, gap, got, want)


@pytest.mark.parametrize("dt,values", [
    ("f32", [1e30, -3e38, 1e-30, 1.4e-45]), ("f32", [1e-40] * 1000), ("f32", [3e38] * 5000),
    ("bf16", [3e38] * 5000), ("bf16", [1e-40] * 999), ("f16", [65504.0] * 5000), ("f16", [6e-8] * 777),
])
def test_sumsq_holds_the_range_of_the_type(gpu, lib, dt, values):
    t = torch.tensor(values, dtype=torch.float64).to(TYPES[dt][1]).cuda()
    got, want = float(sumsq(lib, [t], dt)), exact_sumsq([t])
    assert want > 0 and math.isfinite(want)
    assert near_sum(got, want, t.numel())


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("at", [0, 4500, 9998])
def test_sumsq_shows_what_is_not_finite(gpu, lib, dt, bad, at):
    t = torch.ones(9999, dtype=TYPES[dt][1], device="cuda")
    t[at] = bad
    got = float(sumsq(lib, [t[:1], t], dt))
    assert math.isnan(got) if math.isnan(bad) else got == math.inf


def test_sumsq_same_call_same_bits(gpu, lib):
    _, ts = bucket([100_003, 7, 2_000_001, 0, 513], "f32", 5)
    ws = work()
    got = [sumsq(lib, ts, "f32", ws=ws).view(torch.int64).item() for _ in range(5)]
    assert len(set(got)) == 1


def test_sumsq_counts_a_tensor_as_often_as_it_is_listed(gpu, lib):
    _, ts = bucket([1001], "bf16", 3)
    want = 3 * exact_sumsq(ts)
    assert near_sum(sumsq(lib, ts * 3, "bf16"), want, 3003)


# ---- clip ------------------------------------------------------------------------------------------

def coefficient(sums, scale, max_norm):
    norm = abs(scale) * math.sqrt(math.fsum(sums))
    return norm, scale * min(1.0, max_norm / (norm + 1e-6))


def allowed(want, out_dt, nsum):
    """How far each result may be from `want` (f64); see the head of the file."""
    f = torch.finfo(TYPES[out_dt][1])
    h, c = f.eps / 2, (nsum + 6) * U
    step = {"f64": U, "f32": h + U, "f16": h + 2.0 ** -24 + U, "bf16": h + 2.0 ** -24 + U}[out_dt]
    return want.abs() * (step + c) * (1 + 2 * h) + f.smallest_normal * f.eps / 2 * (1 + 2.0 ** -8)


@pytest.mark.parametrize("dt,out_dt", PAIRS)
@pytest.mark.parametrize("which", list(LISTS))
def test_clip(gpu, lib, which, dt, out_dt):
    # outputs that lie to each other as the gradients do, and outputs that do not
    for gap, out_gap, scale, sums in ((0, 0, 1.0, [4.0]), (3, 3, 1 / 3, [0.3, 1e-9, 700.0]), (1, 2, -2.0, [1e-3]),
                                      (0, 1, 0.7, [1.0]), (2, 0, 0.7, [9.0])):
        _, ts = bucket(LISTS[which], dt, 23 + gap, gap)
        out, outs = bucket(LISTS[which], out_dt, 1, out_gap, pad=7.0)
        norm = clip(lib, outs, out_dt, ts, dt, torch.tensor(sums, dtype=torch.float64, device="cuda"), scale, 1.5)
        want_norm, c = coefficient(sums, scale, 1.5)
        assert abs(float(norm) - want_norm) <= (len(sums) + 2) * U * want_norm
        for t, o in zip(ts, outs):
            want = t.cpu().double() * c
            assert ((o.cpu().double() - want).abs() <= allowed(want, out_dt, len(sums))).all(), (which, gap)
        inside = torch.zeros(out.numel(), dtype=torch.bool)
        for o in outs:
            inside[o.storage_offset():o.storage_offset() + o.numel()] = True
        assert (out.cpu()[~inside].double() == 7.0).all()      # what lies between the outputs stays


@pytest.mark.parametrize("nsum", [2, 63, 64, 65, 1000])
def test_clip_by_many_partial_sums(gpu, lib, nsum):
    sums = [0.001 * (1 + j % 7) for j in range(nsum)]
    _, ts = bucket([3000, 1], "f32", nsum)
    outs = [torch.empty_like(t) for t in ts]
    norm = clip(lib, outs, "f32", ts, "f32", torch.tensor(sums, dtype=torch.float64, device="cuda"), 1.0, 0.01)
    want_norm, c = coefficient(sums, 1.0, 0.01)
    assert abs(float(norm) - want_norm) <= (nsum + 2) * U * want_norm
    for t, o in zip(ts, outs):
        want = t.cpu().double() * c
        assert ((o.cpu().double() - want).abs() <= allowed(want, "f32", nsum)).all()


def test_clip_bits_do_not_depend_on_the_layout(gpu, lib):
    """Adjacent tensors are clipped as one; the results are those of the same tensors apart."""
    numels = [5, 4097, 1, 0, 70_001, 3]
    _, apart = bucket(numels, "bf16", 12, 3, pad=0.0)
    flat = torch.cat(apart)
    together = list(flat.split(numels))
    s = sumsq(lib, apart, "bf16")
    assert torch.equal(sumsq(lib, together, "bf16"), s)      # and the norm's bits do not either
    clip(lib, apart, "bf16", apart, "bf16", s, 0.3, 1.0)
    clip(lib, together, "bf16", together, "bf16", s, 0.3, 1.0)
    assert torch.equal(torch.cat(apart), flat)


@pytest.mark.parametrize("dt,out_dt", PAIRS)
@pytest.mark.parametrize("scale", [1.0, 0.5, -4.0])
def test_clip_by_powers_of_two_is_exact(gpu, lib, dt, out_dt, scale):
    """No norm is above max_norm = infinity, so c = scale: every product is exact, or one rounding of it."""
    _, ts = bucket(EDGES, dt, 31, 1)
    _, outs = bucket(EDGES, out_dt, 2, 2)
    clip(lib, outs, out_dt, ts, dt, cell(9.0), scale, math.inf)
    for t, o in zip(ts, outs):
        want = (t.cpu().double() * scale).to(TYPES[out_dt][1])
        assert torch.equal(o.cpu(), want)


@pytest.mark.parametrize("dt", list(TYPES))
def test_clip_in_place(gpu, lib, dt):
    for sums, max_norm in (([100.0], 1.0), ([0.25], 1.0), ([0.0], 1.0)):
        flat, ts = bucket([5, 0, 4097, 100_001, 1], dt, 41, 3)
        before = [t.cpu().double() for t in ts]
        norm = clip(lib, ts, dt, ts, dt, torch.tensor(sums, dtype=torch.float64, device="cuda"), 1.0, max_norm)
        want_norm, c = coefficient(sums, 1.0, max_norm)
        assert abs(float(norm) - want_norm) <= 3 * U * want_norm
        for t, b in zip(ts, before):
            if c == 1.0:
                assert torch.equal(t.cpu().double(), b)
            else:
                assert ((t.cpu().double() - b * c).abs() <= allowed(b * c, dt, 1)).all()


def test_clip_at_the_ends_of_max_norm(gpu, lib):
    _, ts = bucket([1000, 3], "f32", 51)
    outs = [torch.full_like(t, 5.0) for t in ts]
    assert float(clip(lib, outs, "f32", ts, "f32", cell(2.25), 1.0, 0.0)) == 1.5
    assert all((o == 0).all() for o in outs)                              # max_norm = 0: everything goes
    assert float(clip(lib, outs, "f32", ts, "f32", cell(0.0), 1.0, 1.0)) == 0.0
    assert all(torch.equal(o, t) for o, t in zip(outs, ts))               # norm 0: nothing is clipped
    assert float(clip(lib, outs, "f32", ts, "f32", cell(1e200), 0.0, 1.0)) == 0.0
    assert all((o == 0).all() for o in outs)                              # scale = 0


@pytest.mark.parametrize("dt", ["bf16", "f32", "f64"])
def test_clip_of_gradients_that_exploded(gpu, lib, dt):
    """Norms of 1e41 and more: c is below what 32 bits hold with any precision, the results are not."""
    _, ts = bucket([5000], "f64", 55)
    t = (ts[0] / ts[0].abs().max() * 3e38).to(TYPES[dt][1])
    out = torch.empty_like(t)
    s = sumsq(lib, [t], dt)
    clip(lib, [out], dt, [t], dt, s, 1e-3, 1e-3)
    _, c = coefficient([exact_sumsq([t])], 1e-3, 1e-3)
    assert 0 < c < 1e-40
    want = t.cpu().double() * c
    assert ((out.cpu().double() - want).abs() <= allowed(want, dt, 5000)).all()


@pytest.mark.parametrize("dt,out_dt", PAIRS)
def test_clip_without_a_limit_keeps_what_is_not_finite_to_itself(gpu, lib, dt, out_dt):
    """max_norm = infinity scales and no more, whatever the norm is."""
    t = torch.ones(3000, dtype=TYPES[dt][1], device="cuda")
    t[3], t[4] = math.inf, math.nan
    out = torch.empty(3000, dtype=TYPES[out_dt][1], device="cuda")
    for value in (math.inf, math.nan):
        norm = clip(lib, [out], out_dt, [t], dt, cell(value), 0.5, math.inf)
        assert math.isnan(float(norm)) if math.isnan(value) else float(norm) == math.inf
        got = out.cpu().double()
        assert got[3] == math.inf and got[4].isnan() and int((got == 0.5).sum()) == 2998


@pytest.mark.parametrize("dt,out_dt", PAIRS)
def test_clip_by_a_norm_that_is_not_finite(gpu, lib, dt, out_dt):
    t = torch.ones(5000, dtype=TYPES[dt][1], device="cuda")
    t[77] = math.inf
    t[78] = -math.inf
    out = torch.full((5000,), 9.0, dtype=TYPES[out_dt][1], device="cuda")
    s = sumsq(lib, [t], dt)
    assert float(clip(lib, [out], out_dt, [t], dt, s)) == math.inf        # c = 0: 0, and inf * 0
    got = out.cpu().double()
    assert got[77].isnan() and got[78].isnan() and int((got == 0).sum()) == 4998
    t[4999] = math.nan
    s = sumsq(lib, [t], dt)
    assert math.isnan(float(clip(lib, [out], out_dt, [t], dt, s)))        # c = NaN
    assert out.cpu().double().isnan().all()


def test_clip_overflow_and_subnormal_results(gpu, lib):
    t = torch.tensor([65504.0, 1e-7, 6e-8, -65504.0], dtype=torch.float16, device="cuda")
    o = torch.empty_like(t)
    clip(lib, [o], "f16", [t], "f16", cell(0.0), 4.0, math.inf)
    assert torch.equal(o.cpu(), (t.cpu().double() * 4).to(torch.float16))
    clip(lib, [o], "f16", [t], "f16", cell(0.0), 0.5, math.inf)
    assert torch.equal(o.cpu(), (t.cpu().double() * 0.5).to(torch.float16))
    x = torch.tensor([1.5e-38, 3e-45, 3.4e38], dtype=torch.float32, device="cuda")
    y = torch.empty_like(x)
    clip(lib, [y], "f32", [x], "f32", cell(0.0), 0.25, math.inf)
    assert torch.equal(y.cpu(), (x.cpu().double() * 0.25).float())


# ---- averaging fold --------------------------------------------------------------------------------

def plain_fold(srcs, scale, out_dt):
    acc = srcs[0].cpu().double()
    for s in srcs[1:]:
        acc = acc + s.cpu().double()
    acc = acc * scale
    return (acc.float() if out_dt in ("f16", "bf16") else acc).to(TYPES[out_dt][1])


@pytest.mark.parametrize("dt,out_dt", PAIRS)
@pytest.mark.parametrize("nsrc", [1, 2, 3, 4, 5, 6, 7, 8, 9, 16])
def test_fold(gpu, lib, nsrc, dt, out_dt):
    for k, n in enumerate((1, 2, 7, 9, 255, 1025, 4099, 100_003)):
        off = k % 4                                          # sources and output at different alignments
        srcs = [bucket([n], dt, 100 * nsrc + s, off + s % 3)[1][0] for s in range(nsrc)]
        flat, outs = bucket([n], out_dt, 3, 1 + off, pad=7.0)
        s = fold(lib, outs[0], out_dt, srcs, dt, 1.0 / nsrc)
        want = plain_fold(srcs, 1.0 / nsrc, out_dt)
        assert torch.equal(outs[0].cpu(), want), (n, nsrc)
        assert (flat.cpu()[:1 + off].double() == 7).all() and (flat.cpu()[1 + off + n:].double() == 7).all()
        sq = exact_sumsq([want])
        assert near_sum(s, sq, n)
        again = torch.zeros(n, dtype=TYPES[out_dt][1], device="cuda")
        fold(lib, again, out_dt, srcs, dt, 1.0 / nsrc, want_sum=False)
        assert torch.equal(again.cpu(), want)


@pytest.mark.parametrize("dt", list(TYPES))
def test_fold_into_a_source(gpu, lib, dt):
    for nsrc, into in ((2, 0), (3, 2), (8, 5), (11, 10)):
        srcs = [bucket([50_001], dt, s, 1)[1][0] for s in range(nsrc)]
        want = plain_fold(srcs, 0.25, dt)
        fold(lib, srcs[into], dt, srcs, dt, 0.25)
        assert torch.equal(srcs[into].cpu(), want)


@pytest.mark.parametrize("nsrc", [3, 9])
def test_fold_of_a_source_that_is_listed_twice(gpu, lib, nsrc):
    x = bucket([10_001], "f32", 4, 1)[1][0]
    y = bucket([10_001], "f32", 5, 2)[1][0]
    srcs = [x, y] + [x] * (nsrc - 2)
    want = plain_fold(srcs, 0.5, "f32")
    fold(lib, x, "f32", srcs, "f32", 0.5)
    assert torch.equal(x.cpu(), want)


def large_sources(n, dt, nsrc, off=0):
    g = torch.Generator(device="cuda").manual_seed(n + nsrc)
    return [torch.randn(n + off, generator=g, device="cuda").to(TYPES[dt][1])[off:] for _ in range(nsrc)]


def large_fold(srcs, scale, out_dt):
    """plain_fold with torch's f64 operations on the GPU, which round as the host's do."""
    acc = srcs[0].double()
    for s in srcs[1:]:
        acc = acc + s.double()
    acc = acc * scale
    return (acc.float() if out_dt in ("f16", "bf16") else acc).to(TYPES[out_dt][1])


MIB = 1 << 20
# bytes per source: the burst form takes 64 MiB at a time, then 32 to 64, the rest one vector per thread
BURST = [(5, 32 * MIB), (6, 32 * MIB + 16), (7, 64 * MIB), (8, 64 * MIB + 40 * MIB), (8, 100 * MIB + 24), (5, 31 * MIB)]


@pytest.mark.parametrize("dt", list(TYPES))
@pytest.mark.parametrize("nsrc,nbytes", BURST)
@pytest.mark.parametrize("off", [0, 1])
def test_fold_of_large_blocks(gpu, lib, dt, nsrc, nbytes, off):
    n = nbytes // torch.finfo(TYPES[dt][1]).bits * 8 + off
    srcs = large_sources(n, dt, nsrc, off)
    want = large_fold(srcs, 1.0 / nsrc, dt)
    out = torch.full((n + 2,), 7.0, dtype=TYPES[dt][1], device="cuda")
    s = fold(lib, out[1:n + 1], dt, srcs, dt, 1.0 / nsrc)
    assert torch.equal(out[1:n + 1], want)
    assert float(out[0]) == 7.0 and float(out[-1]) == 7.0
    sq = math.fsum(float((part.double() ** 2).sum()) for part in want.split(1 << 16))
    assert near_sum(s, sq, n + (1 << 16))                 # torch's partial sums are off by up to 2^16 roundings
    fold(lib, srcs[nsrc - 2], dt, srcs, dt, 1.0 / nsrc, want_sum=False)      # into a source
    assert torch.equal(srcs[nsrc - 2], want)


@pytest.mark.parametrize("dt,out_dt", PAIRS)
@pytest.mark.parametrize("nsrc,n", [(2, 40_000_003), (3, 70_000_001), (9, 36_000_007)])
def test_fold_of_more_tiles_than_blocks(gpu, lib, dt, out_dt, nsrc, n):
    srcs = large_sources(n, dt, nsrc)
    out = torch.empty(n, dtype=TYPES[out_dt][1], device="cuda")
    s = fold(lib, out, out_dt, srcs, dt, 0.3)
    want = large_fold(srcs, 0.3, out_dt)
    assert torch.equal(out, want)
    sq = math.fsum(float((part.double() ** 2).sum()) for part in want.split(1 << 16))
    assert near_sum(s, sq, n + (1 << 16))


def test_fold_of_nothing(gpu, lib):
    s, ws = cell(), work()
    assert lib.pgk_grad_fold(None, pgamd.DT_F32, None, 3, 0, pgamd.DT_F32, 1.0, s.data_ptr(), ws.data_ptr(), stream()) == 0
    assert float(s) == 0.0


@pytest.mark.parametrize("dt,out_dt", PAIRS)
def test_fold_of_what_is_not_finite(gpu, lib, dt, out_dt):
    a = torch.ones(3000, dtype=TYPES[dt][1], device="cuda")
    b = a.clone()
    a[5], b[5] = math.inf, -math.inf
    a[6] = math.inf
    b[2999] = math.nan
    out = torch.empty(3000, dtype=TYPES[out_dt][1], device="cuda")
    s = fold(lib, out, out_dt, [a, b], dt, 0.5)
    got = out.cpu().double()
    assert got[5].isnan() and got[6] == math.inf and got[2999].isnan() and int((got == 1).sum()) == 2997
    assert math.isnan(float(s))


def test_fold_keeps_what_32_bits_would_lose(gpu, lib):
    """1e8 + 1 - 1e8 is 1 in a 64-bit sum, 0 in a 32-bit one."""
    srcs = [torch.full((999,), v, device="cuda") for v in (1e8, 1.0, -1e8)]
    out = torch.empty(999, device="cuda")
    assert abs(float(fold(lib, out, "f32", srcs, "f32", 1.0)) - 999.0) == 0.0
    assert (out == 1.0).all()


# ---- a step of them together -------------------------------------------------------------------------

@pytest.mark.parametrize("dt,out_dt", PAIRS)
def test_step_over_buckets(gpu, lib, dt, out_dt):
    """Two buckets are folded from 4 ranks' copies, each with a sum of its own; one clip by the norm of both."""
    numels, ranks = [70_001, 513], 4
    copies = [[bucket([n], dt, 7 * r + b, 1)[1][0] for r in range(ranks)] for b, n in enumerate(numels)]
    means = [torch.empty(n, dtype=TYPES[dt][1], device="cuda") for n in numels]
    sums, ws = cell(n=2), work()
    for b, n in enumerate(numels):
        assert lib.pgk_grad_fold(means[b].data_ptr(), TYPES[dt][0], ptrs(copies[b]), ranks, n, TYPES[dt][0], 1 / ranks,
                                 sums.data_ptr() + 8 * b, ws.data_ptr(), stream()) == 0
    outs = [torch.empty(n, dtype=TYPES[out_dt][1], device="cuda") for n in numels]
    norm = clip(lib, outs, out_dt, means, dt, sums, 1.0, 0.5)
    want_means = [plain_fold(c, 1 / ranks, dt) for c in copies]
    sq = exact_sumsq(want_means)
    want_norm, c = coefficient([sq], 1.0, 0.5)
    assert abs(float(norm) - want_norm) <= sum(numels) * U * want_norm
    assert c < 1.0
    for o, m in zip(outs, want_means):
        want = m.double() * c
        assert ((o.cpu().double() - want).abs() <= allowed(want, out_dt, sum(numels))).all()
    # and the separate pass over the same tensors agrees with the fold's own sums
    assert near_sum(sumsq(lib, means, dt), sq, sum(numels))


def test_step_captured_and_replayed(gpu, lib):
    """Norm and clip in a graph, replayed with new gradients; eager calls with a
    workspace of their own and synchronisations between the replays."""
    numels = [4097, 0, 65_537, 3, 1] + [11] * 300
    flat, ts = bucket(numels, "bf16", 61, 1, pad=0.0)
    out, outs = bucket(numels, "f32", 62, 1, pad=0.0)
    s, norm, ws = cell(), cell(), work()
    lists = ptrs(ts), sizes(ts), ptrs(outs)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        assert lib.pgk_grad_sumsq(lists[0], lists[1], len(ts), pgamd.DT_BF16, s.data_ptr(), ws.data_ptr(), stream()) == 0
        assert lib.pgk_grad_clip(lists[2], pgamd.DT_F32, lists[0], pgamd.DT_BF16, lists[1], len(ts), s.data_ptr(), 1, 0.5,
                                 1.0, norm.data_ptr(), stream()) == 0
    for rep in range(4):
        new, _ = bucket(numels, "bf16", 70 + rep, 1, pad=0.0)
        flat.copy_(new)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed, replayed_norm = out.clone(), float(norm)
        eager_out, eager_outs = bucket(numels, "f32", 63, 1, pad=0.0)
        es = sumsq(lib, ts, "bf16")
        assert float(clip(lib, eager_outs, "f32", ts, "bf16", es, 0.5, 1.0)) == replayed_norm
        assert torch.equal(torch.cat(eager_outs), torch.cat([replayed[o.storage_offset():o.storage_offset() + o.numel()]
                                                             for o in outs]))
        want = exact_sumsq(ts)
        assert near_sum(s, want, n_of(ts))


def test_fold_captured_and_replayed(gpu, lib):
    srcs = [torch.empty(70_003, dtype=torch.float16, device="cuda") for _ in range(5)]
    out = torch.empty(70_003, dtype=torch.float32, device="cuda")
    s, ws, lst = cell(), work(), ptrs(srcs)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        assert lib.pgk_grad_fold(out.data_ptr(), pgamd.DT_F32, lst, 5, 70_003, pgamd.DT_F16, 0.2, s.data_ptr(),
                                 ws.data_ptr(), stream()) == 0
    for rep in range(4):
        for k, t in enumerate(srcs):
            t.copy_(bucket([70_003], "f16", 10 * rep + k)[0])
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = plain_fold(srcs, 0.2, "f32")
        assert torch.equal(out.cpu(), want)
        sq = exact_sumsq([want])
        assert near_sum(s, sq, 70_003)
        torch.ones(1000, device="cuda").sum()
        torch.cuda.synchronize()


def test_two_graphs_that_share_a_workspace(gpu, lib):
    """Replayed one behind the other on one stream, with eager calls on the same workspace between them."""
    ws, side = work(), torch.cuda.Stream()
    sets = [bucket([200_003, 9], "f32", 100 + k)[1] for k in range(2)]
    cells, lists, graphs = [cell() for _ in sets], [(ptrs(ts), sizes(ts)) for ts in sets], []
    torch.cuda.synchronize()
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side), torch.cuda.graph(g, stream=side):
            assert lib.pgk_grad_sumsq(*lists[k], 2, pgamd.DT_F32, cells[k].data_ptr(), ws.data_ptr(), stream()) == 0
        graphs.append(g)
    want = [exact_sumsq(ts) for ts in sets]
    for rep in range(3):
        for c in cells:
            c.fill_(math.nan)
        graphs[0].replay()
        graphs[1].replay()
        eager = sumsq(lib, sets[1], "f32", ws=ws)
        graphs[0].replay()
        torch.cuda.synchronize()
        assert near_sum(cells[0], want[0], 200_012) and near_sum(cells[1], want[1], 200_012)
        assert torch.equal(eager, cells[1])


def test_two_streams_with_a_workspace_each(gpu, lib):
    sets = [bucket([3_000_001, 5, 100_000], "f32", 80 + k)[1] for k in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    cells, works = [cell() for _ in range(2)], [work() for _ in range(2)]
    norms = [cell() for _ in range(2)]
    want = [exact_sumsq(ts) for ts in sets]
    before = [[t.cpu().double() for t in ts] for ts in sets]
    torch.cuda.synchronize()
    for k in range(2):
        with torch.cuda.stream(streams[k]):
            sumsq(lib, sets[k], "f32", cells[k], works[k])
            clip(lib, sets[k], "f32", sets[k], "f32", cells[k], norm=norms[k])
    torch.cuda.synchronize()
    for k in range(2):
        n = n_of(sets[k])
        assert near_sum(cells[k], want[k], n)
        _, c = coefficient([want[k]], 1.0, 1.0)
        for t, b in zip(sets[k], before[k]):
            assert ((t.cpu().double() - b * c).abs() <= allowed(b * c, "f32", n)).all()


def test_a_stream_other_than_the_current_one(gpu, lib):
    """The stream argument is what orders the call, whatever torch's current stream is."""
    _, ts = bucket([1_000_001], "bf16", 91)
    side = torch.cuda.Stream()
    s, ws = cell(), work()
    torch.cuda.synchronize()
    assert lib.pgk_grad_sumsq(ptrs(ts), sizes(ts), 1, pgamd.DT_BF16, s.data_ptr(), ws.data_ptr(), side.cuda_stream) == 0
    side.synchronize()
    want = exact_sumsq(ts)
    assert near_sum(s, want, 1_000_001)


# ---- past 32 bits -------------------------------------------------------------------------------------

def test_a_tensor_past_32_bits(gpu, lib):
    """2^32 + 4099 bf16 gradients, zero but for the first, the last and those around 2^31 and 2^32."""
    n = (1 << 32) + 4099
    t = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    at = [0, (1 << 31) - 1, 1 << 31, (1 << 32) - 1, 1 << 32, n - 1]
    for k, i in enumerate(at):
        t[i] = k + 1
    s = sumsq(lib, [t], "bf16")
    assert float(s) == 1 + 4 + 9 + 16 + 25 + 36
    clip(lib, [t], "bf16", [t], "bf16", cell(0.0), 0.5, math.inf)
    assert [float(t[i]) for i in at] == [0.5, 1.0, 1.5, 2.0, 2.5, 3.0]
    assert int(torch.count_nonzero(t)) == 6
    half = t.clone()
    got = fold(lib, half, "bf16", [half, t], "bf16", 1.0)
    assert [float(half[i]) for i in at] == [1.0, 2.0, 3.0, 4.0, 5.0, 6.0]
    assert float(got) == 91.0 and int(torch.count_nonzero(half)) == 6
