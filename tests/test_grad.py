"""Refusals of the gradient entry points (include/pgk.h, pgk_grad_*): arguments
are checked on the host before anything is launched, so no GPU is needed."""
import ctypes
import math

import pytest

import pgamd

F64, F32, F16, BF16 = pgamd.DT_DOUBLE, pgamd.DT_F32, pgamd.DT_F16, pgamd.DT_BF16
BUF = (ctypes.c_double * 4096)()
BASE = ctypes.addressof(BUF)
SUM, WORK, NORM = BASE, BASE + 1024, BASE + 2048      # places for results; never touched by a refused call


def ptrs(*p):
    return (ctypes.c_void_p * max(len(p), 1))(*p)


def sizes(*n):
    return (ctypes.c_size_t * max(len(n), 1))(*n)


def refused(lib, rc, word):
    assert rc == -1
    msg = (lib.pgk_last_error() or b"").decode()
    assert word in msg, msg


def test_type_codes_extend_the_reference_enum():
    assert (pgamd.DT_INT32, F64, F32, F16, BF16) == (0, 1, 2, 3, 4)


@pytest.mark.parametrize("dt", [0, 5, -1])
def test_other_types_are_refused(lib, dt):
    g, n = ptrs(BASE), sizes(4)
    refused(lib, lib.pgk_grad_sumsq(g, n, 1, dt, SUM, WORK, None), "type")
    refused(lib, lib.pgk_grad_clip(g, dt, g, dt, n, 1, SUM, 1, 1.0, 1.0, None, None), "type")
    refused(lib, lib.pgk_grad_fold(BASE, dt, g, 1, 4, dt, 1.0, None, None, None), "type")


@pytest.mark.parametrize("dt,out", [(F32, BF16), (F32, F64), (F64, F32), (F16, BF16), (BF16, F16), (BF16, F64), (F32, 9)])
def test_type_pairs_that_are_refused(lib, dt, out):
    g, n = ptrs(BASE), sizes(4)
    refused(lib, lib.pgk_grad_clip(g, out, g, dt, n, 1, SUM, 1, 1.0, 1.0, None, None), "output type")
    refused(lib, lib.pgk_grad_fold(BASE, out, g, 1, 4, dt, 1.0, None, None, None), "output type")


def test_gradient_types_stay_out_of_the_reduce_entry_points(lib):
    for dt in (F32, F16, BF16):
        assert lib.pgk_reduce(BASE, BASE, 4, dt, 0, None) == -1
        assert lib.pgk_reduce_multi(BASE, ptrs(BASE), 1, 4, dt, 0, None) == -1


def test_lists(lib):
    g, n = ptrs(BASE), sizes(4)
    refused(lib, lib.pgk_grad_sumsq(g, n, -1, F32, SUM, WORK, None), "list")
    refused(lib, lib.pgk_grad_sumsq(None, n, 1, F32, SUM, WORK, None), "list")
    refused(lib, lib.pgk_grad_sumsq(g, None, 1, F32, SUM, WORK, None), "list")
    refused(lib, lib.pgk_grad_sumsq(ptrs(BASE, None), sizes(4, 1), 2, F32, SUM, WORK, None), "NULL tensor 1")
    refused(lib, lib.pgk_grad_sumsq(g, sizes((1 << 40) + 1), 1, F32, SUM, WORK, None), "elements")
    refused(lib, lib.pgk_grad_sumsq(ptrs(1 << 48), n, 1, F32, SUM, WORK, None), "no device address")
    refused(lib, lib.pgk_grad_clip(None, F32, g, F32, n, 1, SUM, 1, 1.0, 1.0, None, None), "list")
    refused(lib, lib.pgk_grad_clip(ptrs(None), F32, g, F32, n, 1, SUM, 1, 1.0, 1.0, None, None), "NULL tensor 0")
    refused(lib, lib.pgk_grad_fold(BASE, F32, None, 2, 4, F32, 1.0, None, None, None), "NULL list")
    refused(lib, lib.pgk_grad_fold(None, F32, g, 1, 4, F32, 1.0, None, None, None), "NULL")
    refused(lib, lib.pgk_grad_fold(BASE + 512, F32, ptrs(BASE, None), 2, 4, F32, 1.0, None, None, None), "NULL tensor 1")
    for nsrc in (0, 17, -3):
        refused(lib, lib.pgk_grad_fold(BASE, F32, g, nsrc, 4, F32, 1.0, None, None, None), "nsrc")


@pytest.mark.parametrize("dt,es", [(F64, 8), (F32, 4), (F16, 2), (BF16, 2)])
def test_tensors_off_their_elements(lib, dt, es):
    g, n = ptrs(BASE + 256 + es // 2), sizes(4)
    ok = ptrs(BASE)
    refused(lib, lib.pgk_grad_sumsq(g, n, 1, dt, SUM, WORK, None), "multiple of its element")
    refused(lib, lib.pgk_grad_clip(ok, dt, g, dt, n, 1, SUM, 1, 1.0, 1.0, None, None), "multiple of its element")
    refused(lib, lib.pgk_grad_clip(g, dt, ok, dt, n, 1, SUM, 1, 1.0, 1.0, None, None), "multiple of its element")
    refused(lib, lib.pgk_grad_fold(BASE, dt, g, 1, 4, dt, 1.0, None, None, None), "multiple of its element")


def test_places_of_results(lib):
    g, n = ptrs(BASE), sizes(4)
    for bad in (None, BASE + 4):
        refused(lib, lib.pgk_grad_sumsq(g, n, 1, F32, bad, WORK, None), "sumsq")
        refused(lib, lib.pgk_grad_sumsq(g, n, 1, F32, SUM, bad, None), "work")
        refused(lib, lib.pgk_grad_clip(g, F32, g, F32, n, 1, bad, 1, 1.0, 1.0, None, None), "sumsq")
        refused(lib, lib.pgk_grad_fold(BASE, F32, g, 1, 4, F32, 1.0, SUM, bad, None), "work")
    big = (ctypes.c_double * (pgamd.PGK_GRAD_WORK_BYTES // 8))()
    work = ctypes.addressof(big)
    for inside in (work, work + 8, work + pgamd.PGK_GRAD_WORK_BYTES - 8):
        refused(lib, lib.pgk_grad_sumsq(g, n, 1, F32, inside, work, None), "sumsq lies in work")
        refused(lib, lib.pgk_grad_fold(BASE, F32, g, 1, 4, F32, 1.0, inside, work, None), "sumsq lies in work")
    refused(lib, lib.pgk_grad_clip(g, F32, g, F32, n, 1, SUM, 1, 1.0, 1.0, NORM + 4, None), "norm")
    refused(lib, lib.pgk_grad_clip(g, F32, g, F32, n, 1, SUM, 3, 1.0, 1.0, SUM + 16, None), "norm lies in sumsq")
    for nsum in (0, -1):
        refused(lib, lib.pgk_grad_clip(g, F32, g, F32, n, 1, SUM, nsum, 1.0, 1.0, None, None), "partial sums")


def test_scale_and_max_norm(lib):
    g, n = ptrs(BASE), sizes(4)
    for scale in (math.nan, math.inf, -math.inf):
        refused(lib, lib.pgk_grad_clip(g, F32, g, F32, n, 1, SUM, 1, scale, 1.0, None, None), "scale")
        refused(lib, lib.pgk_grad_fold(BASE, F32, g, 1, 4, F32, scale, None, None, None), "scale")
    for max_norm in (math.nan, -1.0, -math.inf):
        refused(lib, lib.pgk_grad_clip(g, F32, g, F32, n, 1, SUM, 1, 1.0, max_norm, None, None), "max_norm")


def test_overlaps(lib):
    n = sizes(64)
    g = ptrs(BASE)
    for off in (4, -4, 252):
        refused(lib, lib.pgk_grad_clip(ptrs(BASE + 1024 + off), F32, ptrs(BASE + 1024), F32, n, 1, SUM, 1, 1.0, 1.0,
                                       None, None), "overlaps")
        refused(lib, lib.pgk_grad_fold(BASE + 1024 + off, F32, ptrs(BASE + 8192, BASE + 1024), 2, 64, F32, 1.0, None,
                                       None, None), "overlaps source 1")
    # widening in place would write over what is still to be read
    refused(lib, lib.pgk_grad_clip(g, F32, g, BF16, n, 1, SUM, 1, 1.0, 1.0, None, None), "overlaps")
    refused(lib, lib.pgk_grad_fold(BASE, F32, g, 1, 64, F16, 1.0, None, None, None), "overlaps source 0")


def test_nothing_to_fold(lib):
    """n = 0 without a sum asked for is a no-op that needs no buffers."""
    assert lib.pgk_grad_fold(None, F32, None, 2, 0, F32, 1.0, None, None, None) == 0


def test_tensor_list():
    """pgamd.tensor_list: what the calls take, from contiguous torch tensors."""
    import torch
    ts = [torch.zeros(5), torch.zeros(0), torch.zeros(2, 3, dtype=torch.bfloat16)]
    p, n, k = pgamd.tensor_list(ts)
    assert k == 3 and list(n) == [5, 0, 6]
    assert p[0] == ts[0].data_ptr() and p[2] == ts[2].data_ptr()
    assert pgamd.tensor_list([])[2] == 0
    with pytest.raises(ValueError, match="tensor 1"):
        pgamd.tensor_list([torch.zeros(4), torch.zeros(4, 4).t()])


def test_group_call_needs_a_handle(lib):
    assert lib.pg_grad_clip(None, F32, None, F32, None, 0, 1.0, 1.0, None, None) == -1
    assert b"NULL handle" in lib.pg_last_error()
