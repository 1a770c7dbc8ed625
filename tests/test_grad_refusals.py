"""Lists and places that the gradient entry points (include/pgk.h, pgk_grad_*) must
not take, because a kernel would read or write where it should not.  Everything is
refused on the host, so no GPU is needed."""
import ctypes
import types

import pytest
import torch

import pgamd

F64, F32, F16, BF16 = pgamd.DT_DOUBLE, pgamd.DT_F32, pgamd.DT_F16, pgamd.DT_BF16


# ---- pgamd.tensor_list -----------------------------------------------------------------------------

def on_gpu(dtype, device="cuda:0", n=4):
    """What tensor_list looks at of a tensor in GPU memory."""
    return types.SimpleNamespace(dtype=dtype, device=device, is_cuda=True, is_contiguous=lambda: True,
                                 data_ptr=lambda: 0x1000, numel=lambda: n)


def test_a_list_with_its_type():
    p, n, k = pgamd.tensor_list([on_gpu(torch.bfloat16), on_gpu(torch.bfloat16, n=0)], BF16)
    assert k == 2 and list(n) == [4, 0] and p[0] == 0x1000
    assert pgamd.tensor_list([], F32)[2] == 0


@pytest.mark.parametrize("dt,dtype", [(F32, torch.bfloat16), (F16, torch.bfloat16), (BF16, torch.float32),
                                      (F64, torch.float32), (F32, torch.int32)])
def test_tensors_of_another_type_than_the_call_gets(dt, dtype):
    """bf16 tensors in a call for f32 would be read to twice their length."""
    right = {F64: torch.float64, F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16}[dt]
    with pytest.raises(ValueError, match=f"tensor 1 is {dtype}"):
        pgamd.tensor_list([on_gpu(right), on_gpu(dtype)], dt)


def test_host_memory_in_a_list_with_its_type():
    with pytest.raises(ValueError, match="tensor 0 is on cpu"):
        pgamd.tensor_list([torch.zeros(4)], F32)


@pytest.mark.parametrize("other", [on_gpu(torch.float32), on_gpu(torch.bfloat16, "cuda:1"),
                                   torch.zeros(4, dtype=torch.bfloat16)])
def test_mixed_lists_on_the_gpu(other):
    """Two types, two devices, or GPU and host memory in one list: no call can take it, whatever type it gets."""
    for ts in ([on_gpu(torch.bfloat16), other], [other, on_gpu(torch.bfloat16)]):
        with pytest.raises(ValueError, match="others are"):
            pgamd.tensor_list(ts)


@pytest.mark.parametrize("dt", [pgamd.DT_INT32, 5, -1])
def test_types_that_no_gradient_has(dt):
    with pytest.raises(ValueError, match="no gradient type"):
        pgamd.tensor_list([], dt)


# ---- places of results and workspace inside the tensors ----------------------------------------------

A, B, C = 0x10_0000_0000, 0x20_0000_0000, 0x30_0000_0000        # addresses far apart; nothing is there to touch
WORK = pgamd.PGK_GRAD_WORK_BYTES
PAIRS = [(F64, F64), (F32, F32), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)]
SIZE = {F64: 8, F32: 4, F16: 2, BF16: 2}


def ptrs(*p):
    return (ctypes.c_void_p * len(p))(*p)


def sizes(*n):
    return (ctypes.c_size_t * len(n))(*n)


def refused(lib, rc, word):
    assert rc == -1
    msg = (lib.pgk_last_error() or b"").decode()
    assert word in msg, msg


@pytest.mark.parametrize("dt", [F64, F32, F16, BF16])
def test_norm_into_its_gradients(lib, dt):
    """The last 8 bytes of a tensor, and a workspace that reaches into it from either side."""
    n = 1000 if dt == F64 else 4000
    end = B + n * SIZE[dt]
    g, ns = ptrs(A, 0, B), sizes(16, 0, n)
    for s in (B, end - 8):
        refused(lib, lib.pgk_grad_sumsq(g, ns, 3, dt, s, C, None), "sumsq lies in tensor 2")
    for w in (B - WORK + 8, end - 8):
        refused(lib, lib.pgk_grad_sumsq(g, ns, 3, dt, C, w, None), "work lies in tensor 2")


@pytest.mark.parametrize("dt,out_dt", PAIRS)
def test_clip_into_its_own_sums(lib, dt, out_dt):
    n = 4000
    g, o, ns = ptrs(A, B), ptrs(A + (1 << 20), C), sizes(16, n)
    end = C + n * SIZE[out_dt]
    for s, nsum in ((C, 1), (end - 8, 1), (C - 24, 4), (end - 8, 9)):
        refused(lib, lib.pgk_grad_clip(o, out_dt, g, dt, ns, 2, s, nsum, 1.0, 1.0, None, None), "sumsq lies in tensor 1")
    s = A + (1 << 21)
    for norm in (C, end - 8, B, B + n * SIZE[dt] - 8):
        refused(lib, lib.pgk_grad_clip(o, out_dt, g, dt, ns, 2, s, 1, 1.0, 1.0, norm, None), "norm lies in tensor 1")
    if dt == out_dt:                                              # in place
        refused(lib, lib.pgk_grad_clip(g, dt, g, dt, ns, 2, B + 8, 1, 1.0, 1.0, None, None), "sumsq lies in tensor 1")


@pytest.mark.parametrize("dt,out_dt", PAIRS)
def test_fold_into_its_own_sum(lib, dt, out_dt):
    n = 4000
    src, s0 = ptrs(A, B), C + (1 << 20)
    for s in (C, C + n * SIZE[out_dt] - 8):
        refused(lib, lib.pgk_grad_fold(C, out_dt, src, 2, n, dt, 1.0, s, s0, None), "sumsq lies in tensor 0")
    refused(lib, lib.pgk_grad_fold(C, out_dt, src, 2, n, dt, 1.0, B + n * SIZE[dt] - 8, s0, None), "sumsq lies in tensor 1")
    refused(lib, lib.pgk_grad_fold(C, out_dt, src, 2, n, dt, 1.0, s0, C + n * SIZE[out_dt] - 8, None), "work lies in tensor 0")
    refused(lib, lib.pgk_grad_fold(C, out_dt, src, 2, n, dt, 1.0, s0, B - WORK + 8, None), "work lies in tensor 1")
