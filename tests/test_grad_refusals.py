"""Lists and places that the gradient entry points (include/pgk.h, pgk_grad_*) must
not take, because a kernel would read or write where it should not.  Everything is
refused on the host, so no GPU is needed."""
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
