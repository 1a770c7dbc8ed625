"""pg_grad_clip (include/pg_ext.h) refuses to run on another device than the
handle's, and on a transport that has no all-reduce."""
import ctypes

import pytest

import pgamd

pytestmark = pytest.mark.gpu


def connect(lib, rank, world, transport):
    h = ctypes.c_void_p()
    pgamd.check(lib.pg_connect_local(rank, world, transport, ctypes.byref(h)), "pg_connect_local")
    return h


def test_another_device_than_the_current_one(gpu, lib):
    """The workspace is allocated on the current device and the kernels run on the handle's: the two must be one.
    With one GPU the handle is the one that says otherwise."""
    x = gpu.full((100,), 3.0, device="cuda")
    gp, ns, k = pgamd.tensor_list([x], pgamd.DT_F32)
    h = connect(lib, 0, 1, pgamd.PG_TRANSPORT_SELF)
    norm = ctypes.c_double(-1.0)
    call = lambda: lib.pg_grad_clip(gp, pgamd.DT_F32, gp, pgamd.DT_F32, ns, k, 1.0, 1.0, ctypes.byref(norm), h)  # noqa: E731
    try:
        here = pgamd.head(h).device
        pgamd.head(h).device = here + 1
        try:
            assert call() == -1
            assert f"the current device is {here}, the handle's {here + 1}" in pgamd.last_error()
        finally:
            pgamd.head(h).device = here
        assert norm.value == -1.0 and bool((x == 3.0).all())
        assert call() == 0 and norm.value == 30.0
    finally:
        lib.pg_close(h)


def test_a_transport_without_an_all_reduce(gpu, lib):
    x = gpu.full((100,), 3.0, device="cuda")
    gp, ns, k = pgamd.tensor_list([x], pgamd.DT_F32)
    h = connect(lib, 0, 2, pgamd.PG_TRANSPORT_LOOPBACK)
    try:
        assert lib.pg_grad_clip(gp, pgamd.DT_F32, gp, pgamd.DT_F32, ns, k, 1.0, 1.0, None, h) == -1
        assert bool((x == 3.0).all())
    finally:
        lib.pg_close(h)
