"""Calls that follow a failed allocation, the library's own or another's in the same
thread: they run as ever, and the failure is not left behind as the thread's last error."""
import ctypes as C

import numpy as np
import pytest

import hale_moe as H

pytestmark = pytest.mark.gpu

HUGE = 1 << 50  # bytes, more than any device has


@pytest.fixture(scope="module")
def hip():
    return C.CDLL("libamdhip64.so.7")


@pytest.fixture
def norm(ctx):
    """An ordinary call, and its check."""
    x = np.linspace(-1, 1, 64).astype(np.float32)
    bufs = [ctx.malloc(n) for n in (256, 256, 64, 8)]
    for b in bufs[:2]:
        b.upload(x)

    def run():
        bufs[2].upload(np.zeros(64, np.int8))
        H.rms_norm_q8_device(ctx, "f32", 1, 64, bufs[0].address, bufs[1].address, 1e-6, bufs[2].address, bufs[3].address)
        u = (x.astype(np.float64) ** 2).reshape(2, 32)
        want = np.rint(127 * u / u.max(1, keepdims=True)).reshape(-1)
        assert (bufs[2].download(np.int8, 64) == want).all()

    yield run
    for b in bufs:
        b.free()


def q4(ctx, bufs=None):
    d = ctx.malloc(256)
    try:
        H.GroupQ4Matrix.from_device(ctx, 1 << 20, 1 << 29, 128, d.address, d.address)  # its bytes are not read: no memory
    finally:
        d.free()


@pytest.mark.parametrize("call", [q4, lambda ctx: ctx.malloc(HUGE),
                                  lambda ctx: H.KvCache(ctx, 4096, 4096, 4096, 256, 1 << 16, 4, 4096)])
def test_a_call_after_one_that_found_no_memory(ctx, hip, norm, call):
    norm()
    with pytest.raises(MemoryError):
        call(ctx)
    assert hip.hipGetLastError() == 0
    with pytest.raises(MemoryError):
        call(ctx)
    norm()


def test_a_call_after_an_error_of_another_library(ctx, hip, norm):
    p = C.c_void_p()
    assert hip.hipMalloc(C.byref(p), C.c_size_t(HUGE)) != 0
    norm()
    hip.hipGetLastError()
