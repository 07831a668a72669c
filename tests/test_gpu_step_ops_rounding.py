"""Rows of the norms that hand on 8 bits are rounded once: results on the GPU against numbers that
a second rounding would change."""
import numpy as np
import pytest

from kv_model import encode
from test_gpu_step_ops import bufs, run_norm  # noqa: F401

pytestmark = pytest.mark.gpu


def rounded(x, dtype):
    """64-bit numbers to the nearest of dtype, ties to even, in one step."""
    if dtype == "f32":
        return x.astype(np.float32).astype(np.float64)
    if dtype == "f16":
        return x.astype(np.float16).astype(np.float64)
    m, e = np.frexp(x)
    return np.ldexp(np.rint(np.ldexp(m, 8)), e - 8)


@pytest.mark.parametrize("dtype,rows", [("f32", 40), ("f16", 120), ("bf16", 400)])
def test_norm_rows_are_rounded_once(ctx, bufs, dtype, rows):
    """y is s w r in 64 bits, off by some 2^-50 of itself: the nearest number of the type but for one that
    near to a border, of which 1.6 million random ones have none (each with a chance of 2^-37 at most)."""
    n = 4096
    rng = np.random.default_rng(rows)
    x = encode(rng.normal(size=(rows, n)) * np.exp(rng.normal(size=(rows, 1))), dtype)[1]
    w = np.exp(0.3 * rng.normal(size=n)).astype(np.float32)
    s = x.astype(np.float64)
    r = 1 / np.sqrt((s * s).mean(1, keepdims=True) + np.float64(np.float32(1e-6)))
    want = s * w.astype(np.float64) * r
    if dtype != "f32":  # numbers that a rounding to f32 first would change are among them
        assert (rounded(want.astype(np.float32).astype(np.float64), dtype) != rounded(want, dtype)).sum() >= 5
    _, y, _, _ = run_norm(ctx, bufs, dtype, x, None, w, 1e-6, 128, want_sum=False)
    assert (y.astype(np.float64) == rounded(want, dtype)).all()


def test_norm_rows_at_the_ends_of_the_types(ctx, bufs):
    """Denormals, zeros and infinities come out as the formula's, rounded once."""
    rng = np.random.default_rng(3)
    for dtype, small in (("f16", 2.0 ** -22), ("bf16", 2.0 ** -131)):
        x = encode(rng.normal(size=(4, 256)), dtype)[1]
        w = (rng.normal(size=256) * small).astype(np.float32)
        w[:8], w[8:16] = 0.0, 3e38
        s = x.astype(np.float64)
        r = 1 / np.sqrt((s * s).mean(1, keepdims=True) + np.float64(np.float32(1e-6)))
        want = s * w.astype(np.float64) * r
        _, y, _, _ = run_norm(ctx, bufs, dtype, x, None, w, 1e-6, 32, want_sum=False)
        step = 2.0 ** -24 if dtype == "f16" else 2.0 ** -133  # of denormals
        low = np.abs(want) < (2.0 ** -14 if dtype == "f16" else 2.0 ** -126)
        assert low[:, 16:].any() and (y[low] == np.rint(want[low] / step) * step).all()
        high = ~low & (np.abs(want) < (65519 if dtype == "f16" else 3.38e38))
        assert (y[high] == rounded(want[high], dtype)).all()
        over = np.abs(want) > (65521 if dtype == "f16" else 3.3962e38)
        assert over.any() and (y[over] == np.inf * np.sign(want[over])).all()
