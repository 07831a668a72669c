"""4-bit products lose no bit of a token's numbers: results on the GPU that are exact but for the last
rounding, against numbers that a part of a token's number left out, or taken twice, would change."""
import numpy as np
import pytest

import hale_moe as H
from kv_model import NP, decode, encode
from test_gpu_step_ops import bufs, q4_model  # noqa: F401
from test_gpu_step_ops_rounding import rounded

pytestmark = pytest.mark.gpu

# kernels of few tokens, of 8 waves and of 4, of rows divided over work-groups; streaming, once and several times over
# the weights; of many tokens
ONE_EACH = [(1, 40, 256, 32, True), (3, 17, 96, 32, False), (5, 100, 8192, 64, True), (3, 40, 14336, 128, True), (16, 63, 2048, 128, False),
            (40, 33, 8224, 32, True), (50, 2000, 1056, 32, True), (5, 6150, 896, 128, True), (37, 4100, 640, 64, False),
            (16, 24580, 2112, 64, True), (16, 16390, 1696, 32, True), (13, 16385, 4224, 128, False),
            (1141, 520, 416, 32, True), (1122, 517, 640, 128, False), (512, 2050, 384, 64, True)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("ntok,rows,cols,group,zeros", ONE_EACH)
def test_q4_keeps_all_bits_of_a_token(ctx, bufs, dtype, ntok, rows, cols, group, zeros):
    """Tokens with one number each that is not 0: every product and sum up to the scale's is exact in f32, so
    a result is (q - zero) x scale rounded to the type, to the bit, wherever the number stands.  f32
    numbers have 19 bits, with 16 + q 24, so that each of three parts of 8 counts; halves 8 (with 4 of
    q - zero and 11 of a scale 23); 8-bit tokens have scales that are powers of two."""
    rng = np.random.default_rng(ntok * rows + cols)
    codes = rng.integers(0, 256, (rows, cols // 2), dtype=np.uint8)
    raw, scales = encode(0.02 * np.exp(0.5 * rng.normal(size=(rows, cols // group))), "f16")
    z = rng.integers(0, 16, (rows, cols // group), dtype=np.uint8) if zeros else None
    m = H.GroupQ4Matrix.new(ctx, rows, cols, group, codes, raw.view(np.uint16), z)
    at, sign = rng.integers(0, cols, ntok), rng.choice([-1.0, 1.0], ntok)
    bits = {"f32": 19, "f16": 8, "bf16": 8, "i8": 7}[dtype]
    x = sign * (rng.integers(1 << (bits - 1), 1 << bits, ntok) | 1)
    if dtype != "i8":
        x = np.ldexp(x, rng.integers(-30 if dtype != "f16" else -12, 10 if dtype != "f16" else 0, ntok))
    wide = np.float64 if dtype == "f32" else np.float32
    full = np.zeros((ntok, cols), wide)
    full[np.arange(ntok), at] = x
    out_type = "f32" if dtype == "i8" else dtype
    out = bufs.put(np.full((ntok, rows), 9, NP[out_type]))
    if dtype == "i8":
        up = np.ldexp(1.0, rng.integers(-8, 8, (ntok, cols // 32))).astype(np.float32)
        m.matmul_q8_device("f32", ntok, bufs.put(full.astype(np.int8)), bufs.put(up), out)
        x = x * up[np.arange(ntok), at // 32]
    else:
        raw_x, back = encode(full, dtype)
        assert (back == full).all()
        m.matmul_device(dtype, ntok, bufs.put(raw_x), out)
    got = decode(bufs.get(out, NP[out_type], ntok * rows), out_type).reshape(ntok, rows).astype(np.float64)
    q = (codes[:, at // 2] >> (4 * (at % 2)).astype(np.uint8) & 15).astype(np.float64)
    q -= 8 if z is None else z[:, at // group]
    exact = lambda v: rounded((q * scales[:, at // group].astype(np.float64)).T * v[:, None], out_type)  # noqa: E731
    assert (got == exact(x)).all(), np.argwhere(got != exact(x))[:5]
    if dtype == "f32":  # without the third part of the numbers hardly one of the results would be this
        two = np.abs(x).astype(np.float32).view(np.uint32)
        top = (two & 0xffff0000).view(np.float32)
        low = ((np.abs(x).astype(np.float32) - top).view(np.uint32) & 0xffff0000).view(np.float32)
        lost = np.sign(x) * (top.astype(np.float64) + low)
        assert ((exact(lost) != exact(x)) | (q.T == 0)).mean() > 0.5
    m.close()


@pytest.mark.parametrize("ntok,rows,cols,group", [(16, 63, 2048, 128), (16, 63, 2048, 32), (16, 1000, 512, 64), (5, 100, 8192, 64), (50, 2000, 1056, 32),
                                                  (5, 6150, 896, 128), (16, 16390, 1696, 32), (13, 16385, 4224, 128), (3, 20000, 1024, 64),
                                                  (1141, 520, 416, 32), (1122, 517, 640, 128), (512, 2050, 384, 64)])
def test_q4_errors_of_f32_tokens_in_the_mean(ctx, bufs, ntok, rows, cols, group):
    """A group's sum of (16 + q) x is some 24 times the root of its squares' sum (16 + q is 24 in the mean of
    squares), and so is (16 + zero) times its sum of x.  Each addition of 32 numbers' first parts rounds at that
    size, group / 32 of them for either sum (those of the second and third parts round 2^-8 below, or in
    64 bits), then the difference and the sum over groups: 2 group / 32 + 2 roundings of at
    most 2^-24 of it each, evenly spread, 2^-24 / sqrt(3) in the mean of squares, and independent."""
    rng = np.random.default_rng(ntok + rows + cols)
    codes = rng.integers(0, 256, (rows, cols // 2), dtype=np.uint8)
    raw, scales = encode(0.02 * np.exp(0.5 * rng.normal(size=(rows, cols // group))) * rng.choice([-1, 1], (rows, cols // group)), "f16")
    z = rng.integers(0, 16, (rows, cols // group), dtype=np.uint8)
    m = H.GroupQ4Matrix.new(ctx, rows, cols, group, codes, raw.view(np.uint16), z)
    x = rng.normal(size=(ntok, cols)).astype(np.float32)
    out = bufs.put(np.zeros((ntok, rows), np.float32))
    m.matmul_device("f32", ntok, bufs.put(x), out)
    got = bufs.get(out, np.float32, ntok * rows).reshape(ntok, rows).astype(np.float64)
    want, _ = q4_model(codes, scales.astype(np.float64), z, group, x)
    size = np.sqrt(np.square(x.astype(np.float64)).reshape(ntok, -1, group).sum(2) @ np.square(24 * scales.astype(np.float64)).T)
    error = np.sqrt(np.square((got - want) / size).mean())
    assert error <= 2.0 ** -24 / np.sqrt(3) * np.sqrt(2 * group / 32 + 2)
    m.close()
