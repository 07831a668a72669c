"""Norms that hand on 8 bits, products of 4-bit weights with group scales, and
rules on logits, on the GPU, against their formulas in 64 bits and more."""
import ctypes as C
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest

import hale_moe as H
from kv_model import EPS, NP, decode, encode

pytestmark = pytest.mark.gpu

SIZE = {"f32": 4, "f16": 2, "bf16": 2}


class Bufs:
    """Device buffers of a test, freed at its end."""

    def __init__(self, ctx):
        self.ctx, self.all = ctx, []

    def put(self, arr, offset=0):
        """A buffer that holds arr from byte `offset` on; its address there."""
        b = self.ctx.malloc(max(offset + arr.nbytes, 4))
        self.all.append(b)
        if arr.nbytes:
            b.upload(arr, offset)
        return b.address + offset

    def set(self, address, arr):
        next(b for b in self.all if b.address == address).upload(arr)

    def get(self, address, dtype, count):
        b = next(b for b in self.all if b.address <= address < b.address + max(b.nbytes, 1))
        return b.download(dtype, count, address - b.address)


@pytest.fixture
def bufs(ctx):
    b = Bufs(ctx)
    yield b
    ctx.synchronize()
    for x in b.all:
        x.free()


def strided(x, stride, fill):
    out = np.full((x.shape[0], stride), fill, x.dtype)
    out[:, :x.shape[1]] = x
    return out


# ---- norms -------------------------------------------------------------------

def norm_model(x, delta, w, eps, block, dtype):
    """s, y in 64 bits, codes, scales in 64 bits.  Products with the weights have
    48 bits and 127 times them 55, which an 80-bit float holds; its quotient is a
    whole number and a half only where that is exact, else off by 2^-57 at most, which
    decides nothing unless the quotient is that near to a border."""
    s = x if delta is None else decode(encode(x + delta, dtype)[0], dtype)
    wide = s.astype(np.longdouble)
    u = (wide * w.astype(np.longdouble)).reshape(len(x), -1, block)
    r = 1 / np.sqrt((s.astype(np.float64) ** 2).mean(1) + np.float32(eps).astype(np.float64))
    top = np.abs(u).max(2, keepdims=True)
    codes = np.rint(np.where(top > 0, 127 * u / np.where(top > 0, top, 1), 0)).astype(np.int8)
    scale = top[:, :, 0].astype(np.float64) * r[:, None] / 127
    return s, u.reshape(x.shape).astype(np.float64) * r[:, None], codes.reshape(x.shape), scale


def run_norm(ctx, bufs, dtype, x, delta, w, eps, block, *, pad=0, offset=0, want_sum=True, want_y=True, in_place=False):
    rows, n = x.shape
    size, stride = SIZE[dtype], n + pad
    put = lambda v: bufs.put(strided(encode(v, dtype)[0], stride, 7), offset * size)  # noqa: E731
    dx, dd = put(x), put(delta) if delta is not None else 0
    fresh = lambda: bufs.put(np.full((rows, stride), 5, NP[dtype]), offset * size)  # noqa: E731
    ds = (dx if in_place else fresh()) if want_sum else 0
    dy = fresh() if want_y else 0
    dw = bufs.put(w.astype(np.float32), 4 * (offset % 4))
    dq, dsc = bufs.put(np.full(rows * n, 99, np.int8), offset), bufs.put(np.full(rows * (n // block), 99, np.float32))
    H.rms_norm_q8_device(ctx, dtype, rows, n, dx, dw, eps, dq, dsc, block=block, d_delta=dd, d_sum=ds, d_y=dy,
                         x_stride=stride, delta_stride=stride, sum_stride=stride, y_stride=stride)
    out = []
    for d, keep in ((ds, 7 if in_place else 5), (dy, 5)):
        if not d:
            out.append(None)
            continue
        raw = bufs.get(d, NP[dtype], rows * stride).reshape(rows, stride)
        assert (raw[:, n:] == np.array(keep).astype(NP[dtype])).all()
        out.append(decode(np.ascontiguousarray(raw[:, :n]), dtype))
    return out[0], out[1], bufs.get(dq, np.int8, rows * n).reshape(rows, n), bufs.get(dsc, np.float32, rows * (n // block)).reshape(rows, -1)


def check_norm(got, x, delta, w, eps, block, dtype):
    s, y, codes, scales = norm_model(x, delta, w, eps, block, dtype)
    gs, gy, gq, gscale = got
    if gs is not None:
        assert (gs == s).all()
    assert (gq == codes).all(), np.argwhere(gq != codes)[:5]
    # the squares' sum, its root and the products in 64 bits: far below half a step of f32
    assert (np.abs(gscale - scales) <= scales * (2.0 ** -24 + 2.0 ** -40) + 2.0 ** -150).all()
    if gy is not None:
        # y in 64 bits, rounded to f32 (2^-24), then to the type
        tol = np.abs(y) * (EPS[dtype] + 2.0 ** -24 + 2.0 ** -40) + (2.0 ** -25 if dtype == "f16" else 2.0 ** -149 if dtype == "f32" else 2.0 ** -134)
        assert (np.abs(gy - y) <= tol).all()


NORMS = [
    # dtype, rows, n, block, delta, pad, offset, in place
    ("f32", 1, 32, 32, False, 0, 0, False),
    ("f32", 1, 2048, 32, True, 0, 0, False),
    ("bf16", 3, 2048, 128, True, 0, 0, True),
    ("f16", 57, 4096, 4096, False, 0, 0, False),
    ("bf16", 5, 96, 96, True, 0, 0, False),
    ("f16", 7, 544, 32, True, 8, 0, True),
    ("bf16", 2, 544, 544, True, 3, 1, False),
    ("f32", 9, 160, 32, True, 1, 3, True),
    ("f32", 2, 4160, 64, True, 0, 0, False),
    ("bf16", 2, 8192, 128, False, 0, 0, False),
    ("f16", 2, 16384, 64, True, 0, 0, False),
    ("bf16", 2, 16352, 32, True, 0, 0, False),
    ("f32", 1, 16384, 16384, True, 0, 0, False),
    ("f32", 70000, 32, 32, True, 0, 0, False),
]


@pytest.mark.parametrize("dtype,rows,n,block,delta,pad,offset,in_place", NORMS)
def test_norm_codes_scales_and_rows(ctx, bufs, dtype, rows, n, block, delta, pad, offset, in_place):
    rng = np.random.default_rng(n + rows)
    ch = np.exp(0.7 * rng.normal(size=n))
    x = encode(rng.normal(size=(rows, n)) * ch, dtype)[1]
    d = encode(0.3 * rng.normal(size=(rows, n)), dtype)[1] if delta else None
    w = np.exp(0.3 * rng.normal(size=n)).astype(np.float32)
    w[::7] *= -1
    got = run_norm(ctx, bufs, dtype, x, d, w, 1e-6, block, pad=pad, offset=offset, in_place=in_place)
    check_norm(got, x, d, w, 1e-6, block, dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_norm_codes_at_borders(ctx, bufs, dtype):
    """Whole numbers around 127 m: a block's quotients are whole numbers and halves."""
    rng = np.random.default_rng(3)
    x = np.zeros((8, 256), np.float32)
    for r in range(8):
        m = [1, 2, 2, 0.25, 0.5, 2, 1, 2][r]
        x[r] = (rng.integers(-127, 128, 256) * m).astype(np.float32)
        x[r, ::32] = 127 * m
        x[r, 1::2] = (rng.integers(-126, 126, 128) + 0.5) * m if m != 0.25 else x[r, 1::2]
    x = encode(x, dtype)[1]
    for block in (32, 64, 128, 256):
        w = np.ones(256, np.float32)
        check_norm(run_norm(ctx, bufs, dtype, x, None, w, 1e-5, block), x, None, w, 1e-5, block, dtype)
        w = np.repeat(np.array([3, 1.5, 7, 0.1], np.float32), 64)  # 127 m times 3 and 7: no exact reciprocal
        check_norm(run_norm(ctx, bufs, dtype, x, None, w, 1e-5, 64), x, None, w, 1e-5, 64, dtype)


def test_norm_extreme_rows(ctx, bufs):
    rng = np.random.default_rng(5)
    x = rng.normal(size=(6, 128)).astype(np.float32)
    x[0] *= 1e37  # squares beyond f32
    x[1] *= 1e-37
    x[2] = 0
    x[3, :64] = 0  # a block of zeros
    x[4, 5] = 3e38
    w = np.ones(128, np.float32)
    got = run_norm(ctx, bufs, "f32", x, None, w, 1e-6, 64)
    check_norm(got, x, None, w, 1e-6, 64, "f32")
    assert (got[3][2] == 0).all() and got[3][3, 0] == 0 and (got[2][3, :64] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_norm_rows_that_are_not_finite(ctx, bufs, dtype):
    rng = np.random.default_rng(6)
    x = encode(rng.normal(size=(5, 256)), dtype)[1]
    x[1, 3], x[2, 200], x[3, 100] = np.nan, np.inf, -np.inf
    w = np.ones(256, np.float32)
    fine = [0, 4]
    for block in (32, 256):
        s, y, q, scale = run_norm(ctx, bufs, dtype, x, None, w, 1e-6, block)
        for r in (1, 2, 3):
            assert np.isnan(scale[r]).all() and (q[r] == 0).all() and np.isnan(y[r]).all()
        check_norm((s[fine], y[fine], q[fine], scale[fine]), x[fine], None, w, 1e-6, block, dtype)
    w[40] = np.inf  # its block only
    _, _, q, scale = run_norm(ctx, bufs, dtype, x, None, w, 1e-6, 32)
    assert np.isnan(scale[0, 1]) and (q[0, 32:64] == 0).all() and np.isfinite(np.delete(scale[0], 1)).all()
    z = np.zeros((1, 64), np.float32)
    _, _, q, scale = run_norm(ctx, bufs, dtype, z, None, w[:64], 0.0, 64)
    assert np.isnan(scale).all() and (q == 0).all()


def test_norm_refusals(ctx, bufs):
    x = bufs.put(np.zeros(4096, np.float32))
    L = H.lib()

    def call(dtype=H.F32, rows=2, n=64, dx=x, xs=64, dd=0, ds=64, w=x, eps=1e-6, block=32, su=0, sus=64, y=0, ys=64, q=x, sc=x):
        return L.hale_rms_norm_q8_device(ctx.handle, dtype, rows, n, dx, xs, dd, ds, w, eps, block, su, sus, y, ys, q, sc)

    for bad in (dict(dtype=H.Q8_0), dict(n=0), dict(n=48), dict(n=16416, xs=16416), dict(block=16), dict(block=128), dict(block=0),
                dict(xs=63), dict(dd=x, ds=63), dict(su=x + 4096, sus=3), dict(y=x + 4096, ys=3), dict(dx=0), dict(w=0), dict(q=0),
                dict(sc=0), dict(dx=x + 2), dict(w=x + 1), dict(sc=x + 2), dict(eps=-1.0), dict(eps=float("nan")),
                dict(su=x, sus=65), dict(su=x + 4096, y=x + 4096), dict(rows=1 << 31)):
        assert call(**bad) == H.EINVAL, bad
    assert call(rows=0, dx=0) == H.OK


# ---- products of 4-bit weights ---------------------------------------------------

def q4_weights(rng, rows, cols, group, zeros, scale_dtype):
    codes = rng.integers(0, 256, (rows, cols // 2), dtype=np.uint8)
    raw, scales = encode(np.exp(0.5 * rng.normal(size=(rows, cols // group))) * 0.02 * rng.choice([-1, 1], (rows, cols // group)), scale_dtype)
    z = rng.integers(0, 16, (rows, cols // group), dtype=np.uint8) if zeros else None
    return codes, raw.view(np.uint16), scales.astype(np.float64), z


def q4_model(codes, scales, z, group, x):
    """The product, and sum scale (16 + q + 16 + zero) |x|, in 64 bits."""
    q = np.stack((codes & 15, codes >> 4), -1).reshape(len(codes), -1).astype(np.float64)
    zz = np.full(scales.shape, 8.0) if z is None else z.astype(np.float64)
    s, zz = np.repeat(scales, group, 1), np.repeat(zz, group, 1)
    x = x.astype(np.float64)
    return x @ (s * (q - zz)).T, np.abs(x) @ (np.abs(s) * (q + zz + 32)).T


def q4_bound(dtype, want, mag, cols, group):
    """Products are exact (16 + q, 5 bits, times at most 11, or three parts of 8).  A group's sums
    are at most 3 * 128 products, each addition off by 2^-23 of the partial sums at most (however the
    matrix unit rounds), 16 + zero times the second sum and the difference by 2^-24 each: against
    `mag`, (3 * 128 + 2) 2^-23.  Between groups a product and a sum each, and the joins of up to 16
    parts: (cols / group + 18) 2^-24.  Then the result's own rounding."""
    rel = (3 * 128 + 2) * 2.0 ** -23 + (cols / group + 18) * 2.0 ** -24
    return mag * rel * 1.01 + EPS[dtype] * np.abs(want) + (2.0 ** -25 if dtype == "f16" else 2.0 ** -126)


Q4 = [
    # dtype, scales, tokens, rows, cols, group, zeros, pad of x, offset of x, pad of out
    ("bf16", "f16", 1, 16, 128, 128, False, 0, 0, 0),
    ("bf16", "f16", 1, 1, 32, 32, True, 0, 0, 0),
    ("f32", "bf16", 1, 17, 96, 32, True, 0, 0, 0),
    ("f16", "f16", 2, 33, 64, 64, True, 0, 0, 0),
    ("f16", "bf16", 5, 40, 192, 64, False, 8, 0, 3),
    ("bf16", "bf16", 7, 100, 1024, 64, True, 3, 1, 0),
    ("f32", "f16", 4, 100, 544, 32, False, 5, 1, 1),
    ("f32", "f16", 16, 63, 2048, 128, True, 0, 0, 0),
    ("f16", "f16", 17, 63, 640, 128, True, 0, 0, 5),
    ("bf16", "f16", 31, 129, 1152, 128, False, 0, 0, 0),
    ("bf16", "f16", 33, 257, 352, 32, True, 0, 0, 0),
    ("f32", "f16", 64, 130, 1088, 64, True, 0, 0, 0),
    ("f16", "f16", 65, 260, 896, 128, False, 0, 0, 0),
    ("bf16", "f16", 130, 300, 1024, 32, False, 0, 0, 0),
    ("f16", "f16", 200, 513, 384, 64, True, 2, 0, 1),
    ("f32", "bf16", 129, 70, 14336, 128, True, 0, 0, 0),
    ("bf16", "f16", 1, 5000, 4096, 128, True, 0, 0, 0),
    ("f16", "f16", 3, 5000, 256, 32, True, 0, 0, 0),
    ("f16", "f16", 1, 20000, 512, 64, False, 0, 0, 0),
]


Q4 += [  # many rows: tokens that fill LDS, and f32 ones that do so twice and three times over
    ("bf16", "f16", 16, 24580, 2112, 64, True, 0, 0, 0), ("f32", "bf16", 16, 16390, 1696, 32, True, 1, 1, 2),
    ("f32", "f16", 13, 16385, 4224, 128, False, 0, 0, 3), ("f16", "f16", 2, 24577, 160, 32, True, 0, 0, 0),
    ("bf16", "f16", 27, 32780, 320, 32, True, 0, 0, 1), ("f32", "f16", 40, 24590, 256, 64, True, 0, 0, 0),
    # many tokens
    ("f16", "f16", 1130, 520, 384, 64, True, 2, 0, 1), ("bf16", "bf16", 965, 1040, 352, 32, False, 0, 0, 0),
    ("f32", "f16", 1141, 520, 416, 32, True, 1, 1, 0), ("bf16", "f16", 1121, 517, 896, 128, True, 1, 1, 1),
    ("f32", "bf16", 1122, 517, 640, 128, False, 0, 0, 0), ("bf16", "bf16", 1901, 2170, 384, 128, True, 0, 0, 0),
    ("bf16", "f16", 40001, 9, 64, 32, True, 0, 0, 0), ("f32", "f16", 1 << 20, 3, 32, 32, False, 0, 0, 0),
    # work-groups of four waves
    ("bf16", "f16", 1, 10250, 1120, 32, True, 0, 0, 0), ("f16", "bf16", 37, 4100, 640, 64, False, 1, 1, 1), ("f32", "f16", 50, 2000, 1056, 32, True, 0, 0, 0),
    ("f32", "f16", 5, 6150, 896, 128, True, 0, 0, 0),
    # few rows of many numbers
    ("bf16", "f16", 3, 40, 14336, 64, True, 0, 0, 0), ("f32", "f16", 5, 100, 8192, 32, True, 0, 0, 1),
    ("f16", "bf16", 40, 33, 8224, 32, False, 0, 0, 0),
]


@pytest.mark.parametrize("dtype,scale_dtype,ntok,rows,cols,group,zeros,xpad,xoff,opad", Q4)
def test_q4_products(ctx, bufs, dtype, scale_dtype, ntok, rows, cols, group, zeros, xpad, xoff, opad):
    rng = np.random.default_rng(rows + cols + ntok)
    codes, raw, scales, z = q4_weights(rng, rows, cols, group, zeros, scale_dtype)
    m = H.GroupQ4Matrix.new(ctx, rows, cols, group, codes, raw, z, scale_dtype)
    back = m.download()
    assert (back[0] == codes).all() and (back[1] == raw).all() and (back[2] == (8 if z is None else z)).all()
    xr, x = encode(rng.normal(size=(ntok, cols)) * np.exp(rng.normal(size=cols)) + 0.5, dtype)
    dx = bufs.put(strided(xr, cols + xpad, 3), xoff * SIZE[dtype])
    out = bufs.put(np.full((ntok, rows + opad), 9, NP[dtype]))
    m.matmul_device(dtype, ntok, dx, out, x_stride=cols + xpad, out_stride=rows + opad)
    got = bufs.get(out, NP[dtype], ntok * (rows + opad)).reshape(ntok, -1)
    assert (got[:, rows:] == np.array(9).astype(NP[dtype])).all()
    got = decode(np.ascontiguousarray(got[:, :rows]), dtype).astype(np.float64)
    want, mag = q4_model(codes, scales, z, group, x)
    assert (np.abs(got - want) <= q4_bound(dtype, want, mag, cols, group)).all()
    m.close()


@pytest.mark.parametrize("dtype,ntok,rows,cols", [("bf16", 2, 40, 14336), ("f32", 16, 100, 4096), ("f16", 40, 33, 8192), ("f32", 16, 16400, 1792)])
def test_q4_calls_in_turn(ctx, bufs, dtype, ntok, rows, cols):
    """Divided rows count their parts in memory of the matrix: eager calls and replays one behind the
    other, of other tokens each time, give the bits of calls apart."""
    rng = np.random.default_rng(cols)
    codes, raw, _, z = q4_weights(rng, rows, cols, 128, True, "f16")
    m = H.GroupQ4Matrix.new(ctx, rows, cols, 128, codes, raw, z)
    xs = [encode(rng.normal(size=(ntok, cols)), dtype)[0] for _ in range(3)]
    dxs, dx = [bufs.put(x) for x in xs], bufs.put(xs[0])
    outs = [bufs.put(np.zeros((ntok, rows), NP[dtype])) for _ in range(4)]
    want = []
    for d, o in zip(dxs, outs):
        m.matmul_device(dtype, ntok, d, o)
        want.append(bufs.get(o, NP[dtype], ntok * rows))
    for _ in range(5):
        for d, o in zip(dxs, outs):
            m.matmul_device(dtype, ntok, d, o)
    assert all((bufs.get(o, NP[dtype], ntok * rows) == w).all() for o, w in zip(outs, want))

    def calls():
        for o in outs:
            m.matmul_device(dtype, ntok, dx, o)

    graph = ctx.capture(calls)
    for x, w in list(zip(xs, want)) * 2:
        bufs.set(dx, x)
        graph.launch()
        assert all((bufs.get(o, NP[dtype], ntok * rows) == w).all() for o in outs)
        m.matmul_device(dtype, ntok, dxs[1], outs[0])
    graph.close()
    m.close()


def test_q4_weights_from_device_memory(ctx, bufs):
    rng = np.random.default_rng(8)
    codes, raw, scales, z = q4_weights(rng, 37, 320, 64, True, "f16")
    m = H.GroupQ4Matrix.from_device(ctx, 37, 320, 64, bufs.put(codes), bufs.put(raw), bufs.put(z | 0xA0))
    back = m.download()
    assert (back[0] == codes).all() and (back[1] == raw).all() and (back[2] == z).all()
    m.close()


@pytest.mark.parametrize("ntok,rows,cols,group,block,zeros,dtype", [
    (1, 16, 128, 128, 32, True, "f32"), (1, 40, 96, 32, 32, False, "f32"), (3, 17, 192, 64, 192, True, "bf16"),
    (5, 100, 544, 32, 544, True, "f16"), (16, 100, 1024, 128, 128, False, "bf16"), (17, 65, 1152, 64, 128, True, "f32"),
    (40, 130, 640, 128, 64, True, "f32"), (100, 257, 512, 64, 32, True, "f16"), (1, 5000, 2048, 128, 32, True, "f32"),
    (130, 300, 896, 128, 896, False, "f32"), (64, 128, 256, 32, 128, True, "bf16"),
    (16, 24600, 1056, 32, 32, True, "f16"), (7, 24577, 640, 128, 640, False, "f32"), (23, 32770, 192, 64, 32, True, "bf16"),
    (965, 1040, 352, 32, 32, True, "f16"), (1130, 520, 640, 128, 64, False, "f32"), (1121, 517, 896, 128, 896, True, "bf16"),
    (1901, 2170, 384, 64, 128, True, "f32"),
    (20, 5200, 416, 32, 32, True, "bf16"), (9, 50, 8192, 128, 64, True, "f32"), (60, 20, 9216, 64, 128, True, "f16"),
])
def test_q4_products_of_8_bit_tokens(ctx, bufs, ntok, rows, cols, group, block, zeros, dtype):
    """Whole numbers up to 128 * 127 * 31 < 2^24 within a unit of 32 to 128 numbers; per unit the
    product of the scales, and a fused product and sum, round by 2^-24 of partial sums of the units'
    magnitudes; then the joins (up to 16 parts) and the result's own rounding."""
    rng = np.random.default_rng(rows + cols + ntok)
    codes, raw, scales, z = q4_weights(rng, rows, cols, group, zeros, "f16")
    m = H.GroupQ4Matrix.new(ctx, rows, cols, group, codes, raw, z)
    q = rng.integers(-127, 128, (ntok, cols), dtype=np.int8)
    xs = np.exp(rng.normal(size=(ntok, cols // block))).astype(np.float32)
    out = bufs.put(np.zeros((ntok, rows), NP[dtype]))
    m.matmul_q8_device(dtype, ntok, bufs.put(q), bufs.put(xs), out, block=block)
    got = decode(bufs.get(out, NP[dtype], ntok * rows), dtype).reshape(ntok, rows).astype(np.float64)
    unit = min(group, block)
    x = q.astype(np.float64) * np.repeat(xs.astype(np.float64), block, 1)
    want, _ = q4_model(codes, scales, z, group, x)
    w = np.stack((codes & 15, codes >> 4), -1).reshape(rows, -1).astype(np.float64)
    w -= 8 if z is None else np.repeat(z.astype(np.float64), group, 1)
    w *= np.repeat(scales, group, 1)
    mag = sum(np.abs(x[:, k:k + unit] @ w[:, k:k + unit].T) for k in range(0, cols, unit))
    tol = mag * (cols / unit + 20) * 2.0 ** -24 * 1.01 + EPS[dtype] * np.abs(want) + (2.0 ** -25 if dtype == "f16" else 0.0)
    assert (np.abs(got - want) <= tol).all()
    m.close()


@pytest.mark.parametrize("dtype,ntok,rows", [("f32", 3, 50), ("bf16", 5, 50), ("f16", 20, 50), ("bf16", 80, 50), ("f32", 70, 50),
                                             ("f16", 9300, 50), ("f32", 9300, 50), ("bf16", 4, 24600), ("f32", 12, 16400)])
def test_q4_tokens_that_are_not_finite_stay_apart(ctx, bufs, dtype, ntok, rows):
    rng = np.random.default_rng(9)
    cols = 256
    codes, raw, _, z = q4_weights(rng, rows, cols, 64, True, "f16")
    m = H.GroupQ4Matrix.new(ctx, rows, cols, 64, codes, raw, z)
    x = rng.normal(size=(ntok, cols)).astype(np.float32)
    outs = []
    for spoil in (False, True):
        if spoil:
            x[1, 7], x[ntok - 1, 255] = np.inf, np.nan
        dx, out = bufs.put(encode(x, dtype)[0]), bufs.put(np.zeros((ntok, rows), NP[dtype]))
        m.matmul_device(dtype, ntok, dx, out)
        outs.append(bufs.get(out, NP[dtype], ntok * rows).reshape(ntok, rows))
    bad = [1, ntok - 1]
    assert not np.isfinite(decode(np.ascontiguousarray(outs[1][bad]), dtype)).any()
    assert (np.delete(outs[0], bad, 0) == np.delete(outs[1], bad, 0)).all()
    m.close()


def test_q4_small_and_large_numbers(ctx, bufs):
    """Numbers from the ends of the types' ranges, whose products stay within f32."""
    rng = np.random.default_rng(10)
    codes, raw, scales, z = q4_weights(rng, 40, 256, 128, True, "bf16")
    m = H.GroupQ4Matrix.new(ctx, 40, 256, 128, codes, raw, z, "bf16")
    for dtype, size in (("f32", 1e33), ("f32", 1e-25), ("bf16", 1e33), ("bf16", 1e-30), ("f16", 200.0), ("f16", 1e-6)):
        xr, x = encode(rng.normal(size=(2, 256)) * size, dtype)
        out = bufs.put(np.zeros((2, 40), NP[dtype]))
        m.matmul_device(dtype, 2, bufs.put(xr), out)
        got = decode(bufs.get(out, NP[dtype], 80), dtype).reshape(2, 40).astype(np.float64)
        want, mag = q4_model(codes, scales, z, 128, x)
        if dtype == "f16":
            want = np.where(np.abs(want) > 65519.9, np.inf * np.sign(want), want)
        ok = np.isfinite(want)
        assert (np.abs(got - want)[ok] <= q4_bound(dtype, want, mag, 256, 128)[ok]).all()
    m.close()


def test_q4_refusals(ctx, bufs):
    d = bufs.put(np.zeros(8192, np.float32))
    L, h = H.lib(), C.c_void_p()
    up = lambda rows=16, cols=128, group=64, st=H.F16, c=d, s=d, z=0: L.hale_q4g_upload_device(ctx.handle, rows, cols, group, st, c, s, z, C.byref(h))  # noqa: E731
    for bad in (dict(rows=0), dict(cols=0), dict(cols=96), dict(group=16), dict(group=256, cols=256), dict(st=H.F32), dict(c=0),
                dict(s=0), dict(s=d + 1), dict(rows=(1 << 30) + 1)):
        assert up(**bad) == H.EINVAL, bad
        assert not h.value
    z = np.full((16, 2), 16, np.uint8)
    with pytest.raises(ValueError):
        H.GroupQ4Matrix.new(ctx, 16, 128, 64, np.zeros((16, 64), np.uint8), np.zeros((16, 2), np.uint16), z)
    with pytest.raises(ValueError):
        H.GroupQ4Matrix.new(ctx, 16, 128, 64, np.zeros((16, 63), np.uint8), np.zeros((16, 2), np.uint16))
    m = H.GroupQ4Matrix.new(ctx, 16, 128, 64, np.zeros((16, 64), np.uint8), np.zeros((16, 2), np.uint16))
    f = lambda dtype=H.F32, n=2, x=d, xs=128, o=d + 4096, os=16: L.hale_q4g_matmul_device(m.handle, dtype, n, x, xs, o, os)  # noqa: E731
    for bad in (dict(dtype=H.Q4_0), dict(x=0), dict(o=0), dict(xs=127), dict(os=15), dict(x=d + 2), dict(o=d + 2), dict(n=(1 << 20) + 1)):
        assert f(**bad) == H.EINVAL, bad
    assert f(n=0, x=0) == H.OK
    q = lambda n=2, block=32, x=d, s=d, dtype=H.F32, o=d + 4096, os=16: L.hale_q4g_matmul_q8_device(m.handle, n, block, x, s, dtype, o, os)  # noqa: E731
    for bad in (dict(block=0), dict(block=16), dict(block=256), dict(x=0), dict(s=0), dict(x=d + 4), dict(s=d + 2), dict(dtype=7), dict(os=15)):
        assert q(**bad) == H.EINVAL, bad
    m.close()


# ---- rules on logits --------------------------------------------------------------

def logits_model(raw, dtype, rules):
    """f32 arithmetic in the documented order; the types' bits."""
    x = decode(raw.reshape(-1), dtype).reshape(raw.shape).astype(np.float32)
    out = raw.copy()
    rows, vocab = raw.shape
    f32 = np.float32
    for r in range(rows):
        named = {}
        hist = rules["tokens"][r]
        for k, tok in enumerate(hist):
            if 0 <= tok < vocab:
                named.setdefault(int(tok), 0)
                named[int(tok)] += k >= rules["prompt"][r]
        bias = {int(t): f32(b) for t, b in rules["bias"][r] if 0 <= t < vocab}
        with np.errstate(all="ignore"):
            for tok in set(named) | set(bias):
                v = x[r, tok]
                if tok in named:
                    rep = f32(rules["repetition"][r])
                    v = v / rep if v > 0 else v * rep
                    if named[tok]:
                        v = (v - f32(rules["frequency"][r]) * f32(named[tok])) - f32(rules["presence"][r])
                if tok in bias:
                    v = v + bias[tok]
                out[r, tok] = encode(np.array([v], np.float32), dtype)[0][0]
        m = rules["mask"][r]
        if m is not None:
            out[r, ~m] = encode(np.array([-np.inf], np.float32), dtype)[0][0]
    return out


def same_bits(a, b, dtype):
    """Equal bits, but for a NaN that was computed with."""
    na, nb = (np.isnan(decode(v.reshape(-1), dtype)).reshape(v.shape) for v in (a, b))
    u = np.uint32 if dtype == "f32" else np.uint16
    return ((a.view(u) == b.view(u)) | (na & nb)).all()


def run_logits(ctx, bufs, dtype, raw, rules, *, pad=0, offset=0, in_place=False, masks=None, mask_row=None):
    rows, vocab = raw.shape
    size = SIZE[dtype]
    start = lambda lists: np.concatenate([[0], np.cumsum([len(v) for v in lists])]).astype(np.int64)  # noqa: E731
    R = H.LogitsRules()
    toks = np.concatenate([np.asarray(v, np.int32) for v in rules["tokens"]] + [np.zeros(0, np.int32)])
    R.tokens, R.token_start, R.ntokens = bufs.put(toks.astype(np.int32)), bufs.put(start(rules["tokens"])), len(toks)
    R.prompt_len = bufs.put(np.asarray(rules["prompt"], np.int64))
    for k in ("repetition", "frequency", "presence"):
        setattr(R, k, bufs.put(np.asarray(rules[k], np.float32)))
    flat = [p for v in rules["bias"] for p in v]
    if flat:
        R.bias_tokens, R.bias = bufs.put(np.array([p[0] for p in flat], np.int32)), bufs.put(np.array([p[1] for p in flat], np.float32))
        R.bias_start, R.nbiases = bufs.put(start(rules["bias"])), len(flat)
    if masks is not None:
        words = (vocab + 31) // 32
        bits = np.zeros((len(masks), (words + 1) * 32), bool)
        bits[:, :vocab] = masks
        R.mask = bufs.put(np.packbits(bits, axis=1, bitorder="little").view(np.uint32))
        R.mask_rows, R.mask_stride = len(masks), words + 1
        if mask_row is not None:
            R.mask_row = bufs.put(np.asarray(mask_row, np.int32))
    stride = vocab + pad
    din = bufs.put(strided(raw, stride, 7), offset * size)
    dout = din if in_place else bufs.put(np.full((rows, stride), 5, NP[dtype]), offset * size)
    H.logits_device(ctx, dtype, rows, vocab, din, R, dout, stride=stride, out_stride=stride)
    got = bufs.get(dout, NP[dtype], rows * stride).reshape(rows, stride)
    assert (got[:, vocab:] == np.array(7 if in_place else 5).astype(NP[dtype])).all()
    return np.ascontiguousarray(got[:, :vocab])


def some_rules(rng, rows, vocab, longest, biases):
    lens = rng.integers(0, longest + 1, rows)
    lens[0] = longest
    tokens = [(rng.random(n) ** 3 * (vocab + 2)).astype(np.int32) - 1 for n in lens]  # some outside the vocabulary
    return dict(tokens=tokens, prompt=[int(rng.integers(0, n + 1)) for n in lens], repetition=rng.uniform(0.5, 2, rows),
                frequency=rng.uniform(-1, 1, rows), presence=rng.uniform(-1, 1, rows),
                bias=[[(int(rng.integers(-2, vocab + 2)), float(rng.normal() * 5)) for _ in range(int(rng.integers(0, biases + 1)))] for _ in range(rows)],
                mask=[None] * rows)


LOGITS = [
    # dtype, rows, vocab, longest history, biases, pad, offset, in place, masks
    ("f32", 1, 1, 3, 2, 0, 0, False, 0),
    ("f32", 1, 50, 40, 0, 0, 0, True, 1),
    ("bf16", 3, 2047, 300, 20, 1, 0, False, 2),
    ("f16", 4, 2048, 1000, 50, 0, 0, True, 0),
    ("bf16", 5, 2056, 100, 3, 8, 0, False, 5),
    ("f16", 2, 4099, 5000, 10, 3, 1, True, 1),
    ("f32", 2, 10000, 20000, 500, 0, 0, False, 2),
    ("f32", 7, 5001, 0, 0, 0, 3, False, 3),
    ("bf16", 300, 1000, 20, 4, 0, 0, False, 10),
    # more biases than a work-group has threads; work-groups of longer slices
    ("f32", 3, 6000, 100, 4000, 0, 0, False, 0), ("f16", 2, 300, 9000, 3000, 0, 0, True, 2),
    ("bf16", 33, 131080, 6000, 1500, 0, 0, False, 7), ("f32", 40, 106003, 200, 30, 2, 1, True, 0),
]


@pytest.mark.parametrize("dtype,rows,vocab,longest,biases,pad,offset,in_place,masks", LOGITS)
def test_logits_rules(ctx, bufs, dtype, rows, vocab, longest, biases, pad, offset, in_place, masks):
    rng = np.random.default_rng(vocab + rows)
    raw = encode(rng.normal(size=(rows, vocab)) * 4, dtype)[0]
    rules = some_rules(rng, rows, vocab, longest, biases)
    table = mask_row = None
    if masks:
        table = rng.random((masks, vocab)) < rng.uniform(0, 1, (masks, 1))
        table[0] = False  # a mask that leaves nothing
        mask_row = rng.integers(-1, masks + 1, rows) if masks != rows else None  # -1 and `masks`: none
        at = mask_row if mask_row is not None else np.arange(rows)
        rules["mask"] = [table[k] if 0 <= k < masks else None for k in at]
    got = run_logits(ctx, bufs, dtype, raw, rules, pad=pad, offset=offset, in_place=in_place, masks=table, mask_row=mask_row)
    assert same_bits(got, logits_model(raw, dtype, rules), dtype)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_logits_that_are_not_finite(ctx, bufs, dtype):
    rng = np.random.default_rng(4)
    x = rng.normal(size=(2, 3000)).astype(np.float32)
    x[:, ::5] = np.nan
    x[:, 1::5], x[:, 2::5] = np.inf, -np.inf
    x[:, 3] = 0.0
    raw = encode(x, dtype)[0]
    if dtype != "f32":
        raw.view(np.uint16)[0, 0] = 0x7FC1 if dtype == "bf16" else 0x7E01  # a NaN's bits stay
    rules = some_rules(rng, 2, 3000, 500, 0)
    rules["tokens"] = [np.array([t for t in v if t != 0], np.int32) for v in rules["tokens"]]
    rules["prompt"] = [min(p, len(v)) for p, v in zip(rules["prompt"], rules["tokens"])]
    rules["bias"] = [[(7, np.inf), (8, -np.inf), (2, np.inf)], []]
    got = run_logits(ctx, bufs, dtype, raw, rules)
    assert same_bits(got, logits_model(raw, dtype, rules), dtype)
    assert got.view(np.uint32 if dtype == "f32" else np.uint16)[0, 0] == raw.view(np.uint32 if dtype == "f32" else np.uint16)[0, 0]


def test_logits_of_two_biases_the_last_counts_and_ranges_are_bounded(ctx, bufs):
    rng = np.random.default_rng(2)
    raw = rng.normal(size=(2, 600)).astype(np.float32)
    rules = some_rules(rng, 2, 600, 0, 0)
    rules["bias"] = [[(5, 1.0), (6, 2.0), (5, 3.0)] * 100 + [(5, -1.5)], [(5, 9.0)]]
    got = run_logits(ctx, bufs, "f32", raw, rules)
    assert same_bits(got, logits_model(raw, "f32", rules), "f32")
    # ranges that leave the lists are cut to them
    R = H.LogitsRules(tokens=bufs.put(np.array([1, 2, 3], np.int32)), token_start=bufs.put(np.array([-5, 2, 1 << 40], np.int64)),
                      ntokens=3, prompt_len=bufs.put(np.array([-3, 1 << 50], np.int64)), presence=bufs.put(np.ones(2, np.float32)),
                      repetition=bufs.put(np.full(2, 2, np.float32)))
    out = bufs.put(np.zeros_like(raw))
    H.logits_device(ctx, "f32", 2, 600, bufs.put(raw), R, out)
    rules = dict(tokens=[[1, 2], [3]], prompt=[0, 1], repetition=[2, 2], frequency=[0, 0], presence=[1, 1], bias=[[], []], mask=[None, None])
    assert same_bits(bufs.get(out, np.float32, 1200).reshape(2, 600), logits_model(raw, "f32", rules), "f32")


def test_logits_without_rules_are_copied(ctx, bufs):
    raw = np.random.default_rng(1).integers(0, 1 << 32, (3, 777), dtype=np.uint64).astype(np.uint32).view(np.float32)
    out = bufs.put(np.zeros_like(raw))
    H.logits_device(ctx, "f32", 3, 777, bufs.put(raw), H.LogitsRules(), out)
    assert (bufs.get(out, np.uint32, raw.size) == raw.view(np.uint32).reshape(-1)).all()


def test_logits_refusals(ctx, bufs):
    d = bufs.put(np.zeros(4096, np.float32))
    L = H.lib()

    def call(dtype=H.F32, rows=2, vocab=64, x=d, xs=64, o=d + 8192, os=64, **k):
        R = H.LogitsRules(**k)
        return L.hale_logits_device(ctx.handle, dtype, rows, vocab, x, xs, C.byref(R), o, os)

    for bad in (dict(dtype=H.Q8_0), dict(x=0), dict(o=0), dict(xs=63), dict(os=63), dict(x=d + 2), dict(o=d + 1), dict(vocab=(1 << 26) + 1),
                dict(o=d, os=65), dict(tokens=d), dict(tokens=d + 2, token_start=d), dict(tokens=d, token_start=d + 4),
                dict(bias_tokens=d), dict(bias_tokens=d, bias=d), dict(mask=d, mask_rows=2, mask_stride=1), dict(mask=d, mask_rows=1, mask_stride=2),
                dict(ntokens=1 << 31), dict(nbiases=1 << 31), dict(repetition=d + 2), dict(prompt_len=d + 4)):
        assert call(**bad) == H.EINVAL, bad
    assert L.hale_logits_device(ctx.handle, H.F32, 2, 64, d, 64, None, d, 64) == H.EINVAL
    assert call(rows=0, x=0) == H.OK and call(vocab=0, x=0) == H.OK


# ---- together ----------------------------------------------------------------------

def test_captured_norm_product_and_rules(ctx, bufs):
    """A norm that hands its codes to a vocabulary product whose logits the rules
    change in place: eager, captured and replayed with other rows in the same buffers."""
    rng = np.random.default_rng(12)
    rows, hidden, vocab = 5, 512, 3001
    codes, raw, scales, z = q4_weights(rng, vocab, hidden, 64, True, "f16")
    head = H.GroupQ4Matrix.new(ctx, vocab, hidden, 64, codes, raw, z)
    w = np.exp(0.2 * rng.normal(size=hidden)).astype(np.float32)
    rules = some_rules(rng, rows, vocab, 50, 5)
    x0, d0 = (encode(rng.normal(size=(rows, hidden)), "bf16")[1] for _ in range(2))
    dx, dd = bufs.put(encode(x0, "bf16")[0]), bufs.put(encode(d0, "bf16")[0])
    dw, dq, ds = bufs.put(w), bufs.put(np.zeros((rows, hidden), np.int8)), bufs.put(np.zeros((rows, hidden // 32), np.float32))
    dsum, dl = bufs.put(np.zeros((rows, hidden), np.uint16)), bufs.put(np.zeros((rows, vocab), np.float32))
    toks = np.concatenate([np.asarray(v, np.int32) for v in rules["tokens"]])
    start = np.concatenate([[0], np.cumsum([len(v) for v in rules["tokens"]])]).astype(np.int64)
    R = H.LogitsRules(tokens=bufs.put(toks), token_start=bufs.put(start), ntokens=len(toks),
                      prompt_len=bufs.put(np.asarray(rules["prompt"], np.int64)),
                      **{k: bufs.put(np.asarray(rules[k], np.float32)) for k in ("repetition", "frequency", "presence")})
    rules["bias"] = [[]] * rows

    def calls():
        H.rms_norm_q8_device(ctx, "bf16", rows, hidden, dx, dw, 1e-6, dq, ds, d_delta=dd, d_sum=dsum)
        head.matmul_q8_device("f32", rows, dq, ds, dl)
        H.logits_device(ctx, "f32", rows, vocab, dl, R, dl)

    def check(x, d):
        s, _, q, sc = norm_model(x, d, w, 1e-6, 32, "bf16")
        assert (decode(bufs.get(dsum, np.uint16, rows * hidden), "bf16").reshape(rows, hidden) == s).all()
        gq = bufs.get(dq, np.int8, rows * hidden).reshape(rows, hidden)
        gs = bufs.get(ds, np.float32, rows * hidden // 32).reshape(rows, -1)
        assert (gq == q).all()
        plain = bufs.put(np.zeros((rows, vocab), np.float32))
        head.matmul_q8_device("f32", rows, bufs.put(gq), bufs.put(gs), plain)  # equal calls give equal bits
        got = bufs.get(dl, np.float32, rows * vocab).reshape(rows, vocab)
        assert same_bits(got, logits_model(bufs.get(plain, np.float32, rows * vocab).reshape(rows, vocab), "f32", rules), "f32")

    calls()
    check(x0, d0)
    graph = ctx.capture(calls)
    for seed in range(4):
        rng = np.random.default_rng(seed)
        x, d = (encode(rng.normal(size=(rows, hidden)) * (seed + 1), "bf16")[1] for _ in range(2))
        for buf, v in ((dx, x), (dd, d)):
            next(b for b in bufs.all if b.address == buf).upload(encode(v, "bf16")[0])
        graph.launch()
        ctx.synchronize()
        check(x, d)
    graph.close()
    head.close()


def test_two_contexts_at_once(ctx, bufs):
    """Two contexts on one device, a thread each, the same calls many times over: each has the
    results of calls apart (divided rows, whose parts are counted in memory of the matrix)."""
    rng = np.random.default_rng(31)
    ntok, rows, cols, vocab = 3, 40, 14336, 5000
    codes, raw, _, z = q4_weights(rng, rows, cols, 128, True, "f16")
    x = rng.normal(size=(ntok, cols)).astype(np.float32)
    w = np.ones(2048, np.float32)
    logits = rng.normal(size=(4, vocab)).astype(np.float32)
    tokens, start = rng.integers(0, vocab, 4000).astype(np.int32), np.array([0, 500, 500, 3000, 4000], np.int64)
    repetition = np.full(4, 1.3, np.float32)

    def work(c, times):
        mine = Bufs(c)
        m = H.GroupQ4Matrix.new(c, rows, cols, 128, codes, raw, z)
        dx, dw, dl = mine.put(x), mine.put(w), mine.put(logits)
        R = H.LogitsRules(tokens=mine.put(tokens), token_start=mine.put(start), ntokens=4000, repetition=mine.put(repetition))
        o, q, s, lo = (mine.put(np.zeros(n, t)) for n, t in ((ntok * rows, np.float32), (7 * 2048, np.int8), (7, np.float32), (4 * vocab, np.float32)))
        for _ in range(times):
            m.matmul_device("f32", ntok, dx, o)
            H.rms_norm_q8_device(c, "f32", 7, 2048, dx, dw, 1e-6, q, s, block=2048)
            H.logits_device(c, "f32", 4, vocab, dl, R, lo)
        got = [mine.get(o, np.float32, ntok * rows), mine.get(q, np.int8, 7 * 2048), mine.get(s, np.float32, 7), mine.get(lo, np.float32, 4 * vocab)]
        m.close()
        for b in mine.all:
            b.free()
        return got

    want = work(ctx, 1)
    other = H.Context(0)
    with ThreadPoolExecutor(2) as pool:
        both = list(pool.map(work, (ctx, other), (200, 200)))
    for got in both:
        assert all((a == b).all() for a, b in zip(got, want))
    other.close()
