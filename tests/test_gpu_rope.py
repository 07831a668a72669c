"""Rotary positions on the GPU (hale_rope_*) against the formula in 64 bits."""
import numpy as np
import pytest

import hale_moe as H
from kv_model import EPS, NP, decode, encode

pytestmark = pytest.mark.gpu

SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def turn(x, pos, freq, factor, layout, r):
    """The rotated rows and, per number, |a| + |b| of its pair, in 64 bits."""
    x = x.astype(np.float64)
    out, mag = x.copy(), np.zeros_like(x)
    ang = pos.astype(np.float64)[:, None] * freq[None]
    c, s = np.cos(ang)[:, None] * factor, np.sin(ang)[:, None] * factor
    ia, ib = (np.arange(r // 2), np.arange(r // 2) + r // 2) if layout == "half" else (np.arange(0, r, 2), np.arange(1, r, 2))
    a, b = x[..., ia], x[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    mag[..., ia] = mag[..., ib] = (np.abs(a) + np.abs(b)) * factor
    return out, mag


def tolerance(dtype, want, mag):
    """The angle in half turns is rounded to f32 (2^-24 of at most 1, times pi),
    sin and cos are within 2 units of 2^-24 times 2, the factor, two products and a sum round once each:
    10 * 2^-24 of |a| + |b|, which covers pi + 4 + 2 and the products of errors; then the
    result's own rounding.  Results below f16's smallest normal number are off by half of 2^-24."""
    tol = mag * 10 * 2.0 ** -24 + EPS[dtype] * np.abs(want)
    return tol + (2.0 ** -25 if dtype == "f16" else 0.0)


def run(ctx, rope, dtype, q, k, pos, in_place=False, pad=0, offset=0):
    """Both sides through strided, offset buffers; what lies between stays."""
    n, hd, size = len(pos), rope.head_dim, SIZE[dtype]
    bp = ctx.malloc(max(4 * n, 4))
    bp.upload(pos.astype(np.int32))
    bufs, args, outs = [bp], [], []
    for x in (q, k):
        heads = 0 if x is None else x.shape[1]
        stride = heads * hd + pad
        total = offset + n * stride
        raw = np.full(total, 77, NP[dtype]) if dtype != "f32" else np.full(total, 77.0, np.float32)
        rows = raw[offset:].reshape(n, stride) if heads else None
        if heads:
            rows[:, :heads * hd] = encode(x, dtype)[0].reshape(n, -1)
        src = ctx.malloc(max(raw.nbytes, 4))
        src.upload(raw)
        dst = src if in_place else ctx.malloc(max(raw.nbytes, 4))
        if not in_place:
            dst.upload(np.full_like(raw, 55))
        bufs += [src, dst]
        args += [(src.address + offset * size if heads else 0, heads, dst.address + offset * size if heads else 0, stride)]
        outs.append((dst, raw, heads, stride, total))
    (dq, nq, oq, sq), (dk, nk, ok, sk) = args
    rope.apply_device(dtype, n, bp.address, dq, nq, oq, dk, nk, ok, q_stride=sq, q_out_stride=sq, k_stride=sk, k_out_stride=sk)
    got = []
    for dst, raw, heads, stride, total in outs:
        if not heads:
            got.append(None)
            continue
        back = dst.download(raw.dtype, total)
        rows = back[offset:].reshape(n, stride)
        keep = raw.dtype.type(77 if in_place else 55)
        assert (back[:offset] == keep).all() and (rows[:, heads * hd:] == keep).all()
        got.append(decode(np.ascontiguousarray(rows[:, :heads * hd]), dtype).reshape(n, heads, hd))
    for b in {id(b): b for b in bufs}.values():
        b.free()
    return got


CASES = [
    # dtype, rows, heads, kv heads, head dim, rotary, layout, scaling, pad, offset, in place
    ("f32", 1, 32, 4, 128, 128, "half", "none", 0, 0, False),
    ("f32", 1, 1, 1, 2, 2, "interleaved", "none", 0, 0, False),
    ("bf16", 33, 32, 8, 128, 64, "interleaved", "parts", 0, 0, False),
    ("f16", 17, 6, 2, 80, 80, "half", "linear", 0, 0, True),
    ("f16", 5, 3, 3, 20, 10, "interleaved", "ntk", 7, 3, True),
    ("bf16", 7, 5, 1, 96, 32, "half", "parts", 3, 1, False),
    ("f32", 9, 4, 2, 36, 6, "half", "ntk", 5, 1, True),
    ("f32", 3, 2, 1, 256, 256, "interleaved", "none", 1, 0, False),
    ("bf16", 1, 64, 8, 112, 112, "half", "none", 0, 0, False),
    ("f16", 300, 3, 1, 64, 64, "half", "none", 4, 4, False),
    ("f32", 2, 3, 1, 1000, 500, "half", "linear", 0, 0, False),
    ("bf16", 65, 1, 1, 15, 2, "interleaved", "none", 0, 0, False),
    ("bf16", 300, 12, 4, 128, 64, "half", "none", 0, 0, True),  # many rows, in 16-byte pieces
    ("f32", 260, 16, 2, 128, 128, "half", "parts", 4, 4, False),
    ("f16", 600, 8, 2, 96, 96, "interleaved", "ntk", 8, 8, False),
    ("bf16", 2100, 3, 1, 80, 16, "interleaved", "linear", 0, 0, False),
    ("f16", 700, 6, 0, 128, 128, "half", "none", 0, 0, True),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c)))
def test_rope_against_64_bits(ctx, case):
    dtype, n, nq, nk, hd, r, layout, scaling, pad, offset, in_place = case
    factor = 1.2 if scaling == "parts" else 1.0
    rope = H.Rope(ctx, hd, 1e6, rotary_dim=r, layout=layout, scaling=scaling, factor=8.0, original_len=8192.0,
                  attention_factor=factor)
    g = np.random.default_rng(n * 131 + hd)
    q, k = (encode(g.standard_normal((n, h, hd)), dtype)[1] if h else None for h in (nq, nk))
    pos = g.integers(0, 1 << 20, n)
    pos[0] = 0
    if n > 2:
        pos[1], pos[2] = 2 ** 31 - 1, -(2 ** 31)  # the ends of what an int32 holds
    got = run(ctx, rope, dtype, q, k, pos, in_place, pad, offset)
    for x, y in zip((q, k), got):
        if x is None:
            continue
        # positions past 2^24 lose more in 64 bits here: the formula's own angle is off by 2^-53 of it
        want, mag = turn(x, pos, rope.frequencies(), factor, layout, r)
        slack = mag * (np.abs(pos)[:, None, None] * 2.0 ** -50)
        assert (np.abs(y - want) <= tolerance(dtype, want, mag) + slack).all()
        if dtype == "f32":
            assert (y[..., r:] == x[..., r:]).all()
    rope.close()


def test_rope_rows_past_a_grid(ctx):
    """More rows than a grid has work-groups: rows about the edge against 64 bits."""
    n, hd, edge = (1 << 24) + 70, 16, (1 << 24) - 1
    rope = H.Rope(ctx, hd, 10000.0)
    freq = np.asarray(rope.frequencies())
    b, pos = ctx.malloc(n * hd * 2), ctx.malloc(n * 4)
    b.upload(np.zeros(n * hd, np.uint16))
    pos.upload(np.arange(n, dtype=np.int32))
    x = {}
    g = np.random.default_rng(5)
    for first in (0, edge - 20, n - 20):
        raw, x[first] = encode(g.standard_normal((20, hd)).astype(np.float32), "bf16")
        b.upload(np.ascontiguousarray(raw.reshape(-1)), first * hd * 2)
    rope.apply_device("bf16", n, pos.address, b.address, 1, b.address, 0, 0, 0)
    for first, v in x.items():
        v = np.asarray(v, np.float64).reshape(20, hd)
        t = (first + np.arange(20))[:, None] * freq
        want = np.concatenate([v[:, :8] * np.cos(t) - v[:, 8:] * np.sin(t), v[:, 8:] * np.cos(t) + v[:, :8] * np.sin(t)], 1)
        got = decode(b.download(np.uint16, 20 * hd, first * hd * 2), "bf16").reshape(20, hd)
        size = np.hypot(np.abs(v[:, :8]), np.abs(v[:, 8:]))
        # result rounded by 2^-8 of it, products and cosines by a few 2^-24
        assert (np.abs(got - want) <= np.abs(want) * 2.0 ** -8 + np.tile(size, 2) * 2.0 ** -20).all(), first
    b.free()
    pos.free()


def test_rope_one_side_and_gradient(ctx):
    """Keys alone; and turning back with negative positions: the transpose, so
    <turn(x), y> = <x, turn back(y)>, and back after forth is the identity."""
    rope = H.Rope(ctx, 64, 1e4)
    g = np.random.default_rng(5)
    x, y = (g.standard_normal((11, 3, 64)).astype(np.float32) for _ in range(2))
    pos = g.integers(0, 5000, 11)
    fx = run(ctx, rope, "f32", None, x, pos)[1]
    by = run(ctx, rope, "f32", y, None, -pos)[0]
    # both sums are of 2112 products; each factor is off by at most 10 * 2^-24 of |a| + |b| <= 2 max
    left, right = (fx.astype(np.float64) * y).sum(), (by.astype(np.float64) * x).sum()
    bound = 2 * 10 * 2.0 ** -24 * (np.abs(x).max() * 2 * np.abs(y).sum() + np.abs(y).max() * 2 * np.abs(x).sum())
    assert abs(left - right) <= bound
    # against differences: the map is linear, so a difference of any size is exact but for roundings
    e = np.zeros_like(x)
    e[4, 1, 9] = 1.0
    col = run(ctx, rope, "f32", None, x + e, pos)[1].astype(np.float64) - fx
    back = run(ctx, rope, "f32", e, None, pos)[0]
    assert (np.abs(col - back) <= 40 * 2.0 ** -24 * (np.abs(x).max() * 2 + 2)).all()
    ident = run(ctx, rope, "f32", fx, None, -pos)[0]
    assert (np.abs(ident - x) <= 4 * 10 * 2.0 ** -24 * np.abs(x).max() * 2).all()
    rope.close()


def test_rope_no_rows_or_heads(ctx):
    rope = H.Rope(ctx, 64, 1e4)
    rope.apply_device("f32", 0, 0, 0, 4, 0)
    rope.apply_device("bf16", 5, 0, 0, 0, 0)
    rope.close()


def test_rope_values_that_are_not_finite_stay_in_their_pairs(ctx):
    rope = H.Rope(ctx, 64, 1e4, rotary_dim=32)
    g = np.random.default_rng(8)
    x = g.standard_normal((3, 2, 64)).astype(np.float32)
    x[1, 0, 5], x[2, 1, 40] = np.nan, np.inf
    got = run(ctx, rope, "f32", x, None, np.array([3, 4, 5]))[0]
    bad = ~np.isfinite(got)
    assert set(map(tuple, np.argwhere(bad))) == {(1, 0, 5), (1, 0, 21), (2, 1, 40)}
    rope.close()


def test_rope_refusals(ctx):
    with pytest.raises(ValueError, match="rotary_dim"):
        H.Rope(ctx, 64, 1e4, rotary_dim=33)
    with pytest.raises(ValueError, match="unknown layout"):
        H.Rope(ctx, 64, 1e4, layout="other")
    rope = H.Rope(ctx, 64, 1e4)
    b = ctx.malloc(4096)
    a = b.address
    with pytest.raises(ValueError, match="not f32"):
        rope.apply_device("q8_0", 1, a, a, 1, a)
    with pytest.raises(ValueError, match="NULL"):
        rope.apply_device("f32", 1, a, 0, 1, a)
    with pytest.raises(ValueError, match="positions"):
        rope.apply_device("f32", 1, 0, a, 1, a)
    with pytest.raises(ValueError, match="below"):
        rope.apply_device("f32", 1, a, a, 2, a, q_stride=127)
    with pytest.raises(ValueError, match="aligned"):
        rope.apply_device("f32", 1, a, a + 2, 1, a + 2)
    with pytest.raises(ValueError, match="different strides"):
        rope.apply_device("f32", 2, a, a, 1, a, q_stride=64, q_out_stride=128)
    with pytest.raises(ValueError, match="frequencies"):
        ctx.check(H.lib().hale_rope_frequencies(rope.handle, (H.C.c_double * 4)(), 4))
    b.free()
    rope.close()


def test_rope_replays_in_a_graph(ctx):
    rope = H.Rope(ctx, 128, 1e6)
    g = np.random.default_rng(3)
    x = g.standard_normal((4, 8, 128)).astype(np.float32)
    bx, bo, bp = ctx.malloc(x.nbytes), ctx.malloc(x.nbytes), ctx.malloc(16)
    graph = ctx.capture(lambda: rope.apply_device("f32", 4, bp.address, bx.address, 8, bo.address))
    for k in range(3):
        pos = g.integers(0, 9999, 4)
        bp.upload(pos.astype(np.int32))
        bx.upload(x * (k + 1))
        graph.launch()
        got = bo.download(np.float32, x.size).reshape(x.shape)
        want = run(ctx, rope, "f32", x * (k + 1), None, pos)[0]
        assert (got.view(np.uint32) == want.view(np.uint32)).all()
    graph.close()
    for b in (bx, bo, bp):
        b.free()
    rope.close()
