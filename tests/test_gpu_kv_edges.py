"""Edges of the paged 8-bit key/value cache on the GPU (hale_kv_*): steps that
fill every list of the plan, graphs around a cache whose buffers grow, queries
that are not finite, values next to the largest number."""
import os

import numpy as np
import pytest

import hale_moe as H
from kv_model import NP, Model, attention_bound, decode, encode
from test_gpu_kv import rig  # noqa: F401

pytestmark = pytest.mark.gpu


def test_one_token_and_a_chunk_under_four_windows_in_both_types(rig):
    """Few and many rows, both over divided contexts, in every view of one step."""
    r = rig(dim=64, heads=8, kv_heads=1, pages=120, seqs=2)
    g = np.random.default_rng(31)
    seqs = [r.create(), r.create()]
    r.step(g, "f32", seqs, [2500, 2000])
    views = [(w, dtype) for w in (0, 1000, 1500, 2000) for dtype in ("f32", "bf16")]
    q = r.put(np.zeros(4500 * 8 * 64, np.float32))
    for w, dtype in views:  # the first call of each makes its view
        r.kv.attention_device(0, dtype, 4500, q.address, q.address, window=w)
    r.step(g, "f32", seqs, [1, 60])
    for w, dtype in views:
        r.check_attention(g, 0, dtype, seqs, [1, 60], window=w)
    r.step(g, "bf16", seqs, [70, 2])  # the other way round
    for w, dtype in views:
        r.check_attention(g, 0, dtype, seqs, [70, 2], window=w)


def test_a_captured_rotation_of_the_steps_positions(rig, ctx):
    """By itself in a graph: replayed for any step, refused once the positions lie
    elsewhere or the cache is gone."""
    r = rig(dim=64)
    rope = H.Rope(ctx, 64, 1e4)
    g = np.random.default_rng(32)
    a = r.create()
    x = g.standard_normal((3, 4, 64)).astype(np.float32)
    src, out = r.put(x), ctx.malloc(x.nbytes)
    turn = lambda: rope.apply_device("f32", 3, r.kv.positions, src.address, 4, out.address)
    graph = ctx.capture(turn)
    for n in (3, 5, 40):
        r.step(g, "f32", [a], [n])
        turn()
        want = out.download(np.float32, x.size).copy()
        for _ in range(2):
            out.upload(np.zeros_like(x))
            graph.launch()
            assert (out.download(np.float32, x.size) == want).all()
    r.kv.reserve(5000)
    with pytest.raises(ValueError, match="grew"):
        graph.launch()
    graph.close()
    graph = ctx.capture(turn)
    r.step(g, "f32", [a], [3])
    graph.launch()
    r.kv.close()
    with pytest.raises(ValueError, match="gone"):
        graph.launch()
    graph.close()
    rope.close()
    out.free()


def set_number(raw, dtype, at, value):
    """A number of an encoded array, given as its bits."""
    raw.view({"f32": np.uint32, "f16": np.uint16, "bf16": np.uint16}[dtype])[at] = value


INF = {"f32": 0x7F800000, "f16": 0x7C00, "bf16": 0x7F80}
SIGN = {"f32": 1 << 31, "f16": 1 << 15, "bf16": 1 << 15}


def attend_raw(r, dtype, raw):
    """Results of queries given as encoded numbers [n][heads][dim]."""
    q, out = r.put(raw.reshape(-1)), r.ctx.malloc(raw.nbytes)
    r.kv.attention_device(0, dtype, raw.shape[0], q.address, out.address)
    got = decode(out.download(NP[dtype], raw.size), dtype).reshape(raw.shape)
    out.free()
    return got


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [1, 60])
def test_every_kind_of_nan_in_a_query(rig, dtype, n):
    """Quiet and signalling, of both signs, with the smallest and largest payloads."""
    r = rig(dim=64, heads=4, kv_heads=2, pages=40)
    g = np.random.default_rng(34)
    a = r.create()
    r.step(g, dtype, [a], [70])
    r.step(g, dtype, [a], [n])
    low = INF[dtype]
    quiet = {"f32": 1 << 22, "f16": 1 << 9, "bf16": 1 << 6}[dtype]
    full = SIGN[dtype] - 1 - low
    clean = encode(g.standard_normal((n, 4, 64)), dtype)[0]
    want = attend_raw(r, dtype, clean)
    for payload in (1, quiet, full - quiet, full):
        for sign in (0, SIGN[dtype]):
            raw = clean.copy()
            set_number(raw, dtype, (n - 1, 2, 33), sign | low | payload)
            got = attend_raw(r, dtype, raw)
            assert np.isnan(got[n - 1, 2]).all(), (hex(payload), sign)
            got[n - 1, 2] = want[n - 1, 2]
            assert (got.view(np.uint32) == want.view(np.uint32)).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("old, n", [(0, 1), (0, 5), (70, 1), (70, 60), (3000, 1), (3000, 20)])
def test_infinite_queries_over_keys_of_one_sign(rig, dtype, old, n):
    """All scores of a row infinite, of one sign: NaN in the row, and in no other."""
    r = rig(dim=64, heads=4, kv_heads=2, pages=60)
    g = np.random.default_rng(33)
    a = r.create()
    for m in (old, n):
        if m:
            r.kv.step([a], [m])
            k = g.standard_normal((m, 2, 64)).astype(np.float32)
            k[:, :, 7] = 3.0 + np.abs(k[:, :, 7])  # codes of one sign, none 0
            r.append(0, dtype, [a], [m], k, g.standard_normal((m, 2, 64)))
    raw = encode(g.standard_normal((n, 4, 64)), dtype)[0]
    clean = attend_raw(r, dtype, raw)
    hit = np.zeros((n, 4), bool)
    for t, h, bits in ((0, 1, INF[dtype]), (0, 2, INF[dtype] | SIGN[dtype]), (n - 1, 3, INF[dtype] | SIGN[dtype])):
        set_number(raw, dtype, (t, h, 7), bits)
        hit[t, h] = True
    got = attend_raw(r, dtype, raw)
    assert np.isnan(got[hit]).all()
    assert (got[~hit].view(np.uint32) == clean[~hit].view(np.uint32)).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("old, n", [(0, 40), (200, 1), (5000, 1), (200, 60), (5000, 40)])
def test_values_next_to_the_largest_number(rig, dtype, old, n):
    """Values up to 3.38e38: sums of them are not finite, their means are."""
    r = rig(dim=64, heads=8, kv_heads=1, pages=100, max_len=6000)
    g = np.random.default_rng(35)
    a = r.create()
    for m in (old, n):
        if m:
            r.kv.step([a], [m])
            v = g.uniform(0.2, 1.0, (m, 1, 64)) * 3.38e38
            r.append(0, dtype, [a], [m], g.standard_normal((m, 1, 64)), v)
    q = encode(g.standard_normal((n, 8, 64)), dtype)[1]
    got = r.attend(0, dtype, q)
    want, mag, prod, total, vtop = r.model.attend(a, 0, q, 0.125)
    assert np.isfinite(got).all()
    assert (np.abs(got.astype(np.float64) - want) <= attention_bound(dtype, mag, prod, total, vtop, 64)).all()


def test_a_graph_is_not_launched_inside_a_capture(rig, ctx):
    r = rig(dim=64)
    g = np.random.default_rng(36)
    a = r.create()
    r.step(g, "f32", [a], [3])
    q, out = r.put(g.standard_normal((3, 4, 64)).astype(np.float32)), ctx.malloc(3 * 4 * 64 * 4)
    call = lambda: r.kv.attention_device(0, "f32", 3, q.address, out.address)
    call()
    want = out.download(np.float32, 3 * 4 * 64).copy()
    graph = ctx.capture(call)
    with pytest.raises(ValueError, match="captur"):
        ctx.capture(graph.launch)
    out.upload(np.zeros(3 * 4 * 64, np.float32))
    graph.launch()
    assert (out.download(np.float32, 3 * 4 * 64) == want).all()
    graph.close()
    out.free()


def test_the_documented_step_runs(ctx):
    """README.md's example of several sequences, as it stands there."""
    with open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "README.md")) as f:
        blocks = f.read().split("```python\n")[1:]
    code = next(b.split("```")[0] for b in blocks if "H.KvCache(" in b)
    g = np.random.default_rng(37)
    heads, kv_heads, dim, n = 8, 2, 64, 6
    x = {name: encode(g.standard_normal((n, h, dim)), "bf16") for name, h in (("q", heads), ("k", kv_heads), ("v", kv_heads))}
    bufs = {name: ctx.malloc(raw.nbytes) for name, (raw, _) in x.items()}
    for name, (raw, _) in x.items():
        bufs[name].upload(raw)
    bufs["out"] = ctx.malloc(x["q"][0].nbytes)
    space = dict(H=H, ctx=ctx, layers=1, layer=0, heads=heads, kv_heads=kv_heads, head_dim=dim, num_pages=8, max_seqs=4,
                 max_len=256, **{name: b.address for name, b in bufs.items()})
    exec(code, space)
    # one token and five, each from position 0: the rotation of both sides and causal attention
    got = decode(bufs["out"].download(np.uint16, x["q"][0].size), "bf16").reshape(n, heads, dim)
    q = decode(bufs["q"].download(np.uint16, x["q"][0].size), "bf16").reshape(n, heads, dim)  # turned in place
    k = decode(bufs["k"].download(np.uint16, x["k"][0].size), "bf16").reshape(n, kv_heads, dim)
    assert (q[0] == x["q"][1][0]).all() and (q[2] != x["q"][1][2]).any()
    model = Model(1, heads, kv_heads, dim)
    for s, at, m in ((0, 0, 1), (1, 1, 5)):
        model.create(s)
        model.append(s, 0, k[at:at + m], x["v"][1][at:at + m])
        want, mag, prod, total, vtop = model.attend(s, 0, q[at:at + m], dim ** -0.5)
        assert (np.abs(got[at:at + m] - want) <= attention_bound("bf16", mag, prod, total, vtop, dim)).all()
    for name in ("rope", "kv"):
        space[name].close()
    for b in bufs.values():
        b.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("size", [1e-27, 1e-33, 1e-38])
@pytest.mark.parametrize("old, n", [(0, 40), (200, 1), (5000, 1), (5000, 40)])
def test_values_next_to_zero(rig, dtype, size, old, n):
    """The smallest values: probabilities are no finer than the documented floor, in which
    scales below 2^-100 count as that."""
    r = rig(dim=64, heads=8, kv_heads=1, pages=100, max_len=6000)
    g = np.random.default_rng(38)
    a = r.create()
    for m in (old, n):
        if m:
            r.kv.step([a], [m])
            r.append(0, dtype, [a], [m], g.standard_normal((m, 1, 64)), g.standard_normal((m, 1, 64)) * size)
    q = encode(g.standard_normal((n, 8, 64)), dtype)[1]
    got = r.attend(0, dtype, q)
    want, mag, prod, total, vtop = r.model.attend(a, 0, q, 0.125)
    bound = attention_bound(dtype, mag, prod, total, np.maximum(vtop, 127 * 2.0 ** -100), 64)
    # numbers below 2^-126 are multiples of 2^-149 (bf16: 2^-133): half a step of the result's rounding,
    # and of each partial sum's, which is held times 2^-10 or less of it
    bound = bound + (2.0 ** -134 if dtype == "bf16" else 2.0 ** -150) + 1024 * 2.0 ** -149
    assert (np.abs(got.astype(np.float64) - want) <= bound).all()
