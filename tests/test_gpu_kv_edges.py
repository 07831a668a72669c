"""Edges of the paged 8-bit key/value cache on the GPU (hale_kv_*): steps that
fill every list of the plan, graphs around a cache whose buffers grow."""
import numpy as np
import pytest

import hale_moe as H
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
