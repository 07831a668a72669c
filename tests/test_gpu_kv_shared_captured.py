"""Captured steps over shared prefixes (hale_kv_share_prefixes) on the GPU: graphs whose replays take
other kernels than the captured step did, and a whole serving step, eager and captured."""
import numpy as np
import pytest

import hale_moe as H
from kv_model import attention_bound, decode, encode
from test_gpu_kv import Rig, rig  # noqa: F401
from test_gpu_kv_shared import family

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim,prompt", [("bf16", 32, 3000), ("f16", 32, 3000), ("f32", 16, 5700)])
@pytest.mark.parametrize("turns", ["apart, shared, apart, shared", "shared, apart, shared"])
def test_a_captured_step_that_comes_to_share_for_many_rows(rig, ctx, dtype, dim, prompt, turns):
    """24 sequences of 16 rows, each in the kernel of few; their shared pages, where there are any, are so
    many that they go to that of many, which a captured step of unrelated sequences launches for
    nothing (the plans: tests/native/kv_shared_worth_check.cpp)."""
    heads, n, ntok = 128, 24, 2
    r = rig(dim=dim, heads=heads, kv_heads=16, pages=400, seqs=n + 1, max_len=6000)
    g = np.random.default_rng(prompt)
    r.kv.reserve(9000)  # the longest step: nothing moves behind a captured one
    r.kv.share_prefixes(64)
    size = n * ntok * heads * dim
    q, out = ctx.malloc(size * 4), ctx.malloc(size * 4)
    graph = None
    for turn in turns.split(", "):
        root = []
        if turn == "apart":
            seqs = [r.create() for _ in range(n)]
            r.step(g, dtype, seqs, [30 * i for i in range(n)])
        else:
            a, seqs = family(r, g, dtype, prompt, n, [5 * i for i in range(n)])
            root = [a]
        r.step(g, dtype, seqs, [ntok] * n)
        raw, x = encode(g.standard_normal((n * ntok, heads, dim)), dtype)
        q.upload(raw.reshape(-1))
        call = lambda: r.kv.attention_device(0, dtype, n * ntok, q.address, out.address)  # noqa: E731
        call()
        eager = out.download(raw.dtype, raw.size)
        graph = graph or ctx.capture(call)
        for _ in range(2):
            out.upload(np.full(raw.size, 9, raw.dtype))
            graph.launch()
            got = out.download(raw.dtype, raw.size)
            assert (got == eager).all()
        got = decode(got, dtype).reshape(n * ntok, heads, dim)
        for i, s in enumerate(seqs):
            at = slice(i * ntok, (i + 1) * ntok)
            want, mag, prod, total, vtop = r.model.attend(s, 0, x[at], dim ** -0.5)
            assert (np.abs(got[at] - want) <= attention_bound(dtype, mag, prod, total, vtop, dim)).all(), (turn, s)
        for s in seqs + root:
            r.free(s)
    graph.close()
    q.free()
    out.free()


def test_a_whole_serving_step_captured(rig, ctx):
    """Norm, projections, rotation, store, attention behind a shared prompt, residual and norm, vocabulary and
    rules, captured in one graph and replayed for later steps, each against the same step's eager calls, to
    the bit (their values: test_gpu_kv_shared.py)."""
    from test_gpu_step_ops import Bufs, q4_weights
    heads, kv_heads, dim, hidden, vocab, n = 8, 2, 64, 512, 1001, 5
    r = rig(dim=dim, heads=heads, kv_heads=kv_heads, pages=100, seqs=10)
    b = Bufs(ctx)
    g = np.random.default_rng(14)
    r.kv.share_prefixes(64)
    _, seqs = family(r, g, "bf16", 200, n, [1, 2, 3, 70, 0])
    made = {}
    for name, rows, cols in (("q", heads * dim, hidden), ("k", kv_heads * dim, hidden), ("v", kv_heads * dim, hidden),
                             ("o", hidden, heads * dim), ("head", vocab, hidden)):
        w = q4_weights(g, rows, cols, 64, True, "f16")
        made[name] = H.GroupQ4Matrix.new(ctx, rows, cols, 64, w[0], w[1], w[3])
    dx, dw = b.put(np.zeros((n, hidden), np.uint16)), b.put(np.exp(0.1 * g.standard_normal(hidden)).astype(np.float32))
    sizes = dict(codes=(np.int8, hidden), scales=(np.float32, hidden // 32), q=(np.uint16, heads * dim), k=(np.uint16, kv_heads * dim),
                 v=(np.uint16, kv_heads * dim), o=(np.uint16, heads * dim), h=(np.uint16, hidden), sum=(np.uint16, hidden),
                 logits=(np.float32, vocab))
    d = {k: b.put(np.zeros((n, w), t)) for k, (t, w) in sizes.items()}
    tokens = b.put(np.array([[5, 6, 5, i] for i in range(n)], np.int32))
    rules = H.LogitsRules(tokens=tokens, token_start=b.put(np.arange(0, 4 * n + 1, 4, dtype=np.int64)), ntokens=4 * n,
                          repetition=b.put(np.full(n, 1.2, np.float32)), presence=b.put(np.full(n, 0.25, np.float32)))
    rope = H.Rope(ctx, dim, 10000.0)

    def calls():
        H.rms_norm_q8_device(ctx, "bf16", n, hidden, dx, dw, 1e-6, d["codes"], d["scales"])
        for name in "qkv":
            made[name].matmul_q8_device("bf16", n, d["codes"], d["scales"], d[name])
        rope.apply_device("bf16", n, r.kv.positions, d["q"], heads, d["q"], d["k"], kv_heads, d["k"])
        r.kv.append_device(0, "bf16", n, d["k"], d["v"])
        r.kv.attention_device(0, "bf16", n, d["q"], d["o"])
        made["o"].matmul_device("bf16", n, d["o"], d["h"])
        H.rms_norm_q8_device(ctx, "bf16", n, hidden, dx, dw, 1e-6, d["codes"], d["scales"], d_delta=d["h"], d_sum=d["sum"])
        made["head"].matmul_q8_device("f32", n, d["codes"], d["scales"], d["logits"])
        H.logits_device(ctx, "f32", n, vocab, d["logits"], rules, d["logits"])

    def results():
        return {k: b.get(a, sizes[k][0], n * sizes[k][1]) for k, a in d.items()}

    graph = None
    for turn in range(4):
        b.set(dx, encode(g.standard_normal((n, hidden)), "bf16")[0])
        b.set(tokens, g.integers(0, vocab, (n, 4)).astype(np.int32))
        r.kv.step(seqs, [1] * n)
        calls()
        want = results()
        assert np.isfinite(want["logits"]).all()
        if graph is None:
            graph = ctx.capture(calls)
        for again in range(2):  # the same step once more, from where the eager one began
            for s in seqs:
                r.kv.seq_truncate(s, r.kv.seq_len(s) - 1)
            r.kv.step(seqs, [1] * n)
            for k, a in d.items():
                b.set(a, np.full(n * sizes[k][1], 7, sizes[k][0]))
            graph.launch()
            got = results()
            assert all((got[k] == want[k]).all() for k in sizes), (turn, again, [k for k in sizes if (got[k] != want[k]).any()])
    graph.close()
    rope.close()
    for m in made.values():
        m.close()
    for x in b.all:
        x.free()
