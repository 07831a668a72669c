"""Attention of sequences that share pages (hale_kv_share_prefixes) on the GPU,
against 64 bits within what its roundings add up to, and the setting beside the
cache's other calls."""
import numpy as np
import pytest

import hale_moe as H
from kv_model import NP, attention_bound, decode, encode
from test_gpu_kv import Rig, rig  # noqa: F401

pytestmark = pytest.mark.gpu


def family(r, g, dtype, prompt, ways, tails):
    """A prompt and its forks, each with a tail of its own."""
    a = r.create()
    r.step(g, dtype, [a], [prompt])
    seqs = r.fork(a, ways)
    if sum(tails):
        r.step(g, dtype, seqs, tails)
    return a, seqs


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [16, 64, 80, 128, 176, 256])
def test_forks_of_one_prompt(rig, dtype, dim):
    r = rig(dim=dim, heads=8, kv_heads=2, pages=200, seqs=12)
    g = np.random.default_rng(dim)
    r.kv.share_prefixes(64)
    _, seqs = family(r, g, dtype, 700, 5, [0, 3, 64, 100, 257])
    r.step(g, dtype, seqs, [1] * 5)
    r.check_attention(g, 0, dtype, seqs, [1] * 5)
    r.step(g, dtype, seqs, [1, 0, 5, 40, 2])
    r.check_attention(g, 0, dtype, seqs, [1, 0, 5, 40, 2], pad=3, offset=1)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (16, 1), (12, 4), (40, 5)])
@pytest.mark.parametrize("ways", [2, 9, 31])
def test_head_groups_and_ways(rig, heads, kv_heads, ways):
    r = rig(dim=32, heads=heads, kv_heads=kv_heads, pages=200, seqs=40)
    g = np.random.default_rng(heads)
    r.kv.share_prefixes(1)
    root, seqs = family(r, g, "bf16", 191, ways, [i % 7 for i in range(ways)])
    r.step(g, "bf16", [root] + seqs, [2] + [1] * ways)
    r.check_attention(g, 0, "bf16", [root] + seqs, [2] + [1] * ways)


@pytest.mark.parametrize("prompt", [63, 64, 65, 127, 128, 1000, 5000])
def test_prompts_of_any_length(rig, prompt):
    r = rig(dim=64, heads=8, kv_heads=1, pages=300, seqs=6, max_len=6000)
    g = np.random.default_rng(prompt)
    r.kv.share_prefixes(64)
    _, seqs = family(r, g, "f16", prompt, 3, [0, 1, 70])
    r.step(g, "f16", seqs, [1, 1, 1])
    r.check_attention(g, 0, "f16", seqs, [1, 1, 1])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_prefixes_within_prefixes(rig, dtype):
    """A system prompt, conversations behind it, answers to each, and one stranger among them."""
    r = rig(layers=2, dim=64, heads=8, kv_heads=2, pages=400, seqs=30, max_len=4096)
    g = np.random.default_rng(4)
    r.kv.share_prefixes(64)
    root, talks = family(r, g, dtype, 330, 3, [200, 0, 900])
    seqs = []
    for t in talks:
        seqs += [t] + r.fork(t, 3)
    stranger = r.create()
    seqs.insert(5, stranger)
    ntok = [1 + i % 3 for i in range(len(seqs))]
    ntok[5] = 150
    r.step(g, dtype, seqs, ntok)
    for layer in (0, 1):
        r.check_attention(g, layer, dtype, seqs, ntok)
    deeper = r.fork(seqs[2], 4)  # a fourth level
    r.step(g, dtype, [seqs[2]] + deeper, [130] * 5)
    again = deeper + r.fork(deeper[0], 2)
    order = [root] + seqs[:3] + again + seqs[3:]
    r.step(g, dtype, order, [1] * len(order))
    r.check_attention(g, 1, dtype, order, [1] * len(order))
    r.check_attention(g, 0, dtype, order, [1] * len(order), window=100)  # windows are computed apart
    order = order[::-1]  # any order of the step is right, neighbours or not
    r.step(g, dtype, order, [1] * len(order))
    r.check_attention(g, 0, dtype, order, [1] * len(order))


@pytest.mark.parametrize("dtype,dim,heads,kv_heads", [("bf16", 128, 16, 2), ("bf16", 128, 32, 4), ("f16", 64, 32, 4), ("f32", 32, 64, 8)])
def test_a_long_prompt_for_many_rows(rig, dtype, dim, heads, kv_heads):
    """Rows over several tiles, pages over many parts; from the second on for the kernel of many rows."""
    r = rig(dim=dim, heads=heads, kv_heads=kv_heads, pages=400, seqs=24, max_len=9000)
    g = np.random.default_rng(5)
    r.kv.share_prefixes(1000)
    _, seqs = family(r, g, dtype, 8100, 20, [3 * i for i in range(20)])
    ntok = [1 + (i % 4) * 2 for i in range(20)]
    r.step(g, dtype, seqs, ntok)
    r.check_attention(g, 0, dtype, seqs, ntok)


def test_sequences_that_diverge_truncate_and_move(rig):
    r = rig(dim=32, heads=4, kv_heads=2, pages=120, seqs=8)
    g = np.random.default_rng(6)
    r.kv.share_prefixes(64)
    root, seqs = family(r, g, "f16", 500, 3, [5, 5, 5])
    r.truncate(seqs[1], 130)  # holds two of the shared pages, the third cut
    r.step(g, "f16", seqs, [3, 200, 1])
    r.check_attention(g, 0, "f16", seqs, [3, 200, 1])
    other = r.copy(seqs[0])  # pages of its own: shares nothing
    order = [seqs[0], other, seqs[2]]
    r.step(g, "f16", order, [1, 1, 1])
    r.free(root)
    assert r.kv.compact() >= 0
    r.check_attention(g, 0, "f16", order, [1, 1, 1])
    r.step(g, "f16", order[::2], [1, 1])
    r.free(seqs[1])
    r.kv.compact()  # pages move behind the step's plan
    r.check_attention(g, 0, "f16", order[::2], [1, 1])
    r.kv.resize(60)
    r.check_attention(g, 0, "f16", order[::2], [1, 1])
    r.check_contents()


def test_the_setting(rig, ctx):
    r = rig(dim=64, heads=8, kv_heads=2, pages=200, seqs=10)
    g = np.random.default_rng(7)
    _, seqs = family(r, g, "f32", 640, 4, [1, 2, 3, 4])
    r.step(g, "f32", seqs, [1] * 4)
    q = encode(g.standard_normal((4, 8, 64)), "f32")[1]
    apart = r.attend(0, "f32", q)
    r.kv.share_prefixes(0)  # as it was: the step stands
    assert (r.attend(0, "f32", q) == apart).all()
    r.kv.share_prefixes(64)
    with pytest.raises(ValueError, match="without a current step"):
        r.attend(0, "f32", q)
    r.kv.step(seqs, [0] * 4)
    for s in seqs:
        r.truncate(s, r.kv.seq_len(s) - 1)

    def again():
        gg = np.random.default_rng(8)
        r.step(gg, "f32", seqs, [1] * 4)
        got = r.attend(0, "f32", q)
        assert (r.attend(0, "f32", q) == got).all()  # equal calls give equal bits
        for s in seqs:
            r.truncate(s, r.kv.seq_len(s) - 1)
        return got

    shared = again()
    r.kv.share_prefixes(641)  # more than they have
    none = again()
    r.kv.share_prefixes(0)
    assert (again() == none).all()
    assert not (none == shared).all() and np.abs(none - shared).max() < 1e-4
    r.kv.share_prefixes(1 << 60)  # beyond any length
    assert (again() == none).all()
    for v in (63, 64):  # pages count
        r.kv.share_prefixes(v)
        assert (again() == shared).all()


@pytest.mark.parametrize("spoil", [np.inf, np.nan])
def test_a_query_that_is_not_finite_spoils_only_its_row(rig, spoil):
    r = rig(dim=64, heads=8, kv_heads=2, pages=100, seqs=10)
    g = np.random.default_rng(9)
    r.kv.share_prefixes(64)
    _, seqs = family(r, g, "f32", 300, 6, [1] * 6)
    r.step(g, "f32", seqs, [1] * 6)
    q = encode(g.standard_normal((6, 8, 64)), "f32")[1]
    clean = r.attend(0, "f32", q)
    q[2, 3, 7] = spoil
    got = r.attend(0, "f32", q)
    assert np.isnan(got[2, 3]).all()
    got[2, 3] = clean[2, 3]
    assert (got == clean).all()


def test_results_in_place_of_queries(rig, ctx):
    r = rig(dim=64, heads=8, kv_heads=2, pages=100, seqs=10)
    g = np.random.default_rng(10)
    r.kv.share_prefixes(64)
    _, seqs = family(r, g, "bf16", 300, 6, [1] * 6)
    stranger = r.create()
    order = seqs[:3] + [stranger] + seqs[3:]
    r.step(g, "bf16", order, [1] * 7)
    raw, x = encode(g.standard_normal((7, 8, 64)), "bf16")
    want = r.attend(0, "bf16", x)
    b = r.put(raw.reshape(-1))
    r.kv.attention_device(0, "bf16", 7, b.address, b.address)
    assert (decode(b.download(raw.dtype, raw.size), "bf16").reshape(want.shape) == want).all()


@pytest.mark.parametrize("dtype,ntok", [("f32", [1] * 6), ("bf16", [1, 3, 1, 40, 1, 1]), ("f16", [20, 20, 1, 1, 0, 2])])
def test_captured_steps_that_share_more_and_less(rig, ctx, dtype, ntok):
    """Captured once, replayed for steps of other forks, of none, and of several prompts."""
    r = rig(dim=64, heads=16, kv_heads=2, pages=500, seqs=20, max_len=8000)
    g = np.random.default_rng(11)
    r.kv.reserve(8000)
    r.kv.share_prefixes(64)
    total = sum(ntok)
    q, out = ctx.malloc(total * 16 * 64 * 4), ctx.malloc(total * 16 * 64 * 4)

    def members(turn):
        if turn == 1:  # nothing in common
            seqs = [r.create() for _ in ntok]
            r.step(g, dtype, seqs, [30 * i for i in range(len(ntok))])
            return seqs, []
        prompts = {0: [400], 2: [3000], 3: [200, 900]}[turn]
        roots, seqs = [], []
        for p in prompts:
            a, got = family(r, g, dtype, p, len(ntok) // len(prompts), [5 * i for i in range(len(ntok) // len(prompts))])
            roots.append(a)
            seqs += got
        return seqs, roots

    graph = None
    for turn in (0, 1, 2, 3, 0):
        seqs, roots = members(turn)
        r.step(g, dtype, seqs, ntok)
        raw, x = encode(g.standard_normal((total, 16, 64)).astype(np.float32), dtype)
        q.upload(raw.reshape(-1))
        call = lambda: r.kv.attention_device(0, dtype, total, q.address, out.address)  # noqa: E731
        call()
        eager = out.download(raw.dtype, raw.size)
        graph = graph or ctx.capture(call)
        for _ in range(2):
            out.upload(np.full(raw.size, 9, raw.dtype))
            graph.launch()
            got = out.download(raw.dtype, raw.size)
            assert (got == eager).all()
            got = decode(got, dtype).reshape(total, 16, 64)
            at = 0
            for s, m in zip(seqs, ntok):
                if m:
                    want, mag, prod, tot, vtop = r.model.attend(s, 0, x[at:at + m], 0.125)
                    assert (np.abs(got[at:at + m] - want) <= attention_bound(dtype, mag, prod, tot, vtop, 64)).all(), (turn, s)
                at += m
        for s in seqs + roots:
            r.free(s)
    seqs, _ = members(0)
    r.kv.share_prefixes(128)
    r.step(g, dtype, seqs, ntok)
    with pytest.raises(ValueError, match="changed"):
        graph.launch()
    graph.close()
    with pytest.raises(ValueError, match="captured"):
        ctx.capture(lambda: r.kv.share_prefixes(0)).close()
    q.free()
    out.free()


def test_what_lies_behind_a_sequence_does_not_matter(rig):
    """Values and scales of former pages, huge ones, beside short tails."""
    r = rig(dim=64, heads=4, kv_heads=1, pages=20, seqs=6)
    g = np.random.default_rng(12)
    a = r.create()
    r.step(g, "f32", [a], [64 * 20], std=1e30)
    r.free(a)
    r.kv.share_prefixes(64)
    _, seqs = family(r, g, "f32", 130, 4, [0, 1, 2, 3])
    r.step(g, "f32", seqs, [1] * 4)
    r.check_attention(g, 0, "f32", seqs, [1] * 4)


def test_a_serving_step_through_norm_products_cache_and_rules(rig, ctx):
    """One decode step of a batch behind a shared prompt, as it is put together: the norm hands
    8 bits to the projections, whose heads are turned, stored and attended with, and a norm hands
    the results to the vocabulary, under rules.  Every link is held to its own inputs."""
    from test_gpu_step_ops import Bufs, logits_model, norm_model, q4_bound, q4_model, q4_weights, same_bits
    heads, kv_heads, dim, hidden, vocab = 8, 2, 64, 512, 1001
    r = rig(dim=dim, heads=heads, kv_heads=kv_heads, pages=100, seqs=10)
    b = Bufs(ctx)
    g = np.random.default_rng(13)
    r.kv.share_prefixes(64)
    _, seqs = family(r, g, "bf16", 200, 5, [1, 2, 3, 70, 0])
    n = len(seqs)
    made = {}
    for name, rows, cols in (("q", heads * dim, hidden), ("k", kv_heads * dim, hidden), ("v", kv_heads * dim, hidden), ("o", hidden, heads * dim),
                             ("head", vocab, hidden)):
        w = q4_weights(g, rows, cols, 64, True, "f16")
        made[name] = (H.GroupQ4Matrix.new(ctx, rows, cols, 64, w[0], w[1], w[3]), w)
    w1 = np.exp(0.1 * g.standard_normal(hidden)).astype(np.float32)
    x = encode(g.standard_normal((n, hidden)), "bf16")[1]
    zero = lambda *shape: b.put(np.zeros(shape, np.uint16))  # noqa: E731
    dx, dw = b.put(encode(x, "bf16")[0]), b.put(w1)
    codes, scales = b.put(np.zeros((n, hidden), np.int8)), b.put(np.zeros((n, hidden // 32), np.float32))
    dq, dk, dv, do, dh = zero(n, heads * dim), zero(n, kv_heads * dim), zero(n, kv_heads * dim), zero(n, heads * dim), zero(n, hidden)
    dsum, dl = zero(n, hidden), b.put(np.zeros((n, vocab), np.float32))
    r.kv.step(seqs, [1] * n)
    H.rms_norm_q8_device(ctx, "bf16", n, hidden, dx, dw, 1e-6, codes, scales)
    for name, d in (("q", dq), ("k", dk), ("v", dv)):
        made[name][0].matmul_q8_device("bf16", n, codes, scales, d)
    rope = H.Rope(ctx, dim, 10000.0)
    rope.apply_device("bf16", n, r.kv.positions, dq, heads, dq, dk, kv_heads, dk)
    r.kv.append_device(0, "bf16", n, dk, dv)
    r.kv.attention_device(0, "bf16", n, dq, do)
    made["o"][0].matmul_device("bf16", n, do, dh)
    got = {k: decode(b.get(d, np.uint16, n * w), "bf16").reshape(n, w)
           for k, d, w in (("q", dq, heads * dim), ("k", dk, kv_heads * dim), ("v", dv, kv_heads * dim), ("o", do, heads * dim), ("h", dh, hidden))}
    _, _, want_codes, _ = norm_model(x, None, w1, 1e-6, 32, "bf16")
    assert (b.get(codes, np.int8, n * hidden).reshape(n, hidden) == want_codes).all()
    # the projection of the values, which nothing turned
    xs = want_codes * np.repeat(b.get(scales, np.float32, n * hidden // 32).reshape(n, -1).astype(np.float64), 32, 1)
    _, _, s, z = made["v"][1]
    want, mag = q4_model(made["v"][1][0], s, z, 64, xs)
    assert (np.abs(got["v"] - want) <= q4_bound("bf16", want, mag, hidden, 64)).all()
    for i, seq in enumerate(seqs):
        r.model.append(seq, 0, got["k"][i].reshape(1, kv_heads, dim), got["v"][i].reshape(1, kv_heads, dim))
        want, mag, prod, total, vtop = r.model.attend(seq, 0, got["q"][i].reshape(1, heads, dim), dim ** -0.5)
        assert (np.abs(got["o"][i].reshape(1, heads, dim) - want) <= attention_bound("bf16", mag, prod, total, vtop, dim)).all()
    want, mag = q4_model(made["o"][1][0], made["o"][1][2], made["o"][1][3], 64, got["o"])
    assert (np.abs(got["h"] - want) <= q4_bound("bf16", want, mag, heads * dim, 64)).all()
    # the residual's addition, the second norm and the vocabulary, in the first one's buffers
    H.rms_norm_q8_device(ctx, "bf16", n, hidden, dx, dw, 1e-6, codes, scales, d_delta=dh, d_sum=dsum)
    made["head"][0].matmul_q8_device("f32", n, codes, scales, dl)
    raw = b.get(dl, np.float32, n * vocab).reshape(n, vocab)
    total = decode(encode(x + got["h"], "bf16")[0], "bf16")
    assert (decode(b.get(dsum, np.uint16, n * hidden), "bf16").reshape(n, hidden) == total).all()
    rules = dict(tokens=[[5, 6, 5, i] for i in range(n)], prompt=[1] * n, repetition=[1.2] * n, frequency=[0.5] * n, presence=[0.25] * n,
                 bias=[[(9, 2.0)]] * n, mask=[None] * n)
    R = H.LogitsRules(tokens=b.put(np.array(rules["tokens"], np.int32)), token_start=b.put(np.arange(0, 4 * n + 1, 4, dtype=np.int64)),
                      ntokens=4 * n, prompt_len=b.put(np.ones(n, np.int64)), repetition=b.put(np.full(n, 1.2, np.float32)),
                      frequency=b.put(np.full(n, 0.5, np.float32)), presence=b.put(np.full(n, 0.25, np.float32)),
                      bias_tokens=b.put(np.full(n, 9, np.int32)), bias=b.put(np.full(n, 2, np.float32)),
                      bias_start=b.put(np.arange(n + 1, dtype=np.int64)), nbiases=n)
    H.logits_device(ctx, "f32", n, vocab, dl, R, dl)
    assert same_bits(b.get(dl, np.float32, n * vocab).reshape(n, vocab), logits_model(raw, "f32", rules), "f32")
    ctx.synchronize()
    rope.close()
    for m, _ in made.values():
        m.close()
    for buf in b.all:
        buf.free()


def test_sharing_of_a_closed_cache_is_refused():
    assert H.lib().hale_kv_share_prefixes(None, 64) == H.EINVAL
