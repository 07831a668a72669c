"""The paged 8-bit key/value cache on the GPU (hale_kv_*): what is stored
against the documented codes, bit for bit; attention against 64 bits, within
what its roundings add up to; pages forked, copied, cut, freed and moved; all
of it together, as a serving loop has it."""
import numpy as np
import pytest

import hale_moe as H
from kv_model import EPS, NP, Model, attention_bound, decode, encode

pytestmark = pytest.mark.gpu


class Rig:
    """A cache beside its model."""

    def __init__(self, ctx, layers=1, heads=4, kv_heads=2, dim=64, pages=64, seqs=8, max_len=4096):
        self.ctx, self.layers, self.shape = ctx, layers, (heads, kv_heads, dim)
        self.kv = H.KvCache(ctx, layers, heads, kv_heads, dim, pages, seqs, max_len)
        self.model = Model(layers, heads, kv_heads, dim)
        self.bufs = []

    def put(self, raw, pad_bytes=0):
        b = self.ctx.malloc(max(raw.nbytes, 16) + pad_bytes)
        b.upload(raw)
        self.bufs.append(b)
        return b

    def create(self):
        s = self.kv.seq_create()
        self.model.create(s)
        return s

    def fork(self, s, n):
        got = self.kv.seq_fork(s, n)
        for f in got:
            self.model.fork(s, f)
        return got

    def copy(self, s):
        c = self.kv.seq_copy(s)
        self.model.fork(s, c)
        return c

    def truncate(self, s, n):
        self.kv.seq_truncate(s, n)
        self.model.truncate(s, n)

    def free(self, s):
        self.kv.seq_free(s)
        del self.model.seqs[s]

    def strided(self, x, dtype, pad, offset):
        """Rows of x [n][heads][dim] with `pad` numbers between, from number `offset` on."""
        n = x.shape[0]
        row = x.shape[1] * x.shape[2]
        raw = np.zeros(offset + n * (row + pad), NP[dtype])
        raw[offset:].reshape(n, row + pad)[:, :row] = encode(x, dtype)[0].reshape(n, row)
        b = self.put(raw)
        return b.address + offset * raw.itemsize, row + pad

    def append(self, layer, dtype, seqs, ntok, k, v, pad=0, offset=0):
        n = int(sum(ntok))
        (dk, sk), (dv, sv) = (self.strided(x, dtype, pad, offset) for x in (k, v))
        self.kv.append_device(layer, dtype, n, dk, dv, k_stride=sk, v_stride=sv)
        at = 0
        for s, m in zip(seqs, ntok):
            self.model.append(s, layer, *(encode(x[at:at + m], dtype)[1] for x in (k, v)))
            at += m

    def step(self, g, dtype, seqs, ntok, std=1.0, pad=0, offset=0):
        """A step whose tokens' keys and values are random, stored in all layers."""
        self.kv.step(seqs, ntok)
        n = int(sum(ntok))
        for layer in range(self.layers):
            k, v = (g.standard_normal((n, *self.shape[1:])) * std * np.exp(0.7 * g.standard_normal((n, 1, 1))) for _ in range(2))
            self.append(layer, dtype, seqs, ntok, k, v, pad, offset)

    def attend(self, layer, dtype, q, scale=None, window=0, pad=0, offset=0):
        n, heads, dim = q.shape
        dq, sq = self.strided(q, dtype, pad, offset)
        row = heads * dim
        out = np.full(offset + n * (row + pad), 7, NP[dtype])
        b = self.put(out)
        self.kv.attention_device(layer, dtype, n, dq, b.address + offset * out.itemsize, scale=scale, window=window,
                                 q_stride=sq, out_stride=row + pad)
        back = b.download(out.dtype, out.size)
        rows = back[offset:].reshape(n, row + pad)
        assert (back[:offset] == 7).all() and (rows[:, row:] == 7).all()  # nothing outside the rows is written
        return decode(np.ascontiguousarray(rows[:, :row]), dtype).reshape(n, heads, dim)

    def check_attention(self, g, layer, dtype, seqs, ntok, window=0, pad=0, offset=0, scale=None, std=1.0):
        heads, _, dim = self.shape
        q = encode(g.standard_normal((int(sum(ntok)), heads, dim)) * std, dtype)[1]
        got = self.attend(layer, dtype, q, scale, window, pad, offset)
        at = 0
        for s, m in zip(seqs, ntok):
            if m:
                want, mag, prod, total, vtop = self.model.attend(s, layer, q[at:at + m], dim ** -0.5 if scale is None else scale, window)
                err = np.abs(got[at:at + m] - want)
                bound = attention_bound(dtype, mag, prod, total, vtop, dim)
                assert np.isfinite(got[at:at + m]).all()
                assert (err <= bound).all(), (s, float((err - bound).max()))
                # a typical error is far below: roundings are of random sign
                typical = 8 * (EPS[dtype] + (2.0 ** -22 if dtype == "f32" else 2.0 ** -11)) * np.sqrt((mag ** 2).mean())
                assert np.sqrt((err ** 2).mean()) <= typical + prod.max() * 2.0 ** -21 * np.sqrt((mag ** 2).mean())
            at += m
        return got

    def check_contents(self):
        for s, layers in self.model.seqs.items():
            n = len(layers[0][0].codes)
            assert self.kv.seq_len(s) == n
            if not n:
                continue
            for layer, (k, v) in enumerate(layers):
                gk, gv = self.kv.read(layer, s, 0, n)
                assert (gk == k.values()).all() and (gv == v.values()).all(), (s, layer)

    def close(self):
        self.kv.close()
        for b in self.bufs:
            b.free()


@pytest.fixture
def rig(ctx):
    made = []

    def make(**kw):
        made.append(Rig(ctx, **kw))
        return made[-1]

    yield make
    for r in made:
        r.close()


# ---- storing -------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 96, 112, 128, 176, 192, 208, 256])
def test_stored_codes_bit_exact(rig, dtype, dim):
    r = rig(dim=dim, heads=3, kv_heads=3, pages=20)
    g = np.random.default_rng(dim)
    a, b = r.create(), r.create()
    for ntok in ([1, 0], [14, 1], [1, 15], [1, 17], [47, 64], [0, 31], [130, 3], [3, 200]):
        r.step(g, dtype, [a, b], ntok, std=10.0 ** g.integers(-3, 3), pad=int(g.integers(0, 4)), offset=int(g.integers(0, 3)))
        r.check_contents()


def test_stored_edges(rig):
    """Zeros, ties, the smallest and largest numbers, what is not finite, a
    block whose scale grows many times, one that is cut and filled again."""
    r = rig(dim=16, heads=1, kv_heads=1, pages=8)
    s = r.create()

    def store(rows):
        x = np.zeros((len(rows), 1, 16), np.float32)
        for i, row in enumerate(rows):
            x[i, 0, :len(row)] = row
        r.kv.step([s], [len(rows)])
        r.append(0, "f32", [s], [len(rows)], x, -x)
        r.check_contents()

    store([[0.0]])
    store([[1e-45, -1e-45], [1e-40, 3e-41]])
    store([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, 126.5, -126.5]])  # scale 1: ties to even
    store([[np.nan, 1.0, -1.0]])
    store([[np.inf, -np.inf, 200.0, -3.0]])
    store([[254.0, 1.0, 3.0, 5.0]])
    store([[3e38, -3.4e38]])
    r.truncate(s, 3)
    store([[1.0, 2.0]])  # keeps the block's large scale
    r.truncate(s, 0)
    store([[1.0, 2.0, -127.0]])
    for k in range(20):
        store([[1.3 ** k, -(1.1 ** k), 0.3]])
    store([[0.1 * i + j for j in range(16)] for i in range(50)])


def test_store_scale_is_a_rounded_quotient(rig):
    # max / 127 with every kind of remainder, codes whose quotients lie next to halves
    r = rig(dim=64, heads=1, kv_heads=1, pages=40)
    s = r.create()
    g = np.random.default_rng(1)
    x = (g.integers(1, 1 << 24, (2048, 1, 64)) * 2.0 ** g.integers(-30, 10, (2048, 1, 1))).astype(np.float32)
    r.kv.step([s], [2048])
    r.append(0, "f32", [s], [2048], x, x[::-1].copy())
    r.check_contents()


# ---- attention -----------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [16, 32, 64, 80, 96, 112, 128, 160, 192, 224, 256])
def test_attention_head_dims(rig, dtype, dim):
    r = rig(dim=dim, heads=6, kv_heads=2, pages=40)
    g = np.random.default_rng(dim + 1)
    seqs = [r.create() for _ in range(3)]
    r.step(g, dtype, seqs, [1, 63, 200])
    r.check_attention(g, 0, dtype, seqs, [1, 63, 200])
    r.step(g, dtype, seqs, [1, 1, 1])
    r.check_attention(g, 0, dtype, seqs, [1, 1, 1])
    r.step(g, dtype, seqs, [0, 2, 9])
    r.check_attention(g, 0, dtype, seqs, [0, 2, 9], pad=3, offset=1)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (7, 7), (16, 1), (17, 1), (33, 1), (64, 2), (40, 8), (12, 4), (150, 1)])
def test_attention_head_groups(rig, heads, kv_heads):
    r = rig(dim=64, heads=heads, kv_heads=kv_heads, pages=40)
    g = np.random.default_rng(heads)
    seqs = [r.create() for _ in range(2)]
    for ntok in ([5, 70], [1, 1], [3, 0], [20, 1]):
        r.step(g, "bf16", seqs, ntok)
        r.check_attention(g, 0, "bf16", seqs, ntok)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 320, 511, 1000])
def test_attention_lengths(rig, n):
    # both sides of a block, a page, a work-group's four pages
    r = rig(dim=64, heads=4, kv_heads=2, pages=40)
    g = np.random.default_rng(n)
    a = r.create()
    if n > 1:
        r.step(g, "f32", [a], [n - 1])
    r.step(g, "f32", [a], [1])
    r.check_attention(g, 0, "f32", [a], [1])


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 200, 4095, 4096, 100000])
def test_attention_windows(rig, window):
    r = rig(dim=64, heads=4, kv_heads=2, pages=60)
    g = np.random.default_rng(window)
    seqs = [r.create() for _ in range(3)]
    r.step(g, "f16", seqs, [10, 300, 700])
    r.check_attention(g, 0, "f16", seqs, [10, 300, 700], window=window)
    r.step(g, "f16", seqs, [1, 1, 1])
    r.check_attention(g, 0, "f16", seqs, [1, 1, 1], window=window)
    r.check_attention(g, 0, "f16", seqs, [1, 1, 1])  # another window of the same step
    r.step(g, "f16", seqs, [6, 5, 0])
    r.check_attention(g, 0, "f16", seqs, [6, 5, 0], window=window)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_long_context_split(rig, dtype):
    # one sequence long enough that its pages go over many work-groups
    r = rig(dim=128, heads=8, kv_heads=1, pages=520, max_len=40000)
    g = np.random.default_rng(2)
    a = r.create()
    r.step(g, dtype, [a], [33000])
    for k in (1, 3, 9):
        r.step(g, dtype, [a], [k])
        r.check_attention(g, 0, dtype, [a], [k])
        r.check_attention(g, 0, dtype, [a], [k], window=9000)


def test_attention_scores_far_apart(rig):
    """Scores of hundreds, of both signs: one key takes all, or the first
    page's maximum is far below a later one's."""
    r = rig(dim=64, heads=2, kv_heads=1, pages=40)
    g = np.random.default_rng(4)
    a = r.create()
    r.kv.step([a], [500])
    k = g.standard_normal((500, 1, 64))
    k[:100] *= 30.0
    k[400:] *= np.linspace(1, 40, 100)[:, None, None]
    r.append(0, "f32", [a], [500], k, g.standard_normal((500, 1, 64)))
    r.check_attention(g, 0, "f32", [a], [500], std=3.0)
    r.check_attention(g, 0, "f32", [a], [500], scale=3.0)
    r.check_attention(g, 0, "f32", [a], [500], scale=1e-3)


def test_attention_zero_and_huge_scales(rig):
    """Blocks of zeros, values of very different magnitude from block to block
    (the accumulators follow the largest scale so far), zero queries."""
    r = rig(dim=64, heads=2, kv_heads=1, pages=40)
    g = np.random.default_rng(6)
    a = r.create()
    n = 400
    k, v = g.standard_normal((n, 1, 64)), g.standard_normal((n, 1, 64))
    k[:16] = 0
    v[:64] = 0
    v[64:80] *= 1e-30
    v[150:] *= 1e25
    r.kv.step([a], [n])
    r.append(0, "f32", [a], [n], k, v)
    r.check_attention(g, 0, "f32", [a], [n])
    r.check_attention(g, 0, "bf16", [a], [n])
    q = np.zeros((n, 2, 64), np.float32)
    got = r.attend(0, "f32", q)
    want, mag, prod, total, vtop = r.model.attend(a, 0, q, 0.125)
    assert (np.abs(got - want) <= attention_bound("f32", mag, prod, total, vtop, 64)).all()
    r.step(g, "f32", [a], [3])  # few rows
    r.check_attention(g, 0, "f32", [a], [3])
    r.check_attention(g, 0, "bf16", [a], [3])


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [5, 60])
def test_a_query_that_is_not_finite_spoils_only_its_row(rig, dtype, n):
    r = rig(dim=64, heads=4, kv_heads=2, pages=40)
    g = np.random.default_rng(7)
    a = r.create()
    r.step(g, dtype, [a], [70])
    r.step(g, dtype, [a], [n])
    q = g.standard_normal((n, 4, 64)).astype(np.float32)
    clean = r.attend(0, dtype, q)
    q[2, 1, 3], q[4, 0, 0], q[n - 1, 3, 63] = np.nan, np.inf, -np.inf
    got = r.attend(0, dtype, q)
    hit = np.zeros((n, 4), bool)
    hit[2, 1] = hit[4, 0] = hit[n - 1, 3] = True
    assert (got[~hit].view(np.uint32) == clean[~hit].view(np.uint32)).all()
    assert np.isnan(got[hit]).all()


@pytest.mark.parametrize("n", [1, 50])
def test_results_in_place_of_queries(rig, n):
    r = rig(dim=64, heads=4, kv_heads=2, pages=40)
    g = np.random.default_rng(8)
    a = r.create()
    r.step(g, "bf16", [a], [900])
    r.step(g, "bf16", [a], [n])
    q = g.standard_normal((n, 4, 64)).astype(np.float32)
    want = r.attend(0, "bf16", q)
    raw = encode(q, "bf16")[0].reshape(-1)
    b = r.put(raw)
    r.kv.attention_device(0, "bf16", n, b.address, b.address)
    assert (decode(b.download(np.uint16, raw.size), "bf16").reshape(q.shape) == want).all()


def test_later_tokens_of_any_size_do_not_reach_earlier_rows(rig):
    """Keys and values behind a row's position, 10^20 times as large as those
    before, in its page and its tile: its result is that of the tokens it sees."""
    r = rig(dim=64, heads=2, kv_heads=1, pages=40)
    g = np.random.default_rng(9)
    for start in (16, 64, 80):  # blocks of their own
        a, n = r.create(), start + 40
        k, v = g.standard_normal((n, 1, 64)), g.standard_normal((n, 1, 64))
        k[start:] *= 1e10
        v[start:] *= 1e20
        r.kv.step([a], [n])
        r.append(0, "f32", [a], [n], k, v)
        q = g.standard_normal((n, 2, 64)).astype(np.float32)
        for dtype in ("f32", "bf16"):
            qd = encode(q, dtype)[1]
            got = r.attend(0, dtype, qd)[:start]
            want, mag, prod, total, vtop = r.model.attend(a, 0, qd, 0.125)
            bound = attention_bound(dtype, mag[:start], prod[:start], total, vtop[:start], 64)
            assert vtop[:start].max() < 1e3 and (np.abs(got - want[:start]) <= bound).all(), (start, dtype)
        r.free(a)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("nseq, ntok, dim, window", [
    (1, 5, 64, 0), (1, 8, 128, 0), (2, 7, 96, 150), (3, 8, 80, 0),  # 33..64 rows, few tiles
    (9, 3, 64, 0), (9, 4, 96, 200), (9, 8, 64, 0), (8, 5, 128, 70),  # and many
    (2, 8, 160, 0), (1, 3, 256, 90)])
def test_rows_between_few_and_many(rig, dtype, nseq, ntok, dim, window):
    r = rig(dim=dim, heads=32, kv_heads=4, pages=200, seqs=12)
    g = np.random.default_rng(11)
    seqs = [r.create() for _ in range(nseq)]
    r.step(g, dtype, seqs, [int(n) for n in g.integers(1, 700, nseq)])
    r.step(g, dtype, seqs, [ntok] * nseq)
    r.check_attention(g, 0, dtype, seqs, [ntok] * nseq, window=window)


@pytest.mark.parametrize("first, second", [("f32", "bf16"), ("f16", "f32")])
def test_types_in_turn_on_one_cache(rig, first, second):
    """Both types' plans of one step, kept over the next; four windows each."""
    r = rig(dim=64, heads=32, kv_heads=4, pages=200, seqs=12)
    g = np.random.default_rng(12)
    seqs = [r.create() for _ in range(9)]
    for ntok in (100, 3, 4):
        r.step(g, first, seqs, [ntok] * 9)
        for window in (0, 33, 65, 120):
            for dtype in (first, second):
                r.check_attention(g, 0, dtype, seqs, [ntok] * 9, window=window)
    b = r.ctx.malloc(36 * 32 * 64 * 4)
    for dtype in (first, second):
        with pytest.raises(ValueError, match="fifth"):
            r.kv.attention_device(0, dtype, 36, b.address, b.address, window=7)
    b.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_captured_join_meets_any_number_of_parts(rig, ctx, dtype):
    """Captured with sequences of few parts, replayed on others of many, and the other
    way round: one of the two joins is fixed by the capture, its parts are not."""
    for lens in ((300, 7000, 300), (7000, 300, 7000)):
        r = rig(dim=64, heads=8, kv_heads=1, pages=260, max_len=8000)
        g = np.random.default_rng(13)
        r.kv.reserve(8000)
        q = ctx.malloc(8 * 64 * 4)
        out = ctx.malloc(8 * 64 * 4)
        graph = None
        for n in lens:
            a = r.create()
            r.step(g, dtype, [a], [n])
            r.step(g, dtype, [a], [1])
            raw, x = encode(g.standard_normal((1, 8, 64)).astype(np.float32), dtype)
            q.upload(raw.reshape(-1))
            r.kv.attention_device(0, dtype, 1, q.address, out.address)
            eager = out.download(raw.dtype, raw.size).copy()
            if graph is None:
                graph = ctx.capture(lambda: r.kv.attention_device(0, dtype, 1, q.address, out.address))
            for _ in range(2):
                graph.launch()
                got = decode(out.download(raw.dtype, raw.size), dtype).reshape(1, 8, 64)
                want, mag, prod, total, vtop = r.model.attend(a, 0, x, 0.125)
                assert (np.abs(got - want) <= attention_bound(dtype, mag, prod, total, vtop, 64)).all(), (n, lens)
            assert np.isfinite(decode(eager, dtype)).all()
            r.free(a)
        graph.close()
        q.free()
        out.free()


@pytest.mark.parametrize("ntok", [1, 40])
def test_pages_past_4_gib(rig, ntok):
    """Pages of 8.5 MB, the sequence's all behind byte 2^32 of the pool."""
    r = rig(layers=64, dim=128, heads=8, kv_heads=8, pages=560, seqs=3, max_len=40000)
    page = 64 * 8 * (64 * 128 * 2 + 128)
    g = np.random.default_rng(14)
    a, b = r.create(), r.create()
    r.kv.step([a], [64 * 515])  # takes the lower pages, stores nothing
    assert 515 * page > 1 << 32
    n = 200
    r.kv.step([b], [n])
    for layer in (0, 63):
        k, v = (g.standard_normal((n, 8, 128)) for _ in range(2))
        r.append(layer, "bf16", [b], [n], k, v)
    r.kv.step([b], [ntok])
    for layer in (0, 63):
        k, v = (g.standard_normal((ntok, 8, 128)) for _ in range(2))
        r.append(layer, "bf16", [b], [ntok], k, v)
        r.check_attention(g, layer, "bf16", [b], [ntok])
    c = r.copy(b)
    r.kv.step([c], [ntok])
    for layer in (0, 63):
        k, v = (g.standard_normal((ntok, 8, 128)) for _ in range(2))
        r.append(layer, "bf16", [c], [ntok], k, v)
        r.check_attention(g, layer, "bf16", [c], [ntok])


def test_a_pool_past_64_bits_is_refused(ctx):
    # 2^39 and a little bytes a page, 2^25 pages: the product wraps to little
    with pytest.raises(MemoryError, match="pages of"):
        H.KvCache(ctx, 4096, 4096, 4096, 256, 1 << 25, 1, 64)


@pytest.mark.parametrize("dtype, ntok", [("bf16", [1, 40, 8]), ("f32", [3, 3, 3]), ("f16", [2] * 9), ("bf16", [3] * 9)])
def test_captured_steps_of_every_kind_of_row(rig, ctx, dtype, ntok):
    """Captured once, replayed over longer sequences, others beside them, twice each."""
    r = rig(dim=64, heads=16, kv_heads=2, pages=260, seqs=12, max_len=8000)
    g = np.random.default_rng(15)
    r.kv.reserve(20000)
    seqs, total = [r.create() for _ in ntok], sum(ntok)
    q, out = ctx.malloc(total * 16 * 64 * 4), ctx.malloc(total * 16 * 64 * 4)
    graph = None
    for grow in (5, 700, 60):
        r.step(g, dtype, seqs, [grow + 3 * i for i in range(len(seqs))])
        r.step(g, dtype, seqs, ntok)
        raw, x = encode(g.standard_normal((total, 16, 64)).astype(np.float32), dtype)
        q.upload(raw.reshape(-1))
        call = lambda: r.kv.attention_device(0, dtype, total, q.address, out.address, window=300)
        call()
        graph = graph or ctx.capture(call)
        for _ in range(2):
            out.upload(np.full(raw.size, 9, raw.dtype))
            graph.launch()
            got = decode(out.download(raw.dtype, raw.size), dtype).reshape(total, 16, 64)
            at = 0
            for s, m in zip(seqs, ntok):
                want, mag, prod, tot, vtop = r.model.attend(s, 0, x[at:at + m], 0.125, 300)
                assert (np.abs(got[at:at + m] - want) <= attention_bound(dtype, mag, prod, tot, vtop, 64)).all(), (grow, s)
                at += m
    graph.close()
    q.free()
    out.free()


@pytest.mark.parametrize("scale", [2.0 ** 127, 3e38, float("inf"), -1.0])
def test_scales_out_of_range_are_refused(rig, ctx, scale):
    r = rig(dim=64, pages=4)
    a = r.create()
    r.kv.step([a], [1])
    x = np.zeros((1, 2, 64), np.float32)
    r.append(0, "f32", [a], [1], x, x)
    b = ctx.malloc(1 << 12)
    with pytest.raises(ValueError, match="below 2\\^127"):
        r.kv.attention_device(0, "f32", 1, b.address, b.address, scale=scale)
    b.free()


def test_what_lies_behind_a_sequence_does_not_matter(rig):
    """Pages that held other sequences' tokens, and tokens that were cut."""
    r = rig(dim=64, heads=4, kv_heads=2, pages=6)
    g = np.random.default_rng(9)
    a = r.create()
    r.step(g, "f32", [a], [384], std=1e30)
    r.free(a)
    b = r.create()
    r.step(g, "f32", [b], [70])
    r.check_attention(g, 0, "f32", [b], [70])
    r.step(g, "f32", [b], [9], std=1e20)
    r.truncate(b, 64)
    r.step(g, "f32", [b], [3])
    r.check_attention(g, 0, "f32", [b], [3])


def test_equal_calls_give_equal_bits(rig):
    r = rig(dim=128, heads=8, kv_heads=2, pages=300, max_len=20000)
    g = np.random.default_rng(10)
    seqs = [r.create() for _ in range(3)]
    r.step(g, "bf16", seqs, [9000, 100, 3000])
    r.step(g, "bf16", seqs, [2, 2, 2])
    q = encode(g.standard_normal((6, 8, 128)), "bf16")[1]
    first = r.attend(0, "bf16", q)
    for _ in range(3):
        assert (r.attend(0, "bf16", q) == first).all()


# ---- pages -------------------------------------------------------------------------

def test_forks_share_until_they_store(rig):
    r = rig(layers=2, dim=64, pages=12, seqs=8)
    g = np.random.default_rng(11)
    a = r.create()
    r.step(g, "f32", [a], [100])
    assert r.kv.pages() == (12, 2)
    f = r.fork(a, 3)
    assert r.kv.pages()[1] == 2
    r.step(g, "f32", [f[0], f[1]], [1, 30])
    assert r.kv.pages()[1] == 5  # a copy of the second page each, and one page more
    r.check_contents()
    r.check_attention(g, 1, "f32", [f[0], f[1]], [1, 30])
    r.step(g, "f32", [a, *f], [1, 1, 1, 1])
    r.check_contents()
    r.check_attention(g, 0, "f32", [a, *f], [1, 1, 1, 1])
    for s in (a, *f):
        r.free(s)
    assert r.kv.pages()[1] == 0


def test_copy_compact_resize(rig):
    r = rig(layers=2, dim=80, pages=20, seqs=8)
    g = np.random.default_rng(12)
    seqs = [r.create() for _ in range(4)]
    r.step(g, "bf16", seqs, [70, 200, 10, 129])
    c = r.copy(seqs[1])
    r.check_contents()
    r.free(seqs[1])
    r.free(seqs[2])
    assert r.kv.pages() == (20, 9)
    assert r.kv.compact() > 0
    assert r.kv.compact() == 0
    r.check_contents()
    live = [seqs[0], seqs[3], c]
    r.kv.resize(10)
    assert r.kv.pages() == (10, 9)
    r.check_contents()
    with pytest.raises(MemoryError, match="pages"):
        r.kv.step(live, [200, 200, 200])
    r.check_contents()
    r.kv.resize(30)
    r.step(g, "bf16", live, [200, 1, 33])
    r.check_contents()
    r.check_attention(g, 1, "bf16", live, [200, 1, 33])
    with pytest.raises(ValueError, match="in use"):
        r.kv.resize(3)


@pytest.mark.parametrize("seed", range(6))
def test_a_serving_loop(rig, seed):
    """Random steps, forks, copies, cuts, frees and compactions over two
    layers, every attention and at the end all contents checked."""
    g = np.random.default_rng(100 + seed)
    dtype = ["f32", "f16", "bf16"][seed % 3]
    dim = [64, 80, 128][seed // 2]
    r = rig(layers=2, dim=dim, heads=6, kv_heads=2, pages=40, seqs=7, max_len=600)
    for _ in range(40):
        live = list(r.model.seqs)
        what = g.integers(0, 10)
        try:
            if not live or what == 0:
                r.create()
            elif what == 1:
                r.free(int(g.choice(live)))
            elif what == 2:
                r.fork(int(g.choice(live)), int(g.integers(1, 3)))
            elif what == 3:
                r.copy(int(g.choice(live)))
            elif what == 4:
                s = int(g.choice(live))
                r.truncate(s, int(g.integers(0, r.kv.seq_len(s) + 1)))
            elif what == 5:
                r.kv.compact()
            else:
                seqs = [s for s in live if g.random() < 0.7]
                ntok = [int(g.integers(0, 5)) if g.random() < 0.7 else int(g.integers(0, 120)) for _ in seqs]
                r.step(g, dtype, seqs, ntok)
                if sum(ntok):
                    r.check_attention(g, int(g.integers(0, 2)), dtype, seqs, ntok, window=int(g.choice([0, 0, 50])))
        except MemoryError:
            pass
        except ValueError as e:
            assert "context overflow" in str(e)
    r.check_contents()


# ---- graphs, streams, several caches ---------------------------------------------------

def test_captured_layers_replay_over_growing_sequences(rig, ctx):
    """Rotation, store and attention of two layers captured once and replayed
    over steps of other lengths and pages, with eager work between."""
    r = rig(layers=2, dim=128, heads=8, kv_heads=2, pages=60, seqs=6)
    rope = H.Rope(ctx, 128, 1e6)
    g = np.random.default_rng(20)
    seqs = [r.create() for _ in range(3)]
    r.kv.reserve(1000)
    r.step(g, "f32", seqs, [61, 5, 300])
    n, (nh, nk, hd) = 3, r.shape
    bq, bk, bv, bo = (ctx.malloc(4 * n * h * hd) for h in (nh, nk, nk, nh))
    rk, rq = ctx.malloc(4 * n * nk * hd), ctx.malloc(4 * n * nh * hd)
    outs = [ctx.malloc(4 * n * nh * hd) for _ in range(2)]

    def layers():
        for layer in range(2):
            rope.apply_device("f32", n, r.kv.positions, bq.address, nh, rq.address, bk.address, nk, rk.address)
            r.kv.append_device(layer, "f32", n, rk.address, bv.address)
            r.kv.attention_device(layer, "f32", n, rq.address, outs[layer].address, window=100 * layer)

    graph = None
    for k in range(8):
        q, kk, v = (g.standard_normal((n, h, hd)).astype(np.float32) for h in (nh, nk, nk))
        for b, x in ((bq, q), (bk, kk), (bv, v)):
            b.upload(x)
        if k == 5:
            r.kv.compact()
        r.kv.step(seqs, [1, 1, 1])
        if k == 0:
            layers()
        else:
            graph = graph or ctx.capture(layers)
            graph.launch()
        kr = rk.download(np.float32, kk.size).reshape(kk.shape)
        qr = rq.download(np.float32, q.size).reshape(q.shape)
        for layer in range(2):
            got = outs[layer].download(np.float32, q.size).reshape(q.shape)
            for i, s in enumerate(seqs):
                r.model.append(s, layer, kr[i:i + 1], v[i:i + 1])
                want, mag, prod, total, vtop = r.model.attend(s, layer, qr[i:i + 1], hd ** -0.5, 100 * layer)
                assert (np.abs(got[i:i + 1] - want) <= attention_bound("f32", mag, prod, total, vtop, hd)).all(), (k, layer, s)
        r.check_contents()
        if k == 2:  # eager work between replays: a longer step of other sequences, which the graph refuses
            extra = r.create()
            r.step(g, "f32", [extra], [700])
            r.check_attention(g, 1, "f32", [extra], [700])
            with pytest.raises(ValueError, match="step"):
                graph.launch()
        if k == 6:
            r.free(extra)
            r.step(g, "f32", [seqs[1]], [40])
    # the buffers grow: the graph is refused from then on
    big = r.create()
    r.step(g, "f32", [big], [1200])
    r.kv.step(seqs, [1, 1, 1])
    with pytest.raises(ValueError, match="grew"):
        graph.launch()
    graph.close()
    rope.close()
    for b in (bq, bk, bv, bo, rk, rq, *outs):
        b.free()


def test_graph_of_a_closed_cache_is_refused(rig, ctx):
    r = rig(dim=64)
    g = np.random.default_rng(21)
    a = r.create()
    r.step(g, "f32", [a], [3])
    q = ctx.malloc(4 * 3 * 4 * 64)
    r.kv.attention_device(0, "f32", 3, q.address, q.address)
    graph = ctx.capture(lambda: r.kv.attention_device(0, "f32", 3, q.address, q.address))
    with pytest.raises(ValueError, match="graphs of the context"):
        r.kv.resize(64)
    r.kv.close()
    with pytest.raises(ValueError, match="gone"):
        graph.launch()
    graph.close()
    q.free()


def test_capture_refusals(rig, ctx):
    r = rig(dim=64)
    g = np.random.default_rng(22)
    a = r.create()
    r.step(g, "f32", [a], [3])
    q = ctx.malloc(4 * 3 * 4 * 64)
    for call in (lambda: r.kv.step([a], [1]), lambda: r.kv.compact(), lambda: r.kv.seq_copy(a), lambda: r.kv.resize(99),
                 lambda: r.kv.attention_device(0, "f32", 3, q.address, q.address, window=5),
                 lambda: r.kv.read_device(0, a, 0, 1, q.address, q.address), lambda: r.kv.reserve(100000),
                 lambda: H.KvCache(ctx, 1, 1, 1, 64, 1, 1, 64), lambda: H.Rope(ctx, 64)):
        with pytest.raises(ValueError, match="captur"):
            ctx.capture(call)
    r.check_contents()
    q.free()


def test_two_caches_of_one_context(rig):
    a, b = rig(dim=64), rig(dim=128, heads=2, kv_heads=2)
    g = np.random.default_rng(23)
    sa, sb = a.create(), b.create()
    for n in (40, 1, 70):
        a.step(g, "f32", [sa], [n])
        b.step(g, "f16", [sb], [n])
        a.check_attention(g, 0, "f32", [sa], [n])
        b.check_attention(g, 0, "f16", [sb], [n])
    a.check_contents()
    b.check_contents()


def test_contexts_side_by_side(ctx):
    """Two contexts on one device, their calls interleaved without waiting."""
    other = H.Context(0)
    rigs = [Rig(c, dim=128, heads=8, kv_heads=2, pages=100) for c in (ctx, other)]
    g = np.random.default_rng(24)
    seqs = [r.create() for r in rigs]
    for n in (900, 1, 5):
        for r, s in zip(rigs, seqs):
            r.step(g, "bf16", [s], [n])
        for r, s in zip(rigs, seqs):
            r.check_attention(g, 0, "bf16", [s], [n])
    for r in rigs:
        r.check_contents()
        r.close()
    other.close()


# ---- refusals ---------------------------------------------------------------------------

def test_refusals(rig, ctx):
    for bad, why in ((dict(dim=24), "head_dim"), (dict(dim=272), "head_dim"), (dict(heads=3), "multiple"),
                     (dict(layers=0), "layers"), (dict(pages=0), "pages"), (dict(seqs=0), "max_seqs"),
                     (dict(max_len=0), "max_len"), (dict(max_len=1 << 30, seqs=65536), "page table")):
        with pytest.raises(ValueError, match=why):
            Rig(ctx, **bad)
    r = rig(dim=64, pages=4, seqs=2, max_len=200)
    kv = r.kv
    b = ctx.malloc(1 << 16)
    p = b.address
    with pytest.raises(ValueError, match="without a current step"):
        kv.append_device(0, "f32", 1, p, p)
    a, c = r.create(), r.create()
    with pytest.raises(MemoryError, match="sequences"):
        kv.seq_create()
    with pytest.raises(ValueError, match="no sequence"):
        kv.seq_free(9)
    with pytest.raises(ValueError, match="holds 0"):
        kv.seq_truncate(a, 1)
    with pytest.raises(ValueError, match="twice"):
        kv.step([a, a], [1, 1])
    with pytest.raises(ValueError, match="overflow"):
        kv.step([a], [201])
    with pytest.raises(ValueError, match="at most 2"):
        kv.step([a, c, 5], [1, 1, 1])
    with pytest.raises(MemoryError, match="pages needed"):
        kv.step([a, c], [200, 65])
    with pytest.raises(ValueError, match="counts"):
        kv.step([a, c], [1])
    kv.step([a, c], [3, 0])
    for call, why in ((lambda: kv.append_device(1, "f32", 3, p, p), "layer 1"),
                      (lambda: kv.append_device(0, "q8_0", 3, p, p), "not f32"),
                      (lambda: kv.append_device(0, "f32", 2, p, p), "the step has 3"),
                      (lambda: kv.append_device(0, "f32", 3, 0, p), "NULL"),
                      (lambda: kv.append_device(0, "f32", 3, p, p, v_stride=127), "below"),
                      (lambda: kv.append_device(0, "f32", 3, p + 2, p), "aligned"),
                      (lambda: kv.attention_device(0, "f32", 3, p, p, scale=0.0), "scale"),
                      (lambda: kv.attention_device(0, "f32", 3, p, p, scale=float("nan")), "scale"),
                      (lambda: kv.attention_device(0, "f32", 4, p, p), "the step has 3"),
                      (lambda: kv.attention_device(0, "f16", 3, p + 1, p), "aligned"),
                      (lambda: kv.attention_device(0, "f16", 3, p, p, out_stride=255), "below"),
                      (lambda: kv.read_device(0, a, 2, 2, p, p), "positions"),
                      (lambda: kv.read_device(0, a, 0, 1, 0, p), "NULL"),
                      (lambda: kv.read_device(3, a, 0, 1, p, p), "layer 3")):
        with pytest.raises(ValueError, match=why):
            call()
    x = np.zeros((3, 2, 64), np.float32)
    r.append(0, "f32", [a, c], [3, 0], x, x)
    for w in (1, 2, 3, 4):
        kv.attention_device(0, "f32", 3, p, p, window=w)
    with pytest.raises(ValueError, match="fifth"):
        kv.attention_device(0, "f32", 3, p, p, window=5)
    kv.seq_truncate(c, 0)  # in the step as well: it ends
    with pytest.raises(ValueError, match="without a current step"):
        kv.attention_device(0, "f32", 3, p, p, window=1)
    kv.step([], [])
    kv.append_device(0, "f32", 0, 0, 0)
    kv.attention_device(0, "f32", 0, 0, 0)
    b.free()
