"""Performance cases of the operators around a paged 8-bit key/value cache:
rotary positions, storing and attending, and moving the cache's pages.

The cache holds keys and values as whole numbers of -127..127 with one f32
scale per block of 16 positions, head, and keys or values, in pages of 64
positions.  A block's scale is max |x| / 127 over its values (rounded to f32),
or its former scale where that is larger; a code is x / scale rounded to the
nearest whole number, ties to even, and the codes a block already held are
rounded anew to a scale that grew.

Each case is one pass of work as a serving program has it done.  Where `own`
is false the pass is computed with elementary torch operations over a plain
paged cache; where it is true, through the library's entry points on one
context, whose stream a device-wide synchronization covers.  Head counts are
those of the repository's benchmark (32 query heads over 4 or 8 key/value
heads of 128) or generic.
"""
import ctypes as C
import math
import os
import sys

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 0, "f16": 1, "bf16": 2}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
PAGE, BLOCK = 64, 16
_CTX = None


def _library():
    """The library's Python view and the program's one context."""
    global _CTX
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "hale-token_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import hale_moe as H
    if _CTX is None:
        _CTX = H.Context(0)
    return H, _CTX


# ---- the cases -------------------------------------------------------------

def listed():
    return [
        # the queries and keys of one decoded token: the smallest call of a step
        dict(name="rope_token_f32", kind="rope", dtype="f32", rows=1, heads=32, kv_heads=4, head_dim=128, rotary=128,
             layout="half", scaling="none", far=4096),
        # a prompt's chunk at far positions, half of each head turned, interleaved pairs, long-context scaling
        dict(name="rope_prompt_bf16", kind="rope", dtype="bf16", rows=2048, heads=32, kv_heads=8, head_dim=128,
             rotary=64, layout="interleaved", scaling="parts", far=131072),
        # five drafted tokens stored behind a conversation, and read back
        dict(name="store_drafts_f32", kind="store", dtype="f32", kv_heads=4, head_dim=128, base=1003, ntok=5),
        # a prompt stored, and read back
        dict(name="store_prompt_bf16", kind="store", dtype="bf16", kv_heads=8, head_dim=128, base=0, ntok=4090),
        # one sequence's next token, at the attention length of the repository's benchmark
        dict(name="attend_1x4096_f32", kind="attend", dtype="f32", heads=32, kv_heads=4, head_dim=128, nseq=1, lo=4095,
             hi=4095, ntok=1, window=0),
        # a serving batch of conversations of very different lengths
        dict(name="attend_batch32_bf16", kind="attend", dtype="bf16", heads=32, kv_heads=8, head_dim=128, nseq=32,
             lo=200, hi=8000, ntok=1, window=0),
        # one very long context
        dict(name="attend_long_bf16", kind="attend", dtype="bf16", heads=32, kv_heads=4, head_dim=128, nseq=1,
             lo=131000, hi=131000, ntok=1, window=0),
        # drafts of a batch checked in one call, narrow heads, a sliding window
        dict(name="attend_drafts_f16", kind="attend", dtype="f16", heads=24, kv_heads=8, head_dim=80, nseq=12, lo=300,
             hi=3000, ntok=5, window=1024),
        # a long prompt's second chunk
        dict(name="attend_prompt_bf16", kind="attend", dtype="bf16", heads=32, kv_heads=4, head_dim=128, nseq=1,
             lo=4000, hi=4000, ntok=2048, window=0),
        # a decode step of a batch through four layers' rotation, store and attention, captured
        dict(name="decode_batch16_bf16", kind="decode", dtype="bf16", heads=32, kv_heads=4, head_dim=128, nseq=16,
             lo=500, hi=3000, layers=4),
        # one prompt forked eight ways, the first token of each, the forks freed
        dict(name="fork_8ways_f32", kind="fork", dtype="f32", heads=32, kv_heads=4, head_dim=128, prompt=1000, ways=8,
             layers=2),
        # a sequence copied to new pages, the old ones freed, the pool compacted
        dict(name="copy_compact_6000", kind="compact", dtype="bf16", kv_heads=4, head_dim=128, length=6000, others=3,
             layers=4),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    """One more case, of the sizes between and around the listed ones."""
    kind = rng.choice(["rope", "rope", "store", "attend", "attend", "attend", "attend", "decode", "fork", "compact"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    hd = rng.choice([64, 80, 96, 112, 128, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 8])
    if kind == "rope":
        return dict(kind=kind, dtype=dtype, rows=int(_log(rng, 1, 3000)), heads=heads, kv_heads=kv, head_dim=hd,
                    rotary=rng.choice([hd, hd, hd // 2, 32]), layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "ntk", "parts"]), far=int(_log(rng, 100, 1000000)))
    if kind == "store":
        return dict(kind=kind, dtype=dtype, kv_heads=kv, head_dim=hd, base=int(_log(rng, 1, 3000)) - 1,
                    ntok=int(_log(rng, 1, 4000)))
    if kind == "attend":
        ntok = int(_log(rng, 1, 1200))
        nseq = max(1, int(_log(rng, 1, max(1.01, min(40, 300 / ntok)))))
        hi = int(_log(rng, 16, min(60000, 600000 / nseq / max(1, ntok / 16))))
        return dict(kind=kind, dtype=dtype, heads=heads, kv_heads=kv, head_dim=hd, nseq=nseq, lo=max(0, hi // 9 - 1),
                    hi=hi, ntok=ntok, window=rng.choice([0, 0, 0, int(_log(rng, 20, 4000))]))
    if kind == "decode":
        return dict(kind=kind, dtype=dtype, heads=heads, kv_heads=kv, head_dim=hd, nseq=int(_log(rng, 1, 32)), lo=50,
                    hi=int(_log(rng, 60, 3000)), layers=rng.choice([1, 2, 4]))
    if kind == "fork":
        return dict(kind=kind, dtype=dtype, heads=heads, kv_heads=kv, head_dim=hd, prompt=int(_log(rng, 10, 3000)),
                    ways=rng.randrange(2, 12), layers=rng.choice([1, 2]))
    return dict(kind=kind, dtype=dtype, kv_heads=kv, head_dim=hd, length=int(_log(rng, 100, 6000)),
                others=rng.randrange(1, 4), layers=rng.choice([1, 2, 4]))


def _lengths(case):
    """The cached lengths of a case's sequences: from lo to hi, in no order."""
    lo, hi, n = case["lo"], case["hi"], case["nseq"]
    if n == 1:
        return [hi]
    return [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** ((0.37 + 0.6180339887 * i) % 1.0))) - 1 for i in range(n)]


# ---- inputs ----------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) % (1 << 62))
    return g


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _keys_values(g, n, case):
    """Keys [n][kv_heads][head_dim], some channels of which are larger, as
    models have them, and values, some tokens of which are larger."""
    kv, hd = case["kv_heads"], case["head_dim"]
    k = _normal(g, n, kv, hd) * torch.exp(0.5 * _normal(g, 1, kv, hd))
    v = _normal(g, n, kv, hd) * torch.exp(0.3 * _normal(g, n, kv, 1))
    t = TORCH[case["dtype"]]
    return k.to(t), v.to(t)


def _queries(g, n, case):
    return (_normal(g, n, case["heads"], case["head_dim"]) * 1.2).to(TORCH[case["dtype"]])


def _rope_inputs(case, seed):
    g = _generator(seed)
    n, t = case["rows"], TORCH[case["dtype"]]
    q = _normal(g, n, case["heads"], case["head_dim"]).to(t)
    k = _normal(g, n, case["kv_heads"], case["head_dim"]).to(t)
    first = int(torch.randint(0, max(1, case["far"] - n), (1,), device="cuda", generator=g))
    return q, k, torch.arange(first, first + n, dtype=torch.int32, device="cuda")


def _store_inputs(case, seed):
    g = _generator(seed)
    return _keys_values(g, case["base"], case), _keys_values(g, case["ntok"], case)


def _attend_inputs(case, seed):
    """Per sequence what is cached and what is new, and the queries."""
    g = _generator(seed)
    old = [_keys_values(g, n, case) for n in _lengths(case)]
    new = [_keys_values(g, case["ntok"], case) for _ in old]
    return old, new, _queries(g, case["ntok"] * len(old), case)


def _decode_inputs(case, seed):
    """Layer by layer: the sequences' cached keys (already turned) and values,
    then the new tokens' queries, keys and values."""
    g = _generator(seed)
    n = case["nseq"]
    for _ in range(case["layers"]):
        old = [_keys_values(g, m, case) for m in _lengths(case)]
        k, v = _keys_values(g, n, case)
        yield old, _queries(g, n, case), k, v


def _fork_inputs(case, seed):
    g = _generator(seed)
    for _ in range(case["layers"]):
        old = _keys_values(g, case["prompt"], case)
        k, v = _keys_values(g, case["ways"], case)
        yield old, _queries(g, case["ways"], case), k, v


def _compact_inputs(case, seed):
    """Layer by layer: the sequence that moves, then the others' contents."""
    g = _generator(seed)
    for _ in range(case["layers"]):
        yield [_keys_values(g, case["length"] + 37 * i, case) for i in range(1 + case["others"])]


# ---- rotary frequencies --------------------------------------------------------

BASE, FACTOR, ORIGINAL, LOW, HIGH = 1e6, 8.0, 8192.0, 1.0, 32.0


def _attention_factor(case):
    return 0.1 * math.log(FACTOR) + 1.0 if case["scaling"] == "parts" else 1.0


def _frequencies(case):
    """The angle per position of each pair, in 64 bits."""
    r = case["rotary"]
    i = torch.arange(r // 2, dtype=torch.float64, device="cuda")
    base = BASE * FACTOR ** (r / (r - 2)) if case["scaling"] == "ntk" else BASE
    f = torch.pow(torch.tensor(base, dtype=torch.float64, device="cuda"), -2 * i / r)
    if case["scaling"] == "linear":
        f = f / FACTOR
    elif case["scaling"] == "parts":  # whole turns in the original length: few are interpolated, many are kept
        keep = ((ORIGINAL * f / (2 * math.pi) - LOW) / (HIGH - LOW)).clamp(0, 1)
        f = f * keep + f / FACTOR * (1 - keep)
    return f


# ---- the plain form --------------------------------------------------------------

def _plain_rope(x, pos, freq, factor, layout, rotary):
    """x [rows][heads][head_dim] turned in 32 bits by angles of 64."""
    angle = pos.double()[:, None] * freq[None]
    c, s = (angle.cos() * factor).float()[:, None], (angle.sin() * factor).float()[:, None]
    y = x.float()
    out = y.clone()
    if layout == "half":
        a, b = y[..., :rotary // 2], y[..., rotary // 2:rotary]
        out[..., :rotary // 2] = a * c - b * s
        out[..., rotary // 2:rotary] = b * c + a * s
    else:
        a, b = y[..., 0:rotary:2], y[..., 1:rotary:2]
        out[..., 0:rotary:2] = a * c - b * s
        out[..., 1:rotary:2] = b * c + a * s
    return out.to(x.dtype)


class _PlainCache:
    """The paged cache in torch: codes [page][layer][block][head][16][dim]."""

    def __init__(self, case, layers, pages):
        kv, hd = case["kv_heads"], case["head_dim"]
        self.codes = [torch.zeros(pages, layers, PAGE // BLOCK, kv, BLOCK, hd, dtype=torch.int8, device="cuda")
                      for _ in range(2)]
        self.scales = [torch.zeros(pages, layers, PAGE // BLOCK, kv, device="cuda") for _ in range(2)]
        self.free, self.refs = list(range(pages - 1, -1, -1)), [0] * pages
        self.seqs, self.next, self.shape = {}, 0, (kv, hd)

    # -- pages
    def create(self):
        self.next += 1
        self.seqs[self.next] = [[], 0]
        return self.next

    def _take(self):
        p = self.free.pop()
        self.refs[p] = 1
        return p

    def _drop(self, p):
        self.refs[p] -= 1
        if not self.refs[p]:
            self.free.append(p)

    def release(self, seq):
        for p in self.seqs.pop(seq)[0]:
            self._drop(p)

    def truncate(self, seq, n):
        pages, _ = self.seqs[seq]
        while len(pages) > (n + PAGE - 1) // PAGE:
            self._drop(pages.pop())
        self.seqs[seq][1] = n

    def fork(self, seq, ways):
        made = []
        for _ in range(ways):
            new = self.create()
            pages, n = self.seqs[seq]
            self.seqs[new] = [list(pages), n]
            for p in pages:
                self.refs[p] += 1
            made.append(new)
        return made

    def _move(self, src, dst):
        if src:
            s, d = (torch.tensor(x, device="cuda") for x in (src, dst))
            for t in self.codes + self.scales:
                t[d] = t[s]

    def copy(self, seq):
        new = self.create()
        pages, n = self.seqs[seq]
        mine = [self._take() for _ in pages]
        self._move(pages, mine)
        self.seqs[new] = [mine, n]
        return new

    def compact(self):
        used = sum(1 for r in self.refs if r)
        holes = [p for p in range(used) if not self.refs[p]]
        late = [p for p in range(used, len(self.refs)) if self.refs[p]]
        self._move(late, holes)
        to = dict(zip(late, holes))
        for s in self.seqs.values():
            s[0] = [to.get(p, p) for p in s[0]]
        for a, b in to.items():
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.free = list(range(len(self.refs) - 1, used - 1, -1))

    # -- steps
    def step(self, seqs, ntok):
        src, dst, page, block, held, row = [], [], [], [], [], []
        self.now, first = [], 0
        for seq, n in zip(seqs, ntok):
            pages, old = self.seqs[seq]
            if n and old % PAGE and self.refs[pages[-1]] > 1:
                p = self._take()
                src.append(pages[-1])
                dst.append(p)
                self._drop(pages[-1])
                pages[-1] = p
            while len(pages) * PAGE < old + n:
                pages.append(self._take())
            for b in range(old // BLOCK, (old + n + BLOCK - 1) // BLOCK):
                page.append(pages[b * BLOCK // PAGE])
                block.append(b % (PAGE // BLOCK))
                held.append(max(0, old - b * BLOCK))
                row.append([first + b * BLOCK + j - old if old <= b * BLOCK + j < old + n else -1
                            for j in range(BLOCK)])
            self.seqs[seq][1] = old + n
            self.now.append((seq, old, n, first))
            first += n
        self._move(src, dst)
        self.touched = [torch.tensor(x, device="cuda") for x in (page, block, held, row)]
        self.positions = torch.cat([torch.arange(old, old + n, device="cuda") for _, old, n, _ in self.now])

    def append(self, layer, k, v):
        page, block, held, row = self.touched
        new = (row >= 0)[:, None, :, None]
        older = (torch.arange(BLOCK, device="cuda")[None] < held[:, None])[:, None, :, None]
        for codes, scales, x in zip(self.codes, self.scales, (k, v)):
            x = x.float()[row.clamp(min=0)].transpose(1, 2)  # [touched][head][16][dim]
            x = torch.where(new & x.isfinite(), x, torch.zeros_like(x))
            had = torch.where(held[:, None] > 0, scales[page, layer, block], torch.zeros((), device="cuda"))
            top = x.abs().amax((-1, -2)).double()
            s = torch.maximum(had, (top / torch.full_like(top, 127.0)).float())  # a quotient, not a product with 1 / 127
            wide = s.double()[..., None, None]
            c = codes[page, layer, block]
            moved = torch.where(wide > 0, (c.double() * had.double()[..., None, None] / wide), torch.zeros_like(wide))
            fresh = torch.where(wide > 0, x.double() / wide, torch.zeros_like(wide))
            c = torch.where(older, moved.round(), torch.where(new, fresh.round().clamp(-127, 127), c.double()))
            codes[page, layer, block] = c.to(torch.int8)
            scales[page, layer, block] = s

    def _whole(self, layer, seq):
        """All keys and values of a sequence: [head][position][dim] f32."""
        pages = torch.tensor(self.seqs[seq][0], device="cuda")
        out = []
        for codes, scales in zip(self.codes, self.scales):
            x = codes[pages, layer].float() * scales[pages, layer][..., None, None]
            out.append(x.permute(2, 0, 1, 3, 4).reshape(self.shape[0], -1, self.shape[1]))
        return out

    def read(self, layer, seq, first, n):
        return tuple(x[:, first:first + n].transpose(0, 1).contiguous() for x in self._whole(layer, seq))

    def attend(self, layer, q, scale, window):
        out = torch.empty_like(q)
        kv, hd = self.shape
        for seq, old, n, first in self.now:
            if not n:
                continue
            k, v = (x[:, :old + n] for x in self._whole(layer, seq))
            x = q[first:first + n].float().view(n, kv, -1, hd).permute(1, 2, 0, 3).reshape(kv, -1, hd)  # [head][group*n]
            score = (x @ k.transpose(1, 2).contiguous() * scale).view(kv, -1, n, old + n)
            at = torch.arange(old + n, device="cuda")
            mine = torch.arange(old, old + n, device="cuda")[:, None]
            hide = at[None] > mine
            if window:
                hide |= at[None] <= mine - window
            score.masked_fill_(hide, -math.inf)
            p = (score - score.amax(-1, keepdim=True)).exp_()
            p = p.div_(p.sum(-1, keepdim=True)).view(kv, -1, old + n)
            y = (p @ v.contiguous()).view(kv, -1, n, hd)
            out[first:first + n] = y.permute(2, 0, 1, 3).reshape(n, -1, hd).to(q.dtype)
        return out


# ---- the library's side -------------------------------------------------------------

def _ptr(t):
    return C.c_void_p(t.data_ptr())


def _ok(status):
    if status:
        _CTX.check(status)


def _own_rope(case):
    H, ctx = _library()
    return H.Rope(ctx, case["head_dim"], BASE, rotary_dim=case["rotary"], layout=case["layout"],
                  scaling=case["scaling"], factor=FACTOR, original_len=ORIGINAL, low=LOW, high=HIGH,
                  attention_factor=_attention_factor(case))


def _own_rope_args(rope, dtype, rows, pos, q, k, qo, ko):
    nh, hd, nk = q.shape[1], q.shape[2], k.shape[1]
    return (rope.handle, CODE[dtype], rows, pos, _ptr(q), nh, nh * hd, _ptr(qo), nh * hd, _ptr(k), nk, nk * hd,
            _ptr(ko), nk * hd)


def _own_cache(case, layers, pages, seqs, longest):
    H, ctx = _library()
    return H.KvCache(ctx, layers, case.get("heads", case["kv_heads"]), case["kv_heads"], case["head_dim"], pages, seqs,
                     longest)


def _own_append_args(kv, layer, dtype, k, v):
    row = k.shape[1] * k.shape[2]
    return kv.handle, layer, CODE[dtype], k.shape[0], _ptr(k), row, _ptr(v), row


def _own_attend_args(kv, layer, dtype, q, out, window):
    row = q.shape[1] * q.shape[2]
    return (kv.handle, layer, CODE[dtype], q.shape[0], _ptr(q), row, q.shape[2] ** -0.5, window, _ptr(out), row)


def _fill(cache, layers, seqs, contents):
    """Stores each sequence's contents[layer][sequence], in either form."""
    n = [k.shape[0] for k, _ in contents[0]]
    if not sum(n):
        return
    cache.step(seqs, n)
    for layer in range(layers):
        k, v = (torch.cat([pair[i] for pair in contents[layer]]).contiguous() for i in range(2))
        if own:
            torch.cuda.synchronize()
            dtype = {v: k for k, v in TORCH.items()}[k.dtype]
            _ok(_library()[0].lib().hale_kv_append_device(*_own_append_args(cache, layer, dtype, k, v)))
            _CTX.synchronize()
        else:
            cache.append(layer, k, v)


def _pages(*lengths):
    return sum(-(-n // PAGE) for n in lengths)


def _cache(case, layers, pages, seqs, longest):
    return _own_cache(case, layers, pages, seqs, longest) if own else _PlainCache(case, layers, pages)


def _new_seq(cache):
    return cache.seq_create() if own else cache.create()


# ---- prepare and run ----------------------------------------------------------------

def prepare(case, seed):
    s = {"kind": case["kind"], "case": case, "lib": _library()[0].lib() if own else None}
    _PREPARE[case["kind"]](s, case, seed)
    torch.cuda.synchronize()
    if own:
        _CTX.synchronize()
    return s


def run(s):
    return _RUN[s["kind"]](s, s["case"])


def _prepare_rope(s, case, seed):
    q, k, pos = _rope_inputs(case, seed)
    if own:
        rope, out = _own_rope(case), (torch.empty_like(q), torch.empty_like(k))
        s.update(rope=rope, out=out, keep=(q, k, pos),
                 args=_own_rope_args(rope, case["dtype"], case["rows"], _ptr(pos), q, k, *out))
    else:
        s.update(q=q, k=k, pos=pos, freq=_frequencies(case))


def _run_rope(s, case):
    if own:
        _ok(s["lib"].hale_rope_device(*s["args"]))
        return s["out"]
    how = (s["pos"], s["freq"], _attention_factor(case), case["layout"], case["rotary"])
    return _plain_rope(s["q"], *how), _plain_rope(s["k"], *how)


def _prepare_store(s, case, seed):
    old, new = _store_inputs(case, seed)
    n = case["base"] + case["ntok"]
    cache = _cache(case, 1, _pages(n) + 3, 2, n)
    seq = _new_seq(cache)
    _fill(cache, 1, [seq], [[old]])
    s.update(cache=cache, seq=seq, new=new)
    if own:
        out = tuple(torch.empty(case["ntok"], case["kv_heads"], case["head_dim"], device="cuda") for _ in range(2))
        s.update(out=out, append=_own_append_args(cache, 0, case["dtype"], *new),
                 read=(cache.handle, 0, seq, case["base"], case["ntok"], _ptr(out[0]), _ptr(out[1])),
                 step=(cache.handle, 1, (C.c_uint32 * 1)(seq), (C.c_uint32 * 1)(case["ntok"])))


def _run_store(s, case):
    if own:
        lib = s["lib"]
        _ok(lib.hale_kv_seq_truncate(s["cache"].handle, s["seq"], case["base"]))
        _ok(lib.hale_kv_step(*s["step"]))
        _ok(lib.hale_kv_append_device(*s["append"]))
        _ok(lib.hale_kv_read_device(*s["read"]))
        return s["out"]
    c = s["cache"]
    c.truncate(s["seq"], case["base"])
    c.step([s["seq"]], [case["ntok"]])
    c.append(0, *s["new"])
    return c.read(0, s["seq"], case["base"], case["ntok"])


def _prepare_attend(s, case, seed):
    old, new, q = _attend_inputs(case, seed)
    total = [k.shape[0] + case["ntok"] for k, _ in old]
    cache = _cache(case, 1, _pages(*total) + 2, len(old), max(total))
    seqs = [_new_seq(cache) for _ in old]
    _fill(cache, 1, seqs, [old])
    _fill(cache, 1, seqs, [new])
    s.update(cache=cache, q=q)
    if own:
        out = torch.empty_like(q)
        s.update(out=out, args=_own_attend_args(cache, 0, case["dtype"], q, out, case["window"]))


def _run_attend(s, case):
    if own:
        _ok(s["lib"].hale_kv_attention_device(*s["args"]))
        return s["out"]
    return s["cache"].attend(0, s["q"], case["head_dim"] ** -0.5, case["window"])


def _rope_case(case):
    return dict(case, rotary=case["head_dim"], layout="half", scaling="none")


def _prepare_decode(s, case, seed):
    layers = list(_decode_inputs(case, seed))
    lens = _lengths(case)
    cache = _cache(case, case["layers"], _pages(*(n + 1 for n in lens)) + 2, len(lens), max(lens) + 1)
    seqs = [_new_seq(cache) for _ in lens]
    _fill(cache, case["layers"], seqs, [layer[0] for layer in layers])
    tokens = [(q, k, v, torch.empty_like(q), torch.empty_like(q), torch.empty_like(k)) for _, q, k, v in layers]
    s.update(cache=cache, seqs=seqs, lens=lens, tokens=tokens)
    if not own:
        s["freq"] = _frequencies(_rope_case(case))
        return
    H, ctx = _library()
    n = len(seqs)
    rope, pos, lib = _own_rope(_rope_case(case)), C.c_void_p(cache.positions), s["lib"]
    s.update(rope=rope, out=torch.empty(len(layers), *tokens[0][0].shape, dtype=tokens[0][0].dtype, device="cuda"),
             step=(cache.handle, n, (C.c_uint32 * n)(*seqs), (C.c_uint32 * n)(*([1] * n))))
    ropes = [_own_rope_args(rope, case["dtype"], n, pos, q, k, qo, ko) for q, k, _, _, qo, ko in tokens]
    appends = [_own_append_args(cache, i, case["dtype"], t[5], t[2]) for i, t in enumerate(tokens)]
    attends = [_own_attend_args(cache, i, case["dtype"], t[4], s["out"][i], 0) for i, t in enumerate(tokens)]

    def layers_of_a_step():
        for a, b, c in zip(ropes, appends, attends):
            _ok(lib.hale_rope_device(*a))
            _ok(lib.hale_kv_append_device(*b))
            _ok(lib.hale_kv_attention_device(*c))

    _ok(lib.hale_kv_step(*s["step"]))
    layers_of_a_step()
    torch.cuda.synchronize()
    ctx.synchronize()
    s["graph"] = ctx.capture(layers_of_a_step)


def _run_decode(s, case):
    cache = s["cache"]
    if own:
        lib = s["lib"]
        for seq, n in zip(s["seqs"], s["lens"]):
            _ok(lib.hale_kv_seq_truncate(cache.handle, seq, n))
        _ok(lib.hale_kv_step(*s["step"]))
        s["graph"].launch()
        return s["out"]
    for seq, n in zip(s["seqs"], s["lens"]):
        cache.truncate(seq, n)
    cache.step(s["seqs"], [1] * len(s["seqs"]))
    out = []
    for i, (q, k, v, *_) in enumerate(s["tokens"]):
        how = (cache.positions, s["freq"], 1.0, "half", case["head_dim"])
        cache.append(i, _plain_rope(k, *how), v)
        out.append(cache.attend(i, _plain_rope(q, *how), case["head_dim"] ** -0.5, 0))
    return torch.stack(out)


def _prepare_fork(s, case, seed):
    layers = list(_fork_inputs(case, seed))
    ways, n = case["ways"], case["prompt"]
    cache = _cache(case, case["layers"], _pages(n + 1) + 2 * ways, 1 + ways, n + 1)
    seq = _new_seq(cache)
    _fill(cache, case["layers"], [seq], [[layer[0]] for layer in layers])
    s.update(cache=cache, seq=seq, tokens=[layer[1:] for layer in layers])
    if own:
        out = torch.empty(len(layers), *layers[0][1].shape, dtype=layers[0][1].dtype, device="cuda")
        s.update(out=out, made=(C.c_uint32 * ways)(), ones=(C.c_uint32 * ways)(*([1] * ways)),
                 append=[_own_append_args(cache, i, case["dtype"], t[2], t[3]) for i, t in enumerate(layers)],
                 attend=[_own_attend_args(cache, i, case["dtype"], t[1], out[i], 0) for i, t in enumerate(layers)])


def _run_fork(s, case):
    cache, ways = s["cache"], case["ways"]
    if own:
        lib, h = s["lib"], cache.handle
        _ok(lib.hale_kv_seq_fork(h, s["seq"], ways, s["made"]))
        _ok(lib.hale_kv_step(h, ways, s["made"], s["ones"]))
        for a, b in zip(s["append"], s["attend"]):
            _ok(lib.hale_kv_append_device(*a))
            _ok(lib.hale_kv_attention_device(*b))
        for seq in s["made"]:
            _ok(lib.hale_kv_seq_free(h, seq))
        return s["out"]
    made = cache.fork(s["seq"], ways)
    cache.step(made, [1] * ways)
    out = []
    for i, (q, k, v) in enumerate(s["tokens"]):
        cache.append(i, k, v)
        out.append(cache.attend(i, q, case["head_dim"] ** -0.5, 0))
    for seq in made:
        cache.release(seq)
    return torch.stack(out)


def _prepare_compact(s, case, seed):
    layers = list(_compact_inputs(case, seed))
    lens = [k.shape[0] for k, _ in layers[0]]
    cache = _cache(case, case["layers"], _pages(lens[0], *lens), 2 + len(lens), max(lens))
    seqs = [_new_seq(cache) for _ in lens]
    _fill(cache, case["layers"], seqs, layers)
    s.update(cache=cache, seq=seqs[0])
    if own:
        shape = (case["layers"], case["length"], case["kv_heads"], case["head_dim"])
        s.update(out=tuple(torch.empty(*shape, device="cuda") for _ in range(2)), new=C.c_uint32(), moved=C.c_size_t())


def _run_compact(s, case):
    cache, n = s["cache"], case["length"]
    if own:
        lib, h = s["lib"], cache.handle
        _ok(lib.hale_kv_seq_copy(h, s["seq"], C.byref(s["new"])))
        _ok(lib.hale_kv_seq_free(h, s["seq"]))
        _ok(lib.hale_kv_compact(h, C.byref(s["moved"])))
        s["seq"] = s["new"].value
        for i in range(case["layers"]):
            _ok(lib.hale_kv_read_device(h, i, s["seq"], 0, n, _ptr(s["out"][0][i]), _ptr(s["out"][1][i])))
        return s["out"]
    new = cache.copy(s["seq"])
    cache.release(s["seq"])
    cache.compact()
    s["seq"] = new
    got = [cache.read(i, new, 0, n) for i in range(case["layers"])]
    return torch.stack([k for k, _ in got]), torch.stack([v for _, v in got])


_PREPARE = dict(rope=_prepare_rope, store=_prepare_store, attend=_prepare_attend, decode=_prepare_decode,
                fork=_prepare_fork, compact=_prepare_compact)
_RUN = dict(rope=_run_rope, store=_run_store, attend=_run_attend, decode=_run_decode, fork=_run_fork,
            compact=_run_compact)


# ---- what a pass cannot do without -------------------------------------------

def _visible(lens, ntok, window):
    """Keys that the queries of each sequence see: their sum over query
    tokens, and how many different ones."""
    pairs = cached = 0
    for n in lens:
        first = max(0, n + 1 - window) if window else 0  # the oldest key of the first query
        cached += n + ntok - first
        p = np.arange(n + 1, n + ntok + 1)
        pairs += int((np.minimum(p, window) if window else p).sum())
    return pairs, cached


def work(case):
    kind, size, kv, hd = case["kind"], SIZE[case["dtype"]], case["kv_heads"], case["head_dim"]
    token = 2 * kv * (hd + 4 / BLOCK)  # the cache's bytes of one position and layer: codes and scales
    if kind == "rope":
        n = case["rows"] * (case["heads"] + kv)
        return {"bytes": 2 * n * hd * size + 4 * case["rows"], "flops": 3 * n * case["rotary"]}
    if kind == "store":  # written, then read back as f32
        n = case["ntok"]
        return {"bytes": n * (2 * kv * hd * (size + 4) + 2 * token), "flops": 4 * n * kv * hd}
    if kind == "compact":  # copied, moved, then read back as f32
        n = case["length"] * case["layers"]
        return {"bytes": n * (5 * token + 8 * kv * hd), "flops": 2 * n * kv * hd}
    q = case["heads"] * hd
    if kind == "attend":
        lens = _lengths(case)
        pairs, cached = _visible(lens, case["ntok"], case["window"])
        return {"bytes": cached * token + 2 * len(lens) * case["ntok"] * q * size, "flops": 4 * q * pairs}
    if kind == "decode":
        n, layers = case["nseq"], case["layers"]
        pairs, cached = _visible(_lengths(case), 1, 0)
        # per token: q and k turned (read, written), k and v stored, q read, the output written
        per = q * size * 4 + kv * hd * size * 4 + token
        return {"bytes": layers * (cached * token + n * per), "flops": layers * (4 * q * pairs + 3 * n * (q + kv * hd))}
    n, layers = case["ways"], case["layers"]
    page = case["prompt"] % PAGE  # the shared page's part, copied for each fork
    per = (2 * q + 2 * kv * hd) * size + token * (1 + 2 * page)
    return {"bytes": layers * (case["prompt"] * token + n * per), "flops": layers * 4 * q * n * (case["prompt"] + 1)}


# ---- the same in 64 bits -----------------------------------------------------

def _stored64(parts):
    """[position][head][dim] in 64 bits as the cache holds what was stored in
    the given order: one array [n][head][dim] after another."""
    codes = scale = None
    for x in parts:
        x = x.float()
        x = torch.where(x.isfinite(), x, torch.zeros_like(x))
        old = 0 if codes is None else codes.shape[0]
        n, (kv, hd) = old + x.shape[0], x.shape[1:]
        blocks = -(-n // BLOCK)
        whole = torch.zeros(blocks * BLOCK, kv, hd, dtype=torch.float64, device="cuda")
        whole[old:n] = x.double()
        top = whole.view(blocks, BLOCK, kv, hd).abs().amax((1, 3))
        need = torch.div(top, torch.full_like(top, 127.0)).float()  # f32, as the scale is held
        grown = need.clone()
        if old:
            m = scale.shape[0]
            if old % BLOCK == 0:
                grown[:m] = scale
            else:
                grown[:m - 1] = scale[:m - 1]
                grown[m - 1] = torch.maximum(scale[m - 1], need[m - 1])
        s = grown.double().repeat_interleave(BLOCK, 0)[:, :, None]
        safe = torch.where(s > 0, s, torch.ones_like(s))
        fresh = (whole / safe).round().clamp(-127, 127) * (s > 0)
        if old:
            was = scale.double().repeat_interleave(BLOCK, 0)[:old, :, None]
            fresh[:old] = (codes * was / safe[:old]).round() * (s[:old] > 0)
        codes, scale = fresh[:n], grown
    return codes * scale.double().repeat_interleave(BLOCK, 0)[:codes.shape[0], :, None]


def _turn64(x, pos, case):
    """Each pair as a complex number times e^(i angle)."""
    f = torch.view_as_complex
    r, x = case["rotary"], x.double()
    turned = x[..., :r]
    if case["layout"] == "half":
        pair = torch.stack((turned[..., :r // 2], turned[..., r // 2:]), -1)
    else:
        pair = turned.reshape(*turned.shape[:-1], r // 2, 2)
    by = torch.polar(torch.full((), _attention_factor(case), dtype=torch.float64, device="cuda"),
                     (pos.double()[:, None] * _frequencies(case))[:, None])
    got = torch.view_as_real(f(pair.contiguous()) * by)
    got = torch.cat((got[..., 0], got[..., 1]), -1) if case["layout"] == "half" else got.flatten(-2)
    return torch.cat((got, x[..., r:]), -1)


def _attend64(q, k, v, window):
    """Queries [n][heads][dim] of the last n positions over all of k, v."""
    n, heads, hd = q.shape
    total, kv = k.shape[:2]
    out = torch.empty(n, heads, hd, dtype=torch.float64, device="cuda")
    back = torch.arange(total - n, total, device="cuda")[:, None] - torch.arange(total, device="cuda")[None]
    seen = (back >= 0) & ((back < window) if window else True)
    for h in range(heads):
        g = h // (heads // kv)
        w = (q[:, h].double() @ k[:, g].t().contiguous()) / math.sqrt(hd)
        w = torch.where(seen, w, torch.full((), -math.inf, dtype=torch.float64, device="cuda")).softmax(-1)
        out[:, h] = w @ v[:, g].contiguous()
    return out


def exact(case, seed):
    kind = case["kind"]
    if kind == "rope":
        q, k, pos = _rope_inputs(case, seed)
        return _turn64(q, pos, case), _turn64(k, pos, case)
    if kind == "store":
        old, new = _store_inputs(case, seed)
        return tuple(_stored64([a, b] if len(a) else [b])[case["base"]:] for a, b in zip(old, new))
    if kind == "compact":
        layers = [layer[0] for layer in _compact_inputs(case, seed)]
        return tuple(torch.stack([_stored64([pair[i]]) for pair in layers]) for i in range(2))
    if kind == "attend":
        old, new, q = _attend_inputs(case, seed)
        out, n = [], case["ntok"]
        for i, (a, b) in enumerate(zip(old, new)):
            k, v = (_stored64([x, y] if len(x) else [y]) for x, y in zip(a, b))
            out.append(_attend64(q[i * n:(i + 1) * n], k, v, case["window"]))
        return torch.cat(out)
    out = []
    if kind == "decode":
        turn, t = _rope_case(case), TORCH[case["dtype"]]
        pos = torch.tensor(_lengths(case), device="cuda")
        for old, q, k, v in _decode_inputs(case, seed):
            q, k = _turn64(q, pos, turn).to(t), _turn64(k, pos, turn).to(t)  # what the rotation hands on
            out.append(torch.cat([_attend64(q[i:i + 1], _stored64([a, k[i:i + 1]]), _stored64([b, v[i:i + 1]]), 0)
                                  for i, (a, b) in enumerate(old)]))
    else:
        for old, q, k, v in _fork_inputs(case, seed):
            out.append(torch.cat([_attend64(q[i:i + 1], _stored64([old[0], k[i:i + 1]]),
                                            _stored64([old[1], v[i:i + 1]]), 0) for i in range(case["ways"])]))
    return torch.stack(out)
