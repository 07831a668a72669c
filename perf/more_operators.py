"""Performance cases of what a step of a serving batch needs around the
quantized layers and the paged cache:

norm    the residual's addition and RMS norm of rows, handing on 8 bits:
        s = x + delta (formed in f32, rounded to the type), u = s w,
        r = 1 / sqrt(mean(s^2) + eps); per block of numbers scale = r max|u| / 127
        and code = 127 u / max|u| rounded to the nearest whole number, ties to
        even; y = r u, rounded to the type.  The codes are returned as they are,
        whole numbers that have to be equal, beside their scales.
q4      products of 4-bit weights that have a scale (and a zero) per group of
        numbers with one to many tokens, given as floats or as 8-bit codes with
        scales: out[t][r] = sum_k scale[r][k / group] (q[r][k] - zero[r][k / group]) x[t][k].
logits  penalties for repeated tokens, biases and grammar masks: a token that
        occurs is divided by the repetition penalty (multiplied where not
        positive), loses frequency times its count and presence among the
        generated ones, gains its bias, and is -inf where the mask has no bit.
prefix  attention of sequences that share a prompt's pages of the 8-bit cache,
        which holds blocks of 16 positions as codes with one f32 scale
        max |x| / 127 (or the block's former scale where that is larger; codes
        are rounded anew to a scale that grew); "step" cases are a whole decode
        step through several layers: positions, stores, attention.

Where `own` is false a pass is computed with elementary torch operations;
where it is true, through the library's entry points on one context, whose
stream a device-wide synchronization covers.  Sizes are those of the
repository's benchmark (hidden 2048 and 4096, 32 query heads over 4 or 8 of
128, a vocabulary of 151936) or generic.
"""
import ctypes as C
import math
import os
import sys

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODE = {"f32": 0, "f16": 1, "bf16": 2}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
PAGE, BLOCK = 64, 16
EPS = 1e-6
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
        # the residual and norm in front of one decoded token's block; the router takes y
        dict(name="norm_1x2048_f32", kind="norm", dtype="f32", rows=1, n=2048, block=32, delta=True, y=True),
        # a prompt's rows
        dict(name="norm_4096x4096_bf16", kind="norm", dtype="bf16", rows=4096, n=4096, block=128, delta=True, y=False),
        # a serving batch, one scale a row, the embedding's rows (no residual yet)
        dict(name="norm_57x4096_f16", kind="norm", dtype="f16", rows=57, n=4096, block=4096, delta=False, y=False),
        # the query projection of one decoded token
        dict(name="q4_token_bf16", kind="q4", dtype="bf16", x8=0, ntok=1, rows=4096, cols=2048, group=128, zeros=True),
        # the vocabulary projection of a generated token
        dict(name="q4_vocab_bf16", kind="q4", dtype="bf16", x8=0, ntok=1, rows=151936, cols=2048, group=64, zeros=True),
        # five drafted tokens through a wide down projection, odd rows, the blocks of 32 that q4_0 has
        dict(name="q4_drafts_f32", kind="q4", dtype="f32", x8=0, ntok=5, rows=1001, cols=14336, group=32, zeros=False),
        # a serving batch's rows as the norm hands them on
        dict(name="q4_batch16_x8", kind="q4", dtype="bf16", x8=32, ntok=16, rows=4096, cols=4096, group=64, zeros=True),
        # a prompt's chunk
        dict(name="q4_prompt_f16", kind="q4", dtype="f16", x8=0, ntok=512, rows=4096, cols=4096, group=128, zeros=False),
        # one sequence's next token
        dict(name="logits_1_f32", kind="logits", dtype="f32", rows=1, vocab=151936, history=3001, biases=20, masks=0),
        # a serving batch, half of it under grammars
        dict(name="logits_64_bf16", kind="logits", dtype="bf16", rows=64, vocab=151936, history=4000, biases=300,
             masks=32),
        # a decode step of eight answers to one prompt through two layers
        dict(name="prefix_step_8x1000_f32", kind="prefix", dtype="f32", heads=32, kv_heads=4, head_dim=128, groups=1,
             ways=8, prompt=1000, lo=0, hi=100, ntok=1, layers=2, step=True),
        # a serving batch behind one long system prompt
        dict(name="prefix_32x8000_bf16", kind="prefix", dtype="bf16", heads=32, kv_heads=8, head_dim=128, groups=1,
             ways=32, prompt=8000, lo=20, hi=600, ntok=1, layers=1, step=False),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng):
    """One more case, of the sizes between and around the listed ones."""
    kind = rng.choice(["norm", "q4", "q4", "logits", "prefix"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "norm":
        block = rng.choice([32, 64, 128, 0])
        n = (block or 32) * max(1, int(_log(rng, 64, 16384)) // (block or 32))
        return dict(kind=kind, dtype=dtype, rows=max(1, int(_log(rng, 1, min(4000, 8e6 / n)))), n=n, block=block or n,
                    delta=rng.random() < 0.7, y=rng.random() < 0.4)
    if kind == "q4":
        group = rng.choice([32, 64, 128])
        cols = group * max(1, int(_log(rng, 128, 14336)) // group)
        ntok = max(1, int(_log(rng, 1, 400)))
        rows = max(1, int(_log(rng, 64, min(150000, 8e9 / ntok / cols))))
        return dict(kind=kind, dtype=dtype, x8=rng.choice([0, 0, 32, 64, 128]) if cols % 128 == 0 else 0, ntok=ntok,
                    rows=rows, cols=cols, group=group, zeros=rng.random() < 0.6)
    if kind == "logits":
        rows = int(_log(rng, 1, 64))
        return dict(kind=kind, dtype=dtype, rows=rows, vocab=int(_log(rng, 500, 151000)),
                    history=int(_log(rng, 1, 6000)), biases=rng.choice([0, int(_log(rng, 1, 300))]),
                    masks=rng.choice([0, 1, (rows + 1) // 2]))
    kv = rng.choice([1, 2, 4, 8])
    ntok = rng.choice([1, 1, 1, 2, 5])
    groups = rng.choice([1, 1, 2, 3])
    ways = max(2, int(_log(rng, 2, 40 / ntok / groups)))
    return dict(kind=kind, dtype=dtype, heads=kv * rng.choice([1, 2, 4, 8]), kv_heads=kv,
                head_dim=rng.choice([64, 80, 128, 128, 128, 256]), groups=groups, ways=ways,
                prompt=int(_log(rng, 65, min(20000, 160000 / ways / groups))), lo=rng.randrange(0, 3),
                hi=int(_log(rng, 4, 400)), ntok=ntok, layers=rng.choice([1, 2]), step=rng.random() < 0.4)


# ---- inputs ----------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) % (1 << 62))
    return g


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _uniform(g, *shape):
    return torch.rand(*shape, device="cuda", generator=g)


def _whole(g, lo, hi, *shape, dtype=torch.int32):
    """Whole numbers of lo .. hi - 1."""
    return torch.randint(lo, hi, shape, device="cuda", generator=g, dtype=dtype)


def _norm_inputs(case, seed):
    """A residual stream, a few channels of which are much larger, the
    block's output that is added to it, and the norm's weights."""
    g, (rows, n), t = _generator(seed), (case["rows"], case["n"]), TORCH[case["dtype"]]
    channel = torch.exp(0.6 * _normal(g, 1, n)) * torch.where(_uniform(g, 1, n) < 0.003, 20.0, 1.0)
    x = (_normal(g, rows, n) * channel).to(t)
    delta = (_normal(g, rows, n) * 0.3).to(t) if case["delta"] else None
    return x, delta, torch.exp(0.3 * _normal(g, n))


def _q4_inputs(case, seed):
    """Codes two to a byte (the first in the low half), scales, zeros or None,
    and the tokens: floats, or codes with scales."""
    g, rows, cols, group, n = _generator(seed), case["rows"], case["cols"], case["group"], case["ntok"]
    codes = _whole(g, 0, 256, rows, cols // 2, dtype=torch.uint8)
    scales = (torch.exp(0.4 * _normal(g, rows, cols // group)) * 0.01).to(torch.float16)
    zeros = _whole(g, 0, 16, rows, cols // group, dtype=torch.uint8) if case["zeros"] else None
    x = _normal(g, n, cols) * torch.exp(0.5 * _normal(g, 1, cols))
    if not case["x8"]:
        return codes, scales, zeros, x.to(TORCH[case["dtype"]]), None
    b = x.view(n, -1, case["x8"])
    s = b.abs().amax(-1) / 127
    return codes, scales, zeros, (b / s[..., None]).round().to(torch.int8).view(n, cols), s


def _logits_inputs(case, seed):
    """Logits, token histories (a few tokens make up most of a text) that
    begin with a prompt, penalties, biases, and masks of which some allow
    nearly all tokens, some a few and one nothing."""
    g, rows, vocab = _generator(seed), case["rows"], case["vocab"]
    logits = (_normal(g, rows, vocab) * 3).to(TORCH[case["dtype"]])
    lens = (case["history"] ** _uniform(g, rows)).long().clamp(1) if rows > 1 else torch.tensor([case["history"]], device="cuda")
    start = torch.zeros(rows + 1, dtype=torch.int64, device="cuda")
    start[1:] = lens.cumsum(0)
    total = int(start[-1])
    tokens = (vocab ** _uniform(g, total)).int() - 1
    prompt = (lens * _uniform(g, rows)).long()
    d = dict(logits=logits, start=start, tokens=tokens, prompt=prompt, repetition=1 + 0.3 * _uniform(g, rows),
             frequency=0.5 * _uniform(g, rows), presence=0.5 * _uniform(g, rows))
    if case["biases"]:
        n = min(case["biases"], vocab)
        first = _whole(g, 0, vocab, rows, 1, dtype=torch.int64)
        stride = next(p for p in (7919, 7907, 7901) if vocab % p)  # no token twice in a row's list
        d["bias_tokens"] = ((first + stride * torch.arange(n, device="cuda")) % vocab).int().view(-1)
        d["bias"] = (_normal(g, rows * n) * 4)
        d["bias_start"] = torch.arange(rows + 1, device="cuda") * n
    if case["masks"]:
        m, words = case["masks"], (vocab + 31) // 32
        odds = 10 ** (-4 * _uniform(g, m, 1))
        odds[m // 2] = 0 if m > 4 else odds[m // 2]
        bits = (_uniform(g, m, words, 32) < odds[..., None]).long() << torch.arange(32, device="cuda")
        d["mask"] = bits.sum(-1).to(torch.int32)  # wraps to the bit pattern
        d["mask_row"] = torch.where(torch.arange(rows, device="cuda") % 2 == 1, -1,
                                    torch.arange(rows, device="cuda") // 2 % m).int()
    return d


def _lengths(case):
    """What each sequence holds behind the prompt: from lo to hi, in no order."""
    lo, hi, n = case["lo"], case["hi"], case["groups"] * case["ways"]
    return [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** ((0.37 + 0.6180339887 * i) % 1.0))) - 1 for i in range(n)]


def _keys_values(g, case, *shape):
    """Keys, some channels of which are larger, as models have them, and
    values, some tokens of which are larger."""
    kv, hd, t = case["kv_heads"], case["head_dim"], TORCH[case["dtype"]]
    k = _normal(g, *shape, kv, hd) * torch.exp(0.5 * _normal(g, kv, hd))
    v = _normal(g, *shape, kv, hd) * torch.exp(0.3 * _normal(g, *shape, kv, 1))
    return k.to(t), v.to(t)


def _prefix_inputs(case, seed):
    """Layer by layer, keys and values of the prompts [groups][prompt], of
    each sequence behind its prompt [sequence][longest] (of which _lengths
    count), of the new tokens [sequence][ntok], and the queries."""
    g, seqs = _generator(seed), case["groups"] * case["ways"]
    for _ in range(case["layers"]):
        yield (_keys_values(g, case, case["groups"], case["prompt"]), _keys_values(g, case, seqs, max(_lengths(case))),
               _keys_values(g, case, seqs, case["ntok"]),
               (_normal(g, seqs * case["ntok"], case["heads"], case["head_dim"]) * 1.2).to(TORCH[case["dtype"]]))


# ---- the plain form --------------------------------------------------------------

def _plain_norm(x, delta, w, block):
    s = x if delta is None else (x.float() + delta.float()).to(x.dtype)
    # in 64 bits: codes next to a border between two whole numbers go by their last bits
    u = s.double() * w.double()
    r = (s.double().square().mean(-1, keepdim=True) + EPS).rsqrt()
    b = u.view(u.shape[0], -1, block)
    top = b.abs().amax(-1, keepdim=True)
    code = torch.where(top > 0, 127 * b / top, torch.zeros_like(b)).round()
    scale = (top * r[..., None] / 127).float()
    return s, (u * r).to(x.dtype), code.to(torch.int8).view_as(s), scale.squeeze(-1)


def _plain_weights(codes, scales, zeros, group, wide):
    """The matrix [rows][cols] in f32 or f64."""
    rows = codes.shape[0]
    q = torch.stack((codes & 15, codes >> 4), -1).view(rows, -1, group).to(wide)
    z = zeros.to(wide)[..., None] if zeros is not None else 8
    return ((q - z) * scales.to(wide)[..., None]).view(rows, -1)


def _plain_q4(codes, scales, zeros, x, xs, case):
    x = x.float()
    if xs is not None:
        x = (x.view(*xs.shape, -1) * xs[..., None]).view(x.shape)
    w = _plain_weights(codes, scales, zeros, case["group"], torch.float32)
    return (x @ w.t().contiguous()).to(TORCH[case["dtype"]])


def _plain_logits(d):
    x = d["logits"].float()
    rows, vocab = x.shape
    at = torch.arange(d["tokens"].numel(), device="cuda")
    row = torch.searchsorted(d["start"], at, right=True) - 1
    place = row * vocab + d["tokens"]
    made = at - d["start"][row] >= d["prompt"][row]  # generated, not of the prompt
    every = torch.bincount(place, minlength=rows * vocab).view(rows, vocab)
    mine = torch.bincount(place[made], minlength=rows * vocab).view(rows, vocab)
    rep = d["repetition"][:, None]
    x = torch.where(every > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - d["frequency"][:, None] * mine - d["presence"][:, None] * (mine > 0)
    if "bias" in d:
        n = d["bias_start"][1:] - d["bias_start"][:-1]
        row = torch.repeat_interleave(torch.arange(rows, device="cuda"), n, output_size=d["bias"].numel())
        x.view(-1)[row * vocab + d["bias_tokens"]] += d["bias"]
    if "mask" in d:
        bits = (d["mask"][..., None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        keep = bits.view(bits.shape[0], -1)[:, :vocab] > 0
        free = d["mask_row"] < 0
        x = torch.where(keep[d["mask_row"].clamp(min=0).long()] | free[:, None], x, -math.inf)
    return x.to(d["logits"].dtype)


def _blocks(x):
    """[..][positions][head][dim] as [..][blocks][16][head][dim] in f64."""
    return x.double().unflatten(-3, (-1, BLOCK))


def _store(codes, scale, x, new):
    """Blocks after the numbers x were stored to them where `new` is true:
    codes [..][blocks][16][head][dim] in f64 and scales [..][blocks][head]."""
    new = new[..., None, None]
    x = _blocks(x)
    top = (x.abs() * new).amax((-3, -1))
    grown = torch.maximum(scale, (top / torch.full_like(top, 127.0)).float())  # a quotient, not a product with 1 / 127
    to = grown.double()[..., None, :, None]
    safe = torch.where(to > 0, to, torch.ones_like(to))
    codes = torch.where(new, x / safe, codes * scale.double()[..., None, :, None] / safe).round()
    return torch.where(to > 0, codes, torch.zeros_like(codes)), grown


def _plain_layer(case, kv, i):
    """One of keys and values of a layer as the cache holds it before the new
    tokens: the prompts' whole pages, [groups][head][position][dim] f32, and what
    lies behind them for each sequence, codes and scales by blocks."""
    (first, held, _), lens = (part[i] for part in kv), torch.tensor(_lengths(case), device="cuda")
    base = case["prompt"] // PAGE * PAGE
    tail, seqs = case["prompt"] - base, case["groups"] * case["ways"]
    size = -(-(tail + max(_lengths(case)) + case["ntok"]) // BLOCK) * BLOCK
    kv_heads, hd = case["kv_heads"], case["head_dim"]
    whole = first[:, :base].float()
    none = torch.zeros(case["groups"], base // BLOCK, kv_heads, device="cuda")
    every = torch.ones(case["groups"], base // BLOCK, BLOCK, dtype=torch.bool, device="cuda")
    c, s = _store(torch.zeros_like(_blocks(whole)), none, whole, every)
    shared = (c.float() * s[..., None, :, None]).flatten(1, 2).transpose(1, 2).contiguous()
    x = torch.zeros(seqs, size, kv_heads, hd, device="cuda")
    x[:, :tail] = first[:, base:].float().repeat_interleave(case["ways"], 0)
    x[:, tail:tail + held.shape[1]] = held.float()
    at = torch.arange(size, device="cuda").expand(seqs, size)
    end = tail + lens[:, None]
    c, s = torch.zeros_like(_blocks(x)), torch.zeros(seqs, size // BLOCK, kv_heads, device="cuda")
    c, s = _store(c, s, x, (at < tail).unflatten(1, (-1, BLOCK)))
    c, s = _store(c, s, x, ((at >= tail) & (at < end)).unflatten(1, (-1, BLOCK)))
    return shared, c, s


def _plain_append(case, layer, new):
    """The layer's own blocks with the new tokens [sequence][ntok] stored."""
    shared, c, s = layer
    n, seqs, size = case["ntok"], c.shape[0], c.shape[1] * BLOCK
    end = case["prompt"] % PAGE + torch.tensor(_lengths(case), device="cuda")[:, None]
    row = torch.arange(seqs, device="cuda")[:, None]
    x = torch.zeros(seqs, size, *new.shape[2:], device="cuda")
    x[row, end + torch.arange(n, device="cuda")] = new.float()
    at = torch.arange(size, device="cuda").expand(seqs, size)
    c, s = _store(c, s, x, ((at >= end) & (at < end + n)).unflatten(1, (-1, BLOCK)))
    return shared, c, s


def _plain_attend(case, keys, values, q):
    (sk, ck, kk), (sv, cv, vv) = keys, values
    own_k, own_v = ((c.float() * s[..., None, :, None]).flatten(1, 2).transpose(1, 2).contiguous()
                    for c, s in ((ck, kk), (cv, vv)))
    groups, ways, n, kv, hd = case["groups"], case["ways"], case["ntok"], case["kv_heads"], case["head_dim"]
    seqs, per = groups * ways, case["heads"] // kv
    x = q.float().view(seqs, n, kv, per, hd).transpose(1, 2).reshape(seqs, kv, n * per, hd) * hd ** -0.5
    mine = x @ own_k.transpose(2, 3).contiguous()  # [sequence][head][row][own position]
    end = case["prompt"] % PAGE + torch.tensor(_lengths(case), device="cuda")
    last = end[:, None] + torch.arange(n, device="cuda").repeat_interleave(per)  # of each row
    mine = mine.masked_fill(torch.arange(mine.shape[-1], device="cuda") > last[:, None, :, None], -math.inf)
    rows = x.view(groups, ways, kv, n * per, hd).transpose(1, 2).reshape(groups, kv, -1, hd)
    score = rows @ sk.transpose(2, 3).contiguous()
    score = score.view(groups, kv, ways, n * per, -1).transpose(1, 2).reshape(seqs, kv, n * per, -1)
    base = score.shape[-1]
    p = torch.cat((score, mine), -1)
    p = (p - p.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    first = p[..., :base].reshape(groups, ways, kv, n * per, base).transpose(1, 2).reshape(groups, kv, -1, base)
    y = (first @ sv).view(groups, kv, ways, n * per, hd).transpose(1, 2).reshape(seqs, kv, n * per, hd)
    y = y + p[..., base:].contiguous() @ own_v
    return y.view(seqs, kv, n, per, hd).transpose(1, 2).reshape(seqs * n, kv * per, hd).to(q.dtype)


# ---- the library's side -------------------------------------------------------------

def _ptr(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


def _ok(status):
    if status:
        _CTX.check(status)


def _own_prefix(case, layers):
    """A cache that shares prefixes, its sequences, and the calls of a layer."""
    H, ctx = _library()
    lib, seqs, n, lens = H.lib(), case["groups"] * case["ways"], case["ntok"], _lengths(case)
    total = [case["prompt"] + m + n for m in lens]
    pages = sum(-(-m // PAGE) for m in total) + case["groups"] * (case["prompt"] // PAGE + 2)
    kv = H.KvCache(ctx, case["layers"], case["heads"], case["kv_heads"], case["head_dim"], pages,
                   seqs + case["groups"], max(total))
    kv.share_prefixes(PAGE)
    row, width = case["kv_heads"] * case["head_dim"], case["heads"] * case["head_dim"]

    def append(i, k, v):
        return (kv.handle, i, CODE[case["dtype"]], k.shape[0], _ptr(k), row, _ptr(v), row)

    def fill(ids, contents):
        """contents[layer]: keys and values of the step's tokens"""
        for i, (k, v) in enumerate(contents):
            k, v = k.contiguous(), v.contiguous()
            torch.cuda.synchronize()
            _ok(lib.hale_kv_append_device(*append(i, k, v)))
            ctx.synchronize()

    roots = [kv.seq_create() for _ in range(case["groups"])]
    kv.step(roots, [case["prompt"]] * len(roots))
    fill(roots, [[x.flatten(0, 1) for x in layer[0]] for layer in layers])
    ids = [s for r in roots for s in kv.seq_fork(r, case["ways"])]
    if sum(lens):
        kv.step(ids, lens)
        at = torch.arange(max(lens), device="cuda") < torch.tensor(lens, device="cuda")[:, None]
        fill(ids, [[x[at] for x in layer[1]] for layer in layers])
    kv.step(ids, [n] * seqs)
    new = [[x.flatten(0, 1) for x in layer[2]] for layer in layers]
    fill(ids, new)
    out = torch.empty(len(layers), *layers[0][3].shape, dtype=layers[0][3].dtype, device="cuda")
    appends = [append(i, *pair) for i, pair in enumerate(new)]
    attends = [(kv.handle, i, CODE[case["dtype"]], seqs * n, _ptr(layer[3]), width, case["head_dim"] ** -0.5, 0,
                _ptr(out[i]), width) for i, layer in enumerate(layers)]
    return dict(cache=kv, ids=ids, new=new, out=out, appends=appends, attends=attends, layers=layers, ctx=ctx)


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


def _prepare_norm(s, case, seed):
    x, delta, w = _norm_inputs(case, seed)
    s.update(x=x, delta=delta, w=w)
    if own:
        rows, n, block = case["rows"], case["n"], case["block"]
        total, y = (torch.empty_like(x) if case[k] else None for k in ("delta", "y"))
        codes = torch.empty(rows, n, dtype=torch.int8, device="cuda")
        scales = torch.empty(rows, n // block, device="cuda")
        s.update(out=(total, y, codes, scales),
                 args=(_library()[1].handle, CODE[case["dtype"]], rows, n, _ptr(x), n, _ptr(delta), n, _ptr(w), EPS,
                       block, _ptr(total), n, _ptr(y), n, _ptr(codes), _ptr(scales)))


def _run_norm(s, case):
    if own:
        _ok(s["lib"].hale_rms_norm_q8_device(*s["args"]))
        total, y, codes, scales = s["out"]
    else:
        total, y, codes, scales = _plain_norm(s["x"], s["delta"], s["w"], case["block"])
    return {"sum": total if case["delta"] else None, "y": y if case["y"] else None, "codes": codes, "scales": scales}


def _prepare_q4(s, case, seed):
    codes, scales, zeros, x, xs = _q4_inputs(case, seed)
    s.update(codes=codes, scales=scales, zeros=zeros, x=x, xs=xs)
    if own:
        H, ctx = _library()
        torch.cuda.synchronize()
        m = H.GroupQ4Matrix.from_device(ctx, case["rows"], case["cols"], case["group"], codes.data_ptr(),
                                        scales.data_ptr(), zeros.data_ptr() if zeros is not None else 0, "f16")
        out = torch.empty(case["ntok"], case["rows"], dtype=TORCH[case["dtype"]], device="cuda")
        if xs is None:
            args = (m.handle, CODE[case["dtype"]], case["ntok"], _ptr(x), case["cols"], _ptr(out), case["rows"])
        else:
            args = (m.handle, case["ntok"], case["x8"], _ptr(x), _ptr(xs), CODE[case["dtype"]], _ptr(out), case["rows"])
        s.update(m=m, out=out, args=args)


def _run_q4(s, case):
    if own:
        call = s["lib"].hale_q4g_matmul_q8_device if case["x8"] else s["lib"].hale_q4g_matmul_device
        _ok(call(*s["args"]))
        return s["out"]
    return _plain_q4(s["codes"], s["scales"], s["zeros"], s["x"], s["xs"], case)


def _prepare_logits(s, case, seed):
    d = _logits_inputs(case, seed)
    s.update(d=d)
    if own:
        H, ctx = _library()
        get = lambda k: d[k].data_ptr() if k in d else 0  # noqa: E731
        rules = H.LogitsRules(tokens=get("tokens"), token_start=get("start"), ntokens=d["tokens"].numel(),
                              prompt_len=get("prompt"), repetition=get("repetition"), frequency=get("frequency"),
                              presence=get("presence"), bias_tokens=get("bias_tokens"), bias=get("bias"),
                              bias_start=get("bias_start"), nbiases=d["bias"].numel() if "bias" in d else 0,
                              mask=get("mask"), mask_rows=case["masks"], mask_stride=(case["vocab"] + 31) // 32,
                              mask_row=get("mask_row"))
        out = torch.empty_like(d["logits"])
        s.update(rules=rules, out=out, args=(ctx.handle, CODE[case["dtype"]], case["rows"], case["vocab"],
                                             _ptr(d["logits"]), case["vocab"], C.byref(rules), _ptr(out), case["vocab"]))


def _run_logits(s, case):
    if own:
        _ok(s["lib"].hale_logits_device(*s["args"]))
        return s["out"]
    return _plain_logits(s["d"])


def _prepare_prefix(s, case, seed):
    layers = list(_prefix_inputs(case, seed))
    if not own:
        held = [[_plain_layer(case, layer[:3], i) for i in (0, 1)] for layer in layers]
        new = [layer[2] for layer in layers]
        if not case["step"]:
            held = [[_plain_append(case, h, x) for h, x in zip(hs, xs)] for hs, xs in zip(held, new)]
        s.update(held=held, new=new, q=[layer[3] for layer in layers])
        return
    s.update(_own_prefix(case, layers))
    lib, seqs = s["lib"], len(s["ids"])
    s["before"] = [case["prompt"] + n for n in _lengths(case)]
    s["args"] = (s["cache"].handle, seqs, (C.c_uint32 * seqs)(*s["ids"]), (C.c_uint32 * seqs)(*([case["ntok"]] * seqs)))

    def layers_of_a_step():
        for a, b in zip(s["appends"], s["attends"]):
            _ok(lib.hale_kv_append_device(*a))
            _ok(lib.hale_kv_attention_device(*b))

    if case["step"]:
        layers_of_a_step()
        s["ctx"].synchronize()
        s["graph"] = s["ctx"].capture(layers_of_a_step)


def _run_prefix(s, case):
    if own:
        lib = s["lib"]
        if not case["step"]:
            for a in s["attends"]:
                _ok(lib.hale_kv_attention_device(*a))
            return s["out"]
        for seq, n in zip(s["ids"], s["before"]):
            _ok(lib.hale_kv_seq_truncate(s["cache"].handle, seq, n))
        _ok(lib.hale_kv_step(*s["args"]))
        s["graph"].launch()
        return s["out"]
    out = []
    for held, new, q in zip(s["held"], s["new"], s["q"]):
        if case["step"]:
            held = [_plain_append(case, h, x) for h, x in zip(held, new)]
        out.append(_plain_attend(case, *held, q))
    return torch.stack(out)


_PREPARE = dict(norm=_prepare_norm, q4=_prepare_q4, logits=_prepare_logits, prefix=_prepare_prefix)
_RUN = dict(norm=_run_norm, q4=_run_q4, logits=_run_logits, prefix=_run_prefix)


# ---- what a pass cannot do without -------------------------------------------

def work(case):
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind == "norm":
        rows, n = case["rows"], case["n"]
        return {"bytes": rows * (n * (size * (1 + 2 * case["delta"] + case["y"]) + 1) + 4 * n // case["block"]) + 4 * n,
                "flops": 8 * rows * n}
    if kind == "q4":
        rows, cols, n = case["rows"], case["cols"], case["ntok"]
        weights = rows * cols // 2 + rows * (cols // case["group"]) * (3 if case["zeros"] else 2)
        x = n * (cols + 4 * cols // case["x8"]) if case["x8"] else n * cols * size
        return {"bytes": weights + x + n * rows * size, "flops": 2 * n * rows * cols}
    if kind == "logits":
        rows, vocab = case["rows"], case["vocab"]
        mean = case["history"] if rows == 1 else (case["history"] - 1) / max(1e-9, math.log(max(2, case["history"])))
        used = min(case["masks"], (rows + 1) // 2)
        return {"bytes": 2 * rows * vocab * size + rows * (4 * mean + 8 * case["biases"]) + used * vocab / 8,
                "flops": rows * (4 * vocab + 4 * mean)}
    kv, hd, n, q = case["kv_heads"], case["head_dim"], case["ntok"], case["heads"] * case["head_dim"]
    token = 2 * kv * (hd + 4 / BLOCK)  # the cache's bytes of one position and layer: codes and scales
    lens, prompt = _lengths(case), case["prompt"]
    cached = case["groups"] * prompt + sum(m + n for m in lens)
    pairs = sum(n * (prompt + m) + n * (n + 1) // 2 for m in lens)
    stored = len(lens) * n * (2 * kv * hd * size + token) if case["step"] else 0
    return {"bytes": case["layers"] * (cached * token + 2 * len(lens) * n * q * size + stored),
            "flops": case["layers"] * 4 * q * pairs}


# ---- the same in 64 bits -----------------------------------------------------

def _exact_norm(case, seed):
    x, delta, w = _norm_inputs(case, seed)
    s = x.double()
    if delta is not None:
        s = (s + delta.double()).float().to(x.dtype).double()
    y = s / torch.sqrt((s * s).sum(-1, keepdim=True) / case["n"] + EPS) * w.double()
    most = y.unflatten(-1, (-1, case["block"])).abs().max(-1).values
    step = (most / 127).float()
    # 127 y / most by the numbers before the row's factor, whose products with the weights are whole in 64 bits
    raw = (s * w.double()).unflatten(-1, (-1, case["block"]))
    by = raw.abs().max(-1, keepdim=True).values
    whole = torch.round(raw * 127 / by.clamp(min=torch.finfo(torch.float64).tiny))
    return {"sum": s if case["delta"] else None, "y": y if case["y"] else None,
            "codes": whole.flatten(-2).to(torch.int8), "scales": step.double()}


def _exact_q4(case, seed):
    codes, scales, zeros, x, xs = _q4_inputs(case, seed)
    x = x.double()
    if xs is not None:
        x *= xs.double().repeat_interleave(case["x8"], -1)
    out = torch.empty(case["ntok"], case["rows"], dtype=torch.float64, device="cuda")
    for a in range(0, case["rows"], 16384):
        c = codes[a:a + 16384].int()
        w = torch.empty(c.shape[0], case["cols"], dtype=torch.float64, device="cuda")
        w[:, 0::2], w[:, 1::2] = c % 16, c // 16
        w -= 8 if zeros is None else zeros[a:a + 16384].double().repeat_interleave(case["group"], 1)
        w *= scales[a:a + 16384].double().repeat_interleave(case["group"], 1)
        out[:, a:a + 16384] = x @ w.t().contiguous()
    return out


def _exact_logits(case, seed):
    d = _logits_inputs(case, seed)
    out = d["logits"].double()
    for r in range(case["rows"]):
        a, b = int(d["start"][r]), int(d["start"][r + 1])
        history = d["tokens"][a:b].long()
        rep, x = float(d["repetition"][r]), out[r]
        seen = history.unique()
        x[seen] = torch.where(x[seen] > 0, x[seen] / rep, x[seen] * rep)
        made, count = history[int(d["prompt"][r]):].unique(return_counts=True)
        x[made] -= float(d["frequency"][r]) * count + float(d["presence"][r])
        if "bias" in d:
            at = slice(int(d["bias_start"][r]), int(d["bias_start"][r + 1]))
            x[d["bias_tokens"][at].long()] += d["bias"][at].double()
        if "mask" in d and int(d["mask_row"][r]) >= 0:
            token = torch.arange(case["vocab"], device="cuda")
            word = d["mask"][int(d["mask_row"][r])][token // 32]
            x[(word >> (token % 32).int()) % 2 == 0] = -math.inf
    return out


def _held64(parts):
    """[position][head][dim] in 64 bits as the cache holds what was stored in
    the given order: one array [n][head][dim] after another."""
    codes = scale = None
    for x in parts:
        if not x.shape[0]:
            continue
        old = 0 if codes is None else codes.shape[0]
        n, (kv, hd) = old + x.shape[0], x.shape[1:]
        blocks = -(-n // BLOCK)
        whole = torch.zeros(blocks * BLOCK, kv, hd, dtype=torch.float64, device="cuda")
        whole[old:n] = x.double()
        top = whole.view(blocks, BLOCK, kv, hd).abs().amax((1, 3))
        grown = torch.div(top, torch.full_like(top, 127.0)).float()  # f32, as the scale is held
        if old:
            grown[:scale.shape[0]] = torch.maximum(scale, grown[:scale.shape[0]])
        s = grown.double().repeat_interleave(BLOCK, 0)[:, :, None]
        s = torch.where(s > 0, s, torch.ones_like(s))
        fresh = (whole / s).round()
        if old:
            fresh[:old] = (codes * scale.double().repeat_interleave(BLOCK, 0)[:old, :, None] / s[:old]).round()
        codes, scale = fresh[:n], grown
    return codes * scale.double().repeat_interleave(BLOCK, 0)[:codes.shape[0], :, None]


def _exact_prefix(case, seed):
    n, heads, kv = case["ntok"], case["heads"], case["kv_heads"]
    layers = []
    for first, held, new, q in _prefix_inputs(case, seed):
        out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
        for i, m in enumerate(_lengths(case)):
            k, v = (_held64([first[j][i // case["ways"]], held[j][i, :m], new[j][i]]) for j in (0, 1))
            unseen = torch.ones(n, k.shape[0], dtype=torch.bool, device="cuda").triu(k.shape[0] - n + 1)
            for h in range(heads):
                g, at = h // (heads // kv), slice(i * n, (i + 1) * n)
                w = (q[at, h].double() @ k[:, g].t().contiguous()) / math.sqrt(case["head_dim"])
                out[at, h] = w.masked_fill(unseen, -math.inf).softmax(-1) @ v[:, g].contiguous()
        layers.append(out)
    return torch.stack(layers)


def exact(case, seed):
    return dict(norm=_exact_norm, q4=_exact_q4, logits=_exact_logits, prefix=_exact_prefix)[case["kind"]](case, seed)
