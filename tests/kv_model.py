"""A plain model of the paged 8-bit key/value cache in numpy, 64 bits: what
each sequence holds, stored the way the library documents it, and attention
over it.  Shared by the GPU tests of the cache."""
import numpy as np

BLOCK = 16
EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step of a rounding, relative


def encode(x, dtype):
    """f32 values as the bytes of a type, and as the f32 values these stand for."""
    x = np.asarray(x, np.float32)
    if dtype == "f32":
        return x.copy(), x
    if dtype == "f16":
        with np.errstate(over="ignore"):
            h = x.astype(np.float16)
        return h, h.astype(np.float32)
    u = np.ascontiguousarray(x).view(np.uint32)
    h = ((u.astype(np.uint64) + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    h = np.where(np.isnan(x), np.uint16(0x7FC0), h)
    return h, decode(h, "bf16")


def decode(raw, dtype):
    if dtype == "f32":
        return raw.view(np.float32)
    if dtype == "f16":
        return raw.view(np.float16).astype(np.float32)
    return (raw.view(np.uint16).astype(np.uint32) << 16).view(np.float32)


NP = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16}


class Stored:
    """One of keys and values of one sequence and layer: codes and scales."""

    def __init__(self, heads, dim):
        self.codes = np.zeros((0, heads, dim))
        self.scales = np.zeros((0, heads), np.float32)

    def copy(self):
        c = Stored(*self.codes.shape[1:])
        c.codes, c.scales = self.codes.copy(), self.scales.copy()
        return c

    def truncate(self, n):
        self.codes = self.codes[:n].copy()
        self.scales = self.scales[:-(-n // BLOCK)].copy()  # a block that is left keeps its scale

    def append(self, x):
        x = np.where(np.isfinite(x), x, np.float32(0)).astype(np.float32)
        old, n = len(self.codes), len(self.codes) + len(x)
        for b in range(old // BLOCK, -(-n // BLOCK)):
            lo, hi = max(old, b * BLOCK), min(n, (b + 1) * BLOCK)
            if lo >= hi:
                continue
            new = x[lo - old:hi - old].astype(np.float64)
            need = (np.abs(new).max((0, 2)) / 127.0).astype(np.float32)
            held = lo - b * BLOCK
            had = self.scales[b] if held else np.zeros_like(need)
            s = np.maximum(had, need)
            wide, safe = s.astype(np.float64)[:, None], np.where(s > 0, s, 1).astype(np.float64)[:, None]
            fresh = np.where(wide > 0, np.clip(np.rint(new / safe), -127, 127), 0.0)
            if held:
                moved = np.rint(self.codes[b * BLOCK:] * had.astype(np.float64)[:, None] / safe)
                self.codes[b * BLOCK:] = np.where(wide > 0, moved, 0.0)
                self.scales[b] = s
            else:
                self.scales = np.concatenate([self.scales, s[None]])
            self.codes = np.concatenate([self.codes, fresh])

    def values(self):
        """f32, as reading back gives them: code times scale, rounded."""
        return (self.codes.astype(np.float32) * np.repeat(self.scales, BLOCK, 0)[:len(self.codes), :, None]).astype(np.float32)

    def exact(self):
        return self.codes * np.repeat(self.scales.astype(np.float64), BLOCK, 0)[:len(self.codes), :, None]


class Model:
    """The sequences of a cache: per layer (keys, values)."""

    def __init__(self, layers, heads, kv_heads, dim):
        self.shape, self.layers = (heads, kv_heads, dim), layers
        self.seqs = {}

    def create(self, s):
        self.seqs[s] = [(Stored(*self.shape[1:]), Stored(*self.shape[1:])) for _ in range(self.layers)]

    def fork(self, s, new):
        self.seqs[new] = [(k.copy(), v.copy()) for k, v in self.seqs[s]]

    def truncate(self, s, n):
        for pair in self.seqs[s]:
            for x in pair:
                x.truncate(n)

    def append(self, s, layer, k, v):
        self.seqs[s][layer][0].append(k)
        self.seqs[s][layer][1].append(v)

    def attend(self, s, layer, q, scale, window=0):
        """q [n][heads][dim], the last n positions' queries.  Returns out, and for
        attention_bound() sum_j p_j |v_j|, per row the largest sum_d |q_d k_d|, the
        number of keys, and per row 127 times the largest scale of the values' blocks it
        sees."""
        k, v = (x.exact() for x in self.seqs[s][layer])
        n, heads, _ = q.shape
        total, kv = k.shape[:2]
        out, mag, prod = (np.zeros(q.shape) for _ in range(3))
        prod, vtop = np.zeros((n, heads)), np.zeros((n, heads))
        scales = np.repeat(self.seqs[s][layer][1].scales.astype(np.float64), BLOCK, 0)[:total]
        pos = np.arange(total - n, total)[:, None]
        at = np.arange(total)[None]
        see = at <= pos
        if window:
            see &= at > pos - window
        for h in range(heads):
            g = h // (heads // kv)
            qh = q[:, h].astype(np.float64)
            x = np.where(see, scale * (qh @ k[:, g].T), -np.inf)
            p = np.exp(x - x.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            out[:, h] = p @ v[:, g]
            mag[:, h] = p @ np.abs(v[:, g])
            vtop[:, h] = 127 * np.where(see, scales[:, g][None], 0.0).max(1)
            prod[:, h] = scale * (np.where(see[:, :, None], 1.0, 0.0) * (np.abs(qh)[:, None] * np.abs(k[:, g])[None])).sum(2).max(1) \
                if n * total * self.shape[2] < 3e6 else scale * np.abs(qh).sum(1) * np.abs(k[:, g]).max()
        return out, mag, prod, k.shape[0], vtop


def attention_bound(dtype, mag, prod, total, vtop, dim):
    """Elementwise error that the kernel's roundings can add up to.

    Score of a key: dim products summed in f32, each sum off by at most 2^-24
    of the partial sums (at most `prod`), the query's parts by 2^-23 of the
    row's largest (f32; within prod * 2^-23 * dim), two factors and the
    subtraction of the maximum by 2^-24 each, of numbers up to 2 prod:
    s = prod (dim + dim * 2 + 8) 2^-24.  A probability is off by e^s - 1 + 2^-22 (exp2)
    relative, its rounding (2^-11 or 2^-23) and that of the values' scale 3 * 2^-24;
    numerator and denominator both, so twice, against sum p |v|; each of the
    at most total + 64 sums of a row adds 2^-24 of it.  The result is
    rounded once more to its type: f16 numbers below 2^-14 are multiples of 2^-24, so
    there the rounding is off by up to 2^-25 however small the result.

    Small probabilities: a probability, times 2^15 over the row's largest and
    times its block's scale over a power of two of at most twice the largest, is held
    in f16, whose step ends at 2^-24: off by 2^-25 more, times a code of up to 127.  Over
    the sum (at least 2^15) that is 2^-39 vtop for each key.  For f16 and bf16 the
    probabilities of many rows are relative to a reference that may lie 2^8 below the
    largest score's: the sum is at least 2^7, and it is 2^-31 vtop."""
    s = prod * (3 * dim + 8) * 2.0 ** -24
    p = np.expm1(s) + 2.0 ** -22 + (2.0 ** -23 if dtype == "f32" else 2.0 ** -11) + 3 * 2.0 ** -24
    rel = 2 * p + (total + 64) * 2.0 ** -24
    floor = total * 2.0 ** (-39 if dtype == "f32" else -31) * vtop[..., None] + (2.0 ** -25 if dtype == "f16" else 0.0)
    return mag * rel[..., None] * 1.01 + EPS[dtype] * mag + floor
