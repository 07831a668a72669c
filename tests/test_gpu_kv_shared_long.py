"""Attention over long shared prefixes of few heads (hale_kv_share_prefixes) on the GPU, whose rows have many
partial results each, against 64 bits within what its roundings add up to."""
import numpy as np
import pytest

from kv_model import encode
from test_gpu_kv import Rig, rig  # noqa: F401
from test_gpu_kv_shared import family

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dim,heads,kv_heads,prompt,ways", [("f16", 128, 2, 2, 11181, 2), ("bf16", 64, 8, 1, 5000, 3), ("f32", 256, 2, 1, 7238, 2),
                                                                  ("bf16", 16, 4, 1, 20000, 3), ("f32", 80, 16, 2, 4500, 2)])
def test_rows_of_many_parts(rig, dtype, dim, heads, kv_heads, prompt, ways):
    r = rig(dim=dim, heads=heads, kv_heads=kv_heads, pages=prompt // 64 + 20, seqs=5, max_len=prompt + 500)
    g = np.random.default_rng(prompt)
    r.kv.share_prefixes(64)
    _, seqs = family(r, g, dtype, prompt, ways, [5 + 100 * i for i in range(ways)])
    ntok = [1 + i % 2 for i in range(ways)]
    r.step(g, dtype, seqs, ntok)
    r.check_attention(g, 0, dtype, seqs, ntok)
    r.check_attention(g, 0, dtype, seqs, ntok, pad=3, offset=1)


def test_rows_of_more_parts_than_are_brought_at_once(rig):
    """Three levels of 337, 341 and 341 pages in parts of four, 258 with the sequence's own
    (tests/native/kv_shared_worth_check.cpp), and sequences that hold fewer of them."""
    r = rig(dim=16, heads=2, kv_heads=1, pages=1100, seqs=8, max_len=66000)
    g = np.random.default_rng(3)
    r.kv.reserve(22000)
    r.kv.share_prefixes(64)
    a, seqs = family(r, g, "f32", 337 * 64, 2, [0, 341 * 64])
    deep = r.fork(seqs[1], 2)
    r.step(g, "f32", deep[1:], [341 * 64])
    order = [seqs[0], deep[0], deep[1]] + r.fork(deep[1], 1)
    r.step(g, "f32", order, [1] * 4)
    r.check_attention(g, 0, "f32", order, [1] * 4)
