"""Attention over short shared prefixes (hale_kv_share_prefixes) on the GPU, of sequences that are long
enough by themselves for sharing to be of use, against 64 bits within what its roundings add up to."""
import numpy as np
import pytest

from kv_model import encode
from test_gpu_kv import Rig, rig  # noqa: F401
from test_gpu_kv_shared import family

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (16, 1), (12, 4), (40, 5)])
@pytest.mark.parametrize("ways", [2, 9, 31])
def test_head_groups_and_ways(rig, heads, kv_heads, ways):
    r = rig(dim=32, heads=heads, kv_heads=kv_heads, pages=300, seqs=40)
    g = np.random.default_rng(heads)
    r.kv.share_prefixes(1)
    root, seqs = family(r, g, "bf16", 191, ways, [300 + i % 7 for i in range(ways)])
    r.step(g, "bf16", [root] + seqs, [2] + [1] * ways)
    r.check_attention(g, 0, "bf16", [root] + seqs, [2] + [1] * ways)


@pytest.mark.parametrize("prompt", [63, 64, 65, 127, 128, 200])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_prompts_of_any_length(rig, prompt, dtype):
    r = rig(dim=64, heads=8, kv_heads=2, pages=100, seqs=6)
    g = np.random.default_rng(prompt)
    r.kv.share_prefixes(64)
    _, seqs = family(r, g, dtype, prompt, 4, [0, 1, 200, 700])
    r.step(g, dtype, seqs, [1, 3, 1, 1])
    r.check_attention(g, 0, dtype, seqs, [1, 3, 1, 1])


def test_steps_around_the_shortest_that_share(rig):
    """Sequences of 255 to 257 positions: below, nothing is shared and results are those of a cache that never
    shares, to the bit."""
    g = np.random.default_rng(1)
    q = encode(g.standard_normal((4, 8, 64)), "f32")[1]
    for tail, shared in ((54, False), (55, False), (56, True)):
        got = []
        for share in (0, 64):
            r = rig(dim=64, heads=8, kv_heads=2, pages=100, seqs=6)
            gg = np.random.default_rng(tail)
            r.kv.share_prefixes(share)
            _, seqs = family(r, gg, "f32", 200, 4, [tail] * 4)
            r.step(gg, "f32", seqs, [1] * 4)
            got.append(r.attend(0, "f32", q))
            r.check_attention(gg, 0, "f32", seqs, [1] * 4)
        assert (got[0] == got[1]).all() != shared
