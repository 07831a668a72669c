"""Norms that hand on 8 bits with their rows in the place of their inputs: every pair of places that the
header allows, against the same call with places of its own, to the bit."""
import numpy as np
import pytest

import hale_moe as H
from kv_model import NP, encode
from test_gpu_step_ops import SIZE, bufs  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,rows,n,block,pad,offset", [("f32", 1, 32, 32, 0, 0), ("bf16", 3, 512, 64, 0, 0), ("f16", 9, 544, 32, 8, 0),
                                                         ("bf16", 5, 544, 544, 3, 1), ("f32", 300, 2080, 32, 0, 0), ("f16", 4, 4128, 32, 0, 0),
                                                         ("bf16", 3, 16352, 32, 0, 0), ("f32", 2, 16384, 16384, 4, 0)])
@pytest.mark.parametrize("places", ["x -", "d -", "- x", "- d", "x d", "d x"])
def test_norm_rows_in_place(ctx, bufs, dtype, rows, n, block, pad, offset, places):
    """places: where the sums and where the normed rows go, x or delta; - elsewhere."""
    rng = np.random.default_rng(n + rows)
    stride, size = n + pad, SIZE[dtype]
    w = bufs.put(np.exp(0.3 * rng.normal(size=n)).astype(np.float32))
    raw = [np.full((rows, stride), 7, NP[dtype]) for _ in range(2)]
    for v in raw:
        v[:, :n] = encode(rng.normal(size=(rows, n)), dtype)[0]
    got = []
    for at in ("- -", places):
        d = {k: bufs.put(v, offset * size) for k, v in zip("xd", raw)}
        fresh = [bufs.put(np.full((rows, stride), 5, NP[dtype]), offset * size) for _ in range(2)]
        ds, dy = (d.get(k, f) for k, f in zip(at.split(), fresh))
        q, s = bufs.put(np.full(rows * n, 99, np.int8)), bufs.put(np.full(rows * n // block, 99, np.float32))
        H.rms_norm_q8_device(ctx, dtype, rows, n, d["x"], w, 1e-6, q, s, block=block, d_delta=d["d"], d_sum=ds, d_y=dy, x_stride=stride,
                             delta_stride=stride, sum_stride=stride, y_stride=stride)
        out = [bufs.get(a, NP[dtype], rows * stride).reshape(rows, stride) for a in (ds, dy)]
        for o, k in zip(out, at.split()):
            assert (o[:, n:] == np.array(5 if k == "-" else 7).astype(NP[dtype])).all()
        got.append([o[:, :n] for o in out] + [bufs.get(q, np.int8, rows * n), bufs.get(s, np.float32, rows * n // block)])
        for k in "xd":  # an input that nothing is put in place of stays
            if k not in at:
                assert (bufs.get(d[k], NP[dtype], rows * stride).reshape(rows, stride) == raw["xd".index(k)]).all()
    assert all((a == b).all() for a, b in zip(*got))
