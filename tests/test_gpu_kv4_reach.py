"""Caches of more heads or sequences than one launch takes, as far as the cache's own
limits allow them."""
import numpy as np
import pytest

from test_gpu_kv4 import Cache, positions

pytestmark = pytest.mark.gpu


# more layers x kv heads than 8191 (in layers, in kv heads, in both), more requests than 65535
@pytest.mark.parametrize("nLayers,nSeq,nKV,W,maxSeq", [(9001, 4, 1, 2, 3), (2, 3, 8200, 3, 2), (101, 2, 90, 2, 5), (3, 2, 8191, 1, 2),
                                                      (1, 131082, 1, 2, 2), (2, 65538, 1, 1, 2)])
def test_reorder_of_many_heads_and_requests(fh, nLayers, nSeq, nKV, W, maxSeq):
    rng = np.random.default_rng(nLayers + nSeq)
    lens = rng.integers(-1, maxSeq + 2, nSeq)
    c = Cache(fh, nLayers, nSeq, nKV, 32, maxSeq, lens=lens)
    for a, dtype in ((c.k, np.uint8), (c.v, np.uint8)):
        a.upload(rng.integers(0, 256, c.dims + (16,), dtype=dtype))
    for a in (c.kd, c.vd):
        a.upload(rng.standard_normal(c.dims + (1,)).astype(np.float16))
    c.weight.upload(rng.random(c.dims, dtype=np.float32))
    c.pos.upload(positions(rng, *c.dims))
    before = c.host()
    parent = rng.integers(-1, W + 1, nSeq).astype(np.int32)
    c.call("reorder", fh.DeviceArray.from_numpy(parent), W)
    s = np.arange(nSeq)
    source = s // W * W + np.where((parent >= 0) & (parent < W), parent, s % W)
    moved = np.arange(maxSeq) < np.clip(lens, 0, maxSeq)[source][:, None]  # [sequence, slot]
    got = c.host()
    for i in (0, 1, 2, 3, 6, 7):
        there = moved[None, :, None] if before[i].ndim == 4 else moved[None, :, None, :, None]
        np.testing.assert_array_equal(got[i], np.where(there, before[i][:, source], before[i]))
    np.testing.assert_array_equal(got[4], before[4][source])
    np.testing.assert_array_equal(got[5], before[5][source])
