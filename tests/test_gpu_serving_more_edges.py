"""The operators over 8-bit pages and shared prefixes and the logits' adjustments at the ends of
their inputs' range, against the 64-bit forms."""
import numpy as np
import pytest

import serving_more_ref as more
from test_gpu_cache8 import decode8
from test_gpu_shared import call

pytestmark = pytest.mark.gpu

TYPES = [("bf16", "bf16"), ("f32", "f32"), ("f32", "bf16")]


def lay(rows, ps=16):
    """Rows [n, ...] of every kv head as pages [P, hkv, ps, ...]: position j in page j / ps."""
    n, hkv = rows.shape[:2]
    pages = np.zeros((-(-n // ps) * ps, hkv, *rows.shape[2:]), rows.dtype)
    pages[:n] = rows
    return np.ascontiguousarray(np.moveaxis(pages.reshape(-1, ps, *pages.shape[1:]), 2, 1))


def both8(rt, q, qk, k, v, out, scale=None, first=0, ps=16):
    """Decode attention over 8-bit rows k, v = (codes [n, hkv, d], scales [n, hkv]) of all sequences of
    q: the paged call's result, and the shared call's, the first `first` positions (whole pages) as a prefix."""
    n, b = k[0].shape[0], q.shape[0]
    kc, vc, ks, vs = (lay(x, ps) for x in (k[0], v[0], k[1], v[1]))
    table = np.tile(np.arange(kc.shape[0], dtype=np.int32), (b, 1))
    cut = first // ps
    y = decode8(rt, q, qk, kc, vc, ks, vs, table, [n] * b, out, scale)
    z = call(rt, q, qk, None, None, (kc, ks, vc, vs), "q8", table[:1], [cut * ps], [0, b], table[:, cut:], [n - cut * ps] * b,
             out, scale)
    return y, z


def rows8(x):
    return more.encode(np.asarray(x, np.float32))


# ---- scales of V's rows ---------------------------------------------------------------

@pytest.mark.parametrize("d,ps", [(64, 16), (128, 16), (256, 16), (96, 16), (128, 7)])
@pytest.mark.parametrize("qk,out", TYPES)
def test_a_value_scale_of_zero_under_the_largest_score(rt, d, ps, qk, out):
    """Keys whose values' scale is 0, whose scores lie hundreds above those of the tiles before: they take all of
    the weight, and the row is what the others have left, next to nothing."""
    rng = np.random.default_rng(d)
    n, hkv = 400, 64  # (and 16 sequences: a wave has several tiles of each)
    k = np.zeros((n, hkv, d), np.float32)
    k[[37, 70, 203, 390], :, 0] = np.array([60, 200, 300, 90])[:, None]
    v = rows8(rng.standard_normal((n, hkv, d)))
    v[1][[37, 70, 203, 390]] = 0
    q = np.zeros((16, hkv, d), np.float32)
    q[:, :, 0] = 1
    for first in (0, 64, 208):
        for y in both8(rt, q, qk, rows8(k), v, out, 1.0, first, ps):
            assert np.isfinite(y).all() and np.abs(y).max() <= 1e-20
