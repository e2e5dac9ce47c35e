"""The attention over a paged cache at the ends of its arguments' ranges: scales of zero and below,
NaN, weights that fall out of f16's range, clamps far above the scores.  Formulas and tolerances as
in test_paged_gpu.py; what differs is derived at each test.
"""
import math  # noqa: F401

import numpy as np
import pytest
from test_paged_gpu import DTS, U, build, check_attn, half_step, ref_attn, torch  # noqa: F401

pytestmark = pytest.mark.gpu

# few queries of a KV head behind the shared rows, one tile of 128 of them, two tiles (the second not full),
# more blocks of queries than SMs, and no shared rows
CALLS = [
    (3, 4, 2, 64, 16, 70, 40),
    (40, 12, 4, 64, 16, 300, 33),
    (20, 14, 2, 96, 32, 513, 60),
    (40, 32, 8, 128, 64, 1000, 90),
    (320, 64, 16, 64, 16, 300, 20),
    (6, 8, 2, 80, 8, 0, 700),
]


def case(jd, torch, dt, B, H, KV, hd, page, prefix_len, top, **kw):
    lens = np.random.default_rng(B + hd).integers(0, top + 1, B)
    lens[0] = top
    kv, q, ln, prefix, max_len = build(jd, torch, getattr(torch, dt), B, H, KV, hd, page, prefix_len, lens,
                                       seed=B + hd, **kw)
    return kv, q, ln, prefix, max_len, lens


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("B,H,KV,hd,page,prefix_len,top", CALLS)
@pytest.mark.parametrize("scale,clamp", [(0.0, 0.0), (0.0, 30.0), (-0.11, 0.0), (-0.3, 30.0), (1e-42, 0.0)])
def test_attn_scale_zero_and_negative(jd, torch, dt, B, H, KV, hd, page, prefix_len, top, scale, clamp):
    """scale 0: every row that counts has the same weight, whatever the masked ones; a negative scale is
    the positive one with -q."""
    kv, q, ln, prefix, max_len, lens = case(jd, torch, dt, B, H, KV, hd, page, prefix_len, top)
    if prefix_len > 200:  # a page outside the pool among the shared ones: its rows are masked
        prefix[1] = -1
    got = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=prefix_len, scale=scale, clamp=clamp)
    check_attn(torch, kv, q if scale >= 0 else -q, lens, got, prefix, prefix_len, scale=abs(scale), clamp=clamp)
