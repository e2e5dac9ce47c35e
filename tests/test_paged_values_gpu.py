"""The attention over a paged cache at the ends of its arguments' ranges: scales of zero and below,
NaN, weights that fall out of f16's range, clamps far above the scores.  Formulas and tolerances as
in test_paged_gpu.py; what differs is derived at each test.
"""
import math

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


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("clamp", [0.0, 30.0, 1000.0])
@pytest.mark.parametrize("B,H,KV,hd,page,prefix_len,top", CALLS[:5])
def test_attn_nan_of_a_shared_row_shows(jd, torch, dt, clamp, B, H, KV, hd, page, prefix_len, top):
    """A NaN in one number of a shared key, at each place of eight: out and lse of every query of that KV
    head are NaN, those of the other heads are not; a NaN of a query stays with the query, and one of an
    idle slot's shows nowhere."""
    kv, q, ln, prefix, max_len, lens = case(jd, torch, dt, B, H, KV, hd, page, prefix_len, top)
    G = H // KV

    def call():
        return jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=prefix_len, clamp=clamp)

    first = prefix_len - prefix_len % 64
    for t in list(range(first - 64, first - 56)) + [0, prefix_len - 1]:
        row = kv.k[prefix[t // page].long(), t % page, KV - 1]
        was = row[5].clone()
        row[5] = float("nan")
        out, lse = call()
        assert bool(torch.isnan(out[:, H - G:]).all()) and bool(torch.isnan(lse[:, H - G:]).all()), t
        assert bool(torch.isfinite(out[:, :H - G]).all()) and bool(torch.isfinite(lse[:, :H - G]).all()), t
        row[5] = was
    q[1, 1, 3] = float("nan")
    ln[0] = -1
    q[0] = float("nan")
    out, lse = call()
    bad = torch.zeros((B, H), dtype=torch.bool, device="cuda")
    bad[1, 1] = True
    assert torch.equal(torch.isnan(lse)[1:], bad[1:]) and torch.equal(torch.isnan(out).all(-1)[1:], bad[1:])
    assert torch.equal(torch.isnan(out).any(-1)[1:], bad[1:])


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("B,H,KV,hd,page,prefix_len,top", CALLS)
@pytest.mark.parametrize("clamp", [30.0, 1000.0])
def test_attn_clamp_of_infinite_scores(jd, torch, dt, B, H, KV, hd, page, prefix_len, top, clamp):
    """Every score is -inf, which the clamp takes to -clamp: all rows that count have the same weight."""
    kv, q, ln, prefix, max_len, lens = case(jd, torch, dt, B, H, KV, hd, page, prefix_len, top)
    if prefix_len > 200:
        prefix[1] = -1
    kv.k[..., 3] = torch.where(kv.k[..., 3].isnan(), kv.k[..., 3], float("inf"))
    q[..., 3] = -1.0
    out, lse = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=prefix_len, clamp=clamp)
    assert bool((out[torch.as_tensor(lens > 0, device="cuda")] != 0).any())
    # the plain formula with scale 0: the same weights, lse without the -clamp
    kv.k[..., 3] = torch.where(kv.k[..., 3].isnan(), kv.k[..., 3], 0.0)
    check_attn(torch, kv, q, lens, (out, lse + clamp), prefix, prefix_len, scale=0.0, clamp=clamp)


@pytest.mark.parametrize("dt", ["float16", "bfloat16"])
@pytest.mark.parametrize("B,H,KV,hd,page,prefix_len,top", CALLS)
def test_attn_many_small_weights(jd, torch, dt, B, H, KV, hd, page, prefix_len, top):
    """One row in 32 has all the weight but 2^-26 for each of the others, and only these have values.  A
    weight is held at 2^7 times its ratio to the running maximum's: in f16, whose smallest step is 2^-24,
    it is off by 2^-25 / 2^7 of the largest at most, and the largest is p of the softmax."""
    kv, q, ln, prefix, max_len, lens = case(jd, torch, dt, B, H, KV, hd, page, prefix_len, top)
    kv.k.masked_fill_(~kv.k.isnan(), 0.0)
    kv.v.masked_fill_(~kv.v.isnan(), 4096.0)
    q.zero_()
    q[..., 0] = 1.0
    for pages, n in [(prefix, prefix_len)] + [(kv.table[b], int(lens[b])) for b in range(B)]:
        t = torch.arange(5, max(5, n), 32, device="cuda")
        kv.k[pages[t // page].long(), t % page, :, 0] = 18.0
        kv.v[pages[t // page].long(), t % page] = 0.0
    out, lse = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=prefix_len, scale=1.0)
    ref, rl, wabs, delta, rows = ref_attn(torch, kv, q, lens, prefix, prefix_len, 1.0, 0.0)
    n = rows.cuda().double()[:, None]
    e = half_step(torch, q.dtype)
    lim = e * ref.abs() + (2 * delta + e + (n + 8) * U)[..., None] * wabs
    if dt == "float16":
        lim = lim + (n * 2.0 ** -32 * 4096 * torch.exp(18.0 - rl))[..., None]
    some = (n > 5)[..., None].expand_as(lim)
    err = (out.double() - ref).abs()
    assert bool((err <= lim)[some].all()), float((err / lim)[some].max())
    assert bool(((lse.double() - rl).abs() <= delta + (n + 8) * U + 2 * U * rl.abs())[some[..., 0]].all())


def top_score(torch, kv, q, lens, prefix, prefix_len, scale, clamp):
    """The largest |score| of each query [n_seqs][heads], in 64 bits."""
    G, P = q.shape[1] // kv.k.shape[2], kv.k.shape[1]
    top = torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
    for b in range(q.shape[0]):
        for pages, n in ((prefix, prefix_len), (kv.table[b], int(lens[b]))):
            if n > 0:
                t = torch.arange(n, device="cuda")
                k = kv.k[pages[t // P].long(), t % P].double().repeat_interleave(G, 1)
                s = (torch.einsum("hd,thd->ht", q[b].double(), k) * scale).abs().amax(-1)
                top[b] = torch.maximum(top[b], clamp * torch.tanh(s / clamp))
    return top


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("B,H,KV,hd,page,prefix_len,top", CALLS)
@pytest.mark.parametrize("clamp,scale_q", [(100.0, 60.0), (500.0, 2.0), (1e3, 2.0), (1e4, 400.0), (1e6, 2.0), (3e38, 2.0)])
def test_attn_wide_clamps(jd, torch, dt, B, H, KV, hd, page, prefix_len, top, clamp, scale_q):
    """Clamps above the scores: what a score is off by goes by the score, not by the clamp.  c tanh(s / c) is
    a polynomial up to |s| = 0.6 c (8 u of the score) and c - 2c / (1 + e^(2 s / c)) above, off by 2^-21 c,
    which is 15 u of a score above c tanh(0.6): 16 u on top of the plain formula's.  16-bit types use the second
    form alone up to a clamp of 512."""
    kv, q, ln, prefix, max_len, lens = case(jd, torch, dt, B, H, KV, hd, page, prefix_len, top, scale_q=scale_q)
    out, lse = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=prefix_len, clamp=clamp)
    scale = 1 / math.sqrt(hd)
    ref, rl, wabs, delta, rows = ref_attn(torch, kv, q, lens, prefix, prefix_len, scale, clamp)
    delta = delta + 16 * U * top_score(torch, kv, q, lens, prefix, prefix_len, scale, clamp)
    if dt != "float32" and clamp <= 512:
        delta = delta + clamp * 2.0 ** -21
    n = rows.cuda().double()[:, None]
    e = half_step(torch, q.dtype)
    vmax = torch.nan_to_num(kv.v.double(), nan=0.0).abs().max()
    lim = max(e, U) * ref.abs() + (2 * delta + e + (n + 8) * U)[..., None] * wabs
    if dt == "float16":
        lim = lim + (n * 2.0 ** -25 * vmax)[..., None]
    some = (n > 0).expand_as(rl)
    err = (out.double() - ref).abs()
    assert bool((err <= lim)[some].all()), float((err / lim)[some].max())
    le = (lse.double() - rl).abs()
    assert bool((le <= delta + (n + 8) * U + 2 * U * rl.abs())[some].all()), float(le[some].max())


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("hd", [8, 24, 56, 72, 104, 120])
@pytest.mark.parametrize("B,H,KV,prefix_len,top", [(2, 4, 2, 150, 200), (40, 12, 4, 300, 33), (100, 8, 2, 500, 9)])
def test_attn_head_dims_of_odd_eights(jd, torch, dt, hd, B, H, KV, prefix_len, top):
    """head_dim an odd multiple of 8: the last step of 16 of the products is half zeros."""
    kv, q, ln, prefix, max_len, lens = case(jd, torch, dt, B, H, KV, hd, 16, prefix_len, top)
    got = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=prefix_len)
    check_attn(torch, kv, q, lens, got, prefix, prefix_len)
