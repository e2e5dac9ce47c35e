"""The paged cache on the GPU: append (head norms, rotation, scatter) and the attention behind a
shared prefix, against their formulas in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of f32, e = finfo(type).eps / 2 half a step
of the stored type (zero extra for f32 beyond u).

append: a stored number is one rounding of a f32 value whose chain is: the sum of squares (a
tree of head_dim + 13 roundings, halved by the root), rsqrt (2 ulp), two products, two products
and a sum: below 32 u of the head's largest |number|, plus e of the result.

attention: delta bounds the error of a score: the dot product of head_dim f32 products
((head_dim + 4) u sum |q k| scale), the f32 chain behind it (8 u of the score, tanh's 2 ulp
included) and ex2.approx (2^-22); with 16-bit types a clamped score is c - 2c / (1 + e^2x), whose
exponential and quotient put it off by 2^-21 c at most; an exponential on the FMA units is within
2^-22 as well.  A weight is off by 2 delta, sums over n rows by n u; with
16-bit types the weights of the second product are rounded once (e each), and in f16 weights
below 2^-24 of the running scale vanish (n 2^-25 of the largest |v|).  So
|out - ref| <= e |ref| + (2 delta + e + (n + 8) u) sum p |v| (+ n 2^-25 max|v| for f16),
|lse - ref| <= delta + (n + 8) u + 2 u |ref|.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTS = ["float32", "float16", "bfloat16"]


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def half_step(torch, dt):
    return 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2


def angles(torch, n, rot):
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    a = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return a.cos().float().cuda(), a.sin().float().cuda()


def make_kv(jd, torch, dt, n_pages, page, kv_heads, hd, table, order="row", fill=None):
    """Pools in page-row-head order, or with the heads outside the rows."""
    shape = (n_pages, page, kv_heads, hd) if order == "row" else (n_pages, kv_heads, page, hd)
    mk = (lambda: torch.full(shape, fill, dtype=dt, device="cuda")) if fill is not None else \
        (lambda: torch.randn(shape, device="cuda").to(dt))
    k, v = mk(), mk()
    if order != "row":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    return jd.PagedKV(k, v, torch.as_tensor(table, dtype=torch.int32, device="cuda"))


# ------------------------------------------------------------------------------------ append
def ref_heads(x, w, eps, cos, sin, pos, rot, norm_pairs):
    """x [n][heads][hd] f64 -> normalised and rotated, f64."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    y = x.copy()
    if rot:
        a = np.arange(0, rot, 2) if norm_pairs else np.arange(rot // 2)
        b = a + 1 if norm_pairs else a + rot // 2
        c, s = cos[pos][:, None].astype(np.float64), sin[pos][:, None].astype(np.float64)
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def close_heads(torch, got, ref, dt):
    got = got.double().cpu().numpy()
    lim = half_step(torch, dt) * np.abs(ref) + 32 * U * np.abs(ref).max(-1, keepdims=True) * 2
    assert np.all(np.abs(got - ref) <= lim), float(np.max(np.abs(got - ref) / lim))


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("cache", DTS)
@pytest.mark.parametrize("heads,kvh,hd,rot,pairs,norm,page,n", [
    (12, 4, 64, 64, False, False, 1, 1),
    (12, 4, 64, 64, False, False, 16, 37),
    (32, 8, 128, 128, True, True, 16, 5),
    (4, 2, 80, 40, False, True, 8, 19),
    (14, 2, 96, 96, True, False, 64, 130),
    (3, 1, 256, 128, False, True, 1024, 9),
    (1, 1, 8, 8, True, True, 2, 300),
    (40, 40, 128, 0, False, True, 32, 3),
])
def test_append(jd, torch, dt, cache, heads, kvh, hd, rot, pairs, norm, page, n):
    torch.manual_seed(n * 7 + hd)
    rng = np.random.default_rng(n + hd)
    dt, cache = getattr(torch, dt), getattr(torch, cache)
    seqs = min(n, 3)
    seq = np.sort(rng.integers(0, seqs, n)).astype(np.int32)
    pos = np.zeros(n, np.int32)
    for s in range(seqs):
        pos[seq == s] = 5 + np.arange((seq == s).sum())
    perm = rng.permutation(n)  # tokens in any order
    seq, pos = seq[perm], pos[perm]
    per = (int(pos.max()) + page) // page
    table = rng.permutation(seqs * per + 2)[:seqs * per].reshape(seqs, per)
    kv = make_kv(jd, torch, cache, seqs * per + 2, page, kvh, hd, table, fill=7.0,
                 order="row" if n % 2 else "head")
    row = torch.randn((n, (heads + 2 * kvh) * hd), device="cuda").to(dt)
    q, k, v = (row[:, a * hd:b * hd].unflatten(1, (b - a, hd)) for a, b in
               ((0, heads), (heads, heads + kvh), (heads + kvh, heads + 2 * kvh)))
    cos, sin = angles(torch, int(pos.max()) + 1, rot) if rot else (None, None)
    w = (torch.rand(hd, device="cuda") + 0.5, torch.rand(hd, device="cuda") + 0.5) if norm else (None, None)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    before = row.clone()
    got = jd.paged_append(kv, q, k, v, torch.from_numpy(seq).cuda(), torch.from_numpy(pos).cuda(), cos, sin,
                          rope_norm=pairs, q_norm=w[0], k_norm=w[1], eps=1e-5, status=status)
    assert int(status) == 0 and torch.equal(row, before)
    h = [x.double().cpu().numpy() for x in (q, k, v)]
    wn = [None if x is None else x.double().cpu().numpy() for x in w]
    cs = (None, None) if cos is None else (cos.cpu().numpy(), sin.cpu().numpy())
    close_heads(torch, got, ref_heads(h[0], wn[0], 1e-5, *cs, pos, rot, pairs), cache)
    pg, r = torch.from_numpy(table[seq, pos // page]).cuda(), torch.from_numpy(pos % page).long().cuda()
    close_heads(torch, kv.k[pg, r], ref_heads(h[1], wn[1], 1e-5, *cs, pos, rot, pairs), cache)
    assert torch.equal(kv.v[pg, r], v.float().to(cache))
    # every other row of the pools is as it was
    kv.k[pg, r] = 7.0
    kv.v[pg, r] = 7.0
    assert bool((kv.k == 7.0).all()) and bool((kv.v == 7.0).all())


def test_append_padding_bad_entries_and_in_place(jd, torch):
    """Padding tokens and entries outside the tables are left out; the others are written, the
    queries in place; each kind of bad entry raises its own flag."""
    n, kvh, hd = 8, 2, 64
    kv = make_kv(jd, torch, torch.float32, 4, 4, kvh, hd, [[0, 1], [2, 9], [3, -5]], fill=7.0)
    q, k, v = (torch.randn((n, 2, hd), device="cuda") for _ in range(3))
    cos, sin = angles(torch, 7, hd)
    for seq, pos, flag in [([0, 1, 0, -1, 2, 0, 1, 0], [0, 1, 2, 3, 3, -1, 3, 5], 0),
                           ([0, 1, 0, -1, 3, 0, 1, 0], [0, 1, 2, 3, 3, -1, 3, 5], 32),
                           ([0, 1, 0, -1, 2, 0, 1, 0], [0, 1, 2, 3, 8, -1, 3, 5], 2),
                           ([0, 1, 0, -1, 2, 0, 1, 0], [0, 1, 2, 3, 7, -1, 3, 5], 2),   # past the angles
                           ([0, 1, 0, -1, 1, 0, 1, 0], [0, 1, 2, 3, 4, -1, 3, 5], 64),
                           ([0, 1, 0, -1, 2, 0, 1, 0], [0, 1, 2, 3, 5, -1, 3, 5], 64)]:
        kv.k.fill_(7.0)
        kv.v.fill_(7.0)
        mine = q.clone()
        st = torch.zeros(1, dtype=torch.int32, device="cuda")
        s, p = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (seq, pos))
        out = jd.paged_append(kv, mine, k, v, s, p, cos, sin, out=mine, status=st)
        assert out is mine and int(st) == flag
        good = [i for i in range(n) if seq[i] >= 0 and pos[i] >= 0 and not (i == 4 and flag)]
        ref = ref_heads(q.double().cpu().numpy()[good], None, 0, cos.cpu().numpy(), sin.cpu().numpy(),
                        np.array(pos)[good], hd, False)
        close_heads(torch, mine[good], ref, torch.float32)
        bad = [i for i in range(n) if i not in good]
        assert torch.equal(mine[bad], q[bad])
        rows = sum(1 for i in good)
        assert int((kv.v != 7.0).any(-1).any(-1).sum()) == rows


def test_append_keys_and_values_only_and_no_tokens(jd, torch):
    kv = make_kv(jd, torch, torch.bfloat16, 2, 4, 2, 64, [[1, 0]], fill=7.0)
    k, v = (torch.randn((3, 2, 64), device="cuda", dtype=torch.bfloat16) for _ in range(2))
    i32 = dict(dtype=torch.int32, device="cuda")
    assert jd.paged_append(kv, None, k, v, torch.zeros(3, **i32), torch.arange(3, 6, **i32)) is None
    assert torch.equal(kv.k[1, 3], k[0]) and torch.equal(kv.k[0, :2], k[1:]) and torch.equal(kv.v[0, :2], v[1:])
    jd.paged_append(kv, None, k[:0], v[:0], torch.zeros(0, **i32), torch.zeros(0, **i32))


def test_append_far_rows(jd, torch):
    """Rows whose offset in the pool passes 2^31 elements."""
    n_pages, page, kvh, hd = 1100, 1024, 16, 128   # 2.3e9 elements a pool
    k = torch.empty((n_pages, page, kvh, hd), dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    kv = jd.PagedKV(k, v, torch.tensor([[n_pages - 1, 0], [n_pages - 2, 1]], dtype=torch.int32, device="cuda"))
    n = 40
    x = torch.randn((n, kvh, hd), device="cuda", dtype=torch.bfloat16)
    y = torch.randn((n, kvh, hd), device="cuda", dtype=torch.bfloat16)
    pos = torch.arange(1000, 1000 + n, dtype=torch.int32, device="cuda")
    seq = torch.zeros(n, dtype=torch.int32, device="cuda")
    jd.paged_append(kv, None, x, y, seq, pos)
    assert torch.equal(torch.cat([k[n_pages - 1, 1000:], k[0, :16]]), x)
    assert torch.equal(torch.cat([v[n_pages - 1, 1000:], v[0, :16]]), y)
    # and the attention reads them: one query for each of two sequences, the second without rows
    q = torch.randn((2, kvh, hd), device="cuda", dtype=torch.bfloat16)
    k[n_pages - 1, :1000] = 0
    v[n_pages - 1, :1000] = 0
    out, lse = jd.paged_attn(kv, q, torch.tensor([1040, 0], dtype=torch.int32, device="cuda"), 1040)
    s = torch.einsum("hd,thd->ht", q[0].double(), torch.cat([k[n_pages - 1], k[0, :16]]).double()) / math.sqrt(hd)
    p = torch.softmax(s, -1)
    ref = torch.einsum("ht,thd->hd", p, torch.cat([v[n_pages - 1], v[0, :16]]).double())
    assert float((out[0].double() - ref).abs().max()) <= 2 ** -8 * float(ref.abs().max()) * 3 + 1e-4
    assert not out[1].any() and bool((lse[1] == float("-inf")).all())


# ------------------------------------------------------------------------------------ attention
def ref_attn(torch, kv, q, lens, prefix, prefix_len, scale, clamp):
    """(out, lse, sum p |v|, delta, rows) in 64 bits, sequence by sequence."""
    B, H, hd = q.shape
    n_pages, P, KV = kv.k.shape[:3]
    G = H // KV
    out = torch.zeros((B, H, hd), dtype=torch.float64, device="cuda")
    wabs = torch.zeros_like(out)
    lse = torch.full((B, H), float("-inf"), dtype=torch.float64, device="cuda")
    delta = torch.zeros((B, H), dtype=torch.float64, device="cuda")
    rows = torch.zeros(B, dtype=torch.int64)

    def gather(pages, n):
        t = torch.arange(n, device="cuda")
        pg, r = pages.long()[t // P], t % P
        ok = (pg >= 0) & (pg < n_pages)
        return kv.k[pg[ok], r[ok]].double(), kv.v[pg[ok], r[ok]].double()

    kp, vp = gather(prefix, prefix_len) if prefix_len else gather(kv.table[0], 0)
    for b in range(B):
        if lens[b] < 0:
            continue
        km, vm = gather(kv.table[b], int(lens[b]))
        k, v = torch.cat([kp, km]).repeat_interleave(G, 1), torch.cat([vp, vm]).repeat_interleave(G, 1)
        rows[b] = k.shape[0]
        if not rows[b]:
            continue
        s = torch.einsum("hd,thd->ht", q[b].double(), k) * scale
        mag = torch.einsum("hd,thd->ht", q[b].double().abs(), k.abs()).amax(-1) * scale
        if clamp:
            s = clamp * torch.tanh(s / clamp)
        lse[b] = torch.logsumexp(s, -1)
        p = torch.exp(s - lse[b][:, None])
        out[b] = torch.einsum("ht,thd->hd", p, v)
        wabs[b] = torch.einsum("ht,thd->hd", p, v.abs())
        delta[b] = (hd + 4) * U * mag + 8 * U * s.abs().amax(-1) * 2 + 2.0 ** -22
    return out, lse, wabs, delta, rows


def check_attn(torch, kv, q, lens, got, prefix=None, prefix_len=0, scale=None, clamp=0.0):
    scale = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    out, lse, wabs, delta, rows = ref_attn(torch, kv, q, lens, prefix, prefix_len, scale, clamp)
    e = half_step(torch, q.dtype)
    if e and clamp:
        delta = delta + clamp * 2.0 ** -21
    n = rows.cuda().double()[:, None]
    vmax = torch.nan_to_num(kv.v.double(), nan=0.0).abs().max()
    lim = max(e, U) * out.abs() + (2 * delta + e + (n + 8) * U)[..., None] * wabs
    if q.dtype == torch.float16:
        lim = lim + (n * 2.0 ** -25 * vmax)[..., None]
    live = torch.tensor([int(x) >= 0 for x in lens], device="cuda")
    go, gl = got[0].double(), got[1].double()
    bad = ((go - out).abs() > lim) | ~torch.isfinite(go)
    assert not bool(bad[live].any()), float(((go - out).abs() / lim.clamp(min=1e-30))[live].max())
    none = (rows.cuda() == 0)[:, None] & live[:, None]
    assert bool(((gl == float("-inf")) == none)[live].all())
    err = (gl - lse).abs()
    some = live[:, None] & ~none
    assert bool((err <= delta + (n + 8) * U + 2 * U * lse.abs())[some.expand_as(err)].all()), float(err[some.expand_as(err)].max())


def build(jd, torch, dt, B, H, KV, hd, page, prefix_len, lens, seed=0, order="row", scale_q=2.0, junk=float("nan")):
    """Shuffled pages; every row that no sequence reaches holds junk."""
    rng = np.random.default_rng(seed)
    torch.manual_seed(seed)
    max_len = max([1] + [int(x) for x in lens])
    per, shared = -(-max_len // page), -(-prefix_len // page)
    perm = rng.permutation(B * per + shared + 1)
    table = perm[shared:shared + B * per].reshape(B, per)
    kv = make_kv(jd, torch, dt, B * per + shared + 1, page, KV, hd, table, order=order)
    reach = torch.zeros(kv.k.shape[:2], dtype=torch.bool, device="cuda")

    def mark(pages, n):
        t = torch.arange(n, device="cuda")
        reach[torch.as_tensor(pages, device="cuda").long()[t // page], t % page] = True

    mark(perm[:shared] if shared else [0], prefix_len)
    for b in range(B):
        mark(table[b], max(0, int(lens[b])))
    for x in (kv.k, kv.v):
        x.masked_fill_(~reach[:, :, None, None], junk)
    prefix = torch.as_tensor(perm[:shared].copy(), dtype=torch.int32, device="cuda")
    q = (torch.randn((B, H, hd), device="cuda") * scale_q).to(dt)
    return kv, q, torch.tensor([int(x) for x in lens], dtype=torch.int32, device="cuda"), prefix, max_len


SHAPES = [(12, 4, 64), (32, 8, 128), (16, 1, 64), (14, 2, 96), (8, 8, 80), (4, 2, 40), (24, 1, 128)]


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("H,KV,hd", SHAPES)
@pytest.mark.parametrize("page,prefix_len,lens", [
    (1, 0, [1]),
    (1, 5, [0]),
    (16, 0, [0, 1, 15, 16, 17, 33]),
    (64, 129, [0, 3, 200, 64]),
    (8, 512, [7, 1, 40, 9, 128, 0, 2, 77]),
    (256, 1000, [300]),
])
def test_attn(jd, torch, dt, H, KV, hd, page, prefix_len, lens):
    dt = getattr(torch, dt)
    kv, q, ln, prefix, max_len = build(jd, torch, dt, len(lens), H, KV, hd, page, prefix_len, lens, seed=hd + page,
                                       order="head" if page == 64 else "row")
    got = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=prefix_len)
    check_attn(torch, kv, q, lens, got, prefix, prefix_len)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("B,H,KV,hd,page,prefix_len,top", [
    (40, 12, 4, 64, 16, 777, 90),       # 120 queries of a KV head: one 128-row tile, not full
    (64, 32, 8, 128, 64, 1500, 130),    # 256 queries
    (97, 12, 4, 64, 1, 300, 60),        # 291 queries: three tiles, the last with 35
    (33, 14, 2, 96, 32, 129, 700),
    (3, 8, 2, 128, 16, 5000, 4000),     # long and few: split over many parts
    (130, 8, 8, 80, 8, 257, 20),        # one query head to a KV head
    (5, 48, 1, 64, 128, 640, 300),
])
@pytest.mark.parametrize("clamp", [0.0, 30.0])
def test_attn_batches(jd, torch, dt, B, H, KV, hd, page, prefix_len, top, clamp):
    dt = getattr(torch, dt)
    lens = np.random.default_rng(B).integers(0, top + 1, B)
    lens[0] = top
    kv, q, ln, prefix, max_len = build(jd, torch, dt, B, H, KV, hd, page, prefix_len, lens, seed=B, scale_q=6.0)
    got = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=prefix_len, clamp=clamp)
    check_attn(torch, kv, q, lens, got, prefix, prefix_len, clamp=clamp)


@pytest.mark.parametrize("dt", [d for d in DTS if d != "float32"])
@pytest.mark.parametrize("B,H,KV,hd,prefix_len,top", [
    (8, 32, 8, 128, 1024, 900),     # own rows beside a few parts
    (8, 32, 8, 128, 1000, 8),
    (64, 32, 8, 128, 1500, 130),    # two tiles of queries
    (64, 32, 8, 128, 300, 2500),    # own rows that outweigh the shared ones
    (40, 32, 4, 64, 5000, 0),
    (320, 64, 16, 64, 140, 40),     # as many blocks of queries as SMs, and more
    (640, 64, 16, 64, 200, 33),
    (3, 16, 1, 80, 9000, 700),
])
def test_attn_shared_rows_and_own_ones_beside_them(jd, torch, dt, B, H, KV, hd, prefix_len, top):
    """Numbers of parts and of SMs for the own rows from all ends of the estimate."""
    dt = getattr(torch, dt)
    lens = np.random.default_rng(B + top).integers(0, top + 1, B)
    lens[0], lens[-1] = top, -1
    kv, q, ln, prefix, max_len = build(jd, torch, dt, B, H, KV, hd, 16, prefix_len, lens, seed=B)
    got = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=prefix_len)
    check_attn(torch, kv, q, lens, got, prefix, prefix_len)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("prefix_len", [0, 70])
@pytest.mark.parametrize("kind", ["few", "many", "none", "one"])
def test_attn_uneven_lengths(jd, torch, dt, prefix_len, kind):
    """Own rows shared out over the CTAs whatever the lengths: many sequences with most of them empty
    or idle, one long among short ones, none with rows."""
    dt = getattr(torch, dt)
    rng = np.random.default_rng(8)
    lens = {"few": rng.integers(-1, 2, 700), "many": rng.integers(0, 300, 300), "none": np.zeros(40, int),
            "one": np.array([0, 3, 6000, 1, 0, 0, 129, 128, -1])}[kind]
    kv, q, ln, prefix, _ = build(jd, torch, dt, len(lens), 8, 2, 64, 16, prefix_len, lens, seed=6)
    max_len = min(6000, kv.table.shape[1] * 16)
    got = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=prefix_len)
    check_attn(torch, kv, q, lens, got, prefix, prefix_len)
    if kind == "few":  # a long table, short rows
        kv2 = kv.with_table(torch.cat([kv.table] + [torch.zeros_like(kv.table)] * 60, 1).contiguous())
        again = jd.paged_attn(kv2, q, ln, 900, prefix=prefix, prefix_len=prefix_len)
        check_attn(torch, kv2, q, lens, again, prefix, prefix_len)


@pytest.mark.parametrize("dt", DTS)
def test_attn_growing_scores(jd, torch, dt):
    """Scores that rise along the rows, so that the running maximum moves all the way, then fall."""
    dt = getattr(torch, dt)
    B, H, KV, hd, n = 50, 8, 2, 64, 900
    kv, q, ln, prefix, max_len = build(jd, torch, dt, B, H, KV, hd, 16, n, [30] * B, seed=3)
    t = torch.arange(n, device="cuda")
    ramp = (torch.cat([torch.linspace(-8, 8, 700), torch.linspace(8, -8, 200)])).cuda()
    pg, r = prefix.long()[t // 16], t % 16
    kv.k[pg, r] = (ramp[:, None, None] * torch.ones((KV, hd), device="cuda")).to(dt)
    q.copy_((torch.rand((B, H, 1), device="cuda") * 2 - 1).expand_as(q).to(dt))
    got = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=n)
    check_attn(torch, kv, q, [30] * B, got, prefix, n)


@pytest.mark.parametrize("dt", DTS)
@pytest.mark.parametrize("prefix_len", [0, 40])
def test_attn_idle_slots_strides_and_bad_entries(jd, torch, dt, prefix_len):
    """Idle slots keep their outputs; q and out as slices of wider rows; a length above max_len is
    cut, a page outside the pool left out, and both are flagged."""
    dt = getattr(torch, dt)
    B, H, KV, hd, page = 6, 8, 2, 64, 8
    lens = [20, -1, 24, 0, 9, -7]
    kv, q, ln, prefix, max_len = build(jd, torch, dt, B, H, KV, hd, page, prefix_len, lens, seed=5)
    wide = torch.full((B, H * hd + 64), 7.0, dtype=dt, device="cuda")
    qw = torch.zeros((B, 2 * H * hd), dtype=dt, device="cuda")
    qs = qw[:, H * hd:].unflatten(1, (H, hd))
    qs.copy_(q)
    out, lse = wide[:, :H * hd].unflatten(1, (H, hd)), torch.full((B, H), 7.0, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = jd.paged_attn(kv, qs, ln, max_len, prefix=prefix, prefix_len=prefix_len, out=out, lse=lse, status=st)
    assert got[0] is out and int(st) == 0
    check_attn(torch, kv, q, lens, got, prefix, prefix_len)
    for b in (1, 5):
        assert bool((out[b] == 7.0).all()) and bool((lse[b] == 7.0).all())
    assert bool((wide[:, H * hd:] == 7.0).all())
    # a length above max_len is cut there
    got = jd.paged_attn(kv, q, ln, 16, prefix=prefix, prefix_len=prefix_len, status=st)
    assert int(st) == 2
    check_attn(torch, kv, q, [min(x, 16) for x in lens], got, prefix, prefix_len)
    # bad pages: left out
    st.zero_()
    kv.table[0, 1] = kv.k.shape[0]
    kv.table[2, 0] = -3
    if prefix_len:
        prefix[2] = 1 << 30
    got = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=prefix_len, status=st)
    assert int(st) == 64
    check_attn(torch, kv, q, lens, got, prefix, prefix_len)


@pytest.mark.parametrize("dt", DTS)
def test_attn_all_slots_idle(jd, torch, dt):
    """Nothing to write, a long prefix all the same: the outputs stay, and the work behind the call finds
    the workspace free."""
    dt = getattr(torch, dt)
    kv, q, ln, prefix, max_len = build(jd, torch, dt, 40, 8, 2, 64, 16, 3000, [20] * 40, seed=7)
    want = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=3000)
    idle = torch.full_like(ln, -1)
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    for _ in range(20):
        jd.paged_attn(kv, q, idle, max_len, prefix=prefix, prefix_len=3000, out=out, lse=lse)
        again = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=3000)  # the same workspace as a rule
        assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
    assert bool((out == 7.0).all()) and bool((lse == 7.0).all())


def test_attn_is_repeatable_and_replays(jd, torch):
    """The same call gives the same bits; a captured append and attention replay on new inputs, on
    another stream, and two graphs that were captured one after the other run in either order."""
    B, H, KV, hd, page = 9, 8, 2, 128, 16
    lens = [5, 30, 0, 17, 64, 1, 2, 33, 48]
    kv, q, ln, prefix, max_len = build(jd, torch, torch.bfloat16, B, H, KV, hd, page, 300, lens, seed=9)
    a = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=300)
    for _ in range(3):
        b = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=300)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    cos, sin = angles(torch, 80, hd)
    x = torch.randn((B, (H + 2 * KV) * hd), device="cuda").to(torch.bfloat16)
    seq = torch.arange(B, dtype=torch.int32, device="cuda")
    pos = torch.tensor([max(0, n - 1) for n in lens], dtype=torch.int32, device="cuda")

    def step(x):
        h = [x[:, :H * hd].unflatten(1, (H, hd)), x[:, H * hd:(H + KV) * hd].unflatten(1, (KV, hd)),
             x[:, (H + KV) * hd:].unflatten(1, (KV, hd))]
        r = jd.paged_append(kv, *h, seq, pos, cos, sin)
        return jd.paged_attn(kv, r, ln, max_len, prefix=prefix, prefix_len=300)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.synchronize()
    x2 = torch.randn_like(x)
    graphs = []
    for src in (x, x2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step(src)
        graphs.append((g, src, res))
    for order in ((0, 1), (1, 0), (1, 1)):
        for i in order:
            g, src, res = graphs[i]
            src.copy_(torch.randn_like(src))
            g.replay()
            torch.cuda.synchronize()
            want = step(src)
            assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1])


@pytest.mark.parametrize("dt", DTS)
def test_attn_nan_of_a_read_row_shows(jd, torch, dt):
    """A NaN in a row that a sequence reads is not hidden; the other sequences do not see it."""
    dt = getattr(torch, dt)
    for prefix_len, clamp in ((0, 0.0), (20, 0.0), (20, 30.0)):
        kv, q, ln, prefix, max_len = build(jd, torch, dt, 3, 4, 2, 64, 8, prefix_len, [9, 9, 9], seed=4)
        kv.k[kv.table[1, 1].long(), 0, 1, 5] = float("nan")
        out, lse = jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=prefix_len, clamp=clamp)
        assert bool(torch.isnan(out[1, 2:]).all()) and bool(torch.isnan(lse[1, 2:]).all())
        assert bool(torch.isfinite(out[[0, 2]]).all()) and bool(torch.isfinite(out[1, :2]).all())


def test_attn_refusals(jd, torch):
    kv, q, ln, prefix, max_len = build(jd, torch, torch.bfloat16, 2, 4, 2, 64, 8, 16, [3, 4], seed=1)
    for call in (lambda: jd.paged_attn(kv, q.float(), ln, max_len, prefix=prefix, prefix_len=16),
                 lambda: jd.paged_attn(kv, q, ln.long(), max_len, prefix=prefix, prefix_len=16),
                 lambda: jd.paged_attn(kv, q, ln.cpu(), max_len, prefix=prefix, prefix_len=16),
                 lambda: jd.paged_attn(kv, q, ln, max_len, prefix=prefix, prefix_len=17),
                 lambda: jd.paged_attn(kv, q, ln, 9, prefix=prefix, prefix_len=16),
                 lambda: jd.paged_attn(kv, q[:1], ln, max_len),
                 lambda: jd.paged_attn(kv, q[:, :3], ln, max_len),
                 lambda: jd.paged_attn(kv, q, ln, max_len, out=q),
                 lambda: jd.PagedKV(kv.k, kv.v.float(), kv.table),
                 lambda: jd.PagedKV(kv.k, kv.v, kv.table.long()),
                 lambda: jd.PagedKV(kv.k, kv.v.transpose(1, 2).contiguous().transpose(1, 2), kv.table)):
        with pytest.raises(jd.JdError):
            call()


def test_two_streams_at_once(jd, torch):
    """Two calls that overlap on the GPU do not share a workspace."""
    kv, q, ln, prefix, max_len = build(jd, torch, torch.bfloat16, 16, 32, 8, 128, 16, 3000, [200] * 16, seed=2)
    q2 = torch.randn_like(q)
    want = [jd.paged_attn(kv, x, ln, max_len, prefix=prefix, prefix_len=3000) for x in (q, q2)]
    ss = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(10):
        got = []
        for s, x in zip(ss, (q, q2)):
            with torch.cuda.stream(s):
                got.append(jd.paged_attn(kv, x, ln, max_len, prefix=prefix, prefix_len=3000))
        torch.cuda.synchronize()
        for g, w in zip(got, want):
            assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
