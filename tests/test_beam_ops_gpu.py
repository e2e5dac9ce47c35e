"""Beam selection and state reordering on the GPU against their definitions.

Selection is compared exactly; the inputs' best candidates are first shown (by the 64-bit
reference alone) to lie further apart than the kernel's log-sum can be off: an exponential within 2 ulp,
its argument |x - max| log2(e) rounded twice in f32, each term then off by 2 |x - max| 2^-24;
the weighted mean of |x - max| is the row's entropy at most, so below log(vocab) < 12; f32
sums of at most 32 terms, the rest in 64 bits: 2^-22 + 24 2^-24 + 32 2^-24 < 5e-6.  A score is
rounded once more to f32."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

LSE = 5e-6


@pytest.fixture(scope="module")
def torch():
    import torch
    return torch


def ref_select(x, cum, beams, n_out, done, eos):
    """Lists of (score, parent, token) by the definition, in 64 bits; rows of logits f64."""
    rows, V = x.shape
    res = []
    for g in range(rows // beams):
        c = []
        for b in range(beams):
            r = g * beams + b
            if not cum[r] > -np.inf:
                continue
            if done is not None and done[r]:
                c.append((cum[r], b, eos))
                continue
            y = np.where(np.isnan(x[r]), -np.inf, x[r])
            m = y.max()
            if m == -np.inf:
                continue
            with np.errstate(invalid="ignore", divide="ignore"):
                lp = np.where(y == np.inf, 0.0, -np.inf) - np.log((y == np.inf).sum()) if m == np.inf else \
                    y - m - np.log(np.exp(y - m).sum())
            # n_out + 1 of a row at least, ties included
            kth = np.sort(lp)[::-1][min(n_out, V - 1)]
            c += [(cum[r] + lp[t], b, int(t)) for t in np.nonzero((lp >= kth) & (lp > -np.inf))[0]]
        c.sort(key=lambda e: (-e[0], e[1], e[2]))
        res.append(c)
    return res


def check_select(jd, torch, logits, cum, beams, n_out, done=None, eos=0):
    got = jd.beam_select(logits, cum, beams, n_out, done=done, eos=eos)
    parent, token, score = (t.cpu().numpy() for t in got)
    ref = ref_select(logits.double().cpu().numpy(), cum.double().cpu().numpy(), beams, n_out,
                     None if done is None else done.cpu().numpy(), eos)
    for g, c in enumerate(ref):
        for a, b in zip(c[:n_out], c[1:n_out + 1]):  # the inputs decide: no near ties between rows
            assert a[1] == b[1] or a[0] - b[0] > 2 * LSE or a[0] == b[0]
        want = c[:n_out] + [(-np.inf, -1, -1)] * (n_out - len(c))
        assert [(int(p), int(t)) for p, t in zip(parent[g], token[g])] == [(p, t) for _, p, t in want]
        for s, (w, _, _) in zip(score[g], want):
            assert s == w or abs(s - w) <= LSE + 2.0 ** -24 * abs(w), (s, w)


@pytest.mark.parametrize("dt", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("groups,beams,V,n_out", [
    (1, 1, 1, 1), (1, 1, 5, 8), (1, 4, 8256, 8), (3, 2, 257, 4), (2, 5, 32001, 10), (2, 3, 50257, 32),
    (64, 8, 1003, 16), (1, 64, 2048, 32), (40, 6, 16385, 12), (1, 1, 131071, 1), (2, 2, 7, 14)])
def test_select(jd, torch, dt, groups, beams, V, n_out):
    torch.manual_seed(groups * 1000 + V)
    n = groups * beams
    wide = torch.randn((n, V + 3), device="cuda") * 3
    wide = wide.to(getattr(torch, dt))
    logits = wide[:, 1:V + 1]  # rows that start between vector boundaries, NaN and peaks beside them
    wide[:, 0], wide[:, V + 1:] = float("nan"), 9e4 if dt == "float32" else 6e4
    cum = -torch.rand(n, device="cuda") * 3 - 5
    check_select(jd, torch, logits, cum, beams, n_out)
    done = (torch.rand(n, device="cuda") < 0.4).int()
    check_select(jd, torch, logits.contiguous(), cum, beams, n_out, done=done, eos=min(2, V - 1))


def test_select_first_step_and_dead_rows(jd, torch):
    """All beams equal at the start: only the first lives; dead rows by -inf or NaN; a group that is dead."""
    torch.manual_seed(0)
    x = torch.randn((1, 600), device="cuda").expand(8, 600).contiguous()
    inf = float("inf")
    cum = torch.tensor([0, -inf, -inf, float("nan"), -inf, -inf, -inf, -inf], device="cuda")
    check_select(jd, torch, x, cum, 4, 8)
    check_select(jd, torch, x, torch.full((8,), -1.5, device="cuda"), 4, 8)  # equal rows: lowest parent first


def test_select_ties_masks_and_infinities(jd, torch):
    V = 9000
    inf, nan = float("inf"), float("nan")
    x = torch.full((6, V), -inf, device="cuda")
    x[0, [5, 77, 8999]] = torch.tensor([1.0, 1.0, 2.0], device="cuda")
    x[1] = 0.25                                    # every logit equal: the lowest tokens
    x[2, 100:200] = torch.arange(100, device="cuda") % 3 - 0.5
    x[2, 50] = nan
    x[3] = nan
    x[4] = torch.linspace(-1, 1, V, device="cuda")
    x[4, [17, 18]] = inf
    x[5] = torch.finfo(torch.float32).min          # the type's lowest value is a value
    x[5, 4000] = -0.0
    x[5, 4001] = 0.0
    cum = torch.tensor([-1.0, -9.0, -2.0, -3.0, -4.0, -5.0], device="cuda")
    for n_out in (1, 7, 32):
        for i in range(6):
            check_select(jd, torch, x[i:i + 1], cum[i:i + 1], 1, n_out)
        check_select(jd, torch, x[[0, 2, 3, 4]], cum[[0, 2, 3, 4]], 4, n_out)
    many = (torch.arange(2 * V, device="cuda") % 2).float().view(2, V)  # thousands of equal best
    check_select(jd, torch, many, cum[[0, 1]], 2, 32)
    # an adversarial slice: all large numbers in few threads' places
    y = torch.randn((1, V), device="cuda")
    y.view(-1)[: 4 * 40] += 50
    check_select(jd, torch, y, cum[:1], 1, 32)


def test_select_replays(jd, torch):
    torch.manual_seed(4)
    x = torch.randn((8, 5000), device="cuda")
    cum = torch.zeros(8, device="cuda")
    jd.beam_select(x, cum, 4, 8)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        res = jd.beam_select(x, cum, 4, 8)
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        cum.copy_(torch.randn_like(cum))
        g.replay()
        torch.cuda.synchronize()
        want = jd.beam_select(x, cum, 4, 8)
        assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_select_refusals(jd, torch):
    x, cum = torch.randn((4, 10), device="cuda"), torch.zeros(4, device="cuda")
    for call in (lambda: jd.beam_select(x, cum, 3, 2), lambda: jd.beam_select(x, cum[:3], 2, 2),
                 lambda: jd.beam_select(x.t(), cum, 2, 2), lambda: jd.beam_select(x.double(), cum, 2, 2),
                 lambda: jd.beam_select(x, cum, 2, 0), lambda: jd.beam_select(x, cum, 2, 40),
                 lambda: jd.beam_select(x, cum, 2, 2, done=cum), lambda: jd.beam_select(x.cpu(), cum, 2, 2),
                 lambda: jd.beam_select(x, cum, 2, 2, done=torch.zeros(4, dtype=torch.int32, device="cuda"), eos=10)):
        with pytest.raises(jd.JdError):
            call()


# ------------------------------------------------------------------------------------ reorder
@pytest.mark.parametrize("groups,beams", [(1, 1), (1, 4), (3, 5), (2, 64)])
def test_reorder(jd, torch, groups, beams):
    """States of any size and alignment; rows as slices of wider ones; negative and bad parents."""
    torch.manual_seed(beams)
    n = groups * beams
    wide = torch.randint(0, beams, (groups, 2 * beams), dtype=torch.int32, device="cuda")
    parent = wide[:, :beams]
    if beams > 3:
        parent[0, 1] = -1
        parent[groups - 1, 3] = -9
    states = []
    for size in (1, 3, 4, 15, 16, 17, 31, 32, 48, 100, 4099, 32768, 32769, 70001):
        for shift in ((0, 0), (1, 0), (0, 5), (3, 11), (8, 8))[: 5 if size < 100 else 4]:
            src = torch.randint(0, 256, (n, size + 16), dtype=torch.uint8, device="cuda")
            dst = torch.full((n, size + 16), 7, dtype=torch.uint8, device="cuda")
            states.append((src[:, shift[0]:shift[0] + size], dst[:, shift[1]:shift[1] + size], dst))
    rows = (parent + torch.arange(groups, device="cuda")[:, None] * beams).flatten()
    keep = (parent < 0).flatten()
    for i in range(0, len(states), 16):
        part = states[i:i + 16]
        want = []
        for s, d, whole in part:
            w = whole.clone()
            off = d.storage_offset()
            w[~keep, off:off + s.shape[1]] = s[rows[~keep]]
            want.append(w)
        st = torch.zeros(1, dtype=torch.int32, device="cuda")
        jd.beam_reorder(parent, [(s, d) for s, d, _ in part], status=st)
        assert int(st) == 0
        for (s, d, whole), w in zip(part, want):
            assert torch.equal(whole, w), (s.shape, s.storage_offset(), d.storage_offset())


def test_reorder_types_bad_parent_and_replay(jd, torch):
    src = [torch.randn((4, 3, 7), device="cuda"), torch.arange(4, dtype=torch.int64, device="cuda"),
           torch.zeros((4, 0), device="cuda")]
    dst = [torch.zeros_like(s) for s in src]
    parent = torch.tensor([[1, 1], [4, 0]], dtype=torch.int32, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    jd.beam_reorder(parent, list(zip(src, dst)), status=st)
    assert int(st) == 32
    for s, d in zip(src[:2], dst[:2]):
        assert torch.equal(d[[0, 1, 3]], s[[1, 1, 2]]) and not d[2].any()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        jd.beam_reorder(parent, list(zip(src, dst)))
    parent.copy_(torch.tensor([[0, 1], [1, 0]]))
    g.replay()
    assert torch.equal(dst[0], src[0][[0, 1, 3, 2]])
    with pytest.raises(jd.JdError):
        jd.beam_reorder(parent, [(src[0], src[0])])
    with pytest.raises(jd.JdError):
        jd.beam_reorder(parent, [(src[0], dst[0].double())])
    with pytest.raises(jd.JdError):
        jd.beam_reorder(parent, [(src[0][:2], dst[0][:2])])
