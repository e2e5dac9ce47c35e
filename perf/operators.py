"""What the device operators of a beam or parallel decode cost: a paged key/value cache that tokens are
appended to (with the heads' norms and the position rotation on the way), the attention of a batch whose
sequences share a long prefix, the beams' selection over the vocabulary, and the reordering of the beams'
states.  Each case is one call on device tensors.

`run` is the plain form in elementary torch operations, or, where `own` is true, the framework's calls.
"""
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def package():
    """The framework's Python binding (its folder's name has a dot, so it is loaded by path)."""
    name = "janus_doe_b200"
    if name not in sys.modules:
        folder = os.path.join(ROOT, "janus.doe_b200")
        spec = importlib.util.spec_from_file_location(name, os.path.join(folder, "__init__.py"),
                                                      submodule_search_locations=[folder])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    return sys.modules[name]


# ------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # four beams of the depth-12 own model (12/4 heads of 64) take one step: f32, pages of one row
        dict(name="append_beams", op="append", tokens=4, heads=12, kv_heads=4, hd=64, rot=64, pair="neox", norm=False,
             dt="f32", cache="f32", page=1, seqs=4, start=512),
        # one decode step of 96 sequences on the 8B host shape, heads normed, into a cache of 16-row pages
        dict(name="append_step", op="append", tokens=96, heads=32, kv_heads=8, hd=128, rot=128, pair="norm", norm=True,
             dt="bf16", cache="bf16", page=16, seqs=96, start=1999),
        # prompts of 7 sequences (ragged, 14,339 tokens in all) written to the cache at once
        dict(name="append_prompts", op="append", tokens=14339, heads=32, kv_heads=8, hd=128, rot=128, pair="neox",
             norm=True, dt="bf16", cache="bf16", page=64, seqs=7, start=0),
        # four beams behind a 512-token prompt on the own model, with its clamp: the smallest call
        dict(name="attn_beams", op="attn", seqs=4, heads=12, kv_heads=4, hd=64, dt="f32", page=1, prefix=512,
             max_len=33, clamp=30.0),
        # 256 samples of one 777-token prompt on the own model (f32 cache and clamp)
        dict(name="attn_samples", op="attn", seqs=256, heads=12, kv_heads=4, hd=64, dt="f32", page=16, prefix=777,
             max_len=247, clamp=30.0),
        # 32 sequences of the 8B host shape behind one 2048-token instruction
        dict(name="attn_batch", op="attn", seqs=32, heads=32, kv_heads=8, hd=128, dt="bf16", page=16, prefix=2048,
             max_len=301, clamp=0.0),
        # no shared part: eight long ragged sequences, half precision
        dict(name="attn_ragged", op="attn", seqs=8, heads=32, kv_heads=8, hd=128, dt="f16", page=32, prefix=0,
             max_len=8191, clamp=0.0),
        # 64 sequences that ask about one document of 32,789 tokens: the largest call
        dict(name="attn_document", op="attn", seqs=64, heads=32, kv_heads=8, hd=128, dt="bf16", page=64, prefix=32789,
             max_len=1000, clamp=0.0),
        # one step of four beams over the own model's vocabulary
        dict(name="select_beams", op="select", groups=1, beams=4, vocab=8256, n_out=8, dt="f32", done=False),
        # 48 prompts with six beams each over the 8B host vocabulary, some beams finished
        dict(name="select_batch", op="select", groups=48, beams=6, vocab=128256, n_out=12, dt="f32", done=True),
        # page tables and token histories of four beams
        dict(name="reorder_tables", op="reorder", groups=1, beams=4, row_bytes="4096,2048,48"),
        # contiguous caches of 32 beams (22 layers of 300 rows of 4 x 64 halves): keys and values
        dict(name="reorder_caches", op="reorder", groups=4, beams=8, row_bytes="3379200,3379200"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


SHAPES = [(12, 4), (32, 8), (4, 2), (8, 8), (16, 1), (14, 2)]


def draw(rng):
    op = rng.choice(["append", "attn", "attn", "select", "reorder"])
    if op == "append":
        heads, kv = rng.choice(SHAPES)
        hd = rng.choice([64, 128, 80, 96])
        dt = rng.choice(["f32", "bf16", "f16"])
        cache = rng.choice([dt, "bf16"])
        tokens = _log(rng, 1, 14000 * 48 * 128 * 2 // ((heads + 2 * kv) * hd * SIZE[dt]))
        tokens = min(tokens, 14000)
        return dict(op="append", tokens=tokens, heads=heads, kv_heads=kv, hd=hd, rot=rng.choice([hd, hd, hd // 2]),
                    pair=rng.choice(["neox", "norm"]), norm=rng.random() < 0.5, dt=dt, cache=cache,
                    page=rng.choice([1, 8, 16, 64, 128]), seqs=min(tokens, _log(rng, 1, 256)), start=rng.randrange(0, 3001))
    if op == "attn":
        heads, kv = rng.choice(SHAPES)
        hd = rng.choice([64, 128, 128, 80, 96])
        dt = rng.choice(["f32", "bf16", "bf16", "f16"])
        seqs = _log(rng, 1, 256)
        # the products of the shared part and the bytes of the own parts stay below the largest case's
        top = int(64 * 32 * 128 * 32000 // (seqs * heads * hd) // (4 if dt == "f32" else 1))
        prefix = 0 if rng.random() < 0.15 else _log(rng, 1, max(1, min(32000, top)))
        most = max(1, min(8192, 64 * 1000 * 8 * 128 * 2 // (seqs * kv * hd * SIZE[dt])))
        return dict(op="attn", seqs=seqs, heads=heads, kv_heads=kv, hd=hd, dt=dt, page=rng.choice([1, 8, 16, 64, 128]),
                    prefix=prefix, max_len=_log(rng, 1, most), clamp=rng.choice([0.0, 0.0, 30.0]))
    if op == "select":
        beams = rng.choice([1, 2, 3, 4, 6, 8, 16])
        vocab = _log(rng, 500, 150000)
        groups = _log(rng, 1, max(1, min(64, 48 * 6 * 128256 // (beams * vocab))))
        return dict(op="select", groups=groups, beams=beams, vocab=vocab, n_out=rng.choice([beams, 2 * beams]),
                    dt=rng.choice(["f32", "bf16", "f16"]), done=rng.random() < 0.5)
    groups, beams = rng.choice([1, 2, 4]), rng.choice([2, 4, 8, 5])
    return dict(op="reorder", groups=groups, beams=beams,
                row_bytes=",".join(str(_log(rng, 4, 6000000 // rng.choice([1, 2, 3]))) for _ in range(rng.choice([1, 2, 3]))))


# ------------------------------------------------------------------------------------ the inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 17)
    return g


def _randn(g, shape, dt, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt)


def _angles(n, rot):
    """cos and sin of pos * 10000^(-2i/rot), in 64 bits, kept in 32 as the engine keeps them."""
    inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    a = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * inv[None, :]
    return a.cos().float().contiguous(), a.sin().float().contiguous()


def prepare(case, seed):
    g = _gen(seed)
    st = dict(case)
    rng = np.random.default_rng(int(seed) + 5)
    if case["op"] == "append":
        n, H, KV, hd, P, B = (case[k] for k in ("tokens", "heads", "kv_heads", "hd", "page", "seqs"))
        # the tokens of a fused projection: q, k and v are slices of one row
        st["qkv"] = _randn(g, (n, (H + 2 * KV) * hd), DT[case["dt"]])
        # how many tokens each sequence has goes by the case alone, so that the pools' sizes do too
        ragged = np.random.default_rng(n * 257 + B)
        cut = np.sort(ragged.choice(np.arange(1, n), B - 1, replace=False)) if B > 1 else np.array([], np.int64)
        counts = np.diff(np.concatenate([[0], cut, [n]]))
        seq = np.repeat(np.arange(B), counts)
        pos = np.concatenate([case["start"] + np.arange(c) for c in counts])
        pages = (case["start"] + int(counts.max()) + P - 1) // P
        first = case["start"] // P
        # only the pages that this call writes exist for each sequence; earlier table entries repeat page 0
        per = pages - first
        table = np.zeros((B, pages), np.int32)
        table[:, first:] = rng.permutation(B * per).reshape(B, per)
        st["table"] = torch.from_numpy(table).cuda()
        st["seq"] = torch.from_numpy(seq.astype(np.int32)).cuda()
        st["pos"] = torch.from_numpy(pos.astype(np.int32)).cuda()
        shape = (B * per, P, KV, hd)
        st["k_pool"] = torch.zeros(shape, dtype=DT[case["cache"]], device="cuda")
        st["v_pool"] = torch.zeros(shape, dtype=DT[case["cache"]], device="cuda")
        st["cos"], st["sin"] = _angles(case["start"] + int(counts.max()), case["rot"])
        st["q_norm"] = _randn(g, (hd,), torch.float32, 0.1) + 1 if case["norm"] else None
        st["k_norm"] = _randn(g, (hd,), torch.float32, 0.1) + 1 if case["norm"] else None
        x = st["qkv"]
        st["q"] = x[:, :H * hd].unflatten(1, (H, hd))
        st["k"] = x[:, H * hd:(H + KV) * hd].unflatten(1, (KV, hd))
        st["v"] = x[:, (H + KV) * hd:].unflatten(1, (KV, hd))
    elif case["op"] == "attn":
        B, H, KV, hd, P = (case[k] for k in ("seqs", "heads", "kv_heads", "hd", "page"))
        dt = DT[case["dt"]]
        st["lens"], lens = _lens(case, seed)
        per = (case["max_len"] + P - 1) // P
        shared = (case["prefix"] + P - 1) // P
        order = rng.permutation(B * per + shared).astype(np.int32)
        st["prefix_table"] = torch.from_numpy(order[:shared].copy()).cuda()
        st["table"] = torch.from_numpy(order[shared:].reshape(B, per).copy()).cuda()
        st["k_pool"] = _randn(g, (B * per + shared, P, KV, hd), dt)
        st["v_pool"] = _randn(g, (B * per + shared, P, KV, hd), dt)
        # queries in the scale that a trained head has: a few positions take most of the weight
        st["q"] = _randn(g, (B, H, hd), dt, 2.0)
    elif case["op"] == "select":
        n, V = case["groups"] * case["beams"], case["vocab"]
        x = torch.randn((n, V), generator=g, device="cuda") * 2.5
        hot = torch.randint(0, V, (n, 8), generator=g, device="cuda")
        x.scatter_add_(1, hot, torch.rand((n, 8), generator=g, device="cuda") * 8 + 2)
        st["logits"] = x.to(DT[case["dt"]])
        st["cum"] = -torch.rand((n,), generator=g, device="cuda") * 3 - 20
        st["done"] = None
        if case["done"]:
            st["done"] = (torch.rand((n,), generator=g, device="cuda") < 0.2).to(torch.int32)
    else:
        n = case["groups"] * case["beams"]
        st["parent"] = torch.randint(0, case["beams"], (case["groups"], case["beams"]), generator=g, device="cuda",
                                     dtype=torch.int32)
        st["src"] = [torch.randint(0, 256, (n, b), generator=g, device="cuda", dtype=torch.uint8)
                     for b in _row_bytes(case)]
        st["dst"] = [torch.zeros_like(s) for s in st["src"]]
    if own and case["op"] in ("append", "attn"):
        st["kv"] = package().PagedKV(st["k_pool"], st["v_pool"], st["table"])
    return st


def _row_bytes(case):
    return [int(b) for b in case["row_bytes"].split(",")]


def _lens(case, seed):
    rng = np.random.default_rng(int(seed) + 11)
    lens = rng.integers(0, case["max_len"] + 1, case["seqs"]).astype(np.int32)
    lens[rng.integers(0, case["seqs"])] = case["max_len"]
    return torch.from_numpy(lens).cuda(), lens


# ------------------------------------------------------------------------------------ one pass
def run(st):
    return {"append": _append, "attn": _attn, "select": _select, "reorder": _reorder}[st["op"]](st)


def _rotate(x, cos, sin, rot, pair):
    """x [n][heads][hd] in f32; cos, sin [n][1][rot / 2]."""
    if pair == "neox":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def _rms(x, w):
    return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * w


def _append(st):
    if own:
        q = package().paged_append(st["kv"], st["q"], st["k"], st["v"], st["seq"], st["pos"], st["cos"], st["sin"],
                                   rope_norm=st["pair"] == "norm", q_norm=st["q_norm"], k_norm=st["k_norm"], eps=1e-5)
        return {"q": q, "k_pool": st["k_pool"], "v_pool": st["v_pool"]}
    q, k, v = st["q"].float(), st["k"].float(), st["v"].float()
    if st["norm"]:
        q, k = _rms(q, st["q_norm"]), _rms(k, st["k_norm"])
    pos, P = st["pos"].long(), st["page"]
    cos, sin = st["cos"][pos][:, None], st["sin"][pos][:, None]
    q, k = _rotate(q, cos, sin, st["rot"], st["pair"]), _rotate(k, cos, sin, st["rot"], st["pair"])
    page = st["table"][st["seq"].long(), pos // P].long()
    dt = st["k_pool"].dtype
    st["k_pool"][page, pos % P] = k.to(dt)
    st["v_pool"][page, pos % P] = v.to(dt)
    return {"q": q.to(dt), "k_pool": st["k_pool"], "v_pool": st["v_pool"]}


def _attn(st):
    scale = 1.0 / math.sqrt(st["hd"])
    if own:
        out, lse = package().paged_attn(st["kv"], st["q"], st["lens"], st["max_len"], prefix=st["prefix_table"],
                                        prefix_len=st["prefix"], scale=scale, clamp=st["clamp"])
        return {"out": out, "lse": lse}
    B, H, KV, hd, P, c = (st[k] for k in ("seqs", "heads", "kv_heads", "hd", "page", "clamp"))
    q = st["q"].float().view(B, KV, H // KV, hd)
    t = torch.arange(st["prefix"], device="cuda")
    page = st["prefix_table"].long()[t // P]
    kp, vp = st["k_pool"][page, t % P].float(), st["v_pool"][page, t % P].float()      # [prefix][KV][hd]
    t = torch.arange(st["max_len"], device="cuda")
    page = st["table"].long()[:, t // P]
    ks, vs = st["k_pool"][page, t % P].float(), st["v_pool"][page, t % P].float()      # [B][max_len][KV][hd]
    s = torch.cat([torch.einsum("bkgd,tkd->bkgt", q, kp), torch.einsum("bkgd,btkd->bkgt", q, ks)], -1) * scale
    if c:
        s = c * torch.tanh(s / c)
    beyond = t[None] >= st["lens"][:, None]
    s[..., st["prefix"]:].masked_fill_(beyond[:, None, None], float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > float("-inf"), m, 0.0))
    total = p.sum(-1, keepdim=True)
    o = torch.einsum("bkgt,tkd->bkgd", p[..., :st["prefix"]], vp)
    o = o + torch.einsum("bkgt,btkd->bkgd", p[..., st["prefix"]:], vs)
    o = o / torch.where(total > 0, total, 1.0)
    return {"out": o.reshape(B, H, hd).to(st["q"].dtype), "lse": (m + torch.log(total)).view(B, H)}


EOS = 2


def _select(st):
    n, V, G, beams, k = st["cum"].numel(), st["vocab"], st["groups"], st["beams"], st["n_out"]
    if own:
        parent, token, score = package().beam_select(st["logits"], st["cum"], beams, k, done=st["done"], eos=EOS)
        return {"parent": parent, "token": token, "score": score}
    # in 64 bits: candidates of different beams lie next to one another
    x = st["logits"].double()
    m = x.amax(-1, keepdim=True)
    s = st["cum"].double()[:, None] + (x - (m + torch.log(torch.exp(x - m).sum(-1, keepdim=True))))
    if st["done"] is not None:
        # a finished beam is one candidate: itself, with the end token and its score
        fin = torch.full((1, V), float("-inf"), dtype=s.dtype, device=s.device)
        fin = fin.expand(n, V).clone()
        fin[:, EOS] = st["cum"].double()
        s = torch.where(st["done"][:, None] != 0, fin, s)
    score, flat = torch.sort(s.view(G, beams * V), dim=-1, descending=True, stable=True)
    score, flat = score[:, :k], flat[:, :k]
    none = score == float("-inf")
    parent = torch.where(none, -1, flat // V).to(torch.int32)
    token = torch.where(none, -1, flat % V).to(torch.int32)
    return {"parent": parent, "token": token, "score": score.float()}


def _reorder(st):
    if own:
        package().beam_reorder(st["parent"], list(zip(st["src"], st["dst"])))
        return st["dst"]
    parent = st["parent"].long()
    rows = (parent + torch.arange(st["groups"], device="cuda")[:, None] * st["beams"]).flatten()
    for s, d in zip(st["src"], st["dst"]):
        d.copy_(s[rows])
    return st["dst"]


# ------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    if case["op"] == "append":
        row = (case["heads"] + 2 * case["kv_heads"]) * case["hd"]
        n = case["tokens"]
        per = row * (SIZE[case["dt"]] + SIZE[case["cache"]]) + case["rot"] * 4 + 12
        flops = n * (case["heads"] + case["kv_heads"]) * (3 * case["rot"] + (4 * case["hd"] if case["norm"] else 0))
        return {"bytes": n * per, "flops": flops}
    if case["op"] == "attn":
        # the own parts' lengths are uniform up to max_len
        keys = case["prefix"] + case["seqs"] * (case["max_len"] / 2)
        pairs = case["seqs"] * (case["prefix"] + case["max_len"] / 2)
        io = case["seqs"] * case["heads"] * (2 * case["hd"] * SIZE[case["dt"]] + 4)
        return {"bytes": int(keys * case["kv_heads"] * case["hd"] * 2 * SIZE[case["dt"]] + io),
                "flops": int(pairs * case["heads"] * case["hd"] * 4)}
    if case["op"] == "select":
        n = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": n * SIZE[case["dt"]], "flops": n * 3}
    return {"bytes": 2 * case["groups"] * case["beams"] * sum(_row_bytes(case)), "flops": 0}


# ------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(case, st)
    if case["op"] == "attn":
        return _exact_attn(case, st)
    if case["op"] == "select":
        return _exact_select(case, st)
    rows = st["parent"].cpu().numpy() + np.arange(case["groups"])[:, None] * case["beams"]
    return [torch.from_numpy(s.cpu().numpy()[rows.reshape(-1)]) for s in st["src"]]


def _exact_append(case, st):
    """Each pair of a head's numbers is one complex number, turned by the position's angle."""
    half = case["rot"] // 2
    first = torch.arange(half, device="cuda") * (2 if case["pair"] == "norm" else 1)
    second = first + (1 if case["pair"] == "norm" else half)
    pos = st["pos"].long()
    turn = torch.complex(st["cos"][pos].double(), st["sin"][pos].double())[:, None, :]
    done = []
    for x, w in ((st["q"], st["q_norm"]), (st["k"], st["k_norm"])):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / case["hd"] + 1e-5) * w.double()
        z = torch.complex(y[..., first], y[..., second]) * turn
        y = y.clone()
        y[..., first], y[..., second] = z.real, z.imag
        done.append(y)
    q, k = done
    P = case["page"]
    row = st["table"].long()[st["seq"].long(), pos // P] * P + pos % P
    pools = []
    for new, pool in ((k, st["k_pool"]), (st["v"].double(), st["v_pool"])):
        flat = pool.double().view(-1, case["kv_heads"], case["hd"])
        flat[row] = new
        pools.append(flat.view(pool.shape))
    return {"q": q, "k_pool": pools[0], "v_pool": pools[1]}


def _exact_attn(case, st):
    B, H, KV, hd, P, c = (case[k] for k in ("seqs", "heads", "kv_heads", "hd", "page", "clamp"))
    lens = st["lens"].tolist()
    flat_k = st["k_pool"].view(-1, KV, hd)
    flat_v = st["v_pool"].view(-1, KV, hd)

    def rows(table, n):
        t = torch.arange(n, device="cuda")
        return table.long()[t // P] * P + t % P

    shared = rows(st["prefix_table"], case["prefix"])
    kp, vp = flat_k[shared].double(), flat_v[shared].double()
    out = torch.zeros((B, H, hd), dtype=torch.float64, device="cuda")
    lse = torch.full((B, H), float("-inf"), dtype=torch.float64, device="cuda")
    for b in range(B):
        if case["prefix"] + lens[b] == 0:
            continue
        mine = rows(st["table"][b], lens[b])
        km, vm = flat_k[mine].double(), flat_v[mine].double()
        for h in range(H):
            j = h // (H // KV)
            q = st["q"][b, h].double()
            s = torch.cat([kp[:, j] @ q, km[:, j] @ q]) / math.sqrt(hd)
            if c:
                s = c * torch.tanh(s / c)
            z = torch.logsumexp(s, 0)
            p = torch.exp(s - z)
            lse[b, h] = z
            out[b, h] = p[:case["prefix"]] @ vp[:, j] + p[case["prefix"]:] @ vm[:, j]
    return {"out": out, "lse": lse}


def _exact_select(case, st):
    G, beams, V, k = case["groups"], case["beams"], case["vocab"], case["n_out"]
    x = st["logits"].double().cpu().numpy()
    cum = st["cum"].double().cpu().numpy()
    done = None if st["done"] is None else st["done"].cpu().numpy()
    parent, token, score = (np.full((G, k), v) for v in (-1, -1, -np.inf))
    parent, token = parent.astype(np.int32), token.astype(np.int32)
    for g in range(G):
        found = []
        for b in range(beams):
            r = g * beams + b
            if done is not None and done[r]:
                found.append((-cum[r], b, EOS))
                continue
            top = x[r].max()
            lp = x[r] - (top + np.log(np.exp(x[r] - top).sum()))
            least = np.partition(lp, V - min(k, V))[V - min(k, V)]
            found += [(-(cum[r] + lp[t]), b, int(t)) for t in np.nonzero(lp >= least)[0]]
        for i, (s, b, t) in enumerate(sorted(found)[:k]):
            parent[g, i], token[g, i], score[g, i] = b, t, -s
    return {"parent": torch.from_numpy(parent), "token": torch.from_numpy(token), "score": torch.from_numpy(score)}
