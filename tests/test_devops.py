"""Refusals of the device operators, on the host only: the _check functions are the first thing
each call runs; the addresses are plain integers and nothing is dereferenced."""
import ctypes as C
import importlib

import pytest

OK, EINVAL, EUNSUPPORTED = 0, -1, -5


@pytest.fixture(scope="module")
def dv(jd):
    m = importlib.import_module("janus_doe_b200.devops")
    m._lib()
    return m


def kv_of(dv, **over):
    d = dict(k=1 << 20, v=1 << 24, dt=30, n_pages=8, page_size=16, n_kv_heads=2, head_dim=64, page_stride=16 * 128,
             row_stride=128, head_stride=64, table=4096, table_stride=4, n_seqs=2)
    d.update(over)
    return dv.JdgPagedKV(**d)


def refused(jd, rc, code, msg):
    assert rc == code
    if code != OK:
        assert msg.encode() in jd.lib().jdg_last_error(None)


KV_CASES = [
    (dict(), OK, ""),
    (dict(dt=8), EUNSUPPORTED, "type"),
    (dict(page_size=12), EINVAL, "power of two"),
    (dict(page_size=2048), EINVAL, "power of two"),
    (dict(page_size=0), EINVAL, "power of two"),
    (dict(head_dim=60), EUNSUPPORTED, "head_dim"),
    (dict(head_dim=264), EUNSUPPORTED, "head_dim"),
    (dict(k=(1 << 20) + 8), EINVAL, "16 bytes"),
    (dict(row_stride=132), EINVAL, "16 bytes"),
    (dict(head_stride=-64), EINVAL, "16 bytes"),
    (dict(k=0), EINVAL, "bad cache"),
    (dict(table=0), EINVAL, "bad cache"),
    (dict(n_pages=0), EINVAL, "bad cache"),
]


def append_of(dv, **over):
    # three tokens of a fused row of 4 + 2 + 2 heads of 64
    q = 1 << 28
    d = dict(q=q, k=q + 512, v=q + 768, dt=30, n_tokens=3, n_heads=4, q_stride=512, k_stride=512, v_stride=512,
             q_out=1 << 29, q_out_stride=256, seq=4096, pos=8192, cos=12288, sin=16384, n_pos=100, rot_dim=64,
             rope_norm=0, q_norm=None, k_norm=None, eps=1e-5, status=None)
    d.update(over)
    return dv.JdgAppendArgs(**d)


@pytest.mark.parametrize("over,code,msg", KV_CASES)
def test_cache_description(jd, dv, over, code, msg):
    f = jd.lib().jdg_paged_append_check
    refused(jd, f(C.byref(kv_of(dv, **over)), C.byref(append_of(dv))), code, msg)


@pytest.mark.parametrize("over,code,msg", [
    (dict(), OK, ""),
    (dict(n_tokens=0), OK, ""),
    (dict(n_heads=0, q=None, q_out=None), OK, ""),
    (dict(rot_dim=0, cos=None, sin=None), OK, ""),
    (dict(q_out=1 << 28, q_out_stride=512), OK, ""),              # the queries in place
    (dict(k=1 << 30, v=1 << 31, q_out=(1 << 28) + 512, q_out_stride=512), OK, ""),  # beside them in the row
    (dict(q_out=(1 << 28) + 512, q_out_stride=512), EINVAL, "overlaps k"),
    (dict(q_out=(1 << 28) + 128, q_out_stride=512), EINVAL, "overlaps q"),
    (dict(q_out=1 << 28, q_out_stride=256), EINVAL, "overlaps q"),
    (dict(q_out=(1 << 28) + 512 + 256, q_out_stride=512), EINVAL, "overlaps"),   # over the values' columns
    (dict(k=1 << 30, v=1 << 31, q_out=(1 << 28) + 1024 + 512, q_out_stride=512), OK, ""),   # beside, a row further
    (dict(k=1 << 30, v=1 << 31, q_out=(1 << 28) - 512, q_out_stride=512), OK, ""),
    (dict(k=1 << 30, v=1 << 31, q_out=(1 << 28) - 256, q_out_stride=512), EINVAL, "overlaps q"),
    (dict(n_tokens=1, q_out=(1 << 28) + 512, q_out_stride=512), EINVAL, "overlaps k"),
    (dict(q_out=1 << 28, q_out_stride=512, dt=0), EINVAL, "overlaps q"),
    (dict(q_out_stride=128), EINVAL, "rows overlap"),
    (dict(rot_dim=68), EINVAL, "rotation"),
    (dict(rot_dim=72), EINVAL, "rotation"),
    (dict(rope_norm=2), EINVAL, "rotation"),
    (dict(sin=None), EINVAL, "rotation"),
    (dict(eps=float("nan")), EINVAL, "rotation"),
    (dict(k=(1 << 28) + 514), EINVAL, "aligned"),
    (dict(v_stride=514), EINVAL, "aligned"),
    (dict(cos=12292), EINVAL, "aligned"),
    (dict(dt=2), EUNSUPPORTED, "type"),
    (dict(n_heads=5000), EUNSUPPORTED, "heads"),
    (dict(seq=None), EINVAL, "bad arguments"),
    (dict(n_tokens=-1), EINVAL, "bad arguments"),
])
def test_append_arguments(jd, dv, over, code, msg):
    f = jd.lib().jdg_paged_append_check
    refused(jd, f(C.byref(kv_of(dv)), C.byref(append_of(dv, **over))), code, msg)


def attn_of(dv, **over):
    d = dict(q=1 << 28, q_stride=256, out=1 << 29, out_stride=256, lse=1 << 27, n_heads=4, prefix=4096, prefix_len=33,
             lens=8192, max_len=64, scale=0.125, clamp=0.0, status=None)
    d.update(over)
    return dv.JdgAttnArgs(**d)


@pytest.mark.parametrize("kv_over,over,code,msg", [
    ({}, dict(), OK, ""),
    ({}, dict(prefix=None, prefix_len=0, lse=None), OK, ""),
    (dict(n_seqs=0), dict(), OK, ""),
    ({}, dict(n_heads=3), EINVAL, "multiple"),
    (dict(head_dim=136, head_stride=136, row_stride=272), dict(), EUNSUPPORTED, "128"),
    ({}, dict(max_len=65), EINVAL, "max_len"),
    ({}, dict(max_len=-1), EINVAL, "bad arguments"),
    ({}, dict(prefix=None), EINVAL, "bad arguments"),
    ({}, dict(lens=None), EINVAL, "bad arguments"),
    ({}, dict(scale=float("inf")), EINVAL, "finite"),
    ({}, dict(scale=float("nan")), EINVAL, "finite"),
    ({}, dict(clamp=-1.0), EINVAL, "finite"),
    ({}, dict(clamp=float("inf")), EINVAL, "finite"),
    ({}, dict(clamp=1e-40), EINVAL, "too small"),
    ({}, dict(q=(1 << 28) + 8), EINVAL, "aligned"),
    ({}, dict(out_stride=260), EINVAL, "aligned"),
    ({}, dict(out_stride=128), EINVAL, "rows overlap"),
    ({}, dict(out=(1 << 28) + 512), EINVAL, "overlaps q"),
    ({}, dict(out=1 << 28), EINVAL, "overlaps q"),
])
def test_attn_arguments(jd, dv, kv_over, over, code, msg):
    kv, a = kv_of(dv, **kv_over), attn_of(dv, **over)
    refused(jd, jd.lib().jdg_paged_attn_check(C.byref(kv), C.byref(a)), code, msg)
    n = jd.lib().jdg_paged_attn_workspace(C.byref(kv), C.byref(a))
    assert (n > 0) == (code == OK) or kv.n_seqs == 0
    if code == OK and n > 16:  # the call itself: a missing or short workspace is refused before anything runs
        refused(jd, jd.lib().jdg_paged_attn(C.byref(kv), C.byref(a), None, n, None), EINVAL, "workspace")
        refused(jd, jd.lib().jdg_paged_attn(C.byref(kv), C.byref(a), 1 << 30, n - 1, None), EINVAL, "workspace")


def select_of(dv, **over):
    d = dict(logits=1 << 28, dt=0, stride=500, groups=2, beams=3, vocab=500, n_out=6, cum=4096, done=None, eos=2,
             parent=8192, token=12288, score=16384)
    d.update(over)
    return dv.JdgSelectArgs(**d)


@pytest.mark.parametrize("over,code,msg", [
    (dict(), OK, ""),
    (dict(logits=(1 << 28) + 4, stride=501), OK, ""),
    (dict(groups=0), OK, ""),
    (dict(n_out=33), EUNSUPPORTED, "n_out"),
    (dict(n_out=0), EINVAL, "bad arguments"),
    (dict(beams=65), EUNSUPPORTED, "beams"),
    (dict(groups=30000), EUNSUPPORTED, "rows"),
    (dict(vocab=0), EINVAL, "bad arguments"),
    (dict(dt=8), EUNSUPPORTED, "type"),
    (dict(logits=(1 << 28) + 2), EINVAL, "misaligned"),
    (dict(done=4096, eos=500), EINVAL, "eos"),
    (dict(done=4096, eos=-1), EINVAL, "eos"),
    (dict(score=None), EINVAL, "bad arguments"),
])
def test_select_arguments(jd, dv, over, code, msg):
    a = select_of(dv, **over)
    refused(jd, jd.lib().jdg_beam_select_check(C.byref(a)), code, msg)
    if code == OK and a.groups:
        n = jd.lib().jdg_beam_select_workspace(C.byref(a))
        assert n > 0
        refused(jd, jd.lib().jdg_beam_select(C.byref(a), 1 << 30, n - 1, None), EINVAL, "workspace")


def reorder_of(dv, states, **over):
    a = dv.JdgReorderArgs(4096, 4, 2, 4, len(states))
    for i, s in enumerate(states):
        a.state[i] = dv.JdgState(*s)
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("states,over,code,msg", [
    ([(1 << 20, 1 << 21, 100, 100, 100)], {}, OK, ""),
    ([], {}, OK, ""),
    ([(1 << 20, 1 << 21, 0, 0, 0)], {}, OK, ""),
    ([(1 << 20, 1 << 20, 100, 100, 100)], {}, EINVAL, "overlaps"),
    ([(1 << 20, (1 << 20) + 799, 100, 100, 100)], {}, EINVAL, "overlaps"),
    ([(1 << 20, (1 << 20) + 800, 100, 100, 100)], {}, OK, ""),
    ([(1 << 20, 1 << 21, 100, 100, 100), (1 << 21, 1 << 22, 8, 8, 8)], {}, EINVAL, "overlaps"),
    ([(1 << 20, 1 << 21, 100, 100, 100), (1 << 22, 1 << 21, 8, 8, 8)], {}, EINVAL, "overlaps"),
    ([(1 << 20, 1 << 21, 100, 100, 99)], {}, EINVAL, "overlap"),
    ([(0, 1 << 21, 100, 100, 100)], {}, EINVAL, "pointers"),
    ([(1 << 20, 1 << 21, 100, 100, 100)], dict(parent_stride=3), EINVAL, "bad arguments"),
    ([(1 << 20, 1 << 21, 100, 100, 100)], dict(n_states=17), EINVAL, "bad arguments"),
    ([(1 << 20, 1 << 50, 1 << 40, 1 << 40, 1 << 40)], dict(beams=64, parent_stride=64), EUNSUPPORTED, "too many bytes"),
])
def test_reorder_arguments(jd, dv, states, over, code, msg):
    a = reorder_of(dv, states, **over)
    refused(jd, jd.lib().jdg_beam_reorder_check(C.byref(a)), code, msg)
