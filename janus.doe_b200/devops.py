"""Device operators on torch tensors: the paged key/value cache (append, attention behind a
shared prefix), the beams' selection and the reordering of their states (include/jdgpu.h).

Every call runs on the tensors' device and its current torch stream, can be captured into a
graph, and takes the workspace it needs from torch's allocator for that stream.  Refused
arguments raise JdError and touch nothing.  No gradients are computed: a call whose inputs require
one warns, unless it is made under torch.no_grad().
"""
import ctypes as C
import warnings

from . import jdgpu
from .jdgpu import JD_BF16, JD_EINVAL, JD_F16, JD_F32, JD_OK, JdError

STATUS_POS, STATUS_SEQ, STATUS_PAGE = 2, 32, 64
MAX_STATES = 16


class JdgPagedKV(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p)] + \
               [(n, C.c_int) for n in ("dt", "n_pages", "page_size", "n_kv_heads", "head_dim")] + \
               [(n, C.c_int64) for n in ("page_stride", "row_stride", "head_stride")] + \
               [("table", C.c_void_p), ("table_stride", C.c_int), ("n_seqs", C.c_int)]


class JdgAppendArgs(C.Structure):
    _fields_ = [("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("dt", C.c_int), ("n_tokens", C.c_int),
                ("n_heads", C.c_int), ("q_stride", C.c_int64), ("k_stride", C.c_int64), ("v_stride", C.c_int64),
                ("q_out", C.c_void_p), ("q_out_stride", C.c_int64), ("seq", C.c_void_p), ("pos", C.c_void_p),
                ("cos", C.c_void_p), ("sin", C.c_void_p), ("n_pos", C.c_int), ("rot_dim", C.c_int),
                ("rope_norm", C.c_int), ("q_norm", C.c_void_p), ("k_norm", C.c_void_p), ("eps", C.c_float),
                ("status", C.c_void_p)]


class JdgAttnArgs(C.Structure):
    _fields_ = [("q", C.c_void_p), ("q_stride", C.c_int64), ("out", C.c_void_p), ("out_stride", C.c_int64),
                ("lse", C.c_void_p), ("n_heads", C.c_int), ("prefix", C.c_void_p), ("prefix_len", C.c_int),
                ("lens", C.c_void_p), ("max_len", C.c_int), ("scale", C.c_float), ("clamp", C.c_float),
                ("status", C.c_void_p)]


class JdgSelectArgs(C.Structure):
    _fields_ = [("logits", C.c_void_p), ("dt", C.c_int), ("stride", C.c_int64)] + \
               [(n, C.c_int) for n in ("groups", "beams", "vocab", "n_out")] + \
               [("cum", C.c_void_p), ("done", C.c_void_p), ("eos", C.c_int), ("parent", C.c_void_p),
                ("token", C.c_void_p), ("score", C.c_void_p)]


class JdgState(C.Structure):
    _fields_ = [("src", C.c_void_p), ("dst", C.c_void_p), ("row_bytes", C.c_int64), ("src_stride", C.c_int64),
                ("dst_stride", C.c_int64)]


class JdgReorderArgs(C.Structure):
    _fields_ = [("parent", C.c_void_p)] + [(n, C.c_int) for n in ("parent_stride", "groups", "beams", "n_states")] + \
               [("state", JdgState * MAX_STATES), ("status", C.c_void_p)]


_fns = None
_torch = None
_dt = None
_stream = None  # device number -> address of its current stream


def _lib():
    global _fns, _torch, _dt, _stream
    if _fns is None:
        import torch
        L = jdgpu.lib()
        P = C.POINTER
        sig = {
            "jdg_paged_append": [P(JdgPagedKV), P(JdgAppendArgs), C.c_void_p],
            "jdg_paged_append_check": [P(JdgPagedKV), P(JdgAppendArgs)],
            "jdg_paged_attn": [P(JdgPagedKV), P(JdgAttnArgs), C.c_void_p, C.c_size_t, C.c_void_p],
            "jdg_paged_attn_check": [P(JdgPagedKV), P(JdgAttnArgs)],
            "jdg_paged_attn_workspace": [P(JdgPagedKV), P(JdgAttnArgs)],
            "jdg_beam_select": [P(JdgSelectArgs), C.c_void_p, C.c_size_t, C.c_void_p],
            "jdg_beam_select_check": [P(JdgSelectArgs)],
            "jdg_beam_select_workspace": [P(JdgSelectArgs)],
            "jdg_beam_reorder": [P(JdgReorderArgs), C.c_void_p],
            "jdg_beam_reorder_check": [P(JdgReorderArgs)],
        }
        for name, args in sig.items():
            f = getattr(L, name)
            f.argtypes = args
            f.restype = C.c_size_t if name.endswith("_workspace") else C.c_int
        _torch = torch
        # the address itself, where torch offers it: a Stream object takes a microsecond to make
        _stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or \
            (lambda dev: torch.cuda.current_stream(dev).cuda_stream)
        _dt = {torch.float32: JD_F32, torch.float16: JD_F16, torch.bfloat16: JD_BF16}
        _fns = L
    return _fns


def _refuse(msg):
    raise JdError(JD_EINVAL, msg)


def _check(rc):
    if rc != JD_OK:
        raise JdError(rc, (jdgpu.lib().jdg_last_error(None) or b"").decode(errors="replace"))


def _dtype(t, name):
    if t.dtype not in _dt:
        _refuse("%s: %s is not float32, float16 or bfloat16" % (name, t.dtype))
    return _dt[t.dtype]


def _ints(t, name, shape, dev):
    """Address of a contiguous int32 tensor of that shape on device number dev."""
    if t.dtype is not _torch.int32 or t.get_device() != dev or t.shape != shape or not t.is_contiguous():
        _refuse("%s: want a contiguous int32 tensor %s on cuda:%d" % (name, tuple(shape), dev))
    return t.data_ptr()


def _floats(t, name, shape, dev):
    if t.dtype is not _torch.float32 or t.get_device() != dev or t.shape != shape or not t.is_contiguous():
        _refuse("%s: want a contiguous float32 tensor %s on cuda:%d" % (name, tuple(shape), dev))
    return t.data_ptr()


def _heads(t, name, n, heads, hd, dev):
    """[n][heads][hd] with the heads of a token contiguous; returns the token stride."""
    if t.get_device() != dev or t.shape != (n, heads, hd):
        _refuse("%s: want [%d][%d][%d] on cuda:%d, got %s on %s" % (name, n, heads, hd, dev, tuple(t.shape), t.device))
    sn, sh, sd = t.stride()
    if (sd != 1 or (heads > 1 and sh != hd)) and t.numel():
        _refuse("%s: the heads of a token must be contiguous" % name)
    return sn if n > 1 else heads * hd


def _forward_only(who, *tensors):
    if _torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                warnings.warn("%s computes no gradients: its results carry none, although an input requires one" % who,
                              stacklevel=3)
                return


def _launch(dev, fn, *args):
    """fn(*args, stream) on the current stream of device number dev, with dev current."""
    if _torch.cuda.current_device() == dev:
        rc = fn(*args, _stream(dev))
    else:
        with _torch.cuda.device(dev):
            rc = fn(*args, _stream(dev))
    if rc:
        _check(rc)


class PagedKV:
    """A paged key/value cache of one layer: pools k, v [n_pages][page_size][n_kv_heads][head_dim]
    (any strides with head_dim contiguous, the same for both) and the sequences' page tables
    [n_seqs][max_pages] (int32).  Position t of sequence s is row t % page_size of page
    table[s][t // page_size].  Holds references, copies nothing."""

    def __init__(self, k, v, table):
        _lib()
        if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device or k.device.type != "cuda":
            _refuse("PagedKV: k and v must be CUDA tensors [n_pages][page_size][n_kv_heads][head_dim] of one type")
        st = [k.stride(i) if k.shape[i] > 1 else 0 for i in range(4)]
        if st != [v.stride(i) if v.shape[i] > 1 else 0 for i in range(4)] or (k.shape[3] > 1 and st[3] != 1):
            _refuse("PagedKV: k and v must have the same strides, head_dim contiguous")
        if table.dim() != 2:
            _refuse("PagedKV: the table must be [n_seqs][max_pages]")
        self.k, self.v, self.table, self.device = k, v, table, k.device
        self.dev, self.dtype = k.get_device(), k.dtype
        self.n_pages, self.page_size, self.n_kv_heads, self.head_dim = k.shape
        self.n_seqs = table.shape[0]
        self.c = JdgPagedKV(k.data_ptr(), v.data_ptr(), _dtype(k, "PagedKV"), *k.shape, *st[:3],
                            _ints(table, "table", table.shape, self.dev), table.shape[1], table.shape[0])
        self.ref = C.byref(self.c)

    def with_table(self, table):
        """The same pools behind another page table."""
        return PagedKV(self.k, self.v, table)


def paged_append(kv, q, k, v, seq, pos, cos=None, sin=None, rope_norm=False, q_norm=None, k_norm=None, eps=1e-5,
                 out=None, status=None):
    """Append tokens to the cache; returns the rotated queries in the cache's type ([n][heads][hd]),
    or None when q is None.  q, k, v: [n][heads][head_dim]; seq, pos: int32 [n] (negative: padding,
    left alone); cos, sin: float32 [n_pos][rot_dim / 2] or None; q_norm, k_norm: float32 [head_dim]
    weights of the heads' RMS norm or None; out: where the queries go (q itself is allowed)."""
    _forward_only("paged_append", q, k, v, cos, sin, q_norm, k_norm)
    hd, kvh, dev, n = kv.head_dim, kv.n_kv_heads, kv.dev, k.shape[0]
    ks, vs = _heads(k, "k", n, kvh, hd, dev), _heads(v, "v", n, kvh, hd, dev)
    if v.dtype is not k.dtype or (q is not None and q.dtype is not k.dtype):
        _refuse("paged_append: q, k and v must have one type")
    qp = qs = op = os_ = heads = 0
    if q is not None:
        if q.dim() != 3:
            _refuse("paged_append: q must be [n][heads][head_dim]")
        heads = q.shape[1]
        qs = _heads(q, "q", n, heads, hd, dev)
        if out is None:
            out, os_ = kv.k.new_empty((n, heads, hd)), heads * hd
        else:
            if out.dtype is not kv.dtype:
                _refuse("paged_append: out must have the cache's type")
            os_ = _heads(out, "out", n, heads, hd, dev)
        qp, op = q.data_ptr(), out.data_ptr()
    rot = n_pos = 0
    cp = sp = None
    if cos is not None:
        if cos.dim() != 2 or sin is None:
            _refuse("paged_append: cos and sin must be [n_pos][rot_dim / 2]")
        n_pos, rot = cos.shape
        cp, sp, rot = _floats(cos, "cos", cos.shape, dev), _floats(sin, "sin", cos.shape, dev), 2 * rot
    if n == 0:
        return out
    a = JdgAppendArgs(qp, k.data_ptr(), v.data_ptr(), _dtype(k, "k"), n, heads, qs, ks, vs, op, os_,
                      _ints(seq, "seq", (n,), dev), _ints(pos, "pos", (n,), dev), cp, sp, n_pos, rot,
                      1 if rope_norm else 0, None if q_norm is None else _floats(q_norm, "q_norm", (hd,), dev),
                      None if k_norm is None else _floats(k_norm, "k_norm", (hd,), dev), eps,
                      None if status is None else _ints(status, "status", (1,), dev))
    _launch(dev, _fns.jdg_paged_append, kv.ref, C.byref(a))
    return out


def paged_attn(kv, q, lens, max_len, prefix=None, prefix_len=0, scale=None, clamp=0.0, out=None, lse=None, status=None):
    """Attention of one query token per sequence: q [n_seqs][heads][head_dim] in the cache's type over
    the prefix_len shared rows behind `prefix` (int32 pages) and each sequence's own lens[s] rows
    (int32; 0: none, negative: an idle slot, left alone) behind its table row.  max_len bounds lens:
    a longer one is cut there, which only status (int32 [1]) tells.  Returns (out, lse)."""
    _forward_only("paged_attn", q, kv.k, kv.v)
    hd, dev, B = kv.head_dim, kv.dev, kv.n_seqs
    if q.dim() != 3:
        _refuse("paged_attn: q must be [n_seqs][heads][head_dim]")
    heads = q.shape[1]
    qs = _heads(q, "q", B, heads, hd, dev)
    if q.dtype is not kv.dtype or (out is not None and out.dtype is not kv.dtype):
        _refuse("paged_attn: q and out must have the cache's type")
    if out is None:
        out, os_ = q.new_empty((B, heads, hd)), heads * hd
    else:
        os_ = _heads(out, "out", B, heads, hd, dev)
    if lse is None:
        lse = q.new_empty((B, heads), dtype=_torch.float32)
        lp = lse.data_ptr()
    else:
        lp = _floats(lse, "lse", (B, heads), dev)
    pp = None
    if prefix_len:
        if prefix is None or prefix.dim() != 1 or prefix.shape[0] * kv.page_size < prefix_len:
            _refuse("paged_attn: prefix must list the pages of %d shared rows" % prefix_len)
        pp = _ints(prefix, "prefix", prefix.shape, dev)
    if B == 0:
        return out, lse
    a = JdgAttnArgs(q.data_ptr(), qs, out.data_ptr(), os_, lp, heads, pp, prefix_len, _ints(lens, "lens", (B,), dev),
                    max_len, hd ** -0.5 if scale is None else scale, clamp,
                    None if status is None else _ints(status, "status", (1,), dev))
    ref = C.byref(a)
    n = _fns.jdg_paged_attn_workspace(kv.ref, ref)
    if not n:
        _check(_fns.jdg_paged_attn_check(kv.ref, ref))
    ws = q.new_empty(n, dtype=_torch.uint8)
    _launch(dev, _fns.jdg_paged_attn, kv.ref, ref, ws.data_ptr(), n)
    return out, lse


def beam_select(logits, cum, beams, n_out, done=None, eos=0):
    """The n_out best continuations of each group of `beams` rows of logits [groups * beams][vocab]:
    (parent, token, score), each [groups][n_out], best first; cum: float32 scores of the rows; done:
    int32, nonzero rows continue only as themselves (token eos).  Places without a continuation
    hold parent = token = -1, score = -inf."""
    L, dev = _lib(), logits.get_device()
    _forward_only("beam_select", logits, cum)
    if logits.dim() != 2 or dev < 0 or beams < 1 or logits.shape[0] % beams or \
            (logits.shape[1] > 1 and logits.stride(1) != 1):
        _refuse("beam_select: logits must be a CUDA tensor [groups * beams][vocab], rows contiguous")
    rows, vocab = logits.shape
    groups = rows // beams
    shape = (groups, max(n_out, 0))
    parent, score = logits.new_empty(shape, dtype=_torch.int32), logits.new_empty(shape, dtype=_torch.float32)
    token = _torch.empty_like(parent)
    if rows == 0:
        return parent, token, score
    a = JdgSelectArgs(logits.data_ptr(), _dtype(logits, "logits"), logits.stride(0) if rows > 1 else vocab,
                      groups, beams, vocab, n_out, _floats(cum, "cum", (rows,), dev),
                      None if done is None else _ints(done, "done", (rows,), dev), eos, parent.data_ptr() or None,
                      token.data_ptr() or None, score.data_ptr() or None)
    ref = C.byref(a)
    n = L.jdg_beam_select_workspace(ref)
    if not n:
        _check(L.jdg_beam_select_check(ref))
    ws = logits.new_empty(n, dtype=_torch.uint8)
    _launch(dev, L.jdg_beam_select, ref, ws.data_ptr(), n)
    return parent, token, score


def beam_reorder(parent, states, status=None):
    """Row i of group g of every dst becomes row parent[g][i] of that group of its src.  parent: int32
    [groups][beams] (rows may be strided; negative: the dst row is left alone); states: (src, dst)
    pairs of tensors [groups * beams][...] whose rows are contiguous; no dst overlaps a src."""
    L, dev = _lib(), parent.get_device()
    _forward_only("beam_reorder", *[src for src, _ in states])
    if parent.dim() != 2 or parent.dtype is not _torch.int32 or dev < 0 or \
            (parent.shape[1] > 1 and parent.stride(1) != 1):
        _refuse("beam_reorder: parent must be a CUDA int32 tensor [groups][beams]")
    groups, beams = parent.shape
    rows = groups * beams
    if len(states) > MAX_STATES:
        _refuse("beam_reorder: at most %d states" % MAX_STATES)
    if rows == 0 or not states:
        return
    a = JdgReorderArgs(parent.data_ptr(), parent.stride(0) if groups > 1 else beams, groups, beams, len(states))
    for i, (src, dst) in enumerate(states):
        if src.shape != dst.shape or src.dtype is not dst.dtype or src.get_device() != dev or \
                dst.get_device() != dev or src.dim() < 1 or src.shape[0] != rows:
            _refuse("beam_reorder: state %d: src and dst must be [%d][...] of one type on cuda:%d" % (i, rows, dev))
        n, es = src.numel(), src.element_size()
        if n and not (src.is_contiguous() or src[0].is_contiguous()) or not (dst.is_contiguous() or dst[0].is_contiguous()):
            _refuse("beam_reorder: state %d: rows must be contiguous" % i)
        size = n // rows * es
        # an empty state has no storage: any address stands in for it, nothing is copied
        a.state[i] = (src.data_ptr() or parent.data_ptr(), dst.data_ptr() or parent.data_ptr(), size,
                      src.stride(0) * es if rows > 1 else size, dst.stride(0) * es if rows > 1 else size)
    if status is not None:
        a.status = _ints(status, "status", (1,), dev)
    _launch(dev, L.jdg_beam_reorder, C.byref(a))
