// jdg_paged.cu — the paged key/value cache: tokens appended on the way from the projections
// (per-head norms, position rotation, scatter), and the attention of one decode step for
// sequences that share a prefix.
#include "jdg_paged_tc.cuh"

using namespace jdg;

// ------------------------------------------------------------------------------------ checks
static int log2_ceil(int n) {
    int s = 0;
    while ((1 << s) < n) s++;
    return s;
}
static bool misaligned(const void *p, size_t bytes) { return ((uintptr_t)p & (bytes - 1)) != 0; }

// whether n rows of `arow` bytes, `as` bytes apart from a on, share a byte with the other rows; rows of
// one buffer may interleave (the same distance, columns apart)
static bool rows_meet(const void *a, int64_t as, int64_t arow, const void *b, int64_t bs, int64_t brow, int64_t n) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    if (x >= y + (uintptr_t)((n - 1) * bs + brow) || y >= x + (uintptr_t)((n - 1) * as + arow)) return false;
    if (as != bs || as <= 0 || n == 1) return true;
    const int64_t d = (int64_t)((y - x) % (uintptr_t)as), off = y >= x ? d : (as - (int64_t)((x - y) % (uintptr_t)as)) % as;
    return off < arow || off + brow > as;
}

static int kv_check(const char *who, const jdg_paged_kv *kv) {
    if (!kv || !kv->k || !kv->v || !kv->table || kv->n_pages < 1 || kv->n_kv_heads < 1 || kv->n_seqs < 0 ||
        kv->table_stride < 0) {
        jdg_set_err(nullptr, "%s: bad cache description", who);
        return JD_EINVAL;
    }
    const int es = devop_size(kv->dt);
    if (!es) {
        jdg_set_err(nullptr, "%s: cache type %d is not f32, f16 or bf16", who, kv->dt);
        return JD_EUNSUPPORTED;
    }
    if (kv->page_size < 1 || kv->page_size > 1024 || (kv->page_size & (kv->page_size - 1))) {
        jdg_set_err(nullptr, "%s: page_size %d is not a power of two up to 1024", who, kv->page_size);
        return JD_EINVAL;
    }
    if (kv->head_dim < 8 || kv->head_dim > 256 || kv->head_dim % 8) {
        jdg_set_err(nullptr, "%s: head_dim %d is not a multiple of 8 up to 256", who, kv->head_dim);
        return JD_EUNSUPPORTED;
    }
    const int64_t al = 16 / es;
    if (kv->page_stride < 0 || kv->row_stride < 0 || kv->head_stride < 0 || kv->page_stride % al ||
        kv->row_stride % al || kv->head_stride % al || misaligned(kv->k, 16) || misaligned(kv->v, 16)) {
        jdg_set_err(nullptr, "%s: cache pointers and strides must be multiples of 16 bytes", who);
        return JD_EINVAL;
    }
    return JD_OK;
}

extern "C" int jdg_paged_append_check(const jdg_paged_kv *kv, const jdg_append_args *a) {
    const char *who = "jdg_paged_append";
    int rc = kv_check(who, kv);
    if (rc != JD_OK) return rc;
    if (!a || a->n_tokens < 0 || a->n_heads < 0 || !a->k || !a->v || !a->seq || !a->pos ||
        (a->n_heads && (!a->q || !a->q_out))) {
        jdg_set_err(nullptr, "%s: bad arguments", who);
        return JD_EINVAL;
    }
    const int es = devop_size(a->dt), hd = kv->head_dim;
    if (!es) {
        jdg_set_err(nullptr, "%s: type %d is not f32, f16 or bf16", who, a->dt);
        return JD_EUNSUPPORTED;
    }
    if (a->n_heads > 4096 || kv->n_kv_heads > 4096) {
        jdg_set_err(nullptr, "%s: more than 4096 heads", who);
        return JD_EUNSUPPORTED;
    }
    if (a->rot_dim < 0 || a->rot_dim > hd || a->rot_dim % 8 || (a->rope_norm != 0 && a->rope_norm != 1) ||
        (a->rot_dim && (!a->cos || !a->sin || a->n_pos < 0)) || !(a->eps >= 0.f)) {
        jdg_set_err(nullptr, "%s: bad rotation or norm (rot_dim %d of head_dim %d)", who, a->rot_dim, hd);
        return JD_EINVAL;
    }
    const int es_out = devop_size(kv->dt);
    if (a->k_stride % 4 || a->v_stride % 4 || a->k_stride < 0 || a->v_stride < 0 || misaligned(a->k, 4 * es) ||
        misaligned(a->v, 4 * es) ||
        (a->n_heads && (a->q_stride % 4 || a->q_out_stride % 4 || a->q_stride < 0 || misaligned(a->q, 4 * es) ||
                        misaligned(a->q_out, 4 * es_out))) ||
        misaligned(a->cos, 16) || misaligned(a->sin, 16) || misaligned(a->q_norm, 16) || misaligned(a->k_norm, 16)) {
        jdg_set_err(nullptr, "%s: q, k, v, q_out must be aligned to 4 elements, cos, sin and norms to 16 bytes", who);
        return JD_EINVAL;
    }
    if (a->n_heads && a->n_tokens) {
        if (a->n_tokens > 1 && a->q_out_stride < (int64_t)a->n_heads * hd) {
            jdg_set_err(nullptr, "%s: q_out rows overlap", who);
            return JD_EINVAL;
        }
        // q_out on top of q: the same numbers, read and written by one thread; anything else is refused
        const int64_t qrow = (int64_t)a->n_heads * hd * es, orow = (int64_t)a->n_heads * hd * es_out,
                      krow = (int64_t)kv->n_kv_heads * hd * es;
        const bool same = a->q == a->q_out && a->dt == kv->dt && (a->q_stride == a->q_out_stride || a->n_tokens == 1);
        const struct {
            const void *x;
            int64_t stride, row;
            const char *name;
        } in[3] = {{same ? nullptr : a->q, a->q_stride * es, qrow, "q"}, {a->k, a->k_stride * es, krow, "k"},
                   {a->v, a->v_stride * es, krow, "v"}};
        for (const auto &t : in)
            if (t.x && rows_meet(a->q_out, a->q_out_stride * es_out, orow, t.x, t.stride, t.row, a->n_tokens)) {
                jdg_set_err(nullptr, "%s: q_out overlaps %s", who, t.name);
                return JD_EINVAL;
            }
    }
    return JD_OK;
}

extern "C" int jdg_paged_attn_check(const jdg_paged_kv *kv, const jdg_attn_args *a) {
    const char *who = "jdg_paged_attn";
    int rc = kv_check(who, kv);
    if (rc != JD_OK) return rc;
    if (!a || a->n_heads < 1 || a->prefix_len < 0 || a->max_len < 0 || !a->q || !a->out || !a->lens ||
        (a->prefix_len && !a->prefix)) {
        jdg_set_err(nullptr, "%s: bad arguments", who);
        return JD_EINVAL;
    }
    if (a->n_heads % kv->n_kv_heads) {
        jdg_set_err(nullptr, "%s: %d heads are not a multiple of %d KV heads", who, a->n_heads, kv->n_kv_heads);
        return JD_EINVAL;
    }
    if (kv->head_dim > 128) {
        jdg_set_err(nullptr, "%s: head_dim %d is above 128", who, kv->head_dim);
        return JD_EUNSUPPORTED;
    }
    if ((int64_t)kv->n_seqs * a->n_heads > (1 << 24) || a->prefix_len > (1 << 29) || a->max_len > (1 << 29) ||
        (int64_t)kv->n_seqs * (a->max_len / kPaTile + 1) > 0x7fffffff) {
        jdg_set_err(nullptr, "%s: too large (%d sequences, %d heads)", who, kv->n_seqs, a->n_heads);
        return JD_EUNSUPPORTED;
    }
    if ((int64_t)a->max_len > (int64_t)kv->table_stride * kv->page_size) {
        jdg_set_err(nullptr, "%s: max_len %d is above the table's %d pages of %d", who, a->max_len, kv->table_stride,
                    kv->page_size);
        return JD_EINVAL;
    }
    if (!(a->clamp >= 0.f) || !(a->scale == a->scale) || a->scale - a->scale != 0.f || a->clamp - a->clamp != 0.f) {
        jdg_set_err(nullptr, "%s: scale and clamp must be finite, clamp not negative", who);
        return JD_EINVAL;
    }
    if (a->clamp > 0.f && !((a->scale < 0.f ? -a->scale : a->scale) / a->clamp < 1e37f)) {
        jdg_set_err(nullptr, "%s: clamp %g is too small for scale %g", who, a->clamp, a->scale);
        return JD_EINVAL;
    }
    const int es = devop_size(kv->dt);
    const int64_t al = 16 / es, row = (int64_t)a->n_heads * kv->head_dim;
    if (a->q_stride % al || a->out_stride % al || a->q_stride < 0 || misaligned(a->q, 16) || misaligned(a->out, 16)) {
        jdg_set_err(nullptr, "%s: q and out must be aligned to 16 bytes", who);
        return JD_EINVAL;
    }
    if (kv->n_seqs > 0) {
        const int64_t n1 = kv->n_seqs - 1;
        if (n1 && a->out_stride < row) {
            jdg_set_err(nullptr, "%s: out rows overlap", who);
            return JD_EINVAL;
        }
        const uintptr_t q0 = (uintptr_t)a->q, o0 = (uintptr_t)a->out;
        if (q0 < o0 + (n1 * a->out_stride + row) * es && o0 < q0 + (n1 * a->q_stride + row) * es) {
            jdg_set_err(nullptr, "%s: out overlaps q", who);
            return JD_EINVAL;
        }
    }
    return JD_OK;
}

// ------------------------------------------------------------------------------------ append
// A head's row is handled by head_dim/(2W) lanes (rounded up to a power of two), 2W numbers each:
// the first and the second of W pairs, so that nothing is exchanged between lanes.  Pairs
// (i, i + rot/2) are two groups of W rot/2 apart, pairs (2i, 2i+1) one group of 2W.  W is 8 for
// 16-bit types where head_dim and rot_dim allow it (16-byte loads), else 4.  A lane goes through
// its heads one after the other, three loads ahead, with the pair's four factors (norm weight
// times cos or sin) formed once for all heads of a kind: two packed products and the norm's
// factor for a pair.  Bound: HBM (each number read and written once).
struct AppendP {
    const void *q, *k, *v;
    void *q_out, *kc, *vc;
    int64_t q_stride, k_stride, v_stride, q_out_stride, page_stride, row_stride, head_stride;
    const int *seq, *pos, *table;
    const float *cos, *sin, *q_norm, *k_norm;
    int n_tokens, n_heads, n_kv, hd, lph_shift, slot_shift, page_shift, n_pages, table_stride, n_seqs, n_pos, rot;
    int rope_norm, wide;
    float eps, inv_hd;
    int *status;
};
constexpr int kApThreads = 128, kApAhead = 3;

// W elements as they lie in memory
template <typename T, int W>
struct RawW {
    static constexpr int N = W * (int)sizeof(T) / 8;  // 8-byte words
    uint2 w[N];
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (N == 1) {
            w[0] = __ldcs(reinterpret_cast<const uint2 *>(p));
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 2) {
                const uint4 x = __ldcs(reinterpret_cast<const uint4 *>(p) + i / 2);
                w[i] = make_uint2(x.x, x.y);
                w[i + 1] = make_uint2(x.z, x.w);
            }
        }
    }
    __device__ __forceinline__ void get(float (&f)[W]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                f[2 * i] = __uint_as_float(w[i].x);
                f[2 * i + 1] = __uint_as_float(w[i].y);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float2 a = unpack2(w[i].x, (const T *)nullptr), b = unpack2(w[i].y, (const T *)nullptr);
                f[4 * i] = a.x;
                f[4 * i + 1] = a.y;
                f[4 * i + 2] = b.x;
                f[4 * i + 3] = b.y;
            }
        }
    }
};
template <typename T, int W>
__device__ __forceinline__ void store_w(T *p, const float (&f)[W]) {
    if constexpr (sizeof(T) == 4 || W == 4) {
#pragma unroll
        for (int i = 0; i < W; i += 4) st4(p + i, make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]));
    } else {
        *reinterpret_cast<uint4 *>(p) = make_uint4(pack2(f[0], f[1], p), pack2(f[2], f[3], p), pack2(f[4], f[5], p),
                                                   pack2(f[6], f[7], p));
    }
}

template <typename TI, typename TC, int W, bool NORM, bool PAIRS>
__global__ __launch_bounds__(kApThreads, 4) void k_paged_append(const __grid_constant__ AppendP p) {
    const int slots = 1 << p.slot_shift, lph = 1 << p.lph_shift;
    const int64_t id = (int64_t)blockIdx.x * kApThreads + threadIdx.x;
    const int tok = (int)(id >> p.slot_shift), s = (int)id & (slots - 1);
    const int u = s & (lph - 1), hstep = slots >> p.lph_shift, h0 = s >> p.lph_shift;
    const int nq = p.n_heads, nqk = nq + p.n_kv, heads = nqk + p.n_kv, n_it = (heads + hstep - 1) / hstep;
    const bool inside = tok < p.n_tokens && 2 * W * u < p.hd;
    const bool turn = 2 * W * u < p.rot;
    const int oa = turn && !PAIRS ? W * u : 2 * W * u;
    const int ob = turn && !PAIRS ? (p.rot >> 1) + W * u : 2 * W * u + W;
    // heads of the token from its q, k and v rows: head h at base + h * head_dim
    const TI *qs = (const TI *)p.q + (int64_t)tok * p.q_stride;
    const TI *ks = (const TI *)p.k + (int64_t)tok * p.k_stride - nq * p.hd;
    const TI *vs = (const TI *)p.v + (int64_t)tok * p.v_stride - nqk * p.hd;
    RawW<TI, W> ra[kApAhead], rb[kApAhead];
    auto fetch = [&](RawW<TI, W> &a, RawW<TI, W> &b, int it) {
        const int h = h0 + it * hstep;
        if (inside && h < heads) {
            const TI *src = (h >= nqk ? vs : h < nq ? qs : ks) + h * p.hd;
            a.load(src + oa);
            b.load(src + ob);
        }
    };
#pragma unroll
    for (int i = 0; i < kApAhead; i++) fetch(ra[i], rb[i], i);
    // where the token goes
    bool live = false;
    int64_t crow = 0;
    int pos = 0;
    if (tok < p.n_tokens) {
        const int sq = p.seq[tok];
        pos = p.pos[tok];
        if (sq >= 0 && pos >= 0) {
            int bad = 0;
            if (sq >= p.n_seqs) bad |= JDG_STATUS_SEQ;
            if ((pos >> p.page_shift) >= p.table_stride || (p.rot && pos >= p.n_pos)) bad |= JDG_STATUS_POS;
            if (!bad) {
                const int page = p.table[(int64_t)sq * p.table_stride + (pos >> p.page_shift)];
                if (page < 0 || page >= p.n_pages) bad |= JDG_STATUS_PAGE;
                crow = (int64_t)page * p.page_stride + (int64_t)(pos & ((1 << p.page_shift) - 1)) * p.row_stride;
            }
            live = !bad && inside;
            if (bad && s == 0 && p.status) atomicOr(p.status, bad);
        }
    }
    // pair j: (x, y) -> (x ca - y sb, y cb + x sa); without norm weights ca = cb = cos, sa = sb = sin
    float ca[W], sa[W], cb[NORM ? W : 1], sb[NORM ? W : 1];
    auto angles = [&]() {
        const int64_t at = (int64_t)pos * (p.rot >> 1) + W * u;
#pragma unroll
        for (int j = 0; j < W; j += 4) {
            *reinterpret_cast<float4 *>(ca + j) = live && turn ? ld4(p.cos + at + j) : make_float4(1.f, 1.f, 1.f, 1.f);
            *reinterpret_cast<float4 *>(sa + j) = live && turn ? ld4(p.sin + at + j) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    if (!NORM) angles();
    int kind = -1;  // whose factors are held: 0 queries, 1 keys
    TC *qd = (TC *)p.q_out + (int64_t)tok * p.q_out_stride;
    TC *kd = (TC *)p.kc + crow, *vd = (TC *)p.vc + crow;
    for (int it0 = 0; it0 < n_it; it0 += kApAhead) {
#pragma unroll
        for (int i = 0; i < kApAhead; i++) {
            const int it = it0 + i;
            if (it >= n_it) break;
            const int h = h0 + it * hstep;
            const bool isv = h >= nqk, isq = h < nq, mine = inside && h < heads;
            float x[W], y[W];
            {
                float a[W], b[W];
                ra[i].get(a);
                rb[i].get(b);
#pragma unroll
                for (int j = 0; j < W; j++) {
                    x[j] = PAIRS ? (j < W / 2 ? a[2 * j % W] : b[2 * j % W]) : a[j];
                    y[j] = PAIRS ? (j < W / 2 ? a[2 * j % W + 1] : b[2 * j % W + 1]) : b[j];
                }
            }
            fetch(ra[i], rb[i], it + kApAhead);
            float inv = 1.f;
            bool normed = false;
            if (NORM) {  // every lane of the head takes part in the sum
                float2 ss = make_float2(0.f, 0.f);
#pragma unroll
                for (int j = 0; j < W; j += 2) {
                    ss = fma2(make_float2(x[j], x[j + 1]), make_float2(x[j], x[j + 1]), ss);
                    ss = fma2(make_float2(y[j], y[j + 1]), make_float2(y[j], y[j + 1]), ss);
                }
                float sum = mine ? ss.x + ss.y : 0.f;
                for (int o = lph >> 1; o; o >>= 1) sum += __shfl_xor_sync(JDG_FULL, sum, o);
                const float *w = isq ? p.q_norm : p.k_norm;
                normed = !isv && w;
                if (normed) inv = rsqrtf(sum * p.inv_hd + p.eps);
                if (mine && !isv && kind != (isq ? 0 : 1)) {
                    kind = isq ? 0 : 1;
                    angles();
#pragma unroll
                    for (int j = 0; j < W; j++) {
                        // place of the pair's two numbers in the head
                        const int px = !turn || PAIRS ? 2 * W * u + (PAIRS ? 2 * j : j) : oa + j;
                        const int py = !turn || PAIRS ? 2 * W * u + (PAIRS ? 2 * j + 1 : W + j) : ob + j;
                        const float wx = w ? w[px] : 1.f, wy = w ? w[py] : 1.f;
                        cb[j] = wy * ca[j];
                        sb[j] = wy * sa[j];
                        ca[j] *= wx;
                        sa[j] *= wx;
                    }
                }
            }
            if (!live || h >= heads) continue;
            if (!isv && turn) {
#pragma unroll
                for (int j = 0; j < W; j += 2) {
                    const float2 xx = make_float2(x[j], x[j + 1]), yy = make_float2(y[j], y[j + 1]);
                    const float2 c1 = make_float2(ca[j], ca[j + 1]), s1 = make_float2(sa[j], sa[j + 1]);
                    const float2 c2 = NORM ? make_float2(cb[j], cb[j + 1]) : c1, s2 = NORM ? make_float2(sb[j], sb[j + 1]) : s1;
                    float2 nx = fma2(xx, c1, mul2(yy, make_float2(-s2.x, -s2.y))), ny = fma2(yy, c2, mul2(xx, s1));
                    if (NORM) {
                        nx = mul2(nx, make_float2(inv, inv));
                        ny = mul2(ny, make_float2(inv, inv));
                    }
                    x[j] = nx.x;
                    x[j + 1] = nx.y;
                    y[j] = ny.x;
                    y[j + 1] = ny.y;
                }
            } else if (NORM && normed) {  // past rot_dim: the norm alone
#pragma unroll
                for (int j = 0; j < W; j++) {
                    x[j] *= inv * ca[j];
                    y[j] *= inv * cb[j];
                }
            }
            float a[W], b[W];
#pragma unroll
            for (int j = 0; j < W; j++) {
                a[j] = PAIRS ? (j & 1 ? y[j / 2] : x[j / 2]) : x[j];
                b[j] = PAIRS ? (j & 1 ? y[(W + j) / 2] : x[(W + j) / 2]) : y[j];
            }
            TC *dst = isq ? qd + h * p.hd : (isv ? vd : kd) + (int64_t)(isv ? h - nqk : h - nq) * p.head_stride;
            store_w(dst + oa, a);
            store_w(dst + ob, b);
        }
    }
}

template <typename TI, typename TC, int W, bool NORM>
static int append_pairs(const AppendP &p, unsigned grid, cudaStream_t st) {
    const char *who = "jdg_paged_append";
    return p.rope_norm ? devop_launch(who, false, k_paged_append<TI, TC, W, NORM, true>, dim3(grid), dim3(kApThreads), 0, st, p)
                       : devop_launch(who, false, k_paged_append<TI, TC, W, NORM, false>, dim3(grid), dim3(kApThreads), 0, st, p);
}
template <typename TI, typename TC, int W>
static int append_w(AppendP p, cudaStream_t st) {
    const int heads = p.n_heads + 2 * p.n_kv;
    p.lph_shift = log2_ceil((p.hd + 2 * W - 1) / (2 * W));
    // threads for each token: a warp where the tokens fill the machine (16 warps an SM), up to one pass
    // over the heads where they are few
    p.slot_shift = 5;
    while ((1 << p.slot_shift) < (heads << p.lph_shift) && ((int64_t)p.n_tokens << p.slot_shift) < 32 * 16 * kDevSMs)
        p.slot_shift++;
    const int64_t threads = (int64_t)p.n_tokens << p.slot_shift;
    const unsigned grid = (unsigned)((threads + kApThreads - 1) / kApThreads);
    return p.q_norm || p.k_norm ? append_pairs<TI, TC, W, true>(p, grid, st) : append_pairs<TI, TC, W, false>(p, grid, st);
}
template <typename TI, typename TC>
static int append_launch(const AppendP &p, cudaStream_t st) {
    if constexpr (sizeof(TI) == 2) {  // groups of 8 need 16-byte rows on both sides
        if (p.hd % 16 == 0 && p.rot % 16 == 0 && p.wide) return append_w<TI, TC, 8>(p, st);
    }
    return append_w<TI, TC, 4>(p, st);
}
template <typename TI>
static int append_cache(const AppendP &p, int dt, cudaStream_t st) {
    return dt == JD_F32   ? append_launch<TI, float>(p, st)
           : dt == JD_F16 ? append_launch<TI, __half>(p, st)
                          : append_launch<TI, __nv_bfloat16>(p, st);
}

extern "C" int jdg_paged_append(const jdg_paged_kv *kv, const jdg_append_args *a, void *stream) {
    int rc = jdg_paged_append_check(kv, a), dev;
    if (rc != JD_OK) return rc;
    if (a->n_tokens == 0) return JD_OK;
    cudaStream_t st = (cudaStream_t)stream;
    rc = devop_stream("jdg_paged_append", st, &dev);
    if (rc != JD_OK) return rc;
    AppendP p = {};
    p.q = a->q; p.k = a->k; p.v = a->v; p.q_out = a->q_out; p.kc = kv->k; p.vc = kv->v;
    p.q_stride = a->q_stride; p.k_stride = a->k_stride; p.v_stride = a->v_stride; p.q_out_stride = a->q_out_stride;
    p.page_stride = kv->page_stride; p.row_stride = kv->row_stride; p.head_stride = kv->head_stride;
    p.seq = a->seq; p.pos = a->pos; p.table = kv->table; p.cos = a->cos; p.sin = a->sin;
    p.q_norm = a->q_norm; p.k_norm = a->k_norm;
    p.n_tokens = a->n_tokens; p.n_heads = a->n_heads; p.n_kv = kv->n_kv_heads; p.hd = kv->head_dim;
    p.page_shift = log2_ceil(kv->page_size); p.n_pages = kv->n_pages; p.table_stride = kv->table_stride;
    p.n_seqs = kv->n_seqs; p.n_pos = a->n_pos; p.rot = a->rot_dim; p.rope_norm = a->rope_norm; p.eps = a->eps;
    p.status = a->status;
    p.inv_hd = 1.f / (float)kv->head_dim;
    const int64_t al = 16 / devop_size(a->dt), alo = 16 / devop_size(kv->dt);
    p.wide = !misaligned(a->k, 16) && !misaligned(a->v, 16) && a->k_stride % al == 0 && a->v_stride % al == 0 &&
             (!a->n_heads || (!misaligned(a->q, 16) && a->q_stride % al == 0 && !misaligned(a->q_out, 16) &&
                              a->q_out_stride % alo == 0));
    return a->dt == JD_F32   ? append_cache<float>(p, kv->dt, st)
           : a->dt == JD_F16 ? append_cache<__half>(p, kv->dt, st)
                             : append_cache<__nv_bfloat16>(p, kv->dt, st);
}

// ------------------------------------------------------------------------------------ attention
// How a call is split.  Queries of a KV head: n_seqs * G rows behind the prefix, G behind a
// sequence's own rows, taken R at a time.  The prefix is cut into equal parts that fill the
// machine; the own rows, whose lengths only the GPU knows, are shared out evenly by the kernel
// itself.  Each (query, part) is (max, sum, out) in the workspace; k_pa_merge joins them.  Where
// there is one part in all, the result is written at once.
static int r_template(int rows) { return rows <= 1 ? 1 : rows <= 2 ? 2 : rows <= 3 ? 3 : rows <= 4 ? 4 : 8; }

static int attn_warps(const PaArgs &p) { return p.f32 && p.hd > 64 && p.r_own <= 4 ? 6 : 4; }  // of a CTA of the warp kernels

// Rows of a part of the prefix in the warp kernels, in tiles of 32: a CTA for each part, 12 warps an SM
// wanted; a tile for each warp where all CTAs then make up no more than that, two otherwise (a part costs
// its write and its read in the join).  12 is what is resident of the 16-bit kernels and of f32 rows of up to 64
// numbers behind up to 4 queries.  Shared memory holds fewer of the other f32 kernels (8 warps at 64 numbers and 8
// queries; above 64, 6, or 4 behind 8 queries): their CTAs run in two or three turns, with so many more parts.
static int chunk_for(int64_t units, int len, int nw) {
    const int64_t want = 12 / nw * kDevSMs, tiles = (len + kPaTile - 1) / kPaTile;
    if (units * ((tiles + nw - 1) / nw) <= want) return nw * kPaTile;
    int64_t n = want / units;
    if (n < 1) n = 1;
    const int64_t c = (tiles + n - 1) / n, least = 2 * nw;
    return (int)(c < least ? least : c) * kPaTile;
}

// Parts of the prefix in the tensor-core kernel, and how many SMs the own rows are shared out over.  That
// kernel leaves no room for others on its SMs, and each part costs the join its write and its read; so more
// parts are not better: fewer leave SMs where the own rows run meanwhile.  Estimated in us: the kernel's
// start, end and steps (a 128 x 128 tile for each stream); own rows in tiles of 32, on the idle SMs beside it
// or on all of them after it; the join's start and (query, part) pairs.  The host knows only a bound of the
// lengths, so it takes the least product of the time t with lengths of half of max_len on average and the
// time without own rows: within 3 % of the best on average where the former holds, as t alone, and within
// 16 % (44 % at most) where max_len is 1024 to 16,384 over lengths of 400 or less (t alone: twice the best).
// The figures are a fit to 332 calls (6 % off on average): 8 to 256 sequences, 300 to 32,789 shared rows, up to
// 1500 own ones, head_dim 64 and 128, many numbers of parts, own rows beside and behind.  Against as many parts
// as SMs and own rows on all of them: 32 sequences x 2048 + 301 rows 20.3 -> 15 us, 32 x 3500 + 700
// 24.3 -> 18.7, 64 x 2048 + 1000 53 -> 38, 64 x 32,789 + 1000 85 -> 70.
static void split_tc(PaArgs *p, int tiles, int64_t prows, int own_units) {
    const float wide = (float)p->hd / 128.f, step = p->hd > 64 ? 2.3f : 1.7f;
    const int units = p->rb_pre * p->KV, most = units < kDevSMs ? kDevSMs / units : 1;
    const int own_tiles = p->max_len ? (p->max_len - 1) / kPaTile + 1 : 0;
    const float own = .5f * (float)p->n_seqs * (float)own_tiles * (float)own_units * wide;
    const bool two = prows > kPtRows;
    float best = 0.f;
    p->np = 0;
    for (int n = 1, last = 0; n <= most && n <= tiles; n++) {
        const int c = (tiles + n - 1) / n;
        if (c == last) continue;  // the same parts
        last = c;
        const int np = (tiles + c - 1) / c, idle = kDevSMs - np * units;
        const float tc = 7.f + step * (float)(two ? c : (c + 1) / 2);
        const float join = 4.5e-4f * wide * (float)np * (float)prows * (float)p->KV;
        float t = tc + 2.5e-3f * own + join;
        int sms = kDevSMs;
        if (idle > 0) {
            const float beside = 5.f + .23f * own / (float)idle;
            const float u = (tc > beside ? tc : beside) + join;
            if (u <= t) t = u, sms = idle;
        }
        const float score = t * (tc + join);
        if (!p->np || score < best) best = score, p->np = np, p->c_pre = c * kPtRows, p->own_sms = sms;
    }
}

static void attn_plan(const jdg_paged_kv *kv, const jdg_attn_args *a, PaArgs *p) {
    const int G = a->n_heads / kv->n_kv_heads;
    p->k = kv->k; p->v = kv->v; p->page_stride = kv->page_stride; p->row_stride = kv->row_stride;
    p->head_stride = kv->head_stride; p->n_pages = kv->n_pages; p->page_shift = log2_ceil(kv->page_size);
    p->table = kv->table; p->table_stride = kv->table_stride; p->q = a->q; p->q_stride = a->q_stride; p->out = a->out;
    p->out_stride = a->out_stride; p->lse = a->lse; p->H = a->n_heads; p->KV = kv->n_kv_heads; p->G = G;
    p->hd = kv->head_dim; p->n_seqs = kv->n_seqs; p->prefix = a->prefix; p->prefix_len = a->prefix_len;
    p->lens = a->lens; p->max_len = a->max_len; p->scale = a->scale; p->clamp = a->clamp; p->status = a->status;
    const int64_t prows = (int64_t)kv->n_seqs * G;
    const bool mma = kv->dt != JD_F32;
    p->r_pre = mma ? (prows <= 8 ? 8 : 16) : r_template(prows > 4 ? 4 : (int)prows);
    p->r_own = mma ? (G <= 8 ? 8 : 16) : r_template(G);
    p->rb_pre = (int)((prows + p->r_pre - 1) / p->r_pre);
    p->rb_own = (G + p->r_own - 1) / p->r_own;
    p->f32 = !mma;
    p->np = p->n_own = 0;
    p->own_sms = kDevSMs;
    // the tensor-core kernel takes a row's maximum before the scale, and masks there: with scale 0 a masked -inf
    // would become NaN, with a negative one the maximum the minimum; both go to the warp kernels, which scale first
    p->tc = a->prefix_len && prows > 16 && (!mma || a->scale > 0.f);
    if (p->tc && !mma) {
        p->rb_pre = (int)((prows + kPfQueries - 1) / kPfQueries);
        p->r_pre = kPfQueries;
        const int64_t units = (int64_t)p->rb_pre * kv->n_kv_heads;
        const int tiles = (a->prefix_len + 31) / 32;
        int64_t splits = 2 * kDevSMs / units;
        splits = splits < 1 ? 1 : splits > tiles ? tiles : splits;
        p->c_pre = (int)((tiles + splits - 1) / splits) * 32;
    } else if (p->tc) {
        p->rb_pre = (int)((prows + 2 * kPtRows - 1) / (2 * kPtRows));
        split_tc(p, (a->prefix_len + kPtRows - 1) / kPtRows, prows, kv->n_kv_heads * p->rb_own);
    } else if (a->prefix_len) {
        // shared and own rows in one launch: the same count of queries at a time
        p->r_pre = p->r_own = p->r_pre > p->r_own ? p->r_pre : p->r_own;
        p->rb_pre = (int)((prows + p->r_pre - 1) / p->r_pre);
        p->rb_own = (G + p->r_own - 1) / p->r_own;
        p->c_pre = chunk_for((int64_t)p->rb_pre * kv->n_kv_heads, a->prefix_len, attn_warps(*p));
    }
    p->r_rows = G < p->r_own ? G : p->r_own;
    if (a->prefix_len) p->np = (a->prefix_len + p->c_pre - 1) / p->c_pre;
    // own rows: shared out over 12 warps of each of their SMs (resident or, some f32 kernels, in turns: see
    // chunk_for); up to two tiles for each warp of a CTA without a prefix go one sequence to a CTA, which then
    // writes the result
    const int nw = attn_warps(*p);
    if (a->max_len && (a->prefix_len || a->max_len > 2 * nw * kPaTile)) {
        p->n_own = 12 / nw * p->own_sms / (kv->n_kv_heads * p->rb_own);
        if (p->n_own < 1) p->n_own = 1;
        if (kv->n_seqs >= 2 * p->n_own && (!p->np || p->tc)) {  // several sequences to a CTA: a warp each
            p->solo = 1;
            p->n_own *= nw;
        }
    }
}

// The workspace: parts of the prefix, pieces of the own rows, the sequences' first pieces and counts.  False:
// none needed.
static bool attn_layout(const jdg_paged_kv *kv, const PaArgs &p, size_t *own, size_t *pieces, size_t *bytes) {
    const size_t part = (size_t)(p.hd + 4) * 4;
    const bool join = p.n_own || p.np > 1 || p.tc;
    *own = join ? (size_t)kv->n_seqs * p.H * p.np * part : 0;
    *pieces = *own + (p.n_own ? (size_t)p.KV * p.rb_own * (p.n_own + kv->n_seqs) * p.r_rows * part : 0);
    *bytes = *pieces + (p.n_own ? (size_t)kv->n_seqs * 8 : 0);
    return join;
}

extern "C" size_t jdg_paged_attn_workspace(const jdg_paged_kv *kv, const jdg_attn_args *a) {
    if (jdg_paged_attn_check(kv, a) != JD_OK) return 0;
    if (kv->n_seqs == 0) return 16;  // nothing to do
    PaArgs p = {};
    attn_plan(kv, a, &p);
    size_t own, pieces, bytes;
    return attn_layout(kv, p, &own, &pieces, &bytes) && bytes > 16 ? bytes : 16;
}

// CTAs of a warp kernel: those of the shared rows (unless another kernel has them), then the own rows'
static int64_t attn_ctas(PaArgs &p, int nw) {
    const int64_t units = (int64_t)p.KV * p.rb_own;
    p.cta_pre = p.np && !p.tc ? p.np * p.KV * p.rb_pre : 0;
    return p.cta_pre + (p.n_own ? p.n_own / (p.solo ? nw : 1) : p.np ? 0 : p.n_seqs) * units;
}
template <int HDP, int R, bool FULL, int TEAM>
static int attn_simt_t(PaArgs p, bool pdl, int dev, cudaStream_t st) {
    using S = PaSimt<HDP, R>;
    const char *who = "jdg_paged_attn";
    int rc = devop_smem<k_pa_simt<HDP, R, FULL, TEAM>>(who, dev, S::kSmem);
    if (rc != JD_OK) return rc;
    const unsigned n = (unsigned)attn_ctas(p, S::kNW);
    return devop_launch(who, pdl, k_pa_simt<HDP, R, FULL, TEAM>, dim3(n), dim3(32 * S::kNW), S::kSmem, st, p);
}
template <int HDP, int R, bool FULL>
static int attn_simt_f(const PaArgs &p, bool pdl, int dev, cudaStream_t st) {
    return p.solo ? attn_simt_t<HDP, R, FULL, 1>(p, pdl, dev, st)
                  : attn_simt_t<HDP, R, FULL, PaSimt<HDP, R>::kNW>(p, pdl, dev, st);
}
template <int HDP, int R>
static int attn_simt(const PaArgs &p, bool pdl, int dev, cudaStream_t st) {
    return p.hd == HDP ? attn_simt_f<HDP, R, true>(p, pdl, dev, st) : attn_simt_f<HDP, R, false>(p, pdl, dev, st);
}
template <int HDP>
static int attn_simt_r(const PaArgs &p, bool pdl, int dev, cudaStream_t st) {
    switch (p.r_own) {
        case 1: return attn_simt<HDP, 1>(p, pdl, dev, st);
        case 2: return attn_simt<HDP, 2>(p, pdl, dev, st);
        case 3: return attn_simt<HDP, 3>(p, pdl, dev, st);
        case 4: return attn_simt<HDP, 4>(p, pdl, dev, st);
        default: return attn_simt<HDP, 8>(p, pdl, dev, st);
    }
}
template <int HDP>
static int attn_f32(const PaArgs &p, int dev, cudaStream_t st) {
    const char *who = "jdg_paged_attn";
    int rc = devop_smem<k_pa_f32<HDP>>(who, dev, PaF32<HDP>::kSmem);
    if (rc != JD_OK) return rc;
    return devop_launch(who, false, k_pa_f32<HDP>, dim3((unsigned)(p.np * p.KV * p.rb_pre)), dim3(32 * kPfWarps),
                        PaF32<HDP>::kSmem, st, p);
}
template <typename T, int HDP, int NQ, bool FULL, int TEAM>
static int attn_mma_t(PaArgs p, bool pdl, int dev, cudaStream_t st) {
    using S = PaMma<HDP>;
    const char *who = "jdg_paged_attn";
    int rc = devop_smem<k_pa_mma<T, HDP, NQ, FULL, TEAM>>(who, dev, S::kSmem);
    if (rc != JD_OK) return rc;
    const unsigned n = (unsigned)attn_ctas(p, S::kNW);
    return devop_launch(who, pdl, k_pa_mma<T, HDP, NQ, FULL, TEAM>, dim3(n), dim3(32 * S::kNW), S::kSmem, st, p);
}
template <typename T, int HDP, int NQ, bool FULL>
static int attn_mma(const PaArgs &p, bool pdl, int dev, cudaStream_t st) {
    return p.solo ? attn_mma_t<T, HDP, NQ, FULL, 1>(p, pdl, dev, st)
                  : attn_mma_t<T, HDP, NQ, FULL, PaMma<HDP>::kNW>(p, pdl, dev, st);
}
template <typename T, int HDP, bool FULL>
static int attn_mma_r(const PaArgs &p, bool pdl, int dev, cudaStream_t st) {
    return p.r_own <= 8 ? attn_mma<T, HDP, 1, FULL>(p, pdl, dev, st) : attn_mma<T, HDP, 2, FULL>(p, pdl, dev, st);
}
template <typename T, int HDP>
static int attn_mma_f(const PaArgs &p, bool pdl, int dev, cudaStream_t st) {
    return p.hd == HDP ? attn_mma_r<T, HDP, true>(p, pdl, dev, st) : attn_mma_r<T, HDP, false>(p, pdl, dev, st);
}
// the warp kernel: own rows, and the shared ones behind few queries
template <typename T>
static int attn_warp(const PaArgs &p, bool pdl, int dev, cudaStream_t st) {
    if constexpr (sizeof(T) == 4)
        return p.hd <= 64 ? attn_simt_r<64>(p, pdl, dev, st) : attn_simt_r<128>(p, pdl, dev, st);
    else
        return p.hd <= 64 ? attn_mma_f<T, 64>(p, pdl, dev, st) : attn_mma_f<T, 128>(p, pdl, dev, st);
}
template <typename T, int HDP, bool FULL, int CLAMP>
static int attn_tc_c(const PaArgs &p, int dev, cudaStream_t st) {
    const char *who = "jdg_paged_attn";
    int rc = devop_smem<k_pa_tc<T, HDP, FULL, CLAMP>>(who, dev, PaTc<HDP>::kSmem);
    if (rc != JD_OK) return rc;
    const unsigned n = (unsigned)(p.np * p.KV * p.rb_pre);
    return devop_launch(who, false, k_pa_tc<T, HDP, FULL, CLAMP>, dim3(n), dim3(kPtThreads), PaTc<HDP>::kSmem, st, p);
}
template <typename T, int HDP, bool FULL>
static int attn_tc(const PaArgs &p, int dev, cudaStream_t st) {
    return p.clamp > kPaWide ? attn_tc_c<T, HDP, FULL, 2>(p, dev, st)
           : p.clamp > 0.f   ? attn_tc_c<T, HDP, FULL, 1>(p, dev, st)
                             : attn_tc_c<T, HDP, FULL, 0>(p, dev, st);
}
// the shared rows behind many queries
template <typename T>
static int attn_shared(const PaArgs &p, int dev, cudaStream_t st) {
    if constexpr (sizeof(T) == 2)
        return p.hd == 64    ? attn_tc<T, 64, true>(p, dev, st)
               : p.hd < 64   ? attn_tc<T, 64, false>(p, dev, st)
               : p.hd == 128 ? attn_tc<T, 128, true>(p, dev, st)
                             : attn_tc<T, 128, false>(p, dev, st);
    else
        return p.hd <= 64 ? attn_f32<64>(p, dev, st) : attn_f32<128>(p, dev, st);
}
template <typename T>
static int attn_run(const PaArgs &p, bool join, int dev, cudaStream_t st) {
    const char *who = "jdg_paged_attn";
    int rc = p.tc ? attn_shared<T>(p, dev, st) : JD_OK;
    if (rc == JD_OK && (!p.tc || p.n_own)) rc = attn_warp<T>(p, p.tc, dev, st);
    if (rc == JD_OK && join) {
        // four warps to a query where there are few
        const int64_t rows = (int64_t)p.n_seqs * p.H;
        rc = rows <= 8 * kDevSMs
                 ? devop_launch(who, true, k_pa_merge<T, 4>, dim3((unsigned)rows), dim3(128), 0, st, p)
                 : devop_launch(who, true, k_pa_merge<T, 1>, dim3((unsigned)((rows + 3) / 4)), dim3(128), 0, st, p);
    }
    return rc;
}

extern "C" int jdg_paged_attn(const jdg_paged_kv *kv, const jdg_attn_args *a, void *workspace, size_t workspace_bytes,
                              void *stream) {
    const char *who = "jdg_paged_attn";
    int rc = jdg_paged_attn_check(kv, a), dev;
    if (rc != JD_OK) return rc;
    if (kv->n_seqs == 0) return JD_OK;
    PaArgs p = {};
    attn_plan(kv, a, &p);
    size_t own, pieces, need;
    const bool join = attn_layout(kv, p, &own, &pieces, &need);
    if (join) {
        if (!workspace || misaligned(workspace, 16) || workspace_bytes < need) {
            jdg_set_err(nullptr, "%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", who, need,
                        workspace ? workspace_bytes : (size_t)0);
            return JD_EINVAL;
        }
        p.part = (float *)workspace;
        if (p.n_own) {
            p.own = (float *)((char *)workspace + own);
            p.pieces = (int2 *)((char *)workspace + pieces);
        }
    }
    cudaStream_t st = (cudaStream_t)stream;
    rc = devop_stream(who, st, &dev);
    if (rc != JD_OK) return rc;
    return kv->dt == JD_F32   ? attn_run<float>(p, join, dev, st)
           : kv->dt == JD_F16 ? attn_run<__half>(p, join, dev, st)
                              : attn_run<__nv_bfloat16>(p, join, dev, st);
}
