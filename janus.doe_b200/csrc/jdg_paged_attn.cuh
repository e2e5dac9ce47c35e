// jdg_paged_attn.cuh — kernels of the attention over a paged cache with a shared prefix.
//
//   s_t = scale q.k_t (clamped: c tanh(s_t / c)),  out = sum_t e^{s_t} v_t / sum_t e^{s_t}
//
// in one pass over the rows with the running maximum m and sum l (kept in base 2):
//   m' = max(m, s),  l' = l 2^{m - m'} + 2^{s - m'},  o' = o 2^{m - m'} + 2^{s - m'} v
// Parts over different rows join by the same rule, so the rows are split over CTAs and the
// shared rows are read for many queries at once.
#pragma once
#include "jdg_devop.cuh"

namespace jdg {

struct PaArgs {
    const void *k, *v;
    int64_t page_stride, row_stride, head_stride;
    int n_pages, page_shift;
    const int *table;
    int table_stride;
    const void *q;
    int64_t q_stride;
    void *out;
    int64_t out_stride;
    float *lse;
    int H, KV, G, hd, n_seqs;
    const int *prefix;
    int prefix_len;
    const int *lens;
    int max_len;
    float scale, clamp;
    int *status;
    // a part of a query is [m, l, -, -, out[hd]]
    float *part;             // parts of the shared rows: [n_seqs * H][np]
    float *own;              // parts of the own rows: [piece][r_rows]; null: no join, the result is written
    int2 *pieces;            // [n_seqs] first piece and count of each sequence, written by the first CTA
    int np;                  // parts of the shared rows
    int c_pre;               // rows of each
    int r_pre, r_own;        // queries that are taken at a time
    int rb_pre, rb_own;      // blocks of queries for each KV head
    int r_rows;              // queries of a block of own rows: min(G, r_own)
    int own_sms;             // SMs that these are shared out over (host)
    int n_own;               // teams that share the own rows of a unit (KV head, block of queries); 0: none
    int solo;                // a team is a warp (else a CTA)
    int cta_pre;             // CTAs of the warp kernel that take shared rows (the first ones)
    int tc, f32;             // the shared rows in a kernel of their own (many queries); f32 cache
};

constexpr int kPaTile = 32;         // cache rows that a warp takes in one go
// The running maximum that the weights are formed against moves only once a score passes it by 2^8 (a published
// variant of the one-pass softmax: after the first tiles nearly none rescales).  Compared as a difference, which
// is exact where the sum with the slack would round.
constexpr float kPaSlack = 8.f;
// The 16-bit kernels round each weight once to the values' type for the second product (the sum l takes it as
// it was): half a step, bf16 2^-8 or f16 2^-11 of sum p |v| at most, about what the rounding of the result adds
// again (bf16, 64 x 32,789 rows: 0.0022 off 64 bits, 0.0017 of it the result's own).  Products of f32 weights would
// be three times the matrix instructions.  f16 ends at 2^-24, so there the weights are held 2^7 times
// higher (up to 2^15 with the slack): what falls below its range is under 2^-32 of the largest weight, not 2^-25.
template <typename T>
constexpr float kPaLift = sizeof(T) == 2 && __is_same(T, __half) ? 7.f : 0.f;

// c tanh(y / c) for |y / c| <= 0.6, u = (y / c)^2: y + y u p(u), an odd polynomial whose largest relative
// error there is least (2^-23.7, fitted by Lawson's iteration).  y / c is only in u: however far c is above y,
// nothing is lost.
constexpr float kPaSmall = 0.6f;
__device__ __forceinline__ float pa_tanh_small(float y, float u) {
    constexpr float p[5] = {-5.89516e-3f, 2.079597e-2f, -5.378383e-2f, 1.3331924e-1f, -3.33333e-1f};
    float q = p[0];
#pragma unroll
    for (int i = 1; i < 5; i++) q = fmaf(q, u, p[i]);
    return fmaf(y * u, q, y);
}
__device__ __forceinline__ float2 pa_tanh_small(float2 y, float2 u) {
    constexpr float p[5] = {-5.89516e-3f, 2.079597e-2f, -5.378383e-2f, 1.3331924e-1f, -3.33333e-1f};
    float2 q = make_float2(p[0], p[0]);
#pragma unroll
    for (int i = 1; i < 5; i++) q = fma2(q, u, make_float2(p[i], p[i]));
    return fma2(mul2(y, u), q, y);
}

// Scores in base 2 from the raw dot products of an f32 cache.  The clamp's tanh: the polynomial where every
// argument of the warp is small (scores below 0.6 clamp, the rule), a third of tanhf's instructions; tanhf
// otherwise.
template <int N>
__device__ __forceinline__ void pa_scores(float (&s)[N], const PaArgs &p) {
    const float lin = p.scale * kLog2e;
    if (!(p.clamp > 0.f)) {
#pragma unroll
        for (int i = 0; i < N; i++) s[i] = s[i] * p.scale * kLog2e;
        return;
    }
    const float in = p.scale / p.clamp, out = p.clamp * kLog2e;
    bool small = true;
#pragma unroll
    for (int i = 0; i < N; i++) small = small && fabsf(s[i] * in) <= kPaSmall;
    if (__all_sync(JDG_FULL, small)) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float x = s[i] * in;
            s[i] = pa_tanh_small(s[i] * lin, x * x);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) s[i] = tanhf(s[i] * in) * out;
    }
}

// length of sequence s's own rows where the result is written: -1 idle, cut at max_len and flagged
__device__ __forceinline__ int pa_len(const PaArgs &p, int s) {
    const int n = p.lens[s];
    if (n > p.max_len && p.status) atomicOr(p.status, JDG_STATUS_POS);
    return n < 0 ? -1 : min(n, p.max_len);
}

__device__ __forceinline__ float *pa_part(const PaArgs &p, int row, int split) {
    return p.part + ((int64_t)row * p.np + split) * (p.hd + 4);
}

// How the own rows are shared out: they are cut into tiles of 32 rows, `sum` in all over the
// sequences; for each unit (KV head, block of queries) n_own teams take equal runs of this list
// (the first few one tile more), so every team has the same work, whatever the lengths.  A team is a
// CTA, whose warps take the tiles in turn and join at the end of each sequence, or, where the
// sequences are many, a warp on its own (256 sequences of 124 rows on average, f32: 24 us against
// 34; 8 of 4,000: the other way round, 37 against 33, for the parts to be joined).  Where sum is less
// than n_own, only sum teams have work: none in between is empty.  The units of a team number c are
// neighbours in the grid: they read the heads of the same cache rows at the same time.  A piece is
// what a team has of a sequence; c + sequence numbers a sequence's pieces without gaps.
struct PaShare {
    int n, each, more;  // teams, tiles of each, teams with one more
    __device__ __forceinline__ PaShare(int n_own, int sum) : n(min(n_own, sum)), each(n ? sum / n : 0), more(sum - each * n) {}
    __device__ __forceinline__ int first(int c) const { return c * each + min(c, more); }
    __device__ __forceinline__ int of(int tile) const {
        const int big = more * (each + 1);
        return tile < big ? tile / (each + 1) : more + (tile - big) / each;
    }
};

// The join of a query's parts: W warps (4 for few queries, else 1) take every W-th batch of eight;
// a lane reads the (m, l) of one part and four numbers of each output, so the kernel is a few trips
// to L2 long.
template <typename T, int W>
__global__ __launch_bounds__(128) void k_pa_merge(const __grid_constant__ PaArgs p) {
    __shared__ float4 so[4][32];
    __shared__ float sm[4], sl[4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = W == 4 ? warp : 0;
    const int row = W == 4 ? blockIdx.x : blockIdx.x * 4 + warp;
    const int s = min(row / p.H, p.n_seqs - 1), h = row - s * p.H, len = pa_len(p, s);
    // before any return: what follows on the stream waits for this kernel alone, and must find the ones before
    // it done even where no query here has anything to write
    dep_wait();
    if (row >= p.n_seqs * p.H || len < 0) return;  // the same for the warps of a query
    const int64_t st = p.hd + 4;
    // parts: np of the shared rows, then the sequence's pieces
    const float *shared = p.part + (int64_t)row * p.np * st, *own = nullptr;
    int n = p.np;
    int64_t own_st = 0;
    if (p.own && len > 0) {
        const int kvh = h / p.G, g = h - kvh * p.G, unit = kvh * p.rb_own + g / p.r_own;
        const int2 pc = p.pieces[s];
        own_st = p.r_rows * st;
        own = p.own + (((int64_t)unit * (p.n_own + p.n_seqs) + pc.x) * p.r_rows + g % p.r_own) * st;
        n += pc.y;
    }
    auto at = [&](int i) { return i < p.np ? shared + i * st : own + (i - p.np) * own_st; };
    const int d = lane * 4;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = sub * 8; i0 < n; i0 += 8 * W) {
        const int nn = min(8, n - i0);
        float4 v[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < nn && d < p.hd) v[j] = ld4(at(i0 + j) + 4 + d);
        const bool in = lane < nn;
        const float2 ml = in ? *reinterpret_cast<const float2 *>(at(i0 + lane)) : make_float2(-INFINITY, 0.f);
        float x = ml.x;
#pragma unroll
        for (int q = 4; q; q >>= 1) x = fmaxf(x, __shfl_xor_sync(JDG_FULL, x, q));
        const float mn = fmaxf(m, __shfl_sync(JDG_FULL, x, 0)), base = mn == -INFINITY ? 0.f : mn, f = ex2(m - base);
        const float w = in ? ex2(ml.x - base) : 0.f;
        float lw = in ? ml.y * w : 0.f;
#pragma unroll
        for (int q = 4; q; q >>= 1) lw += __shfl_xor_sync(JDG_FULL, lw, q);
        l = l * f + __shfl_sync(JDG_FULL, lw, 0);
        o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
        m = mn;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float wj = __shfl_sync(JDG_FULL, w, j);
            if (j < nn && d < p.hd) {
                o.x = fmaf(wj, v[j].x, o.x);
                o.y = fmaf(wj, v[j].y, o.y);
                o.z = fmaf(wj, v[j].z, o.z);
                o.w = fmaf(wj, v[j].w, o.w);
            }
        }
    }
    if (W == 4) {
        so[warp][lane] = o;
        if (lane == 0) {
            sm[warp] = m;
            sl[warp] = l;
        }
        __syncthreads();
        if (warp) return;
        const float mn = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])), base = mn == -INFINITY ? 0.f : mn;
        o = make_float4(0.f, 0.f, 0.f, 0.f);
        l = 0.f;
        m = mn;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float f = ex2(sm[k] - base);
            const float4 x = so[k][lane];
            l = fmaf(f, sl[k], l);
            o = make_float4(fmaf(f, x.x, o.x), fmaf(f, x.y, o.y), fmaf(f, x.z, o.z), fmaf(f, x.w, o.w));
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;  // NaN stays NaN
    if (d < p.hd)
        st4((T *)p.out + (int64_t)s * p.out_stride + (int64_t)h * p.hd + d,
            make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
    if (p.lse && lane == 0) p.lse[row] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
}

// What a CTA works on: R queries from row r0 (of nrows) of KV head kvh, cache rows [t0, t1)
// behind `tab`; split: part of the shared rows, or piece of the own ones.
struct PaWork {
    int kvh, r0, nrows, t0, t1, split, seq;  // seq -1: the shared rows
    int cap;                                 // rows that the table names, whatever the length
    const int *tab;
};
__device__ __forceinline__ void pa_work_shared(const PaArgs &p, int R, PaWork &w) {
    int id = blockIdx.x;  // blocks of queries of the same rows next to one another
    const int rb = id % p.rb_pre;
    id /= p.rb_pre;
    w.kvh = id % p.KV;
    w.split = id / p.KV;
    w.r0 = rb * R;
    w.nrows = min(R, p.n_seqs * p.G - w.r0);
    w.t0 = w.split * p.c_pre;
    w.t1 = min(p.prefix_len, w.t0 + p.c_pre);
    w.cap = w.t1;
    w.seq = -1;
    w.tab = p.prefix;
}
// (sequence, head) of query row i of the work
__device__ __forceinline__ void pa_row(const PaArgs &p, const PaWork &w, int i, int &s, int &h) {
    const int r = w.r0 + i;
    if (w.seq < 0) {
        s = r / p.G;
        h = w.kvh * p.G + (r - s * p.G);
    } else {
        s = w.seq;
        h = w.kvh * p.G + r;
    }
}

// ------------------------------------------------------------------------------------
// What a team of the warp kernels works on: a run of tiles of 32 cache rows of one KV head, for a
// block of queries.
struct PaSpan {
    int seq, seg0;            // first sequence (-1: the shared rows) and its first tile in the list
    int at, end;              // tiles of the list
    int kvh, r0, nrows, base;  // KV head, queries, number of the part (of a piece: less its sequence)
};
// rows that a sequence has (seq -1: of the shared rows, to the end of the span)
__device__ __forceinline__ int pa_rows(const PaArgs &p, const PaSpan &g, int seq) {
    return seq < 0 ? min(p.prefix_len, g.end * kPaTile) : max(0, min(p.lens[seq], p.max_len));
}
__device__ __forceinline__ int pa_tiles_of(int rows) { return (rows + kPaTile - 1) / kPaTile; }
struct PaTile {
    int seq, seg0, rows;  // sequence, its first tile, its rows
    // on to the sequence that has tile i of the list
    __device__ __forceinline__ void seek(const PaArgs &p, const PaSpan &g, int i) {
        for (int n; i >= seg0 + (n = pa_tiles_of(rows));) {
            seg0 += n;
            rows = pa_rows(p, g, ++seq);
        }
    }
};
__device__ __forceinline__ void pa_unit(const PaArgs &p, int unit, PaSpan &g) {
    const int rb = unit % p.rb_own;
    g.kvh = unit / p.rb_own;
    g.r0 = rb * p.r_own;
    g.nrows = min(p.r_own, p.G - g.r0);
}
// (sequence, head) of query i
__device__ __forceinline__ void pa_query(const PaArgs &p, const PaSpan &g, int seq, int i, int &s, int &h) {
    const int r = g.r0 + i;
    s = seq < 0 ? r / p.G : seq;
    h = g.kvh * p.G + (seq < 0 ? r - s * p.G : r);
}
// The span of this team of TEAM warps (the CTA has NW); false: none.  Called by the whole CTA.  To
// share the own rows out, every CTA adds the lengths up for itself (a scan over the sequences: one
// load a thread up to 128 of them).
template <int NW, int TEAM>
__device__ __forceinline__ bool pa_span(const PaArgs &p, int R, PaSpan &g) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if ((int)blockIdx.x < p.cta_pre) {  // shared rows, equal parts; blocks of queries of the same rows side by side
        int id = blockIdx.x * (NW / TEAM) + warp / TEAM;
        const int rb = id % p.rb_pre;
        id /= p.rb_pre;
        g.kvh = id % p.KV;
        g.base = id / p.KV;
        if (g.base >= p.np) return false;
        g.r0 = rb * R;
        g.nrows = min(R, p.n_seqs * p.G - g.r0);
        g.seq = -1;
        g.seg0 = 0;
        g.at = g.base * (p.c_pre / kPaTile);
        g.end = min(pa_tiles_of(p.prefix_len), g.at + p.c_pre / kPaTile);
        return true;
    }
    const int units = p.KV * p.rb_own, b = blockIdx.x - p.cta_pre, row = b / units;
    const int c = row * (NW / TEAM) + warp / TEAM;  // number of the team
    pa_unit(p, b - row * units, g);
    if (!p.own) {  // a sequence to a team: its result
        if (c >= p.n_seqs) return false;
        g.seq = c;
        g.seg0 = g.at = g.base = 0;
        const int n = min(p.lens[c], p.max_len);
        g.end = pa_tiles_of(max(0, n));
        return n >= 0;
    }
    __shared__ int sums[NW], found[NW / TEAM][2];
    constexpr int NT = 32 * NW;
    const int per = (p.n_seqs + NT - 1) / NT, s0 = min(p.n_seqs, tid * per), s1 = min(p.n_seqs, s0 + per);
    int mine = 0;
    for (int s = s0; s < s1; s++) mine += pa_tiles_of(pa_rows(p, g, s));
    int inc = mine;  // inclusive scan
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(JDG_FULL, inc, o);
        if (lane >= o) inc += x;
    }
    if (lane == 31) sums[warp] = inc;
    __syncthreads();
    int before = inc - mine, sum = 0;
#pragma unroll
    for (int k = 0; k < NW; k++) {
        before += k < warp ? sums[k] : 0;
        sum += sums[k];
    }
    const PaShare share(p.n_own, sum);
    if (b == 0) {
        int x = before;
        for (int s = s0; s < s1; s++) {
            const int n = pa_tiles_of(pa_rows(p, g, s));
            const int c0 = n ? share.of(x) : 0;
            p.pieces[s] = make_int2(c0 + s, n ? share.of(x + n - 1) - c0 + 1 : 0);
            x += n;
        }
    }
#pragma unroll
    for (int k = 0; k < NW / TEAM; k++) {  // where each team starts: found by the thread that has the sequence
        const int w = row * (NW / TEAM) + k, at = w < share.n ? share.first(w) : -1;
        if (at >= before && at < before + mine) {
            int x = before, s = s0;
            for (int n; x + (n = pa_tiles_of(pa_rows(p, g, s))) <= at; s++) x += n;
            found[k][0] = s;
            found[k][1] = x;
        }
    }
    __syncthreads();
    if (c >= share.n) return false;
    g.at = share.first(c);
    g.end = share.first(c + 1);
    g.seq = found[warp / TEAM][0];
    g.seg0 = found[warp / TEAM][1];
    g.base = (b - row * units) * (p.n_own + p.n_seqs) + c;
    return true;
}
// Where query i's result for the rows of sequence seq goes: a part, or null: out and lse.
__device__ __forceinline__ float *pa_part_of(const PaArgs &p, const PaSpan &g, int seq, int i, int s, int h) {
    if (seq < 0) return p.part ? pa_part(p, s * p.H + h, g.base) : nullptr;
    return p.own ? p.own + ((int64_t)(g.base + seq) * p.r_rows + i) * (p.hd + 4) : nullptr;
}

// The end of a piece: the parts of the team's warps (m, l behind HDP numbers each, `stride` floats
// from warp to warp; a warp without a tile in the piece has none), joined and written.
template <typename T, int HDP, int NW>  // NW: warps of the team
__device__ __forceinline__ void pa_finish(const PaArgs &p, const PaSpan &g, int seq, const float *mg, int stride, int first,
                                          int count) {
    const int lane = threadIdx.x & 31;
    for (int r = (threadIdx.x >> 5) % NW; r < g.nrows; r += NW) {
        float mx = -INFINITY, sum = 0.f, f[NW];
#pragma unroll
        for (int k = 0; k < NW; k++) {
            f[k] = -INFINITY;
            if ((k - first + NW) % NW < count) f[k] = mg[k * stride + r * (HDP + 2) + HDP];
            mx = fmaxf(mx, f[k]);
        }
        const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
        for (int k = 0; k < NW; k++)
            if ((k - first + NW) % NW < count) {
                f[k] = ex2(f[k] - base);
                sum = fmaf(f[k], mg[k * stride + r * (HDP + 2) + HDP + 1], sum);
            }
        int s, h;
        pa_query(p, g, seq, r, s, h);
        float *part = pa_part_of(p, g, seq, r, s, h);
        if (!part && pa_len(p, s) < 0) continue;
        T *out = (T *)p.out + (int64_t)s * p.out_stride + (int64_t)h * p.hd;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // NaN stays NaN
#pragma unroll
        for (int d = lane; d < HDP; d += 32) {
            float val = 0.f;
#pragma unroll
            for (int k = 0; k < NW; k++)
                if ((k - first + NW) % NW < count) val = fmaf(f[k], mg[k * stride + r * (HDP + 2) + d], val);
            if (d < p.hd) {
                if (part) part[4 + d] = val;
                else out[d] = from_f<T>(val * inv);
            }
        }
        if (lane == 0) {
            if (part) *reinterpret_cast<float2 *>(part) = make_float2(mx, sum);
            else if (p.lse) p.lse[s * p.H + h] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2;
        }
    }
}

// 32 cache rows to shared memory, ROW bytes apart.  off: this lane's row (row number = lane) in
// elements, in the pool even where the row is none of the work's; valid: the rows that are
// (others become zeros, unread).  FULL: head_dim is HDP; pages of 16 rows or more then need one
// exchange for 16 rows, smaller ones an exchange for each row.
template <typename T, int HDP, bool FULL, int ROW>
__device__ __forceinline__ void pa_load32(uint32_t dst, const T *base, int64_t off, uint32_t valid, const PaArgs &p) {
    constexpr int EPC = 16 / (int)sizeof(T);
    const int lane = threadIdx.x & 31;
    if constexpr (FULL) {
        constexpr int cpr = HDP / EPC, rpi = 32 / cpr;
        const int lr = lane / cpr, lc = lane % cpr;
        dst += lr * ROW + lc * 16;
        base += lc * EPC;
        const uint32_t mine = valid >> lr;
        if (p.page_shift >= 4) {
            const int64_t inc = rpi * p.row_stride;
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const T *src = base + __shfl_sync(JDG_FULL, off, half * 16) + lr * p.row_stride;
#pragma unroll
                for (int i = 0; i < 16 / rpi; i++) {
                    const int r = half * 16 + i * rpi;
                    cp16(dst + r * ROW, src, mine >> r & 1u);
                    src += inc;
                }
            }
        } else {
#pragma unroll
            for (int r = 0; r < 32; r += rpi) {
                const T *src = base + __shfl_sync(JDG_FULL, off, r + lr);
                cp16(dst + r * ROW, src, mine >> r & 1u);
            }
        }
    } else {
        const int cpr = p.hd / EPC, rpi = 32 / cpr, lr = lane / cpr, lc = lane - lr * cpr;
        for (int r0 = 0; r0 < 32; r0 += rpi) {
            const int r = r0 + lr;
            const int64_t o = __shfl_sync(JDG_FULL, off, r & 31);
            if (lr < rpi && r < 32) cp16(dst + r * ROW + lc * 16, base + o + lc * EPC, valid >> r & 1u);
        }
    }
}

// The walk over a team's tiles, piece by piece; its NW warps take tiles in turn.  The loads of a warp's
// next tile, of this piece or a later one, are in flight: its keys once this tile's scores are
// done, its values once this tile's outputs are (at the end of a piece: once the values' memory
// has served to join the warps).  Body gives: queries(seq), scores(), weights(valid), values(),
// leave(memory).  A page is looked up a tile before it is needed.
template <typename T, int HDP, bool FULL, int ROW, int NW, int STRIDE, typename Body>
__device__ __forceinline__ void pa_walk(const PaArgs &p, const PaSpan &g, uint8_t *sm, Body &body) {
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % NW, pmask = (1 << p.page_shift) - 1;
    const T *kh = (const T *)p.k + (int64_t)g.kvh * p.head_stride, *vh = (const T *)p.v + (int64_t)g.kvh * p.head_stride;
    const uint32_t ks = (uint32_t)__cvta_generic_to_shared(sm + warp * STRIDE), vs = ks + kPaTile * ROW;
    auto page_of = [&](const PaTile &x, int i) {
        const int *tab = x.seq < 0 ? p.prefix : p.table + (int64_t)x.seq * p.table_stride;
        const int t = (i - x.seg0) * kPaTile + lane;
        return t < x.rows ? tab[t >> p.page_shift] : -1;
    };
    // this lane's row: its place in the pool (in the pool even where the row is none), and the rows that count
    auto place = [&](const PaTile &x, int i, int pg, uint32_t &valid) {
        const int t = (i - x.seg0) * kPaTile + lane;
        const bool in = t < x.rows, ok = in && pg >= 0 && pg < p.n_pages;
        if (in && !ok && p.status) atomicOr(p.status, JDG_STATUS_PAGE);
        valid = __ballot_sync(JDG_FULL, ok);
        return (ok ? (int64_t)pg * p.page_stride : 0) + (int64_t)(t & pmask) * p.row_stride;
    };
    PaTile piece = {g.seq, g.seg0, pa_rows(p, g, g.seq)}, ahead = piece;
    int i = g.at + warp, page = -1;  // this warp's tile; `ahead` and `page` are of the next one, i + NW
    uint32_t valid = 0;
    if (i < g.end) {
        ahead.seek(p, g, i);
        const int64_t off = place(ahead, i, page_of(ahead, i), valid);
        pa_load32<T, HDP, FULL, ROW>(ks, kh, off, valid, p);
        cp_commit();
        pa_load32<T, HDP, FULL, ROW>(vs, vh, off, valid, p);
        cp_commit();
        if (i + NW < g.end) {
            ahead.seek(p, g, i + NW);
            page = page_of(ahead, i + NW);
        }
    }
    for (int first = g.at;;) {
        const int stop = min(g.end, piece.seg0 + pa_tiles_of(piece.rows));
        const bool some = i < stop;
        if (some) body.queries(piece.seq);
        int64_t off = 0;
        uint32_t vnext = 0;
        bool owed = false;  // the next tile's values are still to be asked for
        while (i < stop) {
            const bool more = i + NW < g.end;
            cp_wait<1>();
            __syncwarp();
            body.scores();
            __syncwarp();
            if (more) {
                off = place(ahead, i + NW, page, vnext);
                pa_load32<T, HDP, FULL, ROW>(ks, kh, off, vnext, p);
                if (i + 2 * NW < g.end) {
                    ahead.seek(p, g, i + 2 * NW);
                    page = page_of(ahead, i + 2 * NW);
                }
            }
            cp_commit();
            body.weights(valid);
            cp_wait<1>();
            __syncwarp();
            body.values();
            __syncwarp();
            owed = i + NW >= stop;
            if (!owed) {
                pa_load32<T, HDP, FULL, ROW>(vs, vh, off, vnext, p);
                cp_commit();
            }
            i += NW;
            valid = vnext;
        }
        float *mg = reinterpret_cast<float *>(sm + kPaTile * ROW);  // the values' memory of the team's first warp
        if (some) body.leave(mg + warp * (STRIDE / 4));
        if (NW > 1) __syncthreads();
        else __syncwarp();
        pa_finish<T, HDP, NW>(p, g, piece.seq, mg, STRIDE / 4, (first - g.at) % NW, stop - first);
        if (NW > 1) __syncthreads();
        else __syncwarp();
        if (owed) {
            if (i < g.end) pa_load32<T, HDP, FULL, ROW>(vs, vh, off, vnext, p);
            cp_commit();
        }
        if (stop >= g.end) break;
        first = stop;
        piece.seek(p, g, stop);
    }
    cp_wait<0>();
}

// ------------------------------------------------------------------------------------
// f32 caches: R queries in plain FMAs.  Rows go to shared memory padded by 16 bytes, so 8 lanes
// reading 8 rows meet 8 bank groups.  Scores: lane = row, one chain over the head's numbers for
// each query; output: lane = numbers, rows in order.  Bound: the cache's bytes for up to 4 queries
// (three FMAs a byte), shared memory's reads of the queries beyond.
template <int HDP, int R>
struct PaSimt {
    static constexpr int kNW = HDP == 64 || R > 4 ? 4 : 6;  // warps of a CTA: what shared memory holds
    static constexpr int kRow = HDP * 4 + 16;             // bytes of a row in shared memory
    static constexpr int kTile = kPaTile * kRow;          // one tile of keys or values
    static constexpr int kWarp = 2 * kTile + R * kPaTile * 4 + R * HDP * 4;  // and weights and queries
    static constexpr int kSmem = kNW * kWarp;
};

template <int HDP, int R, bool FULL>
struct PaSimtBody {
    using S = PaSimt<HDP, R>;
    static constexpr int DPL = HDP / 32;  // numbers a lane sums
    const PaArgs &p;
    const PaSpan &g;
    uint8_t *mine;
    float *ws, *qs;
    int lane;
    float m[R], l[R], o[R][DPL], acc[R];

    __device__ __forceinline__ void queries(int seq) {
        __syncwarp();
#pragma unroll
        for (int r = 0; r < R; r++) {
            m[r] = -INFINITY;
            l[r] = 0.f;
            const float *q = nullptr;
            if (r < g.nrows) {
                int s, h;
                pa_query(p, g, seq, r, s, h);
                q = (const float *)p.q + (int64_t)s * p.q_stride + (int64_t)h * p.hd;
            }
#pragma unroll
            for (int d = 0; d < DPL; d++) {
                o[r][d] = 0.f;
                qs[r * HDP + lane * DPL + d] = q && (FULL || lane * DPL + d < p.hd) ? q[lane * DPL + d] : 0.f;
            }
        }
        __syncwarp();
    }
    __device__ __forceinline__ void scores() {
        const int pieces = FULL ? HDP / 4 : p.hd / 4;
#pragma unroll
        for (int r = 0; r < R; r++) acc[r] = 0.f;
        const uint8_t *krow = mine + lane * S::kRow;
#pragma unroll 4
        for (int c = 0; c < pieces; c++) {
            const float4 k = *reinterpret_cast<const float4 *>(krow + c * 16);
#pragma unroll
            for (int r = 0; r < R; r++) acc[r] = dot4(k, *reinterpret_cast<const float4 *>(qs + r * HDP + c * 4), acc[r]);
        }
    }
    __device__ __forceinline__ void weights(uint32_t valid) {
        bool up = false;
        pa_scores(acc, p);
#pragma unroll
        for (int r = 0; r < R; r++) {
            acc[r] = valid >> lane & 1u ? acc[r] : -INFINITY;
            up |= acc[r] - m[r] > kPaSlack;
        }
        if (__any_sync(JDG_FULL, up)) {
#pragma unroll
            for (int r = 0; r < R; r++) {
                const float mn = fmaxf(m[r], warp_max(acc[r]));
                const float f = m[r] == -INFINITY ? 0.f : ex2(m[r] - mn);
                l[r] *= f;
#pragma unroll
                for (int d = 0; d < DPL; d++) o[r][d] *= f;
                m[r] = mn;
            }
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            const float e = acc[r] == -INFINITY ? 0.f : ex2(acc[r] - m[r]);
            l[r] += e;
            ws[r * kPaTile + lane] = e;
        }
    }
    __device__ __forceinline__ void values() {
        const uint8_t *vcol = mine + S::kTile + lane * DPL * 4;
        if (FULL || lane * DPL < p.hd) {
#pragma unroll 2
            for (int i = 0; i < kPaTile; i += 4) {
                float v[4][DPL];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float *vp = reinterpret_cast<const float *>(vcol + (i + j) * S::kRow);
                    if constexpr (DPL == 2) *reinterpret_cast<float2 *>(v[j]) = *reinterpret_cast<const float2 *>(vp);
                    else *reinterpret_cast<float4 *>(v[j]) = *reinterpret_cast<const float4 *>(vp);
                }
#pragma unroll
                for (int r = 0; r < R; r++) {
                    const float4 e = *reinterpret_cast<const float4 *>(ws + r * kPaTile + i);
#pragma unroll
                    for (int d = 0; d < DPL; d++) {
                        o[r][d] = fmaf(e.x, v[0][d], o[r][d]);
                        o[r][d] = fmaf(e.y, v[1][d], o[r][d]);
                        o[r][d] = fmaf(e.z, v[2][d], o[r][d]);
                        o[r][d] = fmaf(e.w, v[3][d], o[r][d]);
                    }
                }
            }
        }
    }
    __device__ __forceinline__ void leave(float *x) {
#pragma unroll
        for (int r = 0; r < R; r++, x += HDP + 2) {
            const float sum = warp_sum(l[r]);
            if (lane == 0) *reinterpret_cast<float2 *>(x + HDP) = make_float2(m[r], sum);
#pragma unroll
            for (int d = 0; d < DPL; d += 2)
                *reinterpret_cast<float2 *>(x + lane * DPL + d) = make_float2(o[r][d], o[r][d + 1]);
        }
    }
};

template <int HDP, int R, bool FULL, int TEAM>
__global__ __launch_bounds__(32 * PaSimt<HDP, R>::kNW, HDP == 64 ? 3 : 1) void k_pa_simt(const __grid_constant__ PaArgs p) {
    using S = PaSimt<HDP, R>;
    extern __shared__ __align__(16) uint8_t pa_sm[];
    dep_trigger();
    PaSpan g;
    if (pa_span<S::kNW, TEAM>(p, R, g)) {
        uint8_t *mine = pa_sm + (threadIdx.x >> 5) * S::kWarp;
        float *ws = reinterpret_cast<float *>(mine + 2 * S::kTile);
        PaSimtBody<HDP, R, FULL> body{p, g, mine, ws, ws + R * kPaTile, (int)(threadIdx.x & 31)};
        pa_walk<float, HDP, FULL, S::kRow, TEAM, S::kWarp>(p, g, TEAM > 1 ? pa_sm : mine, body);
    }
    // a launch that depends on this one may only rely on what came before once this has waited
    dep_wait();
}

// ------------------------------------------------------------------------------------
// f16 / bf16, up to 8 or 16 queries: the same loop with the products as 16 x 8 x 16 matrix
// instructions, cache rows on the 16-row side (S^T = K Q^T, O^T = V^T P^T), so eight queries
// leave nothing of an instruction unused but the queries that are missing.  This path serves few
// queries per cache row, where the cache's bytes bound the time (8 flops a byte for 4 queries)
// and what counts is how few instructions a row needs: 330 for 32 rows of 128 numbers, against
// 810 with the queries on the 16-row side (measured: call 39 -> 35 us for 134 MB, 33
// with its loads further ahead).  P^T is the
// accumulator of S^T transposed in 8 x 8 blocks (movmatrix); nothing goes through memory.
template <typename T>
__device__ __forceinline__ void pa_mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void pa_mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void pa_mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pa_ldsm(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void pa_ldsm_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// Score in base 2, clamped by tanh x = 1 - 2 / (1 + e^2x): off by 2^-21 clamp at most.  Up to a clamp of 512 that is
// 2^-12, below the 2^-11 or 2^-8 that the weights are rounded to next (30 to 50 is usual: 2^-16).  A larger clamp would show
// in scores far below it (they are off by 0.1 at 10^6), so there small arguments take the polynomial: off by 2^-20
// of the score, whatever the clamp.  64 x 32,789 rows, bf16: 108 us in the first form; in the second 103 where all
// scores are below 0.6 clamp, but 161 where they lie on both sides of it and both are formed, which is usual only
// behind a clamp of 30.
constexpr float kPaWide = 512.f;
struct PaScale {
    float mul, c2, cm;  // no clamp: s * mul; clamp: c2 - cm / (1 + 2^(s * mul))
    float in, lin;      // s / clamp, s in base 2
    bool clamped, wide;
    __device__ __forceinline__ explicit PaScale(const PaArgs &p) {
        clamped = p.clamp > 0.f;
        wide = p.clamp > kPaWide;
        in = p.scale / p.clamp;
        lin = p.scale * kLog2e;
        mul = clamped ? 2.f * kLog2e * in : lin;
        c2 = p.clamp * kLog2e;
        cm = 2.f * c2;
    }
    __device__ __forceinline__ float clamp(float s) const {
        return c2 - __fdividef(cm, 1.f + ex2(s * mul));  // 2^x = inf: the quotient is 0
    }
    __device__ __forceinline__ float clamp_wide(float s) const {
        const float x = s * in, big = clamp(s), small = pa_tanh_small(s * lin, x * x);
        return fabsf(x) <= kPaSmall ? small : big;
    }
    // two that are known to be small
    __device__ __forceinline__ float2 clamp_small(float2 s) const {
        const float2 x = mul2(s, make_float2(in, in));
        return pa_tanh_small(mul2(s, make_float2(lin, lin)), mul2(x, x));
    }
};

template <int HDP>
struct PaMma {
    static constexpr int kNW = 4;
    static constexpr int kRow = HDP * 2 + 16;  // ldmatrix: 8 rows meet 8 bank groups
    static constexpr int kTile = kPaTile * kRow;
    static constexpr int kWarp = 2 * kTile;
    static constexpr int kSmem = kNW * kWarp;
};

__device__ __forceinline__ uint32_t pa_trans(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// NQ: blocks of 8 queries.
template <typename T, int HDP, int NQ, bool FULL>
struct PaMmaBody {
    using S = PaMma<HDP>;
    static constexpr int KS = HDP / 16, DT = HDP / 16;
    const PaArgs &p;
    const PaSpan &g;
    const PaScale score;
    uint32_t kfrag, vfrag;
    int qr, qc;
    uint32_t qf[NQ][KS][2];                  // queries as the second operand
    float m[NQ][2], l[NQ][2], o[DT][NQ][4];  // of queries qc, qc + 1 of each block
    float s[2][NQ][4];                       // rows 16 mt + qr (first two) and + 8, queries qc, qc + 1
    uint32_t pf[2][NQ][2];

    __device__ __forceinline__ PaMmaBody(const PaArgs &p_, const PaSpan &g_, uint32_t ks, uint32_t vs)
        : p(p_), g(g_), score(p_) {
        const int lane = threadIdx.x & 31;
        qr = lane >> 2;
        qc = (lane & 3) * 2;
        kfrag = ks + ((lane & 7) + (lane >> 3 & 1) * 8) * S::kRow + (lane >> 4) * 16;
        vfrag = vs + ((lane & 7) + (lane >> 4) * 8) * S::kRow + (lane >> 3 & 1) * 16;
    }
    // query qr of each block, numbers qc, qc + 1 (+ 8) of each 16
    __device__ __forceinline__ void queries(int seq) {
#pragma unroll
        for (int b = 0; b < NQ; b++) {
            const T *q = nullptr;
            if (b * 8 + qr < g.nrows) {
                int sq, h;
                pa_query(p, g, seq, b * 8 + qr, sq, h);
                q = (const T *)p.q + (int64_t)sq * p.q_stride + (int64_t)h * p.hd;
            }
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const int c = k * 16 + j * 8 + qc;
                    qf[b][k][j] = q && (FULL || c < p.hd) ? *reinterpret_cast<const uint32_t *>(q + c) : 0u;
                }
            m[b][0] = m[b][1] = -INFINITY;
            l[b][0] = l[b][1] = 0.f;
#pragma unroll
            for (int d = 0; d < DT; d++) o[d][b][0] = o[d][b][1] = o[d][b][2] = o[d][b][3] = 0.f;
        }
    }
    __device__ __forceinline__ void scores() {
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int b = 0; b < NQ; b++) s[mt][b][0] = s[mt][b][1] = s[mt][b][2] = s[mt][b][3] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
                uint32_t a[4];
                pa_ldsm(a, kfrag + mt * 16 * S::kRow + k * 32);
#pragma unroll
                for (int b = 0; b < NQ; b++) pa_mma16816<T>(s[mt][b], a, qf[b][k][0], qf[b][k][1]);
            }
    }
    __device__ __forceinline__ void weights(uint32_t valid) {
#pragma unroll
        for (int b = 0; b < NQ; b++) {
            if (score.wide) {
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s[mt][b][j] = score.clamp_wide(s[mt][b][j]);
            } else if (score.clamped) {
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s[mt][b][j] = score.clamp(s[mt][b][j]);
            } else {
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s[mt][b][j] *= score.mul;
            }
            if (valid != JDG_FULL) {
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (!(valid >> (mt * 16 + (j >> 1) * 8 + qr) & 1u)) s[mt][b][j] = -INFINITY;
            }
            float x0 = fmaxf(fmaxf(s[0][b][0], s[0][b][2]), fmaxf(s[1][b][0], s[1][b][2]));
            float x1 = fmaxf(fmaxf(s[0][b][1], s[0][b][3]), fmaxf(s[1][b][1], s[1][b][3]));
            if (__any_sync(JDG_FULL, x0 - m[b][0] > kPaSlack + kPaLift<T> || x1 - m[b][1] > kPaSlack + kPaLift<T>)) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) {
                    x0 = fmaxf(x0, __shfl_xor_sync(JDG_FULL, x0, d));
                    x1 = fmaxf(x1, __shfl_xor_sync(JDG_FULL, x1, d));
                }
                x0 = fmaxf(x0 - kPaLift<T>, m[b][0]);
                x1 = fmaxf(x1 - kPaLift<T>, m[b][1]);
                const float f0 = m[b][0] == -INFINITY ? 0.f : ex2(m[b][0] - x0);
                const float f1 = m[b][1] == -INFINITY ? 0.f : ex2(m[b][1] - x1);
                m[b][0] = x0;
                m[b][1] = x1;
                l[b][0] *= f0;
                l[b][1] *= f1;
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    o[d][b][0] *= f0;
                    o[d][b][1] *= f1;
                    o[d][b][2] *= f0;
                    o[d][b][3] *= f1;
                }
            }
            // a query without any score so far (all masked) keeps weight zero
            const float b0 = m[b][0] == -INFINITY ? 0.f : m[b][0], b1 = m[b][1] == -INFINITY ? 0.f : m[b][1];
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
                const float e0 = ex2(s[mt][b][0] - b0), e1 = ex2(s[mt][b][1] - b1);
                const float e2 = ex2(s[mt][b][2] - b0), e3 = ex2(s[mt][b][3] - b1);
                l[b][0] += e0 + e2;
                l[b][1] += e1 + e3;
                pf[mt][b][0] = pa_trans(pack2(e0, e1, (const T *)nullptr));
                pf[mt][b][1] = pa_trans(pack2(e2, e3, (const T *)nullptr));
            }
        }
    }
    __device__ __forceinline__ void values() {
#pragma unroll
        for (int mt = 0; mt < 2; mt++)
#pragma unroll
            for (int d = 0; d < DT; d++) {
                uint32_t a[4];
                pa_ldsm_t(a, vfrag + mt * 16 * S::kRow + d * 32);
#pragma unroll
                for (int b = 0; b < NQ; b++) pa_mma16816<T>(o[d][b], a, pf[mt][b][0], pf[mt][b][1]);
            }
    }
    __device__ __forceinline__ void leave(float *x) {
#pragma unroll
        for (int b = 0; b < NQ; b++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float sum = l[b][j];
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) sum += __shfl_xor_sync(JDG_FULL, sum, d);
                float *y = x + (b * 8 + qc + j) * (HDP + 2);
                if (qr == 0) *reinterpret_cast<float2 *>(y + HDP) = make_float2(m[b][j], sum);
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    y[d * 16 + qr] = o[d][b][j];
                    y[d * 16 + qr + 8] = o[d][b][j + 2];
                }
            }
    }
};

template <typename T, int HDP, int NQ, bool FULL, int TEAM>
__global__ __launch_bounds__(32 * PaMma<HDP>::kNW, 3) void k_pa_mma(const __grid_constant__ PaArgs p) {
    using S = PaMma<HDP>;
    extern __shared__ __align__(16) uint8_t pa_sm[];
    dep_trigger();
    PaSpan g;
    if (pa_span<S::kNW, TEAM>(p, NQ * 8, g)) {
        uint8_t *mine = pa_sm + (threadIdx.x >> 5) * S::kWarp;
        if constexpr (!FULL) {  // the keys' columns past head_dim: zeros for good (the loads never write them; the
                                // values' only reach outputs past head_dim)
            const int cpr = p.hd / 8, nc = HDP / 8 - cpr;
            for (int i = threadIdx.x & 31; i < kPaTile * nc; i += 32)
                *reinterpret_cast<uint4 *>(mine + i / nc * S::kRow + (cpr + i % nc) * 16) = make_uint4(0u, 0u, 0u, 0u);
        }
        const uint32_t ks = (uint32_t)__cvta_generic_to_shared(mine), vs = ks + S::kTile;
        PaMmaBody<T, HDP, NQ, FULL> body(p, g, ks, vs);
        pa_walk<T, HDP, FULL, S::kRow, TEAM, S::kWarp>(p, g, TEAM > 1 ? pa_sm : mine, body);
    }
    // a launch that depends on this one may only rely on what came before once this has waited
    dep_wait();
}

// ------------------------------------------------------------------------------------
// f32 cache, shared rows behind many queries: matrix instructions on three bf16 planes.  An f32
// number is the sum of three bf16 numbers to 2^-26 (x = hi + mid + lo, each the rounding of what
// is left), products of bf16 are exact in f32, and the six products above 2^-26 (hi hi, hi mid,
// mid hi, mid mid, hi lo, lo hi) are summed in f32: the same accuracy as f32 products, at a sixth
// of the instructions' rate, which is still several times the FMA units'.  The CTA splits a tile
// of 32 rows once, into shared memory, for its eight warps of 8 queries (loads of the next tile
// in registers meanwhile); a warp keeps its queries' planes in registers and its outputs to
// itself, so nothing is joined between warps.
constexpr int kPfWarps = 8, kPfQueries = 8 * kPfWarps;
template <int HDP>
struct PaF32 {
    static constexpr int kRow = HDP * 2 + 16;
    static constexpr int kPlane = 32 * kRow;
    static constexpr int kBuf = 6 * kPlane;  // three planes of keys, three of values
    static constexpr int kSmem = 2 * kBuf;
};
// two numbers as three planes of packed pairs
__device__ __forceinline__ void pa_planes(float x, float y, uint32_t (&w)[3]) {
    const __nv_bfloat16 *tag = nullptr;
    w[0] = pack2(x, y, tag);
    float2 h = unpack2(w[0], tag);
    x -= h.x;
    y -= h.y;
    w[1] = pack2(x, y, tag);
    h = unpack2(w[1], tag);
    w[2] = pack2(x - h.x, y - h.y, tag);
}

template <int HDP>
__global__ __launch_bounds__(32 * kPfWarps, HDP == 64 ? 2 : 1) void k_pa_f32(const __grid_constant__ PaArgs p) {
    using S = PaF32<HDP>;
    using B = __nv_bfloat16;
    extern __shared__ __align__(16) uint8_t pa_sm[];
    __shared__ uint8_t flag[2][32];
    constexpr int KS = HDP / 16, DT = HDP / 16, NL = HDP / 32;  // float4 loads of a thread for keys, and for values
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, qr = lane >> 2, qc = (lane & 3) * 2;
    dep_trigger();
    PaWork w;
    pa_work_shared(p, kPfQueries, w);
    const float *kh = (const float *)p.k + (int64_t)w.kvh * p.head_stride;
    const float *vh = (const float *)p.v + (int64_t)w.kvh * p.head_stride;
    // this thread's part of a tile: row tid / 8, numbers 4 (tid % 8) + 32 j
    const int lrow = tid >> 3, lcol = (tid & 7) * 4, pmask = (1 << p.page_shift) - 1;
    float4 rk[NL], rv[NL];
    bool rok = false;
    auto page_of = [&](int t) { return t + lrow < w.t1 ? w.tab[(t + lrow) >> p.page_shift] : -1; };
    auto fetch = [&](int t, int pg) {
        const bool in = t + lrow < w.t1;
        rok = in && pg >= 0 && pg < p.n_pages;
        if (in && !rok && p.status) atomicOr(p.status, JDG_STATUS_PAGE);
        const int64_t off = rok ? (int64_t)pg * p.page_stride + (int64_t)((t + lrow) & pmask) * p.row_stride : 0;
#pragma unroll
        for (int j = 0; j < NL; j++) {
            const bool on = rok && lcol + 32 * j < p.hd;  // zeros for what is not there
            rk[j] = on ? ld4(kh + off + lcol + 32 * j) : make_float4(0.f, 0.f, 0.f, 0.f);
            rv[j] = on ? ld4(vh + off + lcol + 32 * j) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    auto put = [&](int buf) {
        uint8_t *d = pa_sm + buf * S::kBuf + lrow * S::kRow + lcol * 2;
#pragma unroll
        for (int j = 0; j < NL; j++)
#pragma unroll
            for (int kv = 0; kv < 2; kv++) {
                const float4 x = kv ? rv[j] : rk[j];
                uint32_t a[3], b[3];
                pa_planes(x.x, x.y, a);
                pa_planes(x.z, x.w, b);
#pragma unroll
                for (int q = 0; q < 3; q++)
                    *reinterpret_cast<uint2 *>(d + (kv * 3 + q) * S::kPlane + j * 64) = make_uint2(a[q], b[q]);
            }
        if ((tid & 7) == 0) flag[buf][lrow] = rok;
    };
    fetch(w.t0, page_of(w.t0));
    int page = page_of(w.t0 + 32);
    // the planes of this warp's queries as the second operand
    const bool active = warp * 8 < w.nrows;
    uint32_t qf[KS][3][2];
    {
        const float *q = nullptr;
        if (warp * 8 + qr < w.nrows) {
            int s, h;
            pa_row(p, w, warp * 8 + qr, s, h);
            q = (const float *)p.q + (int64_t)s * p.q_stride + (int64_t)h * p.hd;
        }
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int c = k * 16 + j * 8 + qc;
                const float2 x = q && c < p.hd ? *reinterpret_cast<const float2 *>(q + c) : make_float2(0.f, 0.f);
                uint32_t pl[3];
                pa_planes(x.x, x.y, pl);
                qf[k][0][j] = pl[0];
                qf[k][1][j] = pl[1];
                qf[k][2][j] = pl[2];
            }
    }
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[DT][4];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
    put(0);
    __syncthreads();
    const uint32_t base = (uint32_t)__cvta_generic_to_shared(pa_sm);
    const uint32_t kfrag = ((lane & 7) + (lane >> 3 & 1) * 8) * S::kRow + (lane >> 4) * 16;
    const uint32_t vfrag = 3 * S::kPlane + ((lane & 7) + (lane >> 4) * 8) * S::kRow + (lane >> 3 & 1) * 16;
    int buf = 0;
    for (int t = w.t0; t < w.t1; t += 32, buf ^= 1) {
        const bool more = t + 32 < w.t1;
        if (more) {
            fetch(t + 32, page);
            page = page_of(t + 64);
        }
        if (active) {
            const uint32_t tile = base + buf * S::kBuf;
            const uint32_t valid = __ballot_sync(JDG_FULL, flag[buf][lane] != 0);
            float s[2][4];
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
                float lo[4] = {0.f, 0.f, 0.f, 0.f};  // the small products in a sum of their own
                s[mt][0] = s[mt][1] = s[mt][2] = s[mt][3] = 0.f;
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    uint32_t a[3][4];
#pragma unroll
                    for (int q = 0; q < 3; q++) pa_ldsm(a[q], tile + q * S::kPlane + kfrag + mt * 16 * S::kRow + k * 32);
                    pa_mma16816<B>(lo, a[0], qf[k][2][0], qf[k][2][1]);
                    pa_mma16816<B>(s[mt], a[0], qf[k][0][0], qf[k][0][1]);
                    pa_mma16816<B>(lo, a[2], qf[k][0][0], qf[k][0][1]);
                    pa_mma16816<B>(lo, a[1], qf[k][1][0], qf[k][1][1]);
                    pa_mma16816<B>(lo, a[0], qf[k][1][0], qf[k][1][1]);
                    pa_mma16816<B>(lo, a[1], qf[k][0][0], qf[k][0][1]);
                }
#pragma unroll
                for (int j = 0; j < 4; j++) s[mt][j] += lo[j];
            }
            pa_scores(reinterpret_cast<float(&)[8]>(s), p);
            if (valid != JDG_FULL) {
#pragma unroll
                for (int mt = 0; mt < 2; mt++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (!(valid >> (mt * 16 + (j >> 1) * 8 + qr) & 1u)) s[mt][j] = -INFINITY;
            }
            float x[2];
#pragma unroll
            for (int j = 0; j < 2; j++) x[j] = fmaxf(fmaxf(s[0][j], s[0][j + 2]), fmaxf(s[1][j], s[1][j + 2]));
            if (__any_sync(JDG_FULL, x[0] - m[0] > kPaSlack || x[1] - m[1] > kPaSlack)) {
                float f[2];
#pragma unroll
                for (int j = 0; j < 2; j++) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) x[j] = fmaxf(x[j], __shfl_xor_sync(JDG_FULL, x[j], d));
                    x[j] = fmaxf(x[j], m[j]);
                    f[j] = m[j] == -INFINITY ? 0.f : ex2(m[j] - x[j]);
                    m[j] = x[j];
                    l[j] *= f[j];
                }
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int j = 0; j < 4; j++) o[d][j] *= f[j & 1];
            }
            const float b0 = m[0] == -INFINITY ? 0.f : m[0], b1 = m[1] == -INFINITY ? 0.f : m[1];
            uint32_t pf[2][3][2];
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
                const float e0 = ex2(s[mt][0] - b0), e1 = ex2(s[mt][1] - b1), e2 = ex2(s[mt][2] - b0), e3 = ex2(s[mt][3] - b1);
                l[0] += e0 + e2;
                l[1] += e1 + e3;
                uint32_t u[3], v[3];
                pa_planes(e0, e1, u);
                pa_planes(e2, e3, v);
#pragma unroll
                for (int q = 0; q < 3; q++) {
                    pf[mt][q][0] = pa_trans(u[q]);
                    pf[mt][q][1] = pa_trans(v[q]);
                }
            }
#pragma unroll
            for (int mt = 0; mt < 2; mt++)
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    uint32_t a[3][4];
#pragma unroll
                    for (int q = 0; q < 3; q++) pa_ldsm_t(a[q], tile + q * S::kPlane + vfrag + mt * 16 * S::kRow + d * 32);
                    pa_mma16816<B>(o[d], a[0], pf[mt][2][0], pf[mt][2][1]);
                    pa_mma16816<B>(o[d], a[2], pf[mt][0][0], pf[mt][0][1]);
                    pa_mma16816<B>(o[d], a[1], pf[mt][1][0], pf[mt][1][1]);
                    pa_mma16816<B>(o[d], a[0], pf[mt][1][0], pf[mt][1][1]);
                    pa_mma16816<B>(o[d], a[1], pf[mt][0][0], pf[mt][0][1]);
                    pa_mma16816<B>(o[d], a[0], pf[mt][0][0], pf[mt][0][1]);
                }
        }
        if (more) put(buf ^ 1);
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < 2; j++) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[j] += __shfl_xor_sync(JDG_FULL, l[j], d);
        const int r = warp * 8 + qc + j;
        if (r >= w.nrows) continue;
        int s, h;
        pa_row(p, w, r, s, h);
        float *dst = pa_part(p, s * p.H + h, w.split);
        if (lane < 4) *reinterpret_cast<float2 *>(dst) = make_float2(m[j], l[j]);
#pragma unroll
        for (int d = 0; d < DT; d++) {
            if (d * 16 + qr < p.hd) dst[4 + d * 16 + qr] = o[d][j];
            if (d * 16 + qr + 8 < p.hd) dst[4 + d * 16 + qr + 8] = o[d][j + 2];
        }
    }
}

}  // namespace jdg
