// jdg_beam.cu — one step of beam search: the best continuations over beams and vocabulary, and
// the reordering of the beams' states.
//
//   score(r, t) = cum[r] + x_t - log sum_u e^{x_u}          (row r of logits x)
//
// Inside a row the order of the scores is the order of the logits, so a slice of a row needs
// only its n_out largest logits and its (max, sum of exponentials); the scores of these few are
// then formed in 64 bits and ranked over the group.  Candidates of different rows often lie
// closer to one another than 32 bits of a log-softmax can tell.
#include "jdg_devop.cuh"

using namespace jdg;

namespace {

constexpr int kBsThreads = 256, kBsWarps = kBsThreads / 32;
constexpr int kBsMaxOut = 32, kBsMaxBeams = 64;
constexpr int kBsCap = 2048;   // candidates of a slice kept for ranking; more (adversarial rows) go round by round
constexpr int kBsJoin = 1024;  // the same in the join

typedef unsigned long long u64;

// larger float = larger number; NaN and -inf = 0 (never picked)
__device__ __forceinline__ uint32_t ord32(float x) {
    if (!(x > -INFINITY)) return 0u;
    const uint32_t b = __float_as_uint(x + 0.f);  // -0 and 0 are one value
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unord32(uint32_t o) {
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}
__device__ __forceinline__ u64 ord64(double x) {
    if (!(x > -INFINITY)) return 0ull;
    const u64 b = (u64)__double_as_longlong(x + 0.0);
    return (b >> 63) ? ~b : (b | (1ull << 63));
}
__device__ __forceinline__ double unord64(u64 o) {
    return __longlong_as_double((long long)((o >> 63) ? (o & ~(1ull << 63)) : ~o));
}

// slice: logit, then lowest token; 0 = nothing
__device__ __forceinline__ u64 slice_key(float x, int t) {
    const uint32_t o = ord32(x);
    return o ? ((u64)o << 32) | (0xffffffffu - (uint32_t)t) : 0ull;
}

struct SelP {
    const void *logits;
    int64_t stride;
    int beams, vocab, n_out, splits, slice;
    const float *cum;
    const int *done;
    int eos;
    int *parent, *token;
    float *score;
    u64 *keys;      // [row][split][n_out]
    float *smax;    // [row][split]
    double *ssum;   // [row][split]
};

// One slice of one row.  EPT numbers a thread, held in registers: one read of the logits.
// Threshold: the slice's 32 groups of 8 threads each have a largest key; the n_out-th largest of
// these is passed by n_out numbers at least, and by few more (about 15 for n_out 12).  Each warp
// counts for four of the 32 how many are above, and eight threads rank a candidate.
// Measured, 288 x 128,256 f32 (148 MB): call 41 us, of which the join 10.  What a slice waits for is
// the chain of its phases (the loads alone take 18 us, exponentials 6, threshold 3, candidates 9), not
// HBM: with a row's half the bytes (bf16) the call takes as long, and with the next slice on its way
// while one is worked on (CTAs that stay) it took 9 us more.  One warp that sorts the 32 and one
// thread to rank a candidate: 43.6 us.  So sums and products go two at a time and nothing is formed twice.
template <typename T, int EPT>
__global__ __launch_bounds__(kBsThreads, EPT <= 8 ? 6 : 4) void k_beam_slice(const __grid_constant__ SelP p) {
    constexpr int V = 16 / (int)sizeof(T), NV = EPT / V;  // numbers of a 16-byte load, loads a thread
    __shared__ u64 cand[kBsCap];
    __shared__ u64 gmax[32];
    __shared__ float fred[kBsWarps];
    __shared__ double dred[kBsWarps];
    __shared__ u64 thr_s;
    __shared__ int count;
    const int row = blockIdx.y, split = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    dep_trigger();
    if (p.done && p.done[row]) return;
    const T *x = (const T *)p.logits + (int64_t)row * p.stride;
    // slices are cut at 16-byte boundaries of the row as it lies in memory: a row may start between two
    const int skew = (int)(((uintptr_t)x & 15) / sizeof(T));
    const int first = split * p.slice - skew, last = min(p.vocab, first + p.slice);
    float v[EPT];
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int t = first + (i * kBsThreads + tid) * V;
        if (t >= 0 && t + V <= last) {
            const uint4 w = ld_stream_u4(x + t);
            if (V == 4) {
                v[i * V] = __uint_as_float(w.x);
                v[i * V + 1] = __uint_as_float(w.y);
                v[i * V + 2] = __uint_as_float(w.z);
                v[i * V + 3] = __uint_as_float(w.w);
            } else {
                T e[V];
                *reinterpret_cast<uint4 *>(e) = w;
#pragma unroll
                for (int j = 0; j < V; j++) v[i * V + j] = to_f(e[j]);
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; j++) v[i * V + j] = t + j >= 0 && t + j < last ? to_f(x[t + j]) : -INFINITY;
        }
    }
    auto token = [&](int i) { return first + (i / V * kBsThreads + tid) * V + i % V; };
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < EPT; i++) m = fmaxf(m, v[i]);  // NaN is passed over
    int mi = 0;
#pragma unroll
    for (int i = EPT - 1; i >= 0; i--) mi = v[i] == m ? i : mi;  // the thread's first maximum
    const u64 best = slice_key(m, token(mi));
    u64 g = best;
#pragma unroll
    for (int o = 4; o; o >>= 1) {
        const u64 c = __shfl_xor_sync(JDG_FULL, g, o);
        g = c > g ? c : g;
    }
    const float wm = warp_max(m);
    if ((lane & 7) == 0) gmax[tid >> 3] = g;
    if (lane == 0) fred[warp] = wm;
    if (tid == 0) count = 0, thr_s = 0;
    __syncthreads();
    // the one that n_out - 1 others are above (keys are distinct, but for 0); a warp looks at four
    {
        const u64 k = gmax[lane];
#pragma unroll
        for (int i = 0; i < 32 / kBsWarps; i++) {
            const u64 c = __shfl_sync(JDG_FULL, k, warp * (32 / kBsWarps) + i);
            const int above = __popc(__ballot_sync(JDG_FULL, k > c));
            if (lane == 0 && c && above == p.n_out - 1) thr_s = c;
        }
    }
    float mx = fred[0];
#pragma unroll
    for (int w = 1; w < kBsWarps; w++) mx = fmaxf(mx, fred[w]);
    // sum of exponentials: f32 terms, 32 at most in a row, then 64 bits.  The difference is formed first
    // (exact near the maximum, where the weight is)
    float s = 0.f;
    if (mx > -INFINITY && mx < INFINITY) {
        float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < EPT; i += 2) {
            const float2 d = mul2(add2(make_float2(v[i], v[i + 1]), make_float2(-mx, -mx)), make_float2(kLog2e, kLog2e));
            s2 = add2(s2, make_float2(ex2(d.x), ex2(d.y)));
        }
        s = s2.x + s2.y;
        if (!(s == s)) {  // a NaN among them counts as nothing
            s = 0.f;
#pragma unroll
            for (int i = 0; i < EPT; i++) s += v[i] == v[i] ? ex2((v[i] - mx) * kLog2e) : 0.f;
        }
    } else if (mx == INFINITY) {
#pragma unroll
        for (int i = 0; i < EPT; i++) s += v[i] == INFINITY ? 1.f : 0.f;
    }
    double ds = (double)s;
#pragma unroll
    for (int o = 16; o; o >>= 1) ds += __shfl_xor_sync(JDG_FULL, ds, o);
    if (lane == 0) dred[warp] = ds;
    __syncthreads();
    const u64 thr = thr_s;
    if (best && best >= thr) {
        const float tf = thr ? unord32((uint32_t)(thr >> 32)) : -INFINITY;
        uint32_t pass = 0;
#pragma unroll
        for (int i = 0; i < EPT; i++) pass |= v[i] >= tf ? 1u << i : 0u;
        for (; pass; pass &= pass - 1) {  // one or two as a rule; read again (they are in L2)
            const int t = token(__ffs(pass) - 1);
            const u64 k = t >= 0 && t < last ? slice_key(to_f(x[t]), t) : 0ull;
            if (k && k >= thr) {
                const int at = atomicAdd(&count, 1);
                if (at < kBsCap) cand[at] = k;
            }
        }
    }
    __syncthreads();
    const int64_t out = (int64_t)row * p.splits + split;
    if (tid == kBsThreads - 1) {
        double tot = 0;
        for (int w = 0; w < kBsWarps; w++) tot += dred[w];
        p.smax[out] = mx;
        p.ssum[out] = tot;
    }
    u64 *keys = p.keys + out * p.n_out;
    const int n = count;
    if (n <= kBsCap) {
        // rank by counting (keys are distinct)
        for (int i = tid >> 3; i < ((n + 3) & ~3); i += kBsThreads / 8) {  // eight threads a candidate, whole warps
            const u64 k = i < n ? cand[i] : 0ull;
            int r = 0;
            for (int j = tid & 7; j < n; j += 8) r += cand[j] > k;
            r += __shfl_xor_sync(JDG_FULL, r, 1);
            r += __shfl_xor_sync(JDG_FULL, r, 2);
            r += __shfl_xor_sync(JDG_FULL, r, 4);
            if (k && (tid & 7) == 0 && r < p.n_out) keys[r] = k;
        }
        for (int i = n + tid; i < p.n_out; i += kBsThreads) keys[i] = 0;
    } else {
        u64 below = ~0ull;
        for (int r = 0; r < p.n_out; r++) {
            u64 k = 0;
#pragma unroll 1
            for (int i = 0; i < EPT; i++) {
                const int t = token(i);
                const u64 c = t >= 0 && t < last ? slice_key(to_f(x[t]), t) : 0ull;
                if (c < below && c > k) k = c;
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                const u64 c = __shfl_xor_sync(JDG_FULL, k, o);
                k = c > k ? c : k;
            }
            __syncthreads();
            if (lane == 0) gmax[warp] = k;
            __syncthreads();
            for (int w = 0; w < kBsWarps; w++) k = gmax[w] > k ? gmax[w] : k;
            if (tid == 0) keys[r] = k;
            below = k;  // n > n_out: there is always one more
        }
    }
}

// candidate of a group: score in 64 bits, then lowest (parent, slice order)
struct Cand {
    u64 s, t;  // t: larger is earlier
};
__device__ __forceinline__ bool before(const Cand &a, const Cand &b) { return a.s > b.s || (a.s == b.s && a.t > b.t); }

// One CTA joins a group: the rows' sums, then the candidates' scores, threshold and ranks as in the
// slices.  The first kBsHold candidates of a thread are loaded before anything is waited for and
// kept in registers.
constexpr int kBsHold = 8;
__global__ __launch_bounds__(kBsThreads) void k_beam_join(const __grid_constant__ SelP p) {
    __shared__ double lse[kBsMaxBeams];
    __shared__ float rmax[kBsMaxBeams], cums[kBsMaxBeams];
    __shared__ bool fins[kBsMaxBeams];
    __shared__ Cand cand[kBsJoin];
    __shared__ Cand wthr[kBsWarps];
    __shared__ int count;
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = p.splits * p.n_out, total = p.beams * per;
    dep_wait();
    u64 hold[kBsHold];
#pragma unroll
    for (int k = 0; k < kBsHold; k++) {
        const int i = tid + k * kBsThreads;
        hold[k] = i < total ? p.keys[(int64_t)g * total + i] : 0ull;
    }
    // log of the sum of each row, relative to its maximum
    for (int b = warp; b < p.beams; b += kBsWarps) {
        const int64_t row = (int64_t)g * p.beams + b;
        const bool fin = p.done && p.done[row];
        float m = -INFINITY;
        double s = 0;
        if (!fin) {
            for (int i = lane; i < p.splits; i += 32) m = fmaxf(m, p.smax[row * p.splits + i]);
            m = warp_max(m);
            for (int i = lane; i < p.splits; i += 32) {
                const float mi = p.smax[row * p.splits + i];
                // (the slices' factors in f32, as their terms are)
                if (mi > -INFINITY) s += p.ssum[row * p.splits + i] * (mi == m ? 1.0 : (double)ex2((mi - m) * kLog2e));
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(JDG_FULL, s, o);
        }
        if (lane == 0) {
            rmax[b] = m;
            lse[b] = log(s);
            cums[b] = p.cum[row];
            fins[b] = fin;
        }
    }
    if (tid == 0) count = 0;
    __syncthreads();
    // candidate i of the group: row i / per; a finished row's first place holds the row itself
    auto form = [&](int i, u64 k) {
        Cand c = {0, 0};
        const int b = i / per;
        const double cum = (double)cums[b];
        if (fins[b]) {
            if (i == b * per) {
                c.s = ord64(cum);
                c.t = ((u64)(255 - b) << 32) | (0xffffffffu - (uint32_t)p.eos);
            }
            return c;
        }
        if (!k) return c;
        const float x = unord32((uint32_t)(k >> 32));
        c.s = ord64(cum + ((x == rmax[b] ? 0.0 : (double)x - (double)rmax[b]) - lse[b]));
        c.t = ((u64)(255 - b) << 32) | (k & 0xffffffffu);
        return c;
    };
    Cand mine[kBsHold];
#pragma unroll
    for (int k = 0; k < kBsHold; k++) {
        const int i = tid + k * kBsThreads;
        mine[k] = Cand{0, 0};
        if (i < total) mine[k] = form(i, hold[k]);
    }
    // every candidate of this thread
    auto each = [&](auto &&f) {
#pragma unroll
        for (int k = 0; k < kBsHold; k++) f(mine[k]);
#pragma unroll 1
        for (int i = tid + kBsHold * kBsThreads; i < total; i += kBsThreads) f(form(i, p.keys[(int64_t)g * total + i]));
    };
    Cand best = {0, 0};
    each([&](const Cand &c) {
        if (before(c, best)) best = c;
    });
    // the threshold, as in the slices
    Cand k = best;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int d = size >> 1; d; d >>= 1) {
            Cand o;
            o.s = __shfl_xor_sync(JDG_FULL, k.s, d);
            o.t = __shfl_xor_sync(JDG_FULL, k.t, d);
            const bool up = ((lane & size) == 0) == ((lane & d) == 0);
            if (up ? before(o, k) : before(k, o)) k = o;
        }
    k.s = __shfl_sync(JDG_FULL, k.s, p.n_out - 1);
    k.t = __shfl_sync(JDG_FULL, k.t, p.n_out - 1);
    if (lane == 0) wthr[warp] = k;
    __syncthreads();
    Cand thr = wthr[0];
    for (int w = 1; w < kBsWarps; w++)
        if (before(wthr[w], thr)) thr = wthr[w];
    auto put = [&](int r, const Cand &c) {
        const int64_t at = (int64_t)g * p.n_out + r;
        p.parent[at] = c.s ? 255 - (int)(c.t >> 32) : -1;
        p.token[at] = c.s ? (int)(0xffffffffu - (uint32_t)c.t) : -1;
        p.score[at] = c.s ? (float)unord64(c.s) : -INFINITY;
    };
    if (best.s && !before(thr, best)) {
        each([&](const Cand &c) {
            if (c.s && !before(thr, c)) {
                const int at = atomicAdd(&count, 1);
                if (at < kBsJoin) cand[at] = c;
            }
        });
    }
    __syncthreads();
    const int n = count;
    if (n <= kBsJoin) {
        for (int i = tid >> 3; i < ((n + 3) & ~3); i += kBsThreads / 8) {
            const Cand c = i < n ? cand[i] : Cand{0, 0};
            int r = 0;
            for (int j = tid & 7; j < n; j += 8) r += before(cand[j], c);
            r += __shfl_xor_sync(JDG_FULL, r, 1);
            r += __shfl_xor_sync(JDG_FULL, r, 2);
            r += __shfl_xor_sync(JDG_FULL, r, 4);
            if (i < n && (tid & 7) == 0 && r < p.n_out) put(r, c);
        }
        const Cand none = {0, 0};
        for (int i = n + tid; i < p.n_out; i += kBsThreads) put(i, none);
    } else {
        Cand below = {~0ull, ~0ull};
        for (int r = 0; r < p.n_out; r++) {
            Cand c = {0, 0};
            each([&](const Cand &x) {
                if (before(below, x) && before(x, c)) c = x;
            });
#pragma unroll
            for (int d = 16; d; d >>= 1) {
                Cand o;
                o.s = __shfl_xor_sync(JDG_FULL, c.s, d);
                o.t = __shfl_xor_sync(JDG_FULL, c.t, d);
                if (before(o, c)) c = o;
            }
            __syncthreads();
            if (lane == 0) wthr[warp] = c;
            __syncthreads();
            for (int w = 0; w < kBsWarps; w++)
                if (before(wthr[w], c)) c = wthr[w];
            if (tid == 0) put(r, c);
            below = c;
        }
    }
}

// ------------------------------------------------------------------------------------ reorder
constexpr int kRoThreads = 256, kRoChunk = 32768;  // bytes of a row that a CTA copies

struct ReorderP {
    const int *parent;
    int parent_stride, beams, n_states;
    int *status;
    struct {
        const uint8_t *src;
        uint8_t *dst;
        int64_t bytes, src_stride, dst_stride;
        unsigned first;   // first CTA of the state
        unsigned chunks;  // CTAs of a row
    } st[JDG_MAX_STATES];
};

// bytes [sh, sh + 16) of the 32 bytes a, b
__device__ __forceinline__ uint4 shift16(const uint4 &a, const uint4 &b, int sh) {
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (sh & 8) {
#pragma unroll
        for (int i = 0; i < 6; i++) w[i] = w[i + 2];
    }
    if (sh & 4) {
#pragma unroll
        for (int i = 0; i < 5; i++) w[i] = w[i + 1];
    }
    const int bits = (sh & 3) * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                      __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}

// Bytes of rows that may lie anywhere: 16-byte stores at the destination's boundaries, fed by
// 16-byte loads at the source's; a warp shifts by the difference.  Bound: HBM.
__global__ __launch_bounds__(kRoThreads) void k_beam_reorder(const __grid_constant__ ReorderP p) {
    int s = 0;
    while (s + 1 < p.n_states && blockIdx.x >= p.st[s + 1].first) s++;
    const unsigned id = blockIdx.x - p.st[s].first, chunks = p.st[s].chunks;
    const int row = (int)(id / chunks);
    const int64_t c0 = (int64_t)(id - (unsigned)row * chunks) * kRoChunk;
    const int g = row / p.beams, i = row - g * p.beams;
    const int par = p.parent[(int64_t)g * p.parent_stride + i];
    if (par < 0 || par >= p.beams) {
        if (par >= p.beams && p.status && threadIdx.x == 0) atomicOr(p.status, JDG_STATUS_SEQ);
        return;
    }
    const uint8_t *src = p.st[s].src + (int64_t)(g * p.beams + par) * p.st[s].src_stride + c0;
    uint8_t *dst = p.st[s].dst + (int64_t)row * p.st[s].dst_stride + c0;
    const int n = (int)min((int64_t)kRoChunk, p.st[s].bytes - c0), tid = threadIdx.x, lane = tid & 31;
    const int head = min(n, (int)((16 - ((uintptr_t)dst & 15)) & 15));
    const int sh = (int)(((uintptr_t)src + head) & 15);
    if (sh == 0) {
        const int nv = (n - head) >> 4;
        const uint4 *sv = reinterpret_cast<const uint4 *>(src + head);
        uint4 *dv = reinterpret_cast<uint4 *>(dst + head);
        constexpr int U = 8;
        for (int j = tid; j < nv; j += U * kRoThreads) {
            uint4 x[U];
#pragma unroll
            for (int k = 0; k < U; k++)
                if (j + k * kRoThreads < nv) x[k] = ld_stream_u4(sv + j + k * kRoThreads);
#pragma unroll
            for (int k = 0; k < U; k++)
                if (j + k * kRoThreads < nv) dv[j + k * kRoThreads] = x[k];
        }
        const int tail = head + (nv << 4);
        if (tid < head) dst[tid] = src[tid];
        if (tid < n - tail) dst[tail + tid] = src[tail + tid];
        return;
    }
    // destination piece j is bytes [head + 16 j, +16), aligned source pieces j and j + 1 from `base`; the
    // first piece starts sh bytes before src + head, so it is used only where it lies inside the row's bytes
    const uint8_t *base = src + head - sh;
    const int lead = head >= sh ? 0 : 1;                       // first piece whose source is inside
    const int nv = max(lead, (n - head + sh) / 16 - 1);        // pieces j < nv have j + 1 inside too
    constexpr int U = 4;
    for (int j0 = lead + (tid >> 5) * (32 * U); j0 < nv; j0 += U * kRoThreads) {
        uint4 x[U], extra;
#pragma unroll
        for (int k = 0; k < U; k++) {
            const int j = j0 + k * 32 + lane;
            if (j <= nv) x[k] = *reinterpret_cast<const uint4 *>(base + 16 * (int64_t)j);
        }
        const int je = j0 + U * 32;
        if (lane == 31 && je <= nv) extra = *reinterpret_cast<const uint4 *>(base + 16 * (int64_t)je);
#pragma unroll
        for (int k = 0; k < U; k++) {
            // the next piece: the lane above, and for the last lane the next group's first
            const uint4 a = x[k], f = k + 1 < U ? x[k + 1] : extra;
            uint4 b;
            b.x = __shfl_down_sync(JDG_FULL, a.x, 1);
            b.y = __shfl_down_sync(JDG_FULL, a.y, 1);
            b.z = __shfl_down_sync(JDG_FULL, a.z, 1);
            b.w = __shfl_down_sync(JDG_FULL, a.w, 1);
            const int from = k + 1 < U ? 0 : 31;
            const uint32_t fx = __shfl_sync(JDG_FULL, f.x, from), fy = __shfl_sync(JDG_FULL, f.y, from),
                           fz = __shfl_sync(JDG_FULL, f.z, from), fw = __shfl_sync(JDG_FULL, f.w, from);
            if (lane == 31) b = make_uint4(fx, fy, fz, fw);
            const int j = j0 + k * 32 + lane;
            if (j < nv) *reinterpret_cast<uint4 *>(dst + head + 16 * (int64_t)j) = shift16(a, b, sh);
        }
    }
    const int lo = min(n, head + 16 * lead), hi = min(n, head + 16 * nv);
    if (tid < lo) dst[tid] = src[tid];
    if (tid < n - hi) dst[hi + tid] = src[hi + tid];
}

int select_plan(const jdg_select_args *a, SelP *p, int *ept) {
    // a slice is 256 threads x 8 numbers for few rows (latency: more CTAs), x 32 otherwise (fewer
    // candidates to join)
    const int64_t rows = (int64_t)a->groups * a->beams;
    const int v = 16 / devop_size(a->dt);
    const int64_t cols = (int64_t)a->vocab + v - 1;  // a row may start between two 16-byte boundaries
    *ept = rows * ((cols + 8 * kBsThreads - 1) / (8 * kBsThreads)) <= 4 * kDevSMs ? 8 : 32;
    p->slice = *ept * kBsThreads;
    p->splits = (int)((cols + p->slice - 1) / p->slice);
    return JD_OK;
}
size_t select_bytes(const jdg_select_args *a, const SelP &p) {
    return (size_t)a->groups * a->beams * p.splits * ((size_t)p.n_out * 8 + 8 + 8);
}

template <typename T>
int select_run(SelP p, int ept, int groups, cudaStream_t st) {
    const char *who = "jdg_beam_select";
    const dim3 grid(p.splits, groups * p.beams);
    int rc = ept == 8 ? devop_launch(who, false, k_beam_slice<T, 8>, grid, dim3(kBsThreads), 0, st, p)
                      : devop_launch(who, false, k_beam_slice<T, 32>, grid, dim3(kBsThreads), 0, st, p);
    if (rc == JD_OK) rc = devop_launch(who, true, k_beam_join, dim3(groups), dim3(kBsThreads), 0, st, p);
    return rc;
}

bool overlap(const void *a, int64_t na, const void *b, int64_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

}  // namespace

extern "C" int jdg_beam_select_check(const jdg_select_args *a) {
    const char *who = "jdg_beam_select";
    if (!a || !a->logits || !a->cum || !a->parent || !a->token || !a->score || a->groups < 0 || a->beams < 1 ||
        a->vocab < 1 || a->n_out < 1 || a->stride < 0) {
        jdg_set_err(nullptr, "%s: bad arguments", who);
        return JD_EINVAL;
    }
    const int es = devop_size(a->dt);
    if (!es) {
        jdg_set_err(nullptr, "%s: type %d is not f32, f16 or bf16", who, a->dt);
        return JD_EUNSUPPORTED;
    }
    if (a->beams > kBsMaxBeams || a->n_out > kBsMaxOut || (int64_t)a->groups * a->beams > 65535 || a->vocab > (1 << 24)) {
        jdg_set_err(nullptr, "%s: at most %d beams, n_out %d, 65535 rows and 2^24 columns", who, kBsMaxBeams, kBsMaxOut);
        return JD_EUNSUPPORTED;
    }
    if (((uintptr_t)a->logits % es) || (a->done && (a->eos < 0 || a->eos >= a->vocab))) {
        jdg_set_err(nullptr, "%s: misaligned logits, or eos outside the vocabulary", who);
        return JD_EINVAL;
    }
    if (a->groups == 0) return JD_OK;
    const int64_t rows = (int64_t)a->groups * a->beams, outs = (int64_t)a->groups * a->n_out * 4;
    const void *const out[3] = {a->parent, a->token, a->score};
    for (int i = 0; i < 3; i++) {
        // a group's scores may take the place of its rows' own, which are read before
        const bool in_place = out[i] == (const void *)a->cum && i == 2 && a->n_out == a->beams;
        if (overlap(out[i], outs, a->logits, ((rows - 1) * a->stride + a->vocab) * es) ||
            (!in_place && overlap(out[i], outs, a->cum, rows * 4)) || (a->done && overlap(out[i], outs, a->done, rows * 4)) ||
            overlap(out[i], outs, out[(i + 1) % 3], outs)) {
            jdg_set_err(nullptr, "%s: an output overlaps an input or another output", who);
            return JD_EINVAL;
        }
    }
    return JD_OK;
}

extern "C" size_t jdg_beam_select_workspace(const jdg_select_args *a) {
    if (jdg_beam_select_check(a) != JD_OK) return 0;
    SelP p = {};
    int ept;
    p.n_out = a->n_out;
    select_plan(a, &p, &ept);
    const size_t b = select_bytes(a, p);
    return b ? b : 16;
}

extern "C" int jdg_beam_select(const jdg_select_args *a, void *workspace, size_t workspace_bytes, void *stream) {
    const char *who = "jdg_beam_select";
    int rc = jdg_beam_select_check(a), dev, ept;
    if (rc != JD_OK) return rc;
    if (a->groups == 0) return JD_OK;
    SelP p = {};
    p.logits = a->logits; p.stride = a->stride; p.beams = a->beams; p.vocab = a->vocab; p.n_out = a->n_out;
    p.cum = a->cum; p.done = a->done; p.eos = a->eos; p.parent = a->parent; p.token = a->token; p.score = a->score;
    select_plan(a, &p, &ept);
    const size_t need = select_bytes(a, p);
    if (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need) {
        jdg_set_err(nullptr, "%s: workspace of %zu bytes (16-byte aligned) needed, %zu given", who, need,
                    workspace ? workspace_bytes : (size_t)0);
        return JD_EINVAL;
    }
    const size_t parts = (size_t)a->groups * a->beams * p.splits;
    p.keys = (u64 *)workspace;
    p.ssum = (double *)(p.keys + parts * p.n_out);
    p.smax = (float *)(p.ssum + parts);
    cudaStream_t st = (cudaStream_t)stream;
    rc = devop_stream(who, st, &dev);
    if (rc != JD_OK) return rc;
    return a->dt == JD_F32   ? select_run<float>(p, ept, a->groups, st)
           : a->dt == JD_F16 ? select_run<__half>(p, ept, a->groups, st)
                             : select_run<__nv_bfloat16>(p, ept, a->groups, st);
}

extern "C" int jdg_beam_reorder_check(const jdg_reorder_args *a) {
    const char *who = "jdg_beam_reorder";
    if (!a || !a->parent || a->groups < 0 || a->beams < 1 || a->n_states < 0 || a->n_states > JDG_MAX_STATES ||
        a->parent_stride < a->beams) {
        jdg_set_err(nullptr, "%s: bad arguments (at most %d states)", who, JDG_MAX_STATES);
        return JD_EINVAL;
    }
    const int64_t rows = (int64_t)a->groups * a->beams;
    if (rows > (1 << 24)) {
        jdg_set_err(nullptr, "%s: more than 2^24 rows", who);
        return JD_EUNSUPPORTED;
    }
    if (rows == 0) return JD_OK;
    int64_t ctas = 0;
    for (int i = 0; i < a->n_states; i++) {
        const jdg_state &s = a->state[i];
        if (!s.src || !s.dst || s.row_bytes < 0 || s.src_stride < 0 || s.row_bytes > (1ll << 40) ||
            (rows > 1 && s.dst_stride < s.row_bytes)) {
            jdg_set_err(nullptr, "%s: state %d: bad pointers, or rows that overlap", who, i);
            return JD_EINVAL;
        }
        ctas += rows * ((s.row_bytes + kRoChunk - 1) / kRoChunk);
        const int64_t nd = (rows - 1) * s.dst_stride + s.row_bytes;
        if (s.row_bytes && overlap(s.dst, nd, a->parent, ((int64_t)(a->groups - 1) * a->parent_stride + a->beams) * 4)) {
            jdg_set_err(nullptr, "%s: the destination of state %d overlaps the parents", who, i);
            return JD_EINVAL;
        }
        for (int j = 0; j < a->n_states && s.row_bytes; j++) {
            const jdg_state &t = a->state[j];
            if (!t.row_bytes) continue;
            if (overlap(s.dst, nd, t.src, (rows - 1) * t.src_stride + t.row_bytes) ||
                (j != i && overlap(s.dst, nd, t.dst, (rows - 1) * t.dst_stride + t.row_bytes))) {
                jdg_set_err(nullptr, "%s: the destination of state %d overlaps state %d", who, i, j);
                return JD_EINVAL;
            }
        }
    }
    if (ctas > 0x7fffffffll) {
        jdg_set_err(nullptr, "%s: too many bytes for one call", who);
        return JD_EUNSUPPORTED;
    }
    return JD_OK;
}

extern "C" int jdg_beam_reorder(const jdg_reorder_args *a, void *stream) {
    const char *who = "jdg_beam_reorder";
    int rc = jdg_beam_reorder_check(a), dev;
    if (rc != JD_OK) return rc;
    const int64_t rows = (int64_t)a->groups * a->beams;
    ReorderP p = {};
    p.parent = a->parent; p.parent_stride = a->parent_stride; p.beams = a->beams; p.status = a->status;
    unsigned ctas = 0;
    for (int i = 0; i < a->n_states; i++) {
        const jdg_state &s = a->state[i];
        if (!s.row_bytes) continue;
        auto &t = p.st[p.n_states++];
        t.src = (const uint8_t *)s.src; t.dst = (uint8_t *)s.dst; t.bytes = s.row_bytes; t.src_stride = s.src_stride;
        t.dst_stride = s.dst_stride;
        t.first = ctas;
        t.chunks = (unsigned)((s.row_bytes + kRoChunk - 1) / kRoChunk);
        ctas += (unsigned)rows * t.chunks;
    }
    if (!ctas) return JD_OK;
    cudaStream_t st = (cudaStream_t)stream;
    rc = devop_stream(who, st, &dev);
    if (rc != JD_OK) return rc;
    return devop_launch(who, false, k_beam_reorder, dim3(ctas), dim3(kRoThreads), 0, st, p);
}
