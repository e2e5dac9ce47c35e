// jdg_paged_tc.cuh — the shared prefix on the tensor cores (tcgen05), for f16 / bf16 caches.
//
// The queries of one KV head behind a shared prefix are n_seqs * G rows of one matrix Q, so the
// prefix is two matrix products per tile of 128 cache rows: S = Q K^T (128 x 128), O += P V,
// with the running-maximum softmax between them.  A CTA holds up to two tiles of 128 queries and
// walks its share of the prefix:
//   warps 0-3, 4-7   softmax of stream 0 / 1: one query a thread.  S is read from tensor memory
//                    (once for the maximum, once for the weights), P goes back over it as 16-bit
//                    pairs; O is rescaled in tensor memory only when a maximum rises by more
//                    than 2^8 (rare after the first tiles), so there is no correction pass.
//   warp 8           one thread issues every MMA: Q K^T from shared memory, P V with P as the
//                    tensor-memory operand.
//   warps 9-12       copy cache rows to shared memory with 16-byte cp.async, row by row through
//                    the page table (any page size), in the 128-byte swizzle; keys are the
//                    K-major operand and values the MN-major one, both as the cache holds them.
// Two streams keep the tensor core busy: while one stream's softmax runs, the other's products
// do.  With more than 128 queries the streams are the two query tiles and share every cache
// tile; with 128 or fewer, both take the same queries and alternate cache tiles (each then
// writes a part of its own).
//
// Order of the MMAs: P of a stream lies over its S, so S of the next tile may only be written
// once P V has read P.  Both are issued by one thread, and MMAs of one CTA run in issue order;
// the commit behind S covers P V too, so a softmax that sees S knows that O is up to date.
// Every wait is bounded by wall time: on a timeout the CTA flags JDG_STATUS_TIMEOUT, every role
// leaves, the MMAs in flight are waited for (bounded) and the tensor memory is freed.
#pragma once
#include "jdg_async.cuh"
#include "jdg_paged_attn.cuh"

namespace jdg {

constexpr int kPtThreads = 13 * 32, kPtRows = 128;

template <int HDP>
struct PaTc {
    static constexpr int kPanel = kPtRows * 128;          // 64 columns of 128 rows
    static constexpr int kTile = kPanel * (HDP / 64);     // Q, K or V tile
    static constexpr int kSlots = HDP == 64 ? 8 : 5;      // ring of K and V tiles
    static constexpr int kSmem = 1024 + 2 * kTile + kSlots * kTile;
};

// instruction descriptor: D f32, A and B f16 (0) or bf16 (1), M 128, N n; bit 16: B is MN-major
__host__ __device__ constexpr uint32_t pt_idesc(bool bf16, int n, bool b_mn) {
    return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kPtRows >> 4) << 24);
}
// 128-byte swizzle, groups of 8 rows 1024 bytes apart; lbo: stride between 64-column panels (MN-major)
__device__ __forceinline__ uint64_t pt_desc(uint32_t saddr, uint32_t lbo) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)((lbo >> 4) & 0x3FFF) << 16) |
           ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ void pt_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void pt_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void pt_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void pt_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pt_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pt_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void pt_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pt_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pt_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void pt_st32(uint32_t taddr, const float (&v)[32]) {
    const uint32_t *r = reinterpret_cast<const uint32_t *>(v);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
        "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ bool pt_test(uint64_t *bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(done)
                 : "r"(smem_u32(bar)), "r"(parity)
                 : "memory");
    return done != 0;
}
// wait for a phase, at most half a second of wall time or until another role gave up
__device__ __forceinline__ bool pt_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
    if (pt_test(bar, parity)) return true;
    unsigned long long t0, t1;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
    for (;;) {
        uint32_t done;
        asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                     : "=r"(done)
                     : "r"(smem_u32(bar)), "r"(parity)
                     : "memory");
        if (done) return true;
        if (*abort_flag) return false;
        asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t1));
        if (t1 - t0 > 500ull * 1000 * 1000) {
            *abort_flag = 1;
            return false;
        }
    }
}

template <typename T, int HDP, bool FULL>
__global__ __launch_bounds__(kPtThreads, 1) void k_pa_tc(const __grid_constant__ PaArgs p) {
    using C = PaTc<HDP>;
    constexpr int NS = C::kSlots, KS = HDP / 16;
    constexpr bool BF = sizeof(T) == 2 && !__is_same(T, __half);
    extern __shared__ uint8_t pt_raw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pt_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *ring = sm + 2 * C::kTile;
    __shared__ __align__(8) uint64_t full[NS], empty[NS], s_full[2], p_full[2], o_full[2], drained;
    __shared__ uint32_t masks[8][4];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_s;
    volatile int *abort_flag = &abort_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    dep_trigger();
    // work: block of queries, KV head, share of the prefix (blocks of the same rows side by side)
    int id = blockIdx.x;
    const int rb = id % p.rb_pre;
    id /= p.rb_pre;
    const int kvh = id % p.KV, split = id / p.KV;
    const int r0 = rb * 2 * kPtRows, nrows = min(2 * kPtRows, p.n_seqs * p.G - r0);
    const int t0 = split * p.c_pre, t1 = min(p.prefix_len, t0 + p.c_pre), n_tiles = (t1 - t0 + kPtRows - 1) / kPtRows;
    const bool pair = nrows > kPtRows;  // two query tiles; else the streams alternate cache tiles
    const int steps = pair ? 2 * n_tiles : n_tiles;  // step s: stream s & 1, cache tile (pair ? s >> 1 : s)
    if (tid == 0) {
        for (int i = 0; i < NS; i++) {
            mbar_init(&full[i], 4);   // the copy warps
            mbar_init(&empty[i], 1);  // a commit
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);  // the stream's softmax warps
            mbar_init(&o_full[i], 1);
        }
        mbar_init(&drained, 1);
        abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (warp < 8) {
        // queries: 256 rows (zeros past the end), swizzled; without a second tile only 128
        const int n_q = pair ? 2 * kPtRows : kPtRows;
        for (int i = tid; i < n_q * (HDP / 8); i += 256) {
            const int r = i / (HDP / 8), c = i % (HDP / 8);
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (r < nrows && c * 8 < p.hd) {
                const int row = r0 + r, s = row / p.G, h = kvh * p.G + row - s * p.G;
                x = *reinterpret_cast<const uint4 *>((const T *)p.q + (int64_t)s * p.q_stride + (int64_t)h * p.hd + c * 8);
            }
            *reinterpret_cast<uint4 *>(sm + (r >> 7) * C::kTile + (c >> 3) * C::kPanel + (r & 127) * 128 +
                                       (((c & 7) ^ (r & 7)) << 4)) = x;
        }
    } else if (!FULL && warp > 8) {
        // columns past head_dim of every slot: zeros for good (copies never write them)
        const int c0 = p.hd / 8, nc = HDP / 8 - c0;
        for (int i = tid - 9 * 32; i < NS * kPtRows * nc; i += 128) {
            const int r = i / nc, c = c0 + i % nc, row = r & 127;
            *reinterpret_cast<uint4 *>(ring + (r >> 7) * C::kTile + (c >> 3) * C::kPanel + row * 128 +
                                       (((c & 7) ^ (row & 7)) << 4)) = make_uint4(0u, 0u, 0u, 0u);
        }
    }
    fence_proxy_async_smem();
    pt_before();
    __syncthreads();
    pt_after();
    const uint32_t tmem = tmem_slot;
    auto tS = [&](int i) { return tmem + (uint32_t)i * 128; };         // S, and P over it, of stream i
    auto tO = [&](int i) { return tmem + 256 + (uint32_t)i * HDP; };

    if (warp >= 9) {
        // ---------------- copies: slot 2 i holds keys of tile i, slot 2 i + 1 its values ----------------
        const int cw = warp - 9;  // rows 32 cw .. of each tile
        const T *kh = (const T *)p.k + (int64_t)kvh * p.head_stride, *vh = (const T *)p.v + (int64_t)kvh * p.head_stride;
        const int pmask = (1 << p.page_shift) - 1;
        int signalled = 0;
        auto signal = [&](int upto) {  // this warp's rows of the copies before `upto` have landed
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0)
                for (int i = signalled; i < upto; i++) mbar_arrive(&full[i % NS]);
            signalled = upto;
        };
        int64_t off = 0;
        uint32_t valid = 0;
        int page = -1, t = t0 + cw * 32;
        auto page_of = [&](int tt) { return tt + lane < t1 ? p.prefix[(tt + lane) >> p.page_shift] : -1; };
        page = page_of(t);
        bool ok = true;
        for (int i = 0; i < 2 * n_tiles; i++) {
            const int slot = i % NS;
            if (i >= NS) {
                const uint32_t par = (uint32_t)(i / NS - 1) & 1u;
                // (the whole warp decides together) nothing to issue: hand over what is in flight first
                if (!__all_sync(JDG_FULL, pt_test(&empty[slot], par))) {
                    cp_wait<0>();
                    signal(i);
                    ok = pt_wait(&empty[slot], par, abort_flag);
                    if (!__all_sync(JDG_FULL, ok)) break;
                }
                __syncwarp();
            }
            if ((i & 1) == 0) {
                const bool in = t + lane < t1, good = in && page >= 0 && page < p.n_pages;
                if (in && !good && p.status) atomicOr(p.status, JDG_STATUS_PAGE);
                valid = __ballot_sync(JDG_FULL, good);
                off = (good ? (int64_t)page * p.page_stride : 0) + (int64_t)((t + lane) & pmask) * p.row_stride;
                t += kPtRows;
                page = page_of(t);
                if (lane == 0) masks[(i >> 1) & 7][cw] = valid;
            }
            const T *base = i & 1 ? vh : kh;
            const uint32_t dst = smem_u32(ring + slot * C::kTile) + cw * 32 * 128;
            if constexpr (FULL) {
                constexpr int cpr = HDP / 8, rpi = 32 / cpr;
                const int lr = lane / cpr, lc = lane % cpr;
                const uint32_t d0 = dst + (lc >> 3) * C::kPanel + lr * 128, ch = (uint32_t)((lc & 7) ^ lr) << 4;
                const uint32_t mine = valid >> lr;
                base += lc * 8;
                if (p.page_shift >= 4) {
                    const int64_t inc = rpi * p.row_stride;
#pragma unroll
                    for (int half = 0; half < 2; half++) {
                        const T *src = base + __shfl_sync(JDG_FULL, off, half * 16) + lr * p.row_stride;
#pragma unroll
                        for (int k = 0; k < 16 / rpi; k++) {
                            const int r = half * 16 + k * rpi;
                            cp16(d0 + r * 128 + (ch ^ ((r & 7) << 4)), src, mine >> r & 1u);
                            src += inc;
                        }
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 32; r += rpi) {
                        const T *src = base + __shfl_sync(JDG_FULL, off, r + lr);
                        cp16(d0 + r * 128 + (ch ^ ((r & 7) << 4)), src, mine >> r & 1u);
                    }
                }
            } else {
                const int cpr = p.hd / 8, rpi = 32 / cpr, lr = lane / cpr, lc = lane - lr * cpr;
                for (int k = 0; k < 32; k += rpi) {
                    const int r = k + lr;
                    const int64_t o = __shfl_sync(JDG_FULL, off, r & 31);
                    if (lr < rpi && r < 32)
                        cp16(dst + (lc >> 3) * C::kPanel + r * 128 + (((lc & 7) ^ (r & 7)) << 4), base + o + lc * 8,
                             valid >> r & 1u);
                }
            }
            cp_commit();
            if (i + 1 - signalled > 2) {  // two copies stay in flight
                cp_wait<2>();
                signal(i - 1);
            }
        }
        cp_wait<0>();
        signal(2 * n_tiles);
    } else if (warp == 8) {
        // ---------------- MMA thread ----------------
        if (lane == 0) {
            constexpr uint32_t id_s = pt_idesc(BF, kPtRows, false), id_o = pt_idesc(BF, HDP, true);
            const uint32_t q0 = smem_u32(sm), rg = smem_u32(ring);
            auto tile_of = [&](int s) { return pair ? s >> 1 : s; };
            bool ok = true;
            auto scores = [&](int s) {  // S of step s
                const int i = s & 1, x = 2 * tile_of(s), slot = x % NS;
                ok = ok && pt_wait(&full[slot], (uint32_t)(x / NS) & 1u, abort_flag);
                if (!ok) return;
                pt_after();
                const uint32_t a = q0 + (pair ? i * C::kTile : 0), b = rg + slot * C::kTile;
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    const uint32_t o = (k >> 2) * C::kPanel + (k & 3) * 32;
                    pt_mma_ss(tS(i), pt_desc(a + o, 16), pt_desc(b + o, 16), id_s, k > 0);
                }
                pt_commit(&s_full[i]);
                if (!pair || i) pt_commit(&empty[slot]);
            };
            scores(0);
            if (ok && steps > 1) scores(1);
            for (int s = 0; ok && s < steps; s++) {
                const int i = s & 1, x = 2 * tile_of(s) + 1, slot = x % NS;
                ok = pt_wait(&full[slot], (uint32_t)(x / NS) & 1u, abort_flag) &&
                     pt_wait(&p_full[i], (uint32_t)(s >> 1) & 1u, abort_flag);
                if (!ok) break;
                pt_after();
                const uint32_t b = rg + slot * C::kTile;
#pragma unroll
                for (int k = 0; k < kPtRows / 16; k++)
                    pt_mma_ts(tO(i), tS(i) + k * 8, pt_desc(b + k * 2048, C::kPanel), id_o, s > 1 || k > 0);
                if (!pair || i) pt_commit(&empty[slot]);
                if (s + 2 >= steps) pt_commit(&o_full[i]);
                if (s + 2 < steps) scores(s + 2);
            }
            // whatever was issued has run before the tensor memory goes
            pt_commit(&drained);
            int never = 0;
            pt_wait(&drained, 0, &never);
        }
        __syncwarp();
    } else {
        // ---------------- softmax of stream i, query row of this thread ----------------
        const int i = warp >> 2, row = (warp & 3) * 32 + lane;
        const int q = (pair ? i * kPtRows : 0) + row;           // query of the block
        const bool idle = (pair ? i * kPtRows : 0) + (warp & 3) * 32 >= nrows;  // no query in the whole warp
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const PaScale score(p);
        float m = -INFINITY, l = 0.f;
        bool ok = true;
        int n = 0;
        for (int s = i; s < steps; s += 2, n++) {
            ok = pt_wait(&s_full[i], (uint32_t)n & 1u, abort_flag);
            if (!__all_sync(JDG_FULL, ok)) {
                ok = false;
                break;
            }
            if (!idle) {
                pt_after();
                const uint32_t ts = tS(i) + lanes;
                const int tile = pair ? s >> 1 : s;
                uint32_t mk[4];
#pragma unroll
                for (int k = 0; k < 4; k++) mk[k] = *reinterpret_cast<volatile uint32_t *>(&masks[tile & 7][k]);
                float mx = -INFINITY;
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    float v[32];
                    pt_ld32(ts + c * 32, v);
                    pt_ld_wait();
                    if (mk[c] != JDG_FULL) {
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (!(mk[c] >> j & 1u)) v[j] = -INFINITY;
                    }
#pragma unroll
                    for (int j = 0; j < 32; j++) mx = fmaxf(mx, v[j]);
                }
                // the largest score (the clamp rises with its argument, and scale is not negative here)
                mx = mx == -INFINITY ? mx : score.clamped ? score.clamp(mx) : mx * score.mul;
                const bool up = mx > m + kPaSlack;
                if (__any_sync(JDG_FULL, up)) {
                    const float mn = up ? mx : m;
                    const float f = m == -INFINITY ? 0.f : ex2(m - mn);
                    if (n) {  // O of the tiles before, complete with this S
#pragma unroll 1
                        for (int c = 0; c < HDP / 32; c++) {
                            float v[32];
                            pt_ld32(tO(i) + lanes + c * 32, v);
                            pt_ld_wait();
#pragma unroll
                            for (int j = 0; j < 32; j++) v[j] *= f;
                            pt_st32(tO(i) + lanes + c * 32, v);
                        }
                    }
                    l *= f;
                    m = mn;
                }
                const float base = m == -INFINITY ? 0.f : m;
                float2 sum = make_float2(0.f, 0.f);
                const float2 mul = make_float2(score.mul, score.mul), nb = make_float2(-base, -base);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    float v[32];
                    pt_ld32(ts + c * 32, v);
                    pt_ld_wait();
                    uint32_t w[16];
                    if (score.clamped) {
#pragma unroll
                        for (int j = 0; j < 32; j++) v[j] = ex2(score.clamp(v[j]) - base);
                    } else {
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const float2 x = fma2(make_float2(v[j], v[j + 1]), mul, nb);
                            v[j] = ex2(x.x);
                            v[j + 1] = ex2(x.y);
                        }
                    }
                    if (mk[c] != JDG_FULL) {
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (!(mk[c] >> j & 1u)) v[j] = 0.f;
                    }
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        sum = add2(sum, make_float2(v[j], v[j + 1]));
                        // one rounding of each weight to the values' type: below the rounding of the result
                        w[j / 2] = pack2(v[j], v[j + 1], (const T *)nullptr);
                    }
                    pt_st16(ts + c * 16, w);  // over columns of S that have been read
                }
                l += sum.x + sum.y;
                pt_st_wait();
                pt_before();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[i]);
        }
        // the parts: one for each split, two where the streams share the queries
        const int part = split * p.pp + (pair ? 0 : i);
        if (ok && !idle) {
            const bool mine = q < nrows;
            float *dst = nullptr;
            if (mine) {
                const int r = r0 + q, sq = r / p.G, h = kvh * p.G + r - sq * p.G;
                dst = pa_part(p, sq * p.H + h, part);
                *reinterpret_cast<float2 *>(dst) = make_float2(m, l);
                if (pair && p.pp == 2) *reinterpret_cast<float2 *>(dst + p.hd + 4) = make_float2(-INFINITY, 0.f);
            }
            if (n) {
                ok = pt_wait(&o_full[i], 0, abort_flag);
                if (__all_sync(JDG_FULL, ok)) {
                    pt_after();
#pragma unroll 1
                    for (int c = 0; c < HDP / 32; c++) {
                        float v[32];
                        pt_ld32(tO(i) + lanes + c * 32, v);
                        pt_ld_wait();
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            if (mine && c * 32 + j < p.hd) st4(dst + 4 + c * 32 + j, make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]));
                    }
                }
            }
        }
    }
    pt_before();
    __syncthreads();
    if (tid == 0 && *abort_flag && p.status) atomicOr(p.status, JDG_STATUS_TIMEOUT);
    if (warp == 8) {
        pt_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

}  // namespace jdg
