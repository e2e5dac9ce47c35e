// jdg_paged_tc.cuh — the shared prefix on the tensor cores (tcgen05), for f16 / bf16 caches.
//
// The queries of one KV head behind a shared prefix are n_seqs * G rows of one matrix Q, so the
// prefix is two matrix products per tile of 128 cache rows: S = Q K^T (128 x 128), O += P V,
// with the running-maximum softmax between them.  A CTA walks its share of the prefix in two
// streams of four warps, each with its own S, O and statistics:
//   warps 0-3, 4-7   stream 0 / 1: one query a thread, which takes its whole row of S into
//                    registers, finds the maximum and writes P back over S as 16-bit pairs.  Only
//                    when a score passes the running maximum by more than 2^8 (rare after the
//                    first tiles) is O rescaled in tensor memory.  One thread of the stream then
//                    issues O += P V (P is the tensor-memory operand) and the next S (Q and K
//                    from shared memory).
//   warps 8-11       copy cache rows to shared memory with 16-byte cp.async, row by row through
//                    the page table (any page size), in the 128-byte swizzle; keys are the
//                    K-major operand and values the MN-major one, both as the cache holds them.
// While one stream's softmax runs, the other's products do; a stream that issues its own MMAs
// never waits for the other's softmax (256 queries x 1,920 rows: loop of 46 us with one issuing
// thread for both, 40 with two; with the exponentials partly on the FMA units now 35.5).  With more
// than 128 queries the streams are the two query tiles and share every cache tile; with 128 or
// fewer, both take the same queries and alternate cache tiles, and join at the end.
//
// Order of the MMAs: P of a stream lies over its S, so S of the next tile may only be written
// once P V has read P.  Both are issued by one thread, and MMAs of one CTA run in issue order;
// the commit behind S covers P V too, so a softmax that sees S knows that O is up to date.
// Every wait is bounded by wall time: on a timeout the CTA flags JDG_STATUS_TIMEOUT, the roles
// go through the rest of their loops without waiting or issuing, the MMAs in flight are waited
// for (bounded), the parts are left as NaN sums (so out and lse show it, flag or no flag) and the
// tensor memory is freed.
#pragma once
#include "jdg_async.cuh"
#include "jdg_paged_attn.cuh"

namespace jdg {

constexpr int kPtThreads = 12 * 32, kPtRows = 128;
constexpr int kPtCopies = 4, kPtAhead = 2;  // copy warps, 32-row copies each keeps in flight

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
__device__ __forceinline__ void pt_ld16(uint32_t taddr, float (&v)[16]) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
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
// 2^y of two numbers on the FMA units, within 2^-22 (as ex2.approx): y = n + f with n the nearest
// integer (Cody and Waite: the sum with 1.5 2^23 leaves n in the low bits), 2^f by the polynomial of
// degree 5 whose largest relative error on [-1/2, 1/2] is least (fitted by Lawson's iteration), n
// added to the exponent.  Below -126 it stays 2^-126: as good as nothing beside weights of 1.  A NaN
// comes out as the largest number (the row's maximum is what tells of it).
__device__ __forceinline__ float2 pt_exp2(float2 y) {
    asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(y.x));  // -126
    asm("max.NaN.f32 %0, %0, 0fC2FC0000;" : "+f"(y.y));
    const float2 big = make_float2(12582912.f, 12582912.f), nbig = make_float2(-12582912.f, -12582912.f);
    const float2 t = add2(y, big), n = add2(t, nbig), f = add2(y, make_float2(-n.x, -n.y));
    float2 q = make_float2(1.32765e-3f, 1.32765e-3f);
    q = fma2(q, f, make_float2(9.67554e-3f, 9.67554e-3f));
    q = fma2(q, f, make_float2(5.550713e-2f, 5.550713e-2f));
    q = fma2(q, f, make_float2(2.402212e-1f, 2.402212e-1f));
    q = fma2(q, f, make_float2(6.9314697e-1f, 6.9314697e-1f));
    q = fma2(q, f, make_float2(1.00000007f, 1.00000007f));
    return make_float2(__int_as_float(__float_as_int(q.x) + (__float_as_int(t.x) << 23)),
                       __int_as_float(__float_as_int(q.y) + (__float_as_int(t.y) << 23)));
}
// NaN if either is
__device__ __forceinline__ float pt_max(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// one lane of a converged warp, the same each time
__device__ __forceinline__ bool pt_elect() {
    uint32_t yes;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(yes));
    return yes != 0;
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

// CLAMP: 0 none, 1 up to kPaWide, 2 above
template <typename T, int HDP, bool FULL, int CLAMP>
__global__ __launch_bounds__(kPtThreads, 1) void k_pa_tc(const __grid_constant__ PaArgs p) {
    using C = PaTc<HDP>;
    constexpr int NS = C::kSlots, KS = HDP / 16;
    constexpr bool BF = sizeof(T) == 2 && !__is_same(T, __half);
    extern __shared__ uint8_t pt_raw[];
    uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(pt_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *ring = sm + 2 * C::kTile;
    __shared__ __align__(8) uint64_t full[NS], empty[NS], s_full[2], o_full[2], drained[2];
    __shared__ uint32_t masks[8][4];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_s;
    volatile int *abort_flag = &abort_s;
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(JDG_FULL, tid >> 5, 0);  // known to be one value: the MMA operands stay uniform
    dep_trigger();
    // work: block of queries, KV head, share of the prefix (blocks of the same rows side by side)
    int id = blockIdx.x;
    const int rb = id % p.rb_pre;
    id /= p.rb_pre;
    const int kvh = id % p.KV, split = id / p.KV;
    const int r0 = rb * 2 * kPtRows, nrows = min(2 * kPtRows, p.n_seqs * p.G - r0);
    const int t0 = split * p.c_pre, t1 = min(p.prefix_len, t0 + p.c_pre), n_tiles = (t1 - t0 + kPtRows - 1) / kPtRows;
    const bool pair = nrows > kPtRows;  // two query tiles; else the streams alternate cache tiles
    if (tid == 0) {
        for (int i = 0; i < NS; i++) {
            mbar_init(&full[i], 4);              // four 32-row copies
            mbar_init(&empty[i], pair ? 2 : 1);  // a commit of each stream that reads it
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&s_full[i], 1);
            mbar_init(&o_full[i], 1);
            mbar_init(&drained[i], 1);
        }
        abort_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (!FULL && warp >= 8) {
        // columns past head_dim of every slot: zeros for good (copies never write them)
        const int c0 = p.hd / 8, nc = HDP / 8 - c0;
        for (int i = tid - 8 * 32; i < NS * kPtRows * nc; i += 32 * kPtCopies) {
            const int r = i / nc, c = c0 + i % nc, row = r & 127;
            *reinterpret_cast<uint4 *>(ring + (r >> 7) * C::kTile + (c >> 3) * C::kPanel + row * 128 +
                                       (((c & 7) ^ (row & 7)) << 4)) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
    }
    pt_before();
    __syncthreads();
    pt_after();
    const uint32_t tmem = tmem_slot;
    auto tS = [&](int i) { return tmem + (uint32_t)i * 128; };         // S, and P over it, of stream i
    auto tO = [&](int i) { return tmem + 256 + (uint32_t)i * HDP; };

    if (warp >= 8) {
        // ---------------- copies: item 2 j is the keys of tile j, item 2 j + 1 its values; a unit is 32
        // rows of an item, unit u = 4 item + rows / 32, taken in turn by the four warps ----------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const T *kh = (const T *)p.k + (int64_t)kvh * p.head_stride, *vh = (const T *)p.v + (int64_t)kvh * p.head_stride;
        const int pmask = (1 << p.page_shift) - 1, units = 8 * n_tiles;
        auto row_of = [&](int u) { return t0 + (u >> 3) * kPtRows + (u & 3) * 32 + lane; };  // this lane's cache row
        auto page_of = [&](int u) { return row_of(u) < t1 ? p.prefix[row_of(u) >> p.page_shift] : -1; };
        int told = warp - 8, pending = 0;  // first unit not handed over, units in flight
        auto hand_over = [&](int keep) {   // this warp's oldest units have landed, all but `keep`
            fence_proxy_async_smem();
            __syncwarp();
            for (; pending > keep; pending--, told += kPtCopies)
                if (lane == 0) mbar_arrive(&full[(told >> 2) % NS]);
        };
        int page = page_of(warp - 8);
        for (int u = warp - 8; u < units; u += kPtCopies) {
            const int item = u >> 2, slot = item % NS;
            if (item >= NS) {
                const uint32_t par = (uint32_t)(item / NS - 1) & 1u;
                // (the whole warp decides together) nothing to issue: hand over what is in flight first
                if (!__all_sync(JDG_FULL, pt_test(&empty[slot], par))) {
                    cp_wait<0>();
                    hand_over(0);
                    if (!__all_sync(JDG_FULL, pt_wait(&empty[slot], par, abort_flag))) break;
                }
            }
            const int t = row_of(u);
            const bool in = t < t1, good = in && page >= 0 && page < p.n_pages;
            if (in && !good && p.status) atomicOr(p.status, JDG_STATUS_PAGE);
            const uint32_t valid = __ballot_sync(JDG_FULL, good);
            const int64_t off = (good ? (int64_t)page * p.page_stride : 0) + (int64_t)(t & pmask) * p.row_stride;
            page = u + kPtCopies < units ? page_of(u + kPtCopies) : -1;
            if (!(item & 1) && lane == 0) masks[(item >> 1) & 7][u & 3] = valid;
            const T *base = item & 1 ? vh : kh;
            const uint32_t dst = smem_u32(ring + slot * C::kTile) + (u & 3) * 32 * 128;
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
            if (++pending > kPtAhead) {
                cp_wait<kPtAhead>();
                hand_over(kPtAhead);
            }
        }
        cp_wait<0>();
        hand_over(0);
    } else {
        // ---------------- stream i, query row of this thread ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");  // 256 x 216 + 128 x 72 = 384 x 168, the launch's
        const int i = warp >> 2, row = (warp & 3) * 32 + lane;
        const int q = (pair ? i * kPtRows : 0) + row;           // query of the block
        const bool idle = (pair ? i * kPtRows : 0) + (warp & 3) * 32 >= nrows;  // no query in the whole warp
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        // queries: 128 or 256 rows (zeros past the end), swizzled
        for (int k = tid; k < (pair ? 2 : 1) * kPtRows * (HDP / 8); k += 256) {
            const int r = k / (HDP / 8), c = k % (HDP / 8), qq = r0 + r, sq = qq / p.G;
            const bool in = r < nrows && (FULL || c * 8 < p.hd);
            cp16(smem_u32(sm + (r >> 7) * C::kTile + (c >> 3) * C::kPanel + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4)),
                 (const T *)p.q + (in ? (int64_t)sq * p.q_stride + (int64_t)(kvh * p.G + qq - sq * p.G) * p.hd + c * 8 : 0),
                 in);
        }
        cp_commit();
        cp_wait<0>();
        fence_proxy_async_smem();
        asm volatile("bar.sync 3, 256;" ::: "memory");
        // step n of the stream: cache tile (pair ? n : 2 n + i)
        const int steps = pair ? n_tiles : (n_tiles - i + 1) / 2;
        const bool issuer = (warp & 3) == 0;  // the warp whose elected lane issues
        constexpr uint32_t id_s = pt_idesc(BF, kPtRows, false), id_o = pt_idesc(BF, HDP, true);
        const uint64_t dq = pt_desc(smem_u32(sm) + (pair ? i * C::kTile : 0), 16), dk = pt_desc(smem_u32(ring), 16),
                       dv = pt_desc(smem_u32(ring), C::kPanel);
        bool ok = true;
        auto scores = [&](int n) {  // the issuing warp: S of step n
            const int x = 2 * (pair ? n : 2 * n + i), slot = x % NS;
            ok = ok && pt_wait(&full[slot], (uint32_t)(x / NS) & 1u, abort_flag);
            ok = __all_sync(JDG_FULL, ok);
            if (!ok) return;
            pt_after();
            const uint64_t b = dk + (uint64_t)(slot * (C::kTile >> 4));
            if (pt_elect()) {
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    constexpr uint32_t panel = C::kPanel >> 4;
                    const uint64_t o = (k >> 2) * panel + (k & 3) * 2;
                    pt_mma_ss(tS(i), dq + o, b + o, id_s, k > 0);
                }
                pt_commit(&s_full[i]);
                pt_commit(&empty[slot]);
            }
            __syncwarp();
        };
        // the second stream starts half a step late: in step with one another, both softmaxes would share the
        // exponential unit and both products the tensor core, and then wait together
        const bool stagger = n_tiles >= 4;
        if (stagger && i) asm volatile("bar.sync 4, 256;" ::: "memory");
        if (issuer && steps) scores(0);
        const PaScale score(p);
        auto clamped = [&](float v) { return CLAMP == 2 ? score.clamp_wide(v) : score.clamp(v); };
        float m = -INFINITY, l = 0.f;
        for (int n = 0; n < steps; n++) {
            ok = ok && pt_wait(&s_full[i], (uint32_t)n & 1u, abort_flag);
            const bool run = __all_sync(JDG_FULL, ok) && !idle;
            if (run) {
                pt_after();
                const int tile = pair ? n : 2 * n + i;
                const uint32_t ts = tS(i) + lanes;
                uint32_t mk[4];
#pragma unroll
                for (int k = 0; k < 4; k++) mk[k] = *reinterpret_cast<volatile uint32_t *>(&masks[tile & 7][k]);
                const bool partial = (mk[0] & mk[1] & mk[2] & mk[3]) != JDG_FULL;
                if (partial) {  // rows that do not count: -inf into S
#pragma unroll 1
                    for (int c = 0; c < 8; c++) {
                        float v[16];
                        pt_ld16(ts + c * 16, v);
                        pt_ld_wait();
                        const uint32_t bits = (c & 4 ? (c & 2 ? mk[3] : mk[2]) : (c & 2 ? mk[1] : mk[0])) >> ((c & 1) * 16);
#pragma unroll
                        for (int j = 0; j < 16; j++) v[j] = bits >> j & 1u ? v[j] : -INFINITY;
                        pt_st16(ts + c * 16, reinterpret_cast<uint32_t(&)[16]>(v));
                    }
                    pt_st_wait();
                }
                // the whole row of S in registers: its maximum, then the weights against the running one
                float x[4][32];
#pragma unroll
                for (int c = 0; c < 4; c++) pt_ld32(ts + c * 32, x[c]);
                pt_ld_wait();
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int j = 0; j < 32; j++) mx[j & 3] = pt_max(mx[j & 3], x[c][j]);
                float top = pt_max(pt_max(mx[0], mx[1]), pt_max(mx[2], mx[3]));
                if (!(top == top)) l = top;  // a NaN score: the sum, and by it out and lse, are NaN for good
                // (the clamp rises with its argument; scale is positive here; it takes -inf to its lower end, where a
                // row counts at all)
                if (top > -INFINITY || (CLAMP && (mk[0] | mk[1] | mk[2] | mk[3]))) top = CLAMP ? clamped(top) : top * score.mul;
                const bool up = top - m > kPaSlack + kPaLift<T>;
                if (__any_sync(JDG_FULL, up)) {
                    const float mn = up ? top - kPaLift<T> : m;
                    const float f = m == -INFINITY ? 0.f : ex2(m - mn);
                    if (n) {  // O of the tiles before, complete with this S
#pragma unroll 1
                        for (int c = 0; c < HDP / 16; c++) {
                            float ov[16];
                            pt_ld16(tO(i) + lanes + c * 16, ov);
                            pt_ld_wait();
#pragma unroll
                            for (int j = 0; j < 16; j++) ov[j] *= f;
                            pt_st16(tO(i) + lanes + c * 16, reinterpret_cast<uint32_t(&)[16]>(ov));
                        }
                    }
                    l *= f;
                    m = mn;
                }
                const float base = m == -INFINITY ? 0.f : m;
                const float2 mul = make_float2(score.mul, score.mul), nb = make_float2(-base, -base);
                float2 sums[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t w[16];
                    const uint32_t bits = CLAMP && partial ? *reinterpret_cast<volatile uint32_t *>(&masks[tile & 7][c]) : 0u;
                    auto clamped2 = [&](float2 v) { return make_float2(clamped(v.x), clamped(v.y)); };
                    auto weights = [&](auto clamped) {
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            float2 y;
                            if (CLAMP) y = add2(clamped(make_float2(x[c][j], x[c][j + 1])), nb);
                            else y = fma2(make_float2(x[c][j], x[c][j + 1]), mul, nb);
                            if (CLAMP && partial) {  // the clamp has lifted the masked ones as well
                                if (!(bits >> j & 1u)) y.x = -INFINITY;
                                if (!(bits >> (j + 1) & 1u)) y.y = -INFINITY;
                            }
                            // one pair in four on the FMA units (a published division of this softmax's
                            // exponentials): the exponential unit (16 a cycle and SM) bounds it
                            const float2 e = !CLAMP && (j & 6) == 6 ? pt_exp2(y) : make_float2(ex2(y.x), ex2(y.y));
                            sums[(j >> 1) & 1] = add2(sums[(j >> 1) & 1], e);
                            w[j / 2] = pack2(e.x, e.y, (const T *)nullptr);
                        }
                    };
                    if constexpr (CLAMP == 2) {  // far below the clamp (the rule): the polynomial alone
                        float far = 0.f;
#pragma unroll
                        for (int j = 0; j < 32; j++) far = fmaxf(far, fabsf(x[c][j]));
                        if (__all_sync(JDG_FULL, far * score.in <= kPaSmall)) weights([&](float2 v) { return score.clamp_small(v); });
                        else weights(clamped2);
                    } else {
                        weights(clamped2);
                    }
                    pt_st16(ts + c * 16, w);
                }
                const float2 sum = add2(sums[0], sums[1]);
                l += sum.x + sum.y;
                pt_st_wait();
                pt_before();
            }
            asm volatile("bar.sync %0, 128;" ::"r"(1 + i) : "memory");  // P of the whole stream is written
            if (stagger && !i && !n) asm volatile("bar.arrive 4, 256;" ::: "memory");
            if (issuer) {
                const int x = 2 * (pair ? n : 2 * n + i) + 1, slot = x % NS;
                ok = ok && pt_wait(&full[slot], (uint32_t)(x / NS) & 1u, abort_flag);
                ok = __all_sync(JDG_FULL, ok);
                if (ok) {
                    pt_after();
                    const uint64_t b = dv + (uint64_t)(slot * (C::kTile >> 4));
                    if (pt_elect()) {
#pragma unroll
                        for (int k = 0; k < kPtRows / 16; k++)
                            pt_mma_ts(tO(i), tS(i) + k * 8, b + k * 128, id_o, n > 0 || k > 0);
                        pt_commit(&empty[slot]);
                        if (n + 1 == steps) pt_commit(&o_full[i]);
                    }
                    __syncwarp();
                    if (n + 1 < steps) scores(n + 1);
                }
            }
        }
        if (issuer && !ok) {  // whatever was issued runs before the tensor memory goes
            int never = 0;
            if (pt_elect()) pt_commit(&drained[i]);
            __syncwarp();
            pt_wait(&drained[i], 0, &never);
        }
        if (steps) ok = ok && pt_wait(&o_full[i], 0, abort_flag);
        ok = __all_sync(JDG_FULL, ok);
        pt_before();
        asm volatile("bar.sync 3, 256;" ::: "memory");  // both streams are done with the ring
        pt_after();
        const bool gave_up = *abort_flag != 0;  // seen by both streams: a role that fails a wait has set it by now
        // where the streams share the queries, the second leaves its part in shared memory for the first
        constexpr int kSt = HDP + 4;
        float *other = reinterpret_cast<float *>(ring), *ml = other + kPtRows * kSt;
        float f0 = 1.f, f1 = 0.f;
        if (!pair) {
            if (i == 1) {
                ml[2 * row] = m;
                ml[2 * row + 1] = l;
                if (ok && !idle && steps)
                    for (int c = 0; c < HDP; c += 16) {
                        float v[16];
                        pt_ld16(tO(i) + lanes + c, v);
                        pt_ld_wait();
#pragma unroll
                        for (int j = 0; j < 16; j += 4)
                            st4(other + row * kSt + c + j, make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]));
                    }
            }
            asm volatile("bar.sync 3, 256;" ::: "memory");
            if (i == 0 && n_tiles > 1) {
                const float m1 = ml[2 * row], mn = fmaxf(m, m1), base = mn == -INFINITY ? 0.f : mn;
                f0 = ex2(m - base);
                f1 = ex2(m1 - base);
                l = l * f0 + ml[2 * row + 1] * f1;
                m = mn;
            }
        }
        // the part of this split, 32 columns at a time through shared memory, so that a store covers whole lines
        if (gave_up) {
            if (q < nrows && (pair || i == 0)) {
                const int r = r0 + q, sq = r / p.G, h = kvh * p.G + r - sq * p.G;
                *reinterpret_cast<float2 *>(pa_part(p, sq * p.H + h, split)) = make_float2(0.f, __int_as_float(0x7fffffff));
            }
        } else if (!idle && (pair || i == 0)) {
            float *dst = nullptr;
            if (q < nrows) {
                const int r = r0 + q, sq = r / p.G, h = kvh * p.G + r - sq * p.G;
                dst = pa_part(p, sq * p.H + h, split);
                *reinterpret_cast<float2 *>(dst) = make_float2(m, l);
            }
            float *st = ml + 2 * kPtRows + warp * 32 * 36;
            const uint64_t d64 = reinterpret_cast<uint64_t>(dst);
            for (int c = 0; c < HDP; c += 32) {
                float v[2][16];
                pt_ld16(tO(i) + lanes + c, v[0]);
                pt_ld16(tO(i) + lanes + c + 16, v[1]);
                pt_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    float4 x = make_float4(v[j >> 4][j & 15], v[j >> 4][(j & 15) + 1], v[j >> 4][(j & 15) + 2],
                                           v[j >> 4][(j & 15) + 3]);
                    if (!pair && n_tiles > 1) {
                        const float4 y = ld4(other + row * kSt + c + j);
                        x = make_float4(x.x * f0 + y.x * f1, x.y * f0 + y.y * f1, x.z * f0 + y.z * f1, x.w * f0 + y.w * f1);
                    }
                    st4(st + lane * 36 + j, x);
                }
                __syncwarp();
                const int col = c + (lane & 7) * 4;
#pragma unroll
                for (int r = 0; r < 32; r += 4) {
                    float *d = reinterpret_cast<float *>(__shfl_sync(JDG_FULL, d64, r + (lane >> 3)));
                    const float4 x = ld4(st + (r + (lane >> 3)) * 36 + (lane & 7) * 4);
                    if (d && col < p.hd) st4(d + 4 + col, x);
                }
                __syncwarp();
            }
        }
    }
    pt_before();
    __syncthreads();
    if (tid == 0 && *abort_flag && p.status) atomicOr(p.status, JDG_STATUS_TIMEOUT);
    if (warp == 0) {
        pt_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

}  // namespace jdg
