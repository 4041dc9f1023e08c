// Attention over the paged 8-bit cache for many query rows: tcgen05 MMAs on tiles of 2 x 128 packed
// rows x 128 keys (arithmetic: kv_attention.cuh).
//
// One CTA (22 warps) works on one sequence, KV head and tile of 256 packed rows:
//   warps 0-7, 8-15 softmax of row tile 0 / 1, two threads to a row (TMEM lane), 64 keys each: scores
//                   from TMEM, p' back into their place as f16 (the A operand of P V), rare rescales
//                   of O
//   warps 16-19     converters: E4M3 codes -> f16 operands in shared memory, both of K and of V as
//                   rows of 64 dimensions swizzled over 128 bytes (K-major for K, MN-major for V)
//   warp 20         MMA issuer, warp 21 loader (one tensor copy per run of page positions)
// MMA order: S0(0) S1(0), then for each key tile j: P0 V, S0(j+1), P1 V, S1(j+1), so one row tile's
// softmax runs under the other's MMAs; S0(j+1) is complete only after P0 V(j), so a softmax thread
// that has its scores may rescale its row of O without another wait.
#pragma once
#include "kv_attention.cuh"

namespace dfb {

constexpr int kTcKeys = 128;     // keys of one tile
constexpr int kTcRows = 256;     // packed rows of one CTA
constexpr int kTcThreads = 704;
constexpr int kTcRaw = 2;        // raw slots: 128 x HD codes of K or V
constexpr int kTcSlots = 4;      // f16 slots, K and V of successive tiles in turn
constexpr float kTcOff = 7.f, kTcSlack = 8.f;  // p' <= 2^(off + slack) = 2^15 although the maximum is only followed by jumps

template <int HD>
struct TcSmem {
    static constexpr int q = 128 * HD * 2;         // one row tile's queries
    static constexpr int slot = kTcKeys * HD * 2;
    static constexpr int raw = kTcKeys * HD;
    static constexpr int q_off = 0, slot_off = 2 * q, raw_off = slot_off + kTcSlots * slot, sc_off = raw_off + kTcRaw * raw;
    static constexpr int bar_off = sc_off + 4 * 8 * 16;
    static constexpr int n_bars = 2 * kTcRaw + kTcSlots + 12;
    static constexpr int crow_off = bar_off + n_bars * 8 + 32;
    static constexpr int bytes = 1024 + crow_off + kTcRows * 4;
};

__device__ __forceinline__ void tmem_alloc1(uint32_t *holder, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(holder)), "r"(ncols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc1(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void mma1_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mma1_f16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                 "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma1_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),
                 "r"(idesc), "r"(acc)
                 : "memory");
}
// 32 lanes x 32 columns: this thread's lane, columns [col, col + 32).
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float *r) {
    uint32_t *u = reinterpret_cast<uint32_t *>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
          "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]),
          "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]),
          "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
        : "r"(taddr)
        : "memory");
}
// Ties 32 loaded registers to the wait, so that no use of them moves above it.
__device__ __forceinline__ void tmem_ld_wait32(float *r) {
    uint32_t *u = reinterpret_cast<uint32_t *>(r);
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]), "+r"(u[8]), "+r"(u[9]),
                   "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]), "+r"(u[14]), "+r"(u[15]), "+r"(u[16]), "+r"(u[17]), "+r"(u[18]),
                   "+r"(u[19]), "+r"(u[20]), "+r"(u[21]), "+r"(u[22]), "+r"(u[23]), "+r"(u[24]), "+r"(u[25]), "+r"(u[26]), "+r"(u[27]),
                   "+r"(u[28]), "+r"(u[29]), "+r"(u[30]), "+r"(u[31])
                 :
                 : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }
// Two f32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(d)
        : "l"(*reinterpret_cast<const uint64_t *>(&a)), "l"(*reinterpret_cast<const uint64_t *>(&b)), "l"(*reinterpret_cast<const uint64_t *>(&c)));
    return *reinterpret_cast<const float2 *>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<const uint64_t *>(&a)), "l"(*reinterpret_cast<const uint64_t *>(&b)));
    return *reinterpret_cast<const float2 *>(&d);
}
// The factor of a score is kept above 0, so that a masked score of -inf stays -inf where the softmax
// scale is 0 or the product of the scales underflows; every score times this is 0 beside an exponent.
constexpr float kMinFactor = 1.1754944e-38f;
// Whether any of the n threads of a named barrier passes true.
__device__ __forceinline__ bool named_bar_any(uint32_t id, uint32_t n, bool v) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %3, 0;\n\tbarrier.cta.red.or.aligned.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(id), "r"(n), "r"((uint32_t)v)
        : "memory");
    return r != 0;
}
// Bounded wait of one thread (the MMA issuer and single waits); see attn_wait.
__device__ __forceinline__ bool thread_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer();
    while (!mbar_try_wait_sleep(bar, parity, kWaitCheckNs)) {
        if (*abort_flag) return false;
        if (globaltimer() - t0 > kWaitTimeoutNs) {
            *abort_flag = 1;
            return false;
        }
    }
    return true;
}
// MN-major operand, rows (k) of 64 elements (128 bytes) swizzled over 128 bytes: 8-row groups 1024
// bytes apart, 64-element blocks `block` bytes apart.
__device__ __forceinline__ uint64_t mn128_desc(uint32_t smem_addr, uint32_t block) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);
    d |= (uint64_t)(block >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kTcThreads, 1)
    kv_attn_tc_kernel(const dfb_kv_cache c, const dfb_kv_attn a, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const AttnParts parts, bool vec, int32_t *status) {
    using L = TcSmem<HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *sm = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    float4 *sc = reinterpret_cast<float4 *>(sm + L::sc_off);  // [tile & 3][8 runs of 16 keys] ks, log2 vs, 1 / vs, any absent
    uint64_t *bars = reinterpret_cast<uint64_t *>(sm + L::bar_off);
    uint64_t *raw_full = bars, *raw_empty = raw_full + kTcRaw, *conv_full = raw_empty + kTcRaw, *freed = conv_full + kTcSlots;
    uint64_t *bar_s = freed + 2, *bar_pa = bar_s + 2, *bar_pb = bar_pa + 2, *bar_o = bar_pb + 2, *bar_q = bar_o + 2, *bar_drain = bar_q + 1;
    int *shared_i = reinterpret_cast<int *>(bars + L::n_bars);  // abort flag, most keys of a row, TMEM address
    volatile int *abort_flag = shared_i;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int s = blockIdx.z, kvh = blockIdx.y, split = blockIdx.x % parts.splits, tile = blockIdx.x / parts.splits;
    const int rep = a.n_q / c.n_kv;
    const AttnSeq sq = attn_seq(c, a, s, blockIdx.x == 0 && kvh == 0 && tid == 0, status);
    const int row0 = tile * kTcRows, n_packed = sq.n_rows * rep;
    if (row0 >= n_packed) return;
    const bool two = row0 + 128 < n_packed;
    if (tid == 0) {
        shared_i[0] = 0;
        shared_i[1] = 0;
        for (int i = 0; i < kTcRaw; i++) {
            mbar_init(&raw_full[i], 1);
            mbar_init(&raw_empty[i], 4);
        }
        for (int i = 0; i < kTcSlots; i++) {
            mbar_init(&conv_full[i], 4);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&bar_s[i], 1);
            mbar_init(&bar_pa[i], 4);
            mbar_init(&bar_pb[i], 4);
            mbar_init(&freed[i], 1);
            mbar_init(&bar_o[i], 1);
        }
        mbar_init(bar_q, two ? 16 : 8);
        mbar_init(bar_drain, 1);
        fence_barrier_init();
    }
    if (warp == 20) tmem_alloc1(reinterpret_cast<uint32_t *>(&shared_i[2]), 512);
    __syncthreads();
    // keys the tile's rows see
    const int w = tid >> 8, half = (warp >> 2) & 1;  // softmax warps: row tile, half of the keys
    const int R = row0 + w * 128 + (tid & 127);      // this thread's packed row
    int nr = 0;
    if (tid < 2 * kTcRows && R < n_packed) {
        nr = a.vis ? min(max(a.vis[sq.r0 + R / rep], 0), sq.len) : sq.len;
        if (half == 0) atomicMax(&shared_i[1], nr);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const int kend = shared_i[1];
    const uint32_t tmem = (uint32_t)shared_i[2];
    const int n_tiles = (kend + kTcKeys - 1) / kTcKeys;
    const int t0 = (int)((long long)n_tiles * split / parts.splits), nt = (int)((long long)n_tiles * (split + 1) / parts.splits) - t0;

    if (warp < 16) {
        if (w == 0 || two) {
            const int pair = 1 + w * 4 + (warp & 3);  // barrier of the two warps that share 32 rows
            // ── queries: half of the warp's 32 rows as f16, scaled by a power of two ──
            constexpr int LPR = HD / 8, RPI = 32 / LPR;  // lanes of a row (16 bytes each), rows of one load
            const uint32_t tm_s = tmem + w * 128 + ((uint32_t)(warp & 3) << 21), tm_o = tmem + 256 + w * 128 + ((uint32_t)(warp & 3) << 21);
            const int wrow = row0 + w * 128 + (warp & 3) * 32;  // the warp's first packed row
            float *crow = reinterpret_cast<float *>(sm + L::crow_off) + w * 128 + (warp & 3) * 32;
            float cr = fabsf(a.scale) * kLog2e;
            if (nt > 0) {  // (without keys the output goes through this memory right away)
                uint4 raw[LPR / 2];
                const int ch = lane % LPR, r0 = half * 16 + lane / LPR;
                const T *from[LPR / 2];
#pragma unroll
                for (int i = 0; i < LPR / 2; i++) {
                    // (a row that does not exist is read as the last one: what comes of it is not stored)
                    const int r = min(wrow + r0 + i * RPI, n_packed - 1), t = r / rep;
                    from[i] = reinterpret_cast<const T *>(a.q) + (sq.r0 + t) * a.q_tok + (kvh * rep + r - t * rep) * a.q_head + 8 * ch;
                }
                if (vec) {
#pragma unroll
                    for (int i = 0; i < LPR / 2; i++) raw[i] = *reinterpret_cast<const uint4 *>(from[i]);
                } else {
#pragma unroll
                    for (int i = 0; i < LPR / 2; i++)
#pragma unroll
                        for (int e = 0; e < 8; e++) reinterpret_cast<T *>(&raw[i])[e] = from[i][e];
                }
                float up[LPR / 2];
#pragma unroll
                for (int i = 0; i < LPR / 2; i++) up[i] = 1.f;
                if constexpr (!std::is_same<T, __half>::value) {
                    float mx[LPR / 2];
#pragma unroll
                    for (int i = 0; i < LPR / 2; i++) {
                        mx[i] = 0.f;
#pragma unroll
                        for (int e = 0; e < 8; e++) mx[i] = fmaxf(mx[i], fabsf(to_f32<T>(reinterpret_cast<const T *>(&raw[i])[e])));
                    }
#pragma unroll
                    for (int o = 1; o < LPR; o <<= 1)
#pragma unroll
                        for (int i = 0; i < LPR / 2; i++) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
#pragma unroll
                    for (int i = 0; i < LPR / 2; i++) {
                        const int e = (int)(__float_as_uint(mx[i]) >> 23) - 127;
                        up[i] = mx[i] > 0.f && mx[i] < INFINITY ? exp2i(min(max(-e, -126), 60)) : 1.f;
                    }
                    if (ch == 0)
#pragma unroll
                        for (int i = 0; i < LPR / 2; i++) crow[r0 + i * RPI] = 1.f / up[i];
                }
#pragma unroll
                for (int i = 0; i < LPR / 2; i++) {
                    float x[8];
                    const int rt = (warp & 3) * 32 + r0 + i * RPI;
                    const float f = a.scale < 0.f ? -up[i] : up[i];  // a negative scale turns q's sign: the scores' factors stay positive
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = to_f32<T>(reinterpret_cast<const T *>(&raw[i])[e]) * f;
                    uint4 u;
                    u.x = pack_f16(x[0], x[1]); u.y = pack_f16(x[2], x[3]);
                    u.z = pack_f16(x[4], x[5]); u.w = pack_f16(x[6], x[7]);
                    *reinterpret_cast<uint4 *>(sm + L::q_off + w * L::q + (ch / 8) * 16384 + rt * 128 + (((ch & 7) ^ (rt & 7)) << 4)) = u;
                }
                fence_proxy_async_smem();
                named_bar_sync(pair, 64);
                if constexpr (!std::is_same<T, __half>::value) cr *= crow[lane];
                if (lane == 0) mbar_arrive(bar_q);
            }
            // ── key tiles ──
            float M = -INFINITY, l = 0.f;
            for (int j = 0; j < nt; j++) {
                if (!attn_wait(&bar_s[w], j & 1, abort_flag)) break;
                if (wrow >= n_packed) {  // no row of this warp exists: whatever its lanes of P hold, no one reads what comes of it
                    if (lane == 0) mbar_arrive(half ? &bar_pb[w] : &bar_pa[w]);
                    continue;
                }
                tc_fence_after();
                const float4 *g = sc + (j & 3) * 8 + 4 * half;
                const int left = nr - (t0 + j) * kTcKeys - 64 * half;  // keys of this half that the row sees
                const bool cut = __any_sync(0xffffffffu, left < 64 || g[0].w != 0.f);  // (keys of a bad page: rare)
                // 32 scores at a time: all 64 in registers would spill, and the memory behind a spill is L2 here
                float x[32];
                auto fetch = [&](int q) {
                    tmem_ld32(tm_s + 64 * half + 32 * q, x);
                    tmem_ld_wait32(x);
                    if (cut) {
#pragma unroll
                        for (int p = 0; p < 2; p++) {
                            const bool none = g[2 * q + p].y == -INFINITY;
#pragma unroll
                            for (int e = 0; e < 16; e++)
                                if (32 * q + 16 * p + e >= left || none) x[16 * p + e] = -INFINITY;
                        }
                    }
                };
                // the largest t = s fk + lv: by runs, whose factor is not negative
                auto top = [&](int q) {
                    const float4 f = g[2 * q], f1 = g[2 * q + 1];
                    float m[4];
#pragma unroll
                    for (int h = 0; h < 4; h++) {
                        const float *y = x + 8 * h;
                        m[h] = max3(max3(y[0], y[1], y[2]), max3(y[3], y[4], y[5]), fmaxf(y[6], y[7]));
                    }
                    return fmaxf(fmaf(fmaxf(m[0], m[1]), fmaxf(cr * f.x, kMinFactor), f.y), fmaf(fmaxf(m[2], m[3]), fmaxf(cr * f1.x, kMinFactor), f1.y));
                };
                fetch(1);
                float mx = top(1);
                fetch(0);
                mx = fmaxf(mx, top(0)) - kTcOff;
                // follow the maximum only by jumps: most tiles leave M and O as they are, and the two
                // threads of a row need not tell each other more than that
                if (named_bar_any(pair, 64, mx > M + kTcSlack || (M == -INFINITY && mx > M))) {
                    if (half) crow[lane] = mx;
                    named_bar_sync(pair, 64);
                    if (!half) crow[lane] = mx = fmaxf(mx, crow[lane]);
                    named_bar_sync(pair, 64);
                    if (half) mx = crow[lane];
                    const float mn = fmaxf(M, mx), al = mn == -INFINITY ? 1.f : ex2(M - mn);
                    M = mn;
                    l *= al;
                    if (j > 0) {
#pragma unroll
                        for (int i = 0; i < HD / 32; i++) {
                            const uint32_t at = tm_o + half * (HD / 2) + 16 * i;
                            uint32_t u[16];
                            tmem_ld16(at, u);
                            tmem_ld_wait(u);
#pragma unroll
                            for (int e = 0; e < 16; e++) u[e] = __float_as_uint(__uint_as_float(u[e]) * al);
                            tmem_st16(at, u);
                        }
                    }
                }
                const float base = M == -INFINITY ? 0.f : M;
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    if (q == 1) fetch(1);
                    uint32_t u[16];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const float4 f = g[2 * q + h];
                        const float fk = fmaxf(cr * f.x, kMinFactor), add = f.y - base;
                        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const float2 y = fma2(make_float2(x[16 * h + e], x[16 * h + e + 1]), make_float2(fk, fk), make_float2(add, add));
                            const float2 pr = make_float2(ex2(y.x), ex2(y.y));
                            sum = add2(sum, pr);
                            u[8 * h + e / 2] = pack_f16(pr.x, pr.y);
                        }
                        l = fmaf(sum.x + sum.y, f.z, l);
                    }
                    tmem_st16(tm_s + 64 * half + 16 * q, u);  // (below the scores that are still to be fetched)
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(half ? &bar_pb[w] : &bar_pa[w]);
            }
            // ── output ──
            bool ok = true;
            if (nt > 0) ok = attn_wait(&bar_o[w], 0, abort_flag);
            tc_fence_after();
            if (!ok && status) atomicOr(status, DFB_STAT_TIMEOUT);
            // (the query tile is free: its last reader was the last score MMA)
            float *lx = reinterpret_cast<float *>(sm + L::q_off + w * L::q) + (warp & 3) * 64;
            if (nt == 0) named_bar_sync(pair, 64);
            lx[half * 32 + lane] = l;
            named_bar_sync(pair, 64);
            l += lx[(1 - half) * 32 + lane];
            const float inv = l > 0.f ? 1.f / l : 0.f, lw = l > 0.f ? M + log2f(l) : -INFINITY;
            const int own = wrow + lane;  // this thread's packed row
            if (half == 0 && own < n_packed) {
                const size_t row = (size_t)(sq.r0 + own / rep) * a.n_q + kvh * rep + own % rep;
                if (parts.o) parts.w[(size_t)split * a.n_rows * a.n_q + row] = lw;
                else if (a.lse) a.lse[row] = lw * kLn2;
            }
            named_bar_sync(9 + w, 256);  // every lx is read
            // through shared memory, so that rows leave as whole 16-byte columns of consecutive lanes: each
            // warp has half of the dimensions of its rows, in passes of HD bytes
            uint8_t *stage = sm + L::q_off + w * L::q + ((warp & 3) * 2 + half) * 32 * HD;
            auto put = [&](auto zero, int pass) {  // zero's type: of the stored elements
                using E = decltype(zero);
                constexpr int PER = 16 / sizeof(E), N = HD / sizeof(E), CPR = HD / 16;  // elements of a column and of a pass, columns of a row
                const int d0 = half * (HD / 2) + pass * N;
#pragma unroll
                for (int i = 0; i < N / 16; i++) {
                    float o[16] = {};
                    if (nt > 0) {
                        uint32_t u[16];
                        tmem_ld16(tm_o + d0 + 16 * i, u);
                        tmem_ld_wait(u);
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] = __uint_as_float(u[e]);
                    }
#pragma unroll
                    for (int h = 0; h < 16 / PER; h++) {
                        E t[PER];
#pragma unroll
                        for (int e = 0; e < PER; e++) t[e] = from_f32<E>(l > 0.f ? o[PER * h + e] * inv : 0.f);
                        const int ch = i * (16 / PER) + h;
                        *reinterpret_cast<uint4 *>(stage + lane * HD + ((ch ^ (lane & (CPR - 1))) << 4)) = *reinterpret_cast<const uint4 *>(t);
                    }
                }
                __syncwarp();
                const int ch = lane % CPR;
                auto dst = [&](int r) {  // of packed row r
                    const int t = r / rep, tok = sq.r0 + t, head = kvh * rep + r - t * rep;
                    E *d = sizeof(E) == 4 ? reinterpret_cast<E *>(parts.o) + ((size_t)split * a.n_rows * a.n_q + (size_t)tok * a.n_q + head) * HD
                                          : reinterpret_cast<E *>(a.out) + tok * a.out_tok + head * a.out_head;
                    return d + d0 + ch * PER;
                };
                uint4 u[CPR];
#pragma unroll
                for (int i = 0; i < CPR; i++) {
                    const int r = i * (32 / CPR) + lane / CPR;
                    u[i] = *reinterpret_cast<const uint4 *>(stage + r * HD + ((ch ^ (r & (CPR - 1))) << 4));
                }
#pragma unroll
                for (int i = 0; i < CPR; i++) {
                    const int r = wrow + i * (32 / CPR) + lane / CPR;
                    if (r >= n_packed) break;
                    if (sizeof(E) == 4 || vec) *reinterpret_cast<uint4 *>(dst(r)) = u[i];
                    else
#pragma unroll
                        for (int e = 0; e < PER; e++) dst(r)[e] = reinterpret_cast<const E *>(&u[i])[e];
                }
                __syncwarp();
            };
            if (wrow < n_packed) {
                if (parts.o) {
                    put(0.f, 0);
                    put(0.f, 1);
                } else {
                    put(T(0.f), 0);
                }
            }
            tc_fence_before();
        }
    } else {
        if (warp < 20) {
            // ── converters ──
            const int cw = warp - 16;
            for (int n = 0; n < 2 * nt; n++) {
                const int rs = n % kTcRaw, cs = n % kTcSlots, j = n >> 1;
                if (!attn_wait(&raw_full[rs], (n / kTcRaw) & 1, abort_flag)) break;
                // V(j) and K(j + 1) are freed together, by event j + 1 (K(0) by event 0); events alternate
                // between two barriers, and the issuer is never two events ahead of this wait
                const int ev = (n - kTcSlots + 1) >> 1;
                if (n >= kTcSlots && !attn_wait(&freed[ev & 1], (ev >> 1) & 1, abort_flag)) break;
                const uint8_t *src = sm + L::raw_off + rs * L::raw;
                uint8_t *dst = sm + L::slot_off + cs * L::slot;
                const float4 *g = sc + (j & 3) * 8;
                const int left = kend - (t0 + j) * kTcKeys;
                const bool is_v = n & 1;
                // eight lanes of a shared-memory phase take four 16-byte columns of two rows whose swizzles
                // do not meet, for the loads and for the stores
                const int c0 = lane & 3, pr = lane >> 3, sel = (lane >> 2) & 1;
                const int row8 = HD == 128 ? pr ^ (sel * 5) : 2 * pr + sel;
                constexpr int IT = HD / 16;  // 16-byte pieces per thread
                uint4 v[IT];
#pragma unroll
                for (int it = 0; it < IT; it++) {
                    const int o8 = HD == 128 ? cw + 4 * (it >> 1) : cw + 4 * it, hc = HD == 128 ? it & 1 : 0;
                    const int r = o8 * 8 + row8;
                    const int ch = HD == 128 ? (c0 + 4 * hc) ^ (r & 7) : c0 ^ ((r >> 1) & 3);
                    v[it] = *reinterpret_cast<const uint4 *>(src + r * HD + 16 * ch);
                    // codes of absent keys are not numbers to be multiplied by a weight of 0
                    if (is_v && (r >= left || g[r >> 4].y == -INFINITY)) v[it] = make_uint4(0, 0, 0, 0);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&raw_empty[rs]);
#pragma unroll
                for (int it = 0; it < IT; it++) {
                    const int o8 = HD == 128 ? cw + 4 * (it >> 1) : cw + 4 * it, hc = HD == 128 ? it & 1 : 0;
                    const int r = o8 * 8 + row8;
                    uint8_t *d = dst + hc * 16384 + r * 128;
                    uint4 lo, hi;
                    lo.x = e4m3x2_f16x2(v[it].x, 0); lo.y = e4m3x2_f16x2(v[it].x, 1);
                    lo.z = e4m3x2_f16x2(v[it].y, 0); lo.w = e4m3x2_f16x2(v[it].y, 1);
                    hi.x = e4m3x2_f16x2(v[it].z, 0); hi.y = e4m3x2_f16x2(v[it].z, 1);
                    hi.z = e4m3x2_f16x2(v[it].w, 0); hi.w = e4m3x2_f16x2(v[it].w, 1);
                    *reinterpret_cast<uint4 *>(d + (((2 * c0) ^ (r & 7)) << 4)) = lo;
                    *reinterpret_cast<uint4 *>(d + (((2 * c0 + 1) ^ (r & 7)) << 4)) = hi;
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&conv_full[cs]);
            }
        } else if (warp == 20) {
            // ── MMA issuer ──
            if (lane == 0 && nt > 0) {
                const uint32_t id_s = idesc_f16(128, kTcKeys), id_o = idesc_f16(128, HD) | (1u << 16);  // V is MN-major
                const uint32_t base = smem_u32(sm);
                const uint64_t dq = sw128_desc(base + L::q_off), dk = sw128_desc(base + L::slot_off), dv = mn128_desc(base + L::slot_off, 16384);
                auto score = [&](int w, int n) {
                    const uint64_t da = dq + w * (L::q >> 4), db = dk + (n % kTcSlots) * (L::slot >> 4);
#pragma unroll
                    for (int k = 0; k < HD / 16; k++) {
                        const uint32_t off = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
                        mma1_f16_ss(tmem + w * 128, da + off, db + off, id_s, k > 0);
                    }
                };
                auto value = [&](int w, int n, int half, bool add) {
                    const uint64_t db = dv + (n % kTcSlots) * (L::slot >> 4);
#pragma unroll
                    for (int i = 0; i < kTcKeys / 32; i++) {
                        const int k = half * (kTcKeys / 32) + i;
                        mma1_f16_ts(tmem + 256 + w * 128, tmem + w * 128 + 64 * half + 8 * i, db + (2048 >> 4) * k, id_o, add || i > 0);
                    }
                };
                auto ready = [&](uint64_t *b, int ph) {
                    const bool ok = thread_wait(b, ph, abort_flag);
                    tc_fence_after();
                    return ok;
                };
                auto filled = [&](int n) { return ready(&conv_full[n % kTcSlots], (n / kTcSlots) & 1); };
                bool ok = ready(bar_q, 0) && filled(0);
                if (ok) {
                    score(0, 0);
                    mma1_commit(&bar_s[0]);
                    if (two) {
                        score(1, 0);
                        mma1_commit(&bar_s[1]);
                    }
                    mma1_commit(&freed[0]);
                }
                for (int j = 0; ok && j < nt; j++) {
                    const int nv = 2 * j + 1, nk = 2 * j + 2;
                    const bool more = j + 1 < nt;
                    ok = filled(nv);
                    for (int w = 0; ok && w < (two ? 2 : 1); w++) {
                        if (!(ok = ready(&bar_pa[w], j & 1))) break;
                        value(w, nv, 0, j > 0);
                        if (!(ok = ready(&bar_pb[w], j & 1))) break;
                        value(w, nv, 1, true);
                        if (!more) mma1_commit(&bar_o[w]);
                        else {
                            if (w == 0 && !(ok = filled(nk))) break;
                            score(w, nk);
                            mma1_commit(&bar_s[w]);
                        }
                    }
                    if (ok && more) mma1_commit(&freed[(j + 1) & 1]);  // (the last commit is bar_o's, which the softmax warps wait for)
                }
                if (!ok) {  // let what was issued end before TMEM is freed
                    mma1_commit(bar_drain);
                    spin_bounded(bar_drain, 0);
                }
            }
            __syncwarp();
        } else if (warp == 21) {
            // ── loader ──
            const int box = min(c.page, kKeyTile), nb = kTcKeys / box;
            int pid = 0, issued = 0;
            float ks = 1.f, vs = 1.f;
            for (int n = 0; n < 2 * nt; n++) {
                const int rs = n % kTcRaw, j = n >> 1, b0 = (j * nb) % 32;
                if (!(n & 1) && b0 == 0) {
                    const int key = ((t0 + j) * nb + lane) * box;
                    pid = -1;
                    if (key < kend) {
                        pid = c.pages[(size_t)s * c.max_pages + key / c.page];
                        if (pid < 0 || pid >= c.n_pages) {
                            if (status) atomicOr(status, DFB_STAT_PAGE);
                            pid = -1;
                        }
                    }
                    ks = vs = 1.f;
                    if (pid >= 0) {
                        ks = c.k_scale[(size_t)pid * c.n_kv + kvh];
                        vs = c.v_scale[(size_t)pid * c.n_kv + kvh];  // (first used after the tile's copies are under way)
                    }
                }
                if (n >= kTcRaw && !attn_wait(&raw_empty[rs], (n / kTcRaw - 1) & 1, abort_flag)) break;
                uint8_t *dst = sm + L::raw_off + rs * L::raw;
                int n_ok = 0;
                for (int b = 0; b < nb; b++) {
                    const int p = __shfl_sync(0xffffffffu, pid, b0 + b);
                    if (p < 0) continue;
                    n_ok++;
                    if (lane == 0)
                        tma_load_2d(dst + b * box * HD, n & 1 ? &tm_v : &tm_k, 0, (p * c.n_kv + kvh) * c.page + (((t0 + j) * nb + b) * box) % c.page,
                                    &raw_full[rs]);
                }
                if (!(n & 1)) {
                    // (the entry's last readers, the softmax of tile j - 4, ended before K of tile j - 1 was converted)
                    const int src = b0 + (lane & 7) * 16 / box;
                    const int gp = __shfl_sync(0xffffffffu, pid, src);
                    const float gk = __shfl_sync(0xffffffffu, ks, src), gv = fmaxf(__shfl_sync(0xffffffffu, vs, src), 5.421010862427522e-20f);
                    const bool holes = __any_sync(0xffffffffu, gp < 0);
                    if (lane < 8) sc[(j & 3) * 8 + lane] = make_float4(gk, gp < 0 ? -INFINITY : log2f(gv), 1.f / gv, holes ? 1.f : 0.f);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive_expect_tx(&raw_full[rs], n_ok * box * HD);
                issued = n + 1;
            }
            if (*abort_flag)
                for (int n = max(0, issued - kTcRaw); n < issued; n++) spin_bounded(&raw_full[n % kTcRaw], (n / kTcRaw) & 1);
        }
    }
    __syncthreads();
    if (warp == 20) {
        tc_fence_after();
        tmem_dealloc1(tmem, 512);
    }
}

}  // namespace dfb
