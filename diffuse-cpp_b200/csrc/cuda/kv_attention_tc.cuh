// Attention over the paged 8-bit cache for many query rows: tcgen05 MMAs on tiles of 2 x 128 packed
// rows x 128 keys (arithmetic: kv_attention.cuh).
//
// A persistent CTA per SM (14 warps) takes work items -- a sequence, KV head, tile of 256 packed rows
// and part of the keys -- in turn:
//   warps 0-3, 4-7  softmax of row tile 0 / 1, a thread to a row (TMEM lane): scores from TMEM, p' back
//                   into their place as f16 (the A operand of P V), rare rescales of O, the output
//   warps 8-11      converters: E4M3 codes -> f16 operands in shared memory, both of K and of V as
//                   rows of 64 dimensions swizzled over 128 bytes (K-major for K, MN-major for V);
//                   an item's queries
//   warp 12         MMA issuer, warp 13 loader (one tensor copy per run of page positions)
// MMA order: S0(0) S1(0), then for each key tile j: P0 V, S0(j+1), P1 V, S1(j+1), so one row tile's
// softmax runs under the other's MMAs; S0(j+1) is complete only after P0 V(j), so a softmax thread
// that has its scores may rescale its row of O without another wait.  Tile "j + 1" of an item's last
// tile is the next item's first: loader, converters and issuer run ahead across items, and only the
// softmax warps see an item's end.  With one item per CTA, loading page ids, queries and the first
// tile took 13000 of an item's 43000 cycles (6 key tiles) and writing the output 6000.
#pragma once
#include "kv_attention.cuh"

namespace dfb {

constexpr int kTcKeys = 128;     // keys of one tile
constexpr int kTcRows = 256;     // packed rows of one CTA
constexpr int kTcThreads = 512;  // (two warps do nothing: registers are handed out to four warps at a time)
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
    static constexpr int n_bars = 2 * kTcRaw + kTcSlots + 13;
    static constexpr int crow_off = bar_off + n_bars * 8 + 32;
    static constexpr int bytes = 1024 + crow_off + 2 * kTcRows;
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

// 32 bytes to global memory in one store.
__device__ __forceinline__ void store32(void *p, const uint32_t (&u)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]),
                 "r"(u[6]), "r"(u[7])
                 : "memory");
}
// 32 bytes of elements E of one output row; align: what the row's address is a multiple of (32, 16, or the element).
template <typename E>
__device__ __forceinline__ void store_row32(E *p, int align, const uint32_t (&u)[8]) {
    if (align == 32) store32(p, u);
    else if (align == 16) {
        reinterpret_cast<uint4 *>(p)[0] = make_uint4(u[0], u[1], u[2], u[3]);
        reinterpret_cast<uint4 *>(p)[1] = make_uint4(u[4], u[5], u[6], u[7]);
    } else
#pragma unroll
        for (int e = 0; e < 32 / (int)sizeof(E); e++) p[e] = reinterpret_cast<const E *>(u)[e];
}

// One work item; every warp of the CTA works out the same.
struct TcItem {
    int s, kvh, split;
    AttnSeq sq;
    int row0, n_packed, kend, t0, nt;
    bool two;
};
struct TcGrid {
    int tiles, items;  // row tiles of a sequence (at most), work items
};
// The idx-th item; false if it has no rows.  Called by whole warps.
__device__ __forceinline__ bool tc_item(const dfb_kv_cache &c, const dfb_kv_attn &a, const AttnParts &parts, const TcGrid &grid, int rep, int idx,
                                        int32_t *status, TcItem &it) {
    const int per = grid.tiles * parts.splits, lane = threadIdx.x & 31;
    const int x = idx % per, y = idx / per;
    it.split = x % parts.splits;
    it.kvh = y % c.n_kv;
    it.s = y / c.n_kv;
    it.sq = attn_seq(c, a, it.s, x == 0 && it.kvh == 0 && threadIdx.x == 0, status);
    it.row0 = x / parts.splits * kTcRows;
    it.n_packed = it.sq.n_rows * rep;
    if (it.row0 >= it.n_packed) return false;
    it.two = it.row0 + 128 < it.n_packed;
    it.kend = it.sq.len;
    if (a.vis) {  // the most keys any of the item's tokens sees
        const int last = (min(it.row0 + kTcRows, it.n_packed) - 1) / rep;
        int n = 0;
        for (int t = it.row0 / rep + lane; t <= last; t += 32) n = max(n, a.vis[it.sq.r0 + t]);
        it.kend = min(it.kend, max(0, __reduce_max_sync(0xffffffffu, n)));
    }
    const int n = (it.kend + kTcKeys - 1) / kTcKeys;
    it.t0 = (int)((long long)n * it.split / parts.splits);
    it.nt = (int)((long long)n * (it.split + 1) / parts.splits) - it.t0;
    return true;
}

template <typename T, int HD>
__global__ void __launch_bounds__(kTcThreads, 1)
    kv_attn_tc_kernel(const dfb_kv_cache c, const dfb_kv_attn a, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const AttnParts parts, const TcGrid grid, bool vec, int out_align, int32_t *status) {
    using L = TcSmem<HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *sm = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    float4 *sc = reinterpret_cast<float4 *>(sm + L::sc_off);  // [tile & 3][8 runs of 16 keys] ks, log2 vs, 1 / vs, any absent
    uint64_t *bars = reinterpret_cast<uint64_t *>(sm + L::bar_off);
    uint64_t *raw_full = bars, *raw_empty = raw_full + kTcRaw, *conv_full = raw_empty + kTcRaw, *freed = conv_full + kTcSlots;
    uint64_t *bar_s = freed + 2, *bar_pa = bar_s + 2, *bar_pb = bar_pa + 2, *bar_o = bar_pb + 2, *bar_q = bar_o + 2, *bar_drain = bar_q + 2;
    int *shared_i = reinterpret_cast<int *>(bars + L::n_bars);  // abort flag, TMEM address
    volatile int *abort_flag = shared_i;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rep = a.n_q / c.n_kv;
    if (tid == 0) {
        shared_i[0] = 0;
        for (int i = 0; i < kTcRaw; i++) {
            mbar_init(&raw_full[i], 1);
            mbar_init(&raw_empty[i], 4);
        }
        for (int i = 0; i < kTcSlots; i++) mbar_init(&conv_full[i], 4);
        for (int i = 0; i < 2; i++) {
            mbar_init(&bar_s[i], 1);
            mbar_init(&bar_pa[i], 4);
            mbar_init(&bar_pb[i], 4);
            mbar_init(&freed[i], 1);
            mbar_init(&bar_o[i], 1);
            mbar_init(&bar_q[i], 4);
        }
        mbar_init(bar_drain, 1);
        fence_barrier_init();
    }
    if (warp == 12) tmem_alloc1(reinterpret_cast<uint32_t *>(&shared_i[1]), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = (uint32_t)shared_i[1];
    TcItem it;

    if (warp < 8) {
        // ── softmax ──
        const int w = warp >> 2;  // row tile
        const uint32_t tm_s = tmem + w * 128 + ((uint32_t)(warp & 3) << 21), tm_o = tm_s + 256;
        // exponents of the queries' scales, by the parity of the item: one is written while the other may still be read
        const int8_t *crow = reinterpret_cast<const int8_t *>(sm + L::crow_off) + w * 128 + (warp & 3) * 32 + lane;
        int odd = 0;
        uint32_t ph_s = 0, ph_o = 0;
        int g = 0;  // key tiles of the CTA so far
        bool ok = true;
        for (int idx = blockIdx.x; ok && idx < grid.items; idx += gridDim.x) {
            if (!tc_item(c, a, parts, grid, rep, idx, status, it)) continue;
            odd ^= it.nt > 0;
            if (w == 1 && !it.two) {
                g += it.nt;
                continue;
            }
            const int wrow = it.row0 + w * 128 + (warp & 3) * 32;  // the warp's first packed row
            const bool dead = wrow >= it.n_packed;  // no row of this warp exists: whatever its lanes of P hold, no one reads what comes of it
            const int R = min(wrow + lane, it.n_packed - 1), tok = it.sq.r0 + R / rep, head = it.kvh * rep + R % rep;
            int left = (a.vis ? min(max(a.vis[tok], 0), it.sq.len) : it.sq.len) - it.t0 * kTcKeys;  // keys of the tile that the row sees
            float cr = fabsf(a.scale) * kLog2e, M = -INFINITY, l = 0.f;
            for (int j = 0; j < it.nt; j++, g++, left -= kTcKeys) {
                if (!(ok = attn_wait(&bar_s[w], ph_s, abort_flag))) break;
                ph_s ^= 1;
                if (dead) {
                    if (lane == 0) {
                        mbar_arrive(&bar_pa[w]);
                        mbar_arrive(&bar_pb[w]);
                    }
                    continue;
                }
                tc_fence_after();
                if (!std::is_same<T, __half>::value && j == 0) cr *= exp2i(crow[odd * kTcRows]);
                const float4 *gs = sc + (g & 3) * 8;
                const bool cut = __any_sync(0xffffffffu, left < kTcKeys || gs[0].w != 0.f);  // (keys of a bad page: rare)
                // Scores come 32 at a time, twice (for the maximum, for the exponentials), the next 32 under way:
                // a loop that the instruction cache next to the scheduler holds beside the other roles' loops,
                // and no spills (the memory behind a spill is L2: 227 KB of shared memory are in use).
                float xa[32], xb[32];
                auto mask = [&](float (&x)[32], int q) {
                    if (cut)
#pragma unroll
                        for (int p = 0; p < 2; p++) {
                            const int n = gs[2 * q + p].y == -INFINITY ? 0 : left - 32 * q - 16 * p;
#pragma unroll
                            for (int e = 0; e < 16; e++)
                                if (e >= n) x[16 * p + e] = -INFINITY;
                        }
                };
                float mx = -INFINITY;
                // the largest t = s fk + lv: by runs, whose factor is not negative
                auto top = [&](const float (&x)[32], int q) {
#pragma unroll
                    for (int p = 0; p < 2; p++) {
                        const float4 f = gs[2 * q + p];
                        const float *y = x + 16 * p;
                        const float m0 = max3(max3(y[0], y[1], y[2]), max3(y[3], y[4], y[5]), fmaxf(y[6], y[7]));
                        const float m1 = max3(max3(y[8], y[9], y[10]), max3(y[11], y[12], y[13]), fmaxf(y[14], y[15]));
                        mx = fmaxf(mx, fmaf(fmaxf(m0, m1), fmaxf(cr * f.x, kMinFactor), f.y));
                    }
                };
                tmem_ld32(tm_s, xa);
#pragma unroll 1
                for (int q = 0; q < 4; q += 2) {
                    tmem_ld_wait32(xa);
                    tmem_ld32(tm_s + 32 * q + 32, xb);
                    mask(xa, q);
                    top(xa, q);
                    tmem_ld_wait32(xb);
                    tmem_ld32(tm_s + ((32 * q + 64) & 127), xa);  // (in the end the first ones again)
                    mask(xb, q + 1);
                    top(xb, q + 1);
                }
                mx -= kTcOff;
                // follow the maximum only by jumps: most tiles leave M and O as they are
                if (__any_sync(0xffffffffu, mx > M + kTcSlack || (M == -INFINITY && mx > M))) {
                    const float mn = fmaxf(M, mx), al = mn == -INFINITY ? 1.f : ex2(M - mn);
                    M = mn;
                    l *= al;
                    if (j > 0) {
#pragma unroll
                        for (int i = 0; i < HD / 16; i++) {
                            uint32_t u[16];
                            tmem_ld16(tm_o + 16 * i, u);
                            tmem_ld_wait(u);
#pragma unroll
                            for (int e = 0; e < 16; e++) u[e] = __float_as_uint(__uint_as_float(u[e]) * al);
                            tmem_st16(tm_o + 16 * i, u);
                        }
                    }
                }
                const float base = M == -INFINITY ? 0.f : M;
                auto exps = [&](const float (&x)[32], int q) {
                    uint32_t u[16];
#pragma unroll
                    for (int p = 0; p < 2; p++) {
                        const float4 f = gs[2 * q + p];
                        const float fk = fmaxf(cr * f.x, kMinFactor), add = f.y - base;
                        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                        for (int e = 0; e < 16; e += 2) {
                            const float2 y = fma2(make_float2(x[16 * p + e], x[16 * p + e + 1]), make_float2(fk, fk), make_float2(add, add));
                            const float2 pr = make_float2(ex2(y.x), ex2(y.y));
                            sum = add2(sum, pr);
                            u[8 * p + e / 2] = pack_f16(pr.x, pr.y);
                        }
                        l = fmaf(sum.x + sum.y, f.z, l);
                    }
                    tmem_st16(tm_s + 16 * q, u);  // (below the scores that are still to come)
                };
#pragma unroll 1
                for (int q = 0; q < 4; q += 2) {
                    tmem_ld_wait32(xa);
                    tmem_ld32(tm_s + 32 * q + 32, xb);
                    mask(xa, q);
                    exps(xa, q);
                    tmem_ld_wait32(xb);
                    if (q == 0) tmem_ld32(tm_s + 64, xa);
                    mask(xb, q + 1);
                    exps(xb, q + 1);
                    // each half of the tile's keys on its own: its P V starts under the other's exponentials
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(q ? &bar_pb[w] : &bar_pa[w]);
                }
            }
            if (!ok) break;
            // ── output ──
            if (it.nt > 0) {
                if (!(ok = attn_wait(&bar_o[w], ph_o, abort_flag))) break;
                ph_o ^= 1;
                tc_fence_after();
            }
            if (!dead) {
                const bool mine = wrow + lane < it.n_packed;
                const size_t row = (size_t)tok * a.n_q + head, part = (size_t)it.split * a.n_rows * a.n_q + row;
                const float inv = l > 0.f ? 1.f / l : 0.f;
                if (mine) {
                    const float lw = l > 0.f ? M + log2f(l) : -INFINITY;
                    if (parts.o) parts.w[part] = lw;
                    else if (a.lse) a.lse[row] = lw * kLn2;
                }
#pragma unroll
                for (int i = 0; i < HD / 16; i++) {
                    uint32_t o[16], u[8];
                    if (it.nt > 0) {
                        tmem_ld16(tm_o + 16 * i, o);
                        tmem_ld_wait(o);
                    }
                    if (!mine) continue;
                    if (parts.o) {
#pragma unroll
                        for (int h = 0; h < 2; h++) {
#pragma unroll
                            for (int e = 0; e < 8; e++) u[e] = l > 0.f ? __float_as_uint(__uint_as_float(o[8 * h + e]) * inv) : 0;
                            store_row32(parts.o + part * HD + 16 * i + 8 * h, 16, u);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 16; e++) reinterpret_cast<T *>(u)[e] = from_f32<T>(l > 0.f ? __uint_as_float(o[e]) * inv : 0.f);
                        store_row32(reinterpret_cast<T *>(a.out) + tok * a.out_tok + head * a.out_head + 16 * i, out_align, u);
                    }
                }
                tc_fence_before();
            }
        }
        if (!ok && lane == 0 && status) atomicOr(status, DFB_STAT_TIMEOUT);
    } else if (warp < 12) {
        // ── converters ──
        const int cw = warp - 8;
        int n = 0, odd = 0, seen[2] = {0, 0};  // code tiles so far, parity of the item, score phases of each row tile so far
        bool ok = true;
        for (int idx = blockIdx.x; ok && idx < grid.items; idx += gridDim.x) {
            if (!tc_item(c, a, parts, grid, rep, idx, status, it)) continue;
            odd ^= it.nt > 0;
            for (int i = 0; ok && i < 2 * it.nt; i++, n++) {
                if (i == 1) {
                    // the item's queries as f16, scaled by a power of two: a quarter of each row tile per
                    // warp, once the last scores of the item before are there
                    constexpr int LPR = HD / 8, RPI = 32 / LPR, NL = 8;  // lanes of a row (16 bytes each), rows of one load, loads in flight
                    for (int w = 0; ok && w < (it.two ? 2 : 1); w++) {
                        if (seen[w] > 0 && !(ok = attn_wait(&bar_s[w], (seen[w] - 1) & 1, abort_flag))) break;
                        seen[w] += it.nt;
                        const int ch = lane % LPR;
#pragma unroll 1
                        for (int b = 0; b < 32; b += NL * RPI) {
                            uint4 raw[NL];
                            const T *from[NL];
#pragma unroll
                            for (int i = 0; i < NL; i++) {
                                // (a row that does not exist is read as the last one: what comes of it is not stored)
                                const int r = min(it.row0 + w * 128 + cw * 32 + b + i * RPI + lane / LPR, it.n_packed - 1), t = r / rep;
                                from[i] = reinterpret_cast<const T *>(a.q) + (it.sq.r0 + t) * a.q_tok + (it.kvh * rep + r - t * rep) * a.q_head + 8 * ch;
                            }
                            if (vec) {
#pragma unroll
                                for (int i = 0; i < NL; i++) raw[i] = *reinterpret_cast<const uint4 *>(from[i]);
                            } else {
#pragma unroll
                                for (int i = 0; i < NL; i++)
#pragma unroll
                                    for (int e = 0; e < 8; e++) reinterpret_cast<T *>(&raw[i])[e] = from[i][e];
                            }
                            float up[NL];
#pragma unroll
                            for (int i = 0; i < NL; i++) up[i] = 1.f;
                            if constexpr (!std::is_same<T, __half>::value) {
                                float mx[NL];
#pragma unroll
                                for (int i = 0; i < NL; i++) {
                                    mx[i] = 0.f;
#pragma unroll
                                    for (int e = 0; e < 8; e++) mx[i] = fmaxf(mx[i], fabsf(to_f32<T>(reinterpret_cast<const T *>(&raw[i])[e])));
                                }
#pragma unroll
                                for (int o = 1; o < LPR; o <<= 1)
#pragma unroll
                                    for (int i = 0; i < NL; i++) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], o));
#pragma unroll
                                for (int i = 0; i < NL; i++) {
                                    const int e = (int)(__float_as_uint(mx[i]) >> 23) - 127;
                                    const int eu = mx[i] > 0.f && mx[i] < INFINITY ? min(max(-e, -126), 60) : 0;
                                    up[i] = exp2i(eu);
                                    if (ch == 0) reinterpret_cast<int8_t *>(sm + L::crow_off)[odd * kTcRows + w * 128 + cw * 32 + b + i * RPI + lane / LPR] = (int8_t)-eu;
                                }
                            }
#pragma unroll
                            for (int i = 0; i < NL; i++) {
                                float x[8];
                                const int rt = cw * 32 + b + i * RPI + lane / LPR;
                                const float f = a.scale < 0.f ? -up[i] : up[i];  // a negative scale turns q's sign: the scores' factors stay positive
#pragma unroll
                                for (int e = 0; e < 8; e++) x[e] = to_f32<T>(reinterpret_cast<const T *>(&raw[i])[e]) * f;
                                uint4 u;
                                u.x = pack_f16(x[0], x[1]); u.y = pack_f16(x[2], x[3]);
                                u.z = pack_f16(x[4], x[5]); u.w = pack_f16(x[6], x[7]);
                                *reinterpret_cast<uint4 *>(sm + L::q_off + w * L::q + (ch / 8) * 16384 + rt * 128 + (((ch & 7) ^ (rt & 7)) << 4)) = u;
                            }
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bar_q[w]);
                    }
                    if (!ok) break;
                }
                const int rs = n % kTcRaw, cs = n % kTcSlots, g = n >> 1;
                if (!(ok = attn_wait(&raw_full[rs], (n / kTcRaw) & 1, abort_flag))) break;
                // V(g) and K(g + 1) are freed together, by event g + 1 (K(0) by event 0); events alternate
                // between two barriers, and the issuer is never two events ahead of this wait
                const int ev = (n - kTcSlots + 1) >> 1;
                if (n >= kTcSlots && !(ok = attn_wait(&freed[ev & 1], (ev >> 1) & 1, abort_flag))) break;
                const uint8_t *src = sm + L::raw_off + rs * L::raw;
                uint8_t *dst = sm + L::slot_off + cs * L::slot;
                const float4 *gs = sc + (g & 3) * 8;
                const int left = it.kend - (it.t0 + (i >> 1)) * kTcKeys;
                const bool edge = (i & 1) && (left < kTcKeys || gs[0].w != 0.f);
                // eight lanes of a shared-memory phase take four 16-byte columns of two rows whose swizzles
                // do not meet, for the loads and for the stores
                const int c0 = lane & 3, pr = lane >> 3, sel = (lane >> 2) & 1;
                const int row8 = HD == 128 ? pr ^ (sel * 5) : 2 * pr + sel;
                constexpr int IT = HD / 16;  // 16-byte pieces per thread, four at a time
#pragma unroll 1
                for (int k0 = 0; k0 < IT; k0 += 4) {
                    uint4 v[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int k = k0 + i, r = (HD == 128 ? cw + 4 * (k >> 1) : cw + 4 * k) * 8 + row8;
                        const int ch = HD == 128 ? (c0 + 4 * (k & 1)) ^ (r & 7) : c0 ^ ((r >> 1) & 3);
                        v[i] = *reinterpret_cast<const uint4 *>(src + r * HD + 16 * ch);
                        // codes of absent keys are not numbers to be multiplied by a weight of 0
                        if (edge && (r >= left || gs[r >> 4].y == -INFINITY)) v[i] = make_uint4(0, 0, 0, 0);
                    }
                    if (k0 + 4 == IT) {
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&raw_empty[rs]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int k = k0 + i, r = (HD == 128 ? cw + 4 * (k >> 1) : cw + 4 * k) * 8 + row8;
                        uint8_t *d = dst + (HD == 128 ? (k & 1) * 16384 : 0) + r * 128;
                        uint4 lo, hi;
                        lo.x = e4m3x2_f16x2(v[i].x, 0); lo.y = e4m3x2_f16x2(v[i].x, 1);
                        lo.z = e4m3x2_f16x2(v[i].y, 0); lo.w = e4m3x2_f16x2(v[i].y, 1);
                        hi.x = e4m3x2_f16x2(v[i].z, 0); hi.y = e4m3x2_f16x2(v[i].z, 1);
                        hi.z = e4m3x2_f16x2(v[i].w, 0); hi.w = e4m3x2_f16x2(v[i].w, 1);
                        *reinterpret_cast<uint4 *>(d + (((2 * c0) ^ (r & 7)) << 4)) = lo;
                        *reinterpret_cast<uint4 *>(d + (((2 * c0 + 1) ^ (r & 7)) << 4)) = hi;
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&conv_full[cs]);
            }
        }
    } else if (warp == 12) {
        // ── MMA issuer ──
        const uint32_t id_s = idesc_f16(128, kTcKeys), id_o = idesc_f16(128, HD) | (1u << 16);  // V is MN-major
        const uint32_t base = smem_u32(sm);
        const uint64_t dq = sw128_desc(base + L::q_off), dk = sw128_desc(base + L::slot_off), dv = mn128_desc(base + L::slot_off, 16384);
        // Every instruction of the issuing thread beside an MMA costs about ten cycles (its scheduler has
        // five busy warps): the loop over an item's tiles holds nothing but waits, MMAs and commits.
        bool ok = true;
        auto ready = [&](uint64_t *b, uint32_t ph) {
            ok = ok && thread_wait(b, ph, abort_flag);
            tc_fence_after();
        };
        auto value_of = [&](int g) { return dv + (g & 1 ? 3 : 1) * (L::slot >> 4); };  // V(g) is in slot (2 g + 1) % 4
        auto key_of = [&](int g) { return dk + (g & 1 ? 2 : 0) * (L::slot >> 4); };    // K(g) in slot 2 g % 4
        auto wait_value = [&](int g) { ready(&conv_full[g & 1 ? 3 : 1], (g >> 1) & 1); };
        auto wait_key = [&](int g) { ready(&conv_full[g & 1 ? 2 : 0], (g >> 1) & 1); };
        static_assert(kTcSlots == 4, "slots of K and V");
        uint32_t ph_p[2] = {0, 0}, ph_q[2] = {0, 0};
        auto value = [&](int w, uint64_t d, bool first) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                ready(half ? &bar_pb[w] : &bar_pa[w], ph_p[w]);
                if (!ok) return;
#pragma unroll
                for (int i = 0; i < kTcKeys / 32; i++)
                    mma1_f16_ts(tmem + 256 + w * 128, tmem + w * 128 + 32 * half + 8 * i, d + (2048 >> 4) * (4 * half + i), id_o, !(first && half == 0 && i == 0));
            }
            ph_p[w] ^= 1;
        };
        auto score = [&](int w, uint64_t d) {
            if (!ok) return;
#pragma unroll
            for (int k = 0; k < HD / 16; k++) {
                const uint32_t off = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
                mma1_f16_ss(tmem + w * 128, dq + w * (L::q >> 4) + off, d + off, id_s, k > 0);
            }
            mma1_commit(&bar_s[w]);
        };
        auto queries = [&](int w) {
            ready(&bar_q[w], ph_q[w]);
            ph_q[w] ^= 1;
        };
        int idx = (int)blockIdx.x - (int)gridDim.x, g = 0;
        auto next = [&] {  // the next item with keys (all lanes)
            do idx += gridDim.x;
            while (idx < grid.items && !(tc_item(c, a, parts, grid, rep, idx, status, it) && it.nt > 0));
            return idx < grid.items;
        };
        bool have = next();
        if (have && lane == 0) {
            wait_key(0);
            queries(0);
            score(0, key_of(0));
            if (it.two) {
                queries(1);
                score(1, key_of(0));
            }
            if (ok) mma1_commit(&freed[0]);
        }
        while (have) {
            const int nt = it.nt;
            const bool two = it.two;
            have = next();
            if (lane == 0 && ok) {
                for (int t = 0; t + 1 < nt && ok; t++, g++) {
                    const uint64_t d = value_of(g), dn = key_of(g + 1);
                    wait_value(g);
                    value(0, d, t == 0);
                    wait_key(g + 1);
                    score(0, dn);
                    if (two) {
                        value(1, d, t == 0);
                        score(1, dn);
                    }
                    if (ok) mma1_commit(&freed[(g + 1) & 1]);
                }
                const uint64_t d = value_of(g), dn = key_of(g + 1);  // the item's last tile, the next one's first
                wait_value(g);
                value(0, d, nt == 1);
                if (ok) mma1_commit(&bar_o[0]);
                if (have) {
                    wait_key(g + 1);
                    queries(0);
                    score(0, dn);
                }
                if (two) {
                    value(1, d, nt == 1);
                    if (ok) mma1_commit(&bar_o[1]);
                }
                if (have) {
                    if (it.two) {
                        queries(1);
                        score(1, dn);
                    }
                    if (ok) mma1_commit(&freed[(g + 1) & 1]);  // (the CTA's last commits are bar_o's, which the softmax warps wait for)
                }
                g++;
            }
            if (!__shfl_sync(0xffffffffu, ok, 0)) break;
        }
        if (!ok && lane == 0) {  // let what was issued end before TMEM is freed
            mma1_commit(bar_drain);
            spin_bounded(bar_drain, 0);
        }
        __syncwarp();
    } else if (warp == 13) {
        // ── loader ──
        const int box = min(c.page, kKeyTile), sh_box = __ffs(box) - 1, nb = kTcKeys >> sh_box, sh_page = __ffs(c.page) - 1;
        int n = 0;
        bool ok = true;
        for (int idx = blockIdx.x; ok && idx < grid.items; idx += gridDim.x) {
            if (!tc_item(c, a, parts, grid, rep, idx, status, it)) continue;
            int pid = 0;
            float ks = 1.f, vs = 1.f;
            for (int i = 0; i < 2 * it.nt; i++, n++) {
                const int rs = n % kTcRaw, j = i >> 1, b0 = (j * nb) & 31, g = n >> 1;
                if (!(i & 1) && b0 == 0) {
                    const int key = ((it.t0 + j) * nb + lane) << sh_box;
                    pid = -1;
                    if (key < it.kend) {
                        pid = c.pages[(size_t)it.s * c.max_pages + (key >> sh_page)];
                        if (pid < 0 || pid >= c.n_pages) {
                            if (status) atomicOr(status, DFB_STAT_PAGE);
                            pid = -1;
                        }
                    }
                    ks = vs = 1.f;
                    if (pid >= 0) {
                        ks = c.k_scale[(size_t)pid * c.n_kv + it.kvh];
                        vs = c.v_scale[(size_t)pid * c.n_kv + it.kvh];  // (first used after the tile's copies are under way)
                    }
                }
                if (n >= kTcRaw && !(ok = attn_wait(&raw_empty[rs], (n / kTcRaw - 1) & 1, abort_flag))) break;
                uint8_t *dst = sm + L::raw_off + rs * L::raw;
                int n_ok = 0;
                for (int b = 0; b < nb; b++) {
                    const int p = __shfl_sync(0xffffffffu, pid, b0 + b);
                    if (p < 0) continue;
                    n_ok++;
                    if (lane == 0)
                        tma_load_2d(dst + b * box * HD, i & 1 ? &tm_v : &tm_k, 0,
                                    ((p * c.n_kv + it.kvh) << sh_page) + ((((it.t0 + j) * nb + b) << sh_box) & (c.page - 1)), &raw_full[rs]);
                }
                if (!(i & 1)) {
                    // (the entry's last readers, the softmax of tile g - 4, ended before K of tile g - 1 was converted)
                    const int src = b0 + ((lane & 7) * 16 >> sh_box);
                    const int gp = __shfl_sync(0xffffffffu, pid, src);
                    const float gk = __shfl_sync(0xffffffffu, ks, src), gv = fmaxf(__shfl_sync(0xffffffffu, vs, src), 5.421010862427522e-20f);
                    const bool holes = __any_sync(0xffffffffu, gp < 0);
                    if (lane < 8) sc[(g & 3) * 8 + lane] = make_float4(gk, gp < 0 ? -INFINITY : log2f(gv), 1.f / gv, holes ? 1.f : 0.f);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive_expect_tx(&raw_full[rs], n_ok * box * HD);
            }
        }
        if (*abort_flag)  // let the copies in flight land before the block goes
            for (int i = max(0, n - kTcRaw); i < n; i++) spin_bounded(&raw_full[i % kTcRaw], (i / kTcRaw) & 1);
    }
    __syncthreads();
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc1(tmem, 512);
    }
}

}  // namespace dfb
