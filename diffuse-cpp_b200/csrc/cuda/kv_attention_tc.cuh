// Attention over the paged 8-bit cache for many query rows: tcgen05 MMAs on tiles of 2 x 128 packed
// rows x 128 keys (arithmetic: kv_attention.cuh).
//
// A persistent CTA per SM (24 warps) takes work items -- a sequence, KV head, tile of 256 packed rows
// and part of the keys -- in turn:
//   warps 0-7, 8-15 softmax of row tile 0 / 1, two threads to a row (TMEM lane), 64 keys each: scores
//                   from TMEM, p' back into their place as f16 (the A operand of P V), rare rescales
//                   of O, the output
//   warps 16-19     converters: E4M3 codes -> f16 operands in shared memory, both of K and of V as
//                   rows of 64 dimensions swizzled over 128 bytes (K-major for K, MN-major for V);
//                   an item's queries
//   warp 20         MMA issuer
//   warp 21         loader (one tensor copy per run of page positions); works the items out for all
//   warp 22         the rows of items without a key
// MMA order: S0(0) S1(0), then for each key tile j: P0 V, S0(j+1), P1 V, S1(j+1), so one row tile's
// softmax runs under the other's MMAs; S0(j+1) is complete only after P0 V(j), so a softmax thread
// that has its scores may rescale its row of O without another wait.  Tile "j + 1" of an item's last
// tile is the next item's first: loader, converters and issuer run ahead across items, and only the
// softmax warps see an item's end.  With one item per CTA, loading page ids, queries and the first
// tile took 13000 of an item's 43000 cycles (6 key tiles) and writing the output 6000.
//
// Bound: the softmax warps' issue slots (2.7 us for the exponentials, maxima and sums of a key tile's
// 256 x 128 scores; the MMAs and hand-overs alone need 1.9), then an item's queries and output (6 us).
// hd 128: 64 sequences of 256 rows x 32 heads over 768 keys 315 to 337 us (655 to 612 TFLOP/s), 32 rows of
// 28 / 4 heads over 131072 keys, split in 37 parts, 97 us (620 TFLOP/s).
#pragma once
#include "kv_attention.cuh"

namespace dfb {

constexpr int kTcKeys = 128;     // keys of one tile
constexpr int kTcRows = 256;     // packed rows of one CTA
constexpr int kTcThreads = 768;  // 80 registers each (one warp does nothing: registers go to four warps at a time)
// Raw slots (128 x HD codes of K or V) and f16 slots, K and V of successive tiles in turn.  Two tiles of
// codes in flight hide memory's latency (with one, 64 x 256 x 768 took 276 us without any softmax);
// the f16 slots hold what an MMA may read and one more.
constexpr int kTcRaw = 4, kTcSlots = 3;
constexpr float kTcOff = 7.f, kTcSlack = 8.f;  // p' <= 2^(off + slack) = 2^15 although the maximum is only followed by jumps

// One work item with keys, as the loader describes it in shared memory; nt < 0: there are no more.
struct TcItem {
    int s, kvh, split, r0, len, row0, n_packed, kend, t0, nt;
};
constexpr int kTcItems = 4;       // entries
constexpr int kTcItemUsers = 21;  // warps that read them

template <int HD>
struct TcSmem {
    static constexpr int q = 128 * HD * 2;         // one row tile's queries
    static constexpr int slot = kTcKeys * HD * 2;
    static constexpr int raw = kTcKeys * HD;
    static constexpr int q_off = 0, slot_off = 2 * q, raw_off = slot_off + kTcSlots * slot, sc_off = raw_off + kTcRaw * raw;
    static constexpr int bar_off = sc_off + 4 * 8 * 16;
    static constexpr int n_bars = 2 * kTcRaw + kTcSlots + 15 + 2 * kTcItems;
    static constexpr int item_off = bar_off + n_bars * 8 + 16;
    static constexpr int crow_off = item_off + kTcItems * (int)sizeof(TcItem);
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
// D (+)= A B^T with A from shared memory / from TMEM; D, A: TMEM columns.  A kernel that takes all 512
// columns has them from address 0 on, so they are constants here: operands that the compiler can
// keep in uniform registers issue without a move per operand.
template <int D, bool ADD>
__device__ __forceinline__ void mma1_f16_ss(uint64_t a, uint64_t b, uint32_t idesc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(D), "l"(a), "l"(b),
                 "r"(idesc), "n"((int)ADD)
                 : "memory");
}
template <int D, int A>
__device__ __forceinline__ void mma1_f16_ts(uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(D), "r"(A), "l"(b),
                 "r"(idesc), "r"((int)add)
                 : "memory");
}
template <int I>
using Int = std::integral_constant<int, I>;
// f(Int<0>), ..., f(Int<N - 1>)
template <int N, int I = 0, typename F>
__device__ __forceinline__ void unrolled(F &&f) {
    if constexpr (I < N) {
        f(Int<I>());
        unrolled<N, I + 1>(f);
    }
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
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
__device__ __forceinline__ void tmem_st1(uint32_t taddr, float v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(__float_as_uint(v)) : "memory");
}
__device__ __forceinline__ float tmem_ld1(uint32_t taddr) {
    uint32_t v;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;" : "=r"(v) : "r"(taddr) : "memory");
    return __uint_as_float(v);
}
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
// The factor of a score is kept above 0, so that a masked score of -inf stays -inf where the softmax
// scale is 0 or the product of the scales underflows; every score times this is 0 beside an exponent.
constexpr float kMinFactor = 1.1754944e-38f;
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

// One arrival on the mbarrier once this thread's cp.async so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
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

struct TcGrid {
    int tiles, items;  // row tiles of a sequence (at most), work items
};
// The idx-th item; false if it has no rows.  Called by a whole warp.
__device__ __forceinline__ bool tc_item(const dfb_kv_cache &c, const dfb_kv_attn &a, const AttnParts &parts, const TcGrid &grid, int rep, int idx,
                                        int32_t *status, TcItem &it) {
    const int per = grid.tiles * parts.splits, lane = threadIdx.x & 31;
    const int x = idx % per, y = idx / per;
    it.split = x % parts.splits;
    it.kvh = y % c.n_kv;
    it.s = y / c.n_kv;
    const AttnSeq sq = attn_seq(c, a, it.s, x == 0 && it.kvh == 0 && lane == 0, status);
    it.r0 = sq.r0;
    it.len = it.kend = sq.len;
    it.row0 = x / parts.splits * kTcRows;
    it.n_packed = sq.n_rows * rep;
    if (it.row0 >= it.n_packed) return false;
    if (a.vis) {  // the most keys any of the item's tokens sees
        const int last = (min(it.row0 + kTcRows, it.n_packed) - 1) / rep;
        int n = 0;
        for (int t = it.row0 / rep + lane; t <= last; t += 32) n = max(n, a.vis[it.r0 + t]);
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
    uint64_t *bar_s = freed + 2, *bar_pa = bar_s + 2, *bar_pb = bar_pa + 2, *bar_o = bar_pb + 2, *bar_q = bar_o + 2, *bar_raw_q = bar_q + 2, *item_full = bar_raw_q + 2,
             *item_empty = item_full + kTcItems, *bar_drain = item_empty + kTcItems;
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
            mbar_init(&bar_q[i], 8);
            mbar_init(&bar_raw_q[i], 128);
        }
        for (int i = 0; i < kTcItems; i++) {
            mbar_init(&item_full[i], 1);
            mbar_init(&item_empty[i], kTcItemUsers);
        }
        mbar_init(bar_drain, 1);
        fence_barrier_init();
    }
    if (warp == 20) tmem_alloc1(reinterpret_cast<uint32_t *>(&shared_i[1]), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = 0;  // (all 512 columns are this CTA's)
    const volatile TcItem *items = reinterpret_cast<const volatile TcItem *>(sm + L::item_off);

    if (warp < 16) {
        // ── softmax ──
        const int w = warp >> 3, half = (warp >> 2) & 1;  // row tile, half of its keys
        const int pair = 1 + w * 4 + (warp & 3);          // barrier of the two warps that share 32 rows
        const uint32_t tm_s = tmem + w * 128 + 64 * half + ((uint32_t)(warp & 3) << 21);  // this half's scores; 64 ^: the other's
        const uint32_t tm_o = tmem + 256 + w * 128 + half * (HD / 2) + ((uint32_t)(warp & 3) << 21);  // this half of the dimensions
        const int in_tile = w * 128 + (warp & 3) * 32;  // the warp's first row in the item
        uint32_t ph_s = 0, ph_o = 0, ph_q = 0;
        int g = 0;  // key tiles of the CTA so far
        bool ok = true;
        // Half of the warp's 32 query rows of item k as f16 operands.  bf16 rows whose largest value f16
        // holds with room to spare above and below are converted as they are (what f16's subnormals then cut
        // off is below 2^-21 of it), others are scaled to [1, 2) first; a negative softmax scale turns q's
        // sign: the scores' factors stay positive.
        auto queries = [&](int k) {
            const volatile TcItem *it = items + (k & (kTcItems - 1));
            if (!(ok = attn_wait(&item_full[k & (kTcItems - 1)], (k / kTcItems) & 1, abort_flag))) return;
            if (it->nt < 0 || (w == 1 && it->row0 + 128 >= it->n_packed)) return;
            if (!(ok = attn_wait(&bar_raw_q[w], ph_q, abort_flag))) return;
            ph_q ^= 1;
            constexpr int LPR = HD / 8, RPI = 32 / LPR;  // lanes of a row (16 bytes each), rows of one round
            const int ch = lane % LPR;
            if ((!std::is_same<T, __half>::value || a.scale < 0.f) && it->row0 + in_tile < it->n_packed) {
#pragma unroll 2
                for (int x = 0; x < 16 / RPI; x++) {
                    const int rt = (warp & 3) * 32 + half * 16 + x * RPI + lane / LPR;
                    uint4 *at = reinterpret_cast<uint4 *>(sm + L::q_off + w * L::q + (ch / 8) * 16384 + rt * 128 + (((ch ^ rt) & 7) << 4));
                    uint4 u = *at;
                    if constexpr (!std::is_same<T, __half>::value) {
                        const __nv_bfloat162 *h = reinterpret_cast<const __nv_bfloat162 *>(&u);
                        const __nv_bfloat162 m = __hmax2(__hmax2(__habs2(h[0]), __habs2(h[1])), __hmax2(__habs2(h[2]), __habs2(h[3])));
                        const uint32_t mb = *reinterpret_cast<const uint32_t *>(&m);
                        uint32_t mx = max(mb & 0xffffu, mb >> 16);  // bits of a magnitude: ordered like the magnitudes
                        int eu = 0;
                        // all rows of the round within [2^-3, 2^14): no lane above, one lane of each row above the lower end
                        const uint32_t above = __ballot_sync(0xffffffffu, mx >= (124u << 7));
                        bool plain = !__any_sync(0xffffffffu, mx >= (141u << 7));
#pragma unroll
                        for (int r = 0; r < RPI; r++) plain = plain && (above >> (r * LPR) & ((1u << LPR) - 1)) != 0;
                        if (!plain) {
#pragma unroll
                            for (int o = 1; o < LPR; o <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                            const int e = (int)(mx >> 7) - 127;  // (128: inf or NaN)
                            eu = mx != 0 && e < 128 && (e < -3 || e > 13) ? min(max(-e, -126), 60) : 0;
                        }
                        if (ch == 0) reinterpret_cast<int8_t *>(sm + L::crow_off)[(k & 1) * kTcRows + w * 128 + rt] = (int8_t)-eu;
                        const uint32_t v[4] = {u.x, u.y, u.z, u.w};
                        uint32_t o[4];
                        const float f = exp2i(eu);
#pragma unroll
                        for (int p = 0; p < 4; p++) {
                            float lo = __uint_as_float(v[p] << 16), hi = __uint_as_float(v[p] & 0xffff0000u);
                            if (!plain) {
                                lo *= f;
                                hi *= f;
                            }
                            o[p] = pack_f16(lo, hi);
                        }
                        u = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                    if (a.scale < 0.f) { u.x ^= 0x80008000u; u.y ^= 0x80008000u; u.z ^= 0x80008000u; u.w ^= 0x80008000u; }
                    *at = u;
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&bar_q[w]);
        };
        queries(0);
        for (int k = 0; ok; k++) {
            const volatile TcItem *it = items + (k & (kTcItems - 1));  // (published: queries(k) has waited)
            const int nt = it->nt;
            if (nt < 0) break;
            if (w == 1 && it->row0 + 128 >= it->n_packed) {  // no row tile 1
                g += nt;
                queries(k + 1);
            } else {
                const bool dead = it->row0 + in_tile >= it->n_packed;  // no row of this warp exists: no one reads what comes of its lanes
                float cr = fabsf(a.scale) * kLog2e, M = -INFINITY, l = 0.f;
                int left;  // keys of this half of the tile that the row sees
                {
                    const int len = it->len;
                    left = len;
                    if (a.vis) left = min(max(a.vis[it->r0 + min(it->row0 + in_tile + lane, it->n_packed - 1) / rep], 0), len);
                    left -= it->t0 * kTcKeys + 64 * half;
                }
                for (int j = 0; j < nt; j++, g++, left -= kTcKeys) {
                    if (!(ok = attn_wait(&bar_s[w], ph_s, abort_flag))) break;
                    ph_s ^= 1;
                    if (dead) {
                        if (lane == 0) mbar_arrive(half ? &bar_pb[w] : &bar_pa[w]);
                        continue;
                    }
                    tc_fence_after();
                    // exponents of the queries' scales, by the parity of the item: one is written while the other may still be read
                    if (!std::is_same<T, __half>::value && j == 0)
                        cr *= exp2i(reinterpret_cast<const int8_t *>(sm + L::crow_off)[(k & 1) * kTcRows + in_tile + lane]);
                    const float4 *gs = sc + (g & 3) * 8 + 4 * half;
                    const bool cut = __any_sync(0xffffffffu, left < 64 || gs[0].w != 0.f);  // (keys of a bad page: rare)
                    // 32 scores at a time: 64 would spill, and the memory behind a spill is L2 (227 KB of shared
                    // memory are in use)
                    float x[32];
                    auto fetch = [&](int q) {
                        tmem_ld32(tm_s + 32 * q, x);
                        tmem_ld_wait32(x);
                        if (cut)
#pragma unroll
                            for (int p = 0; p < 2; p++) {
                                const int n = gs[2 * q + p].y == -INFINITY ? 0 : left - 32 * q - 16 * p;
#pragma unroll
                                for (int e = 0; e < 16; e++)
                                    if (e >= n) x[16 * p + e] = -INFINITY;
                            }
                    };
                    // the largest t = s fk + lv: by runs, whose factor is not negative
                    auto top = [&](int q, float mx) {
#pragma unroll
                        for (int p = 0; p < 2; p++) {
                            const float4 f = gs[2 * q + p];
                            const float *y = x + 16 * p;
                            const float m0 = max3(max3(y[0], y[1], y[2]), max3(y[3], y[4], y[5]), max3(y[6], y[7], y[8]));
                            const float m1 = max3(max3(y[9], y[10], y[11]), max3(y[12], y[13], y[14]), y[15]);
                            mx = fmaxf(mx, fmaf(fmaxf(m0, m1), fmaxf(cr * f.x, kMinFactor), f.y));
                        }
                        return mx;
                    };
                    fetch(1);
                    float mx = top(1, -INFINITY);
                    fetch(0);
                    mx = top(0, mx) - kTcOff;
                    // follow the maximum only by jumps: most tiles leave M and O as they are, and the two
                    // threads of a row need not tell each other more than that
                    if (named_bar_any(pair, 64, mx > M + kTcSlack || (M == -INFINITY && mx > M))) {
                        tmem_st1(tm_s + 16, mx);  // (a column whose score both threads' registers hold)
                        tmem_st_wait();
                        tc_fence_before();
                        named_bar_sync(pair, 64);
                        tc_fence_after();
                        mx = fmaxf(mx, tmem_ld1((tm_s ^ 64) + 16));
                        tc_fence_before();
                        named_bar_sync(pair, 64);  // both are read before P is written there
                        tc_fence_after();
                        const float mn = fmaxf(M, mx), al = mn == -INFINITY ? 1.f : ex2(M - mn);
                        M = mn;
                        l *= al;
                        if (j > 0) {
#pragma unroll 1
                            for (int i = 0; i < HD / 32; i++) {
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
#pragma unroll 1
                    for (int q = 0; q < 2; q++) {
                        if (q) fetch(1);
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
                    }
                    if (j + 1 == nt) {  // the row's sum, through a column that P leaves free, before the next item's scores can come
                        tmem_st1(tm_s + 32, l);
                        tmem_st_wait();
                        tc_fence_before();
                        named_bar_sync(pair, 64);
                        tc_fence_after();
                        l += tmem_ld1((tm_s ^ 64) + 32);
                        tc_fence_before();
                        named_bar_sync(pair, 64);
                    }
                    tmem_st_wait();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(half ? &bar_pb[w] : &bar_pa[w]);
                }
                if (!ok) break;
                queries(k + 1);  // (under the last tile's P V)
                // ── output ──
                if (!ok || !(ok = attn_wait(&bar_o[w], ph_o, abort_flag))) break;
                ph_o ^= 1;
                tc_fence_after();
                if (!dead) {
                    const int R = it->row0 + in_tile + lane;
                    const bool mine = R < it->n_packed;
                    const int t = R / rep, tok = it->r0 + t, head = it->kvh * rep + R - t * rep;
                    const size_t row = (size_t)tok * a.n_q + head, part = (size_t)it->split * a.n_rows * a.n_q + row;
                    const float inv = l == 0.f ? 0.f : 1.f / l;  // (NaN stays NaN)
                    if (half == 0 && mine) {
                        const float lw = l == 0.f ? -INFINITY : M + log2f(l);
                        if (parts.o) parts.w[part] = lw;
                        else if (a.lse) a.lse[row] = lw * kLn2;
                    }
#pragma unroll 1
                    for (int i = 0; i < HD / 32; i++) {
                        uint32_t o[16], u[8];
                        tmem_ld16(tm_o + 16 * i, o);
                        tmem_ld_wait(o);
                        if (!mine) continue;
                        const int d0 = half * (HD / 2) + 16 * i;
                        if (parts.o) {
#pragma unroll
                            for (int h = 0; h < 2; h++) {
#pragma unroll
                                for (int e = 0; e < 8; e++) u[e] = __float_as_uint(__uint_as_float(o[8 * h + e]) * inv);
                                store_row32(parts.o + part * HD + d0 + 8 * h, 16, u);
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 16; e++) reinterpret_cast<T *>(u)[e] = from_f32<T>(__uint_as_float(o[e]) * inv);
                            store_row32(reinterpret_cast<T *>(a.out) + tok * a.out_tok + head * a.out_head + d0, out_align, u);
                        }
                    }
                    tc_fence_before();
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[k & (kTcItems - 1)]);
        }
        if (!ok && lane == 0 && status) atomicOr(status, DFB_STAT_TIMEOUT);
    } else if (warp < 20) {
        // ── converters ──
        const int cw = warp - 16;
        int n = 0;  // code tiles so far
        bool ok = true;
        for (int k = 0; ok; k++) {
            const volatile TcItem *it = items + (k & (kTcItems - 1));
            if (!(ok = attn_wait(&item_full[k & (kTcItems - 1)], (k / kTcItems) & 1, abort_flag))) break;
            const int nt = it->nt;
            if (nt < 0) break;
            for (int i = 0; ok && i < 2 * nt; i++, n++) {
                if (i == 0) {
                    // the item's queries into place, once the last scores of the item before are there; the
                    // softmax warps turn them into operands when they have landed
                    constexpr int LPR = HD / 8, RPI = 32 / LPR;  // lanes of a row (16 bytes each), rows of one round
                    const int ch = lane % LPR, n_packed = it->n_packed, row0 = it->row0 + cw * 32 + lane / LPR, n_w = it->row0 + 128 < n_packed ? 2 : 1;
                    const T *q = reinterpret_cast<const T *>(a.q) + it->r0 * a.q_tok + it->kvh * rep * a.q_head + 8 * ch;
                    const int last = (n >> 1) - 1;  // the tile before the item: event `last` says that its scores are there
                    if (last >= 0 && !(ok = attn_wait(&freed[last & 1], (last >> 1) & 1, abort_flag))) break;
                    for (int w = 0; w < n_w; w++) {
                        uint8_t *dst = sm + L::q_off + w * L::q + (ch / 8) * 16384 + (cw * 32 + lane / LPR) * 128;
#pragma unroll 4
                        for (int x = 0; x < 32 / RPI; x++) {
                            // (a row that does not exist is read as the last one: what comes of it is not stored)
                            const int r = min(row0 + w * 128 + x * RPI, n_packed - 1), t = r / rep;
                            const T *from = q + t * a.q_tok + (r - t * rep) * a.q_head;
                            uint8_t *at = dst + x * RPI * 128 + (((ch ^ (cw * 32 + lane / LPR + x * RPI)) & 7) << 4);
                            if (vec) cp_async16(at, from);
                            else
#pragma unroll
                                for (int e = 0; e < 8; e++) reinterpret_cast<T *>(at)[e] = from[e];
                        }
                        // (cp.async's arrival does not wait for plain stores, nor order them)
                        if (vec) cp_async_arrive(&bar_raw_q[w]);
                        else mbar_arrive(&bar_raw_q[w]);
                    }
                }
                const int rs = n % kTcRaw, cs = n % kTcSlots, g = n >> 1;
                if (!(ok = attn_wait(&raw_full[rs], (n / kTcRaw) & 1, abort_flag))) break;
                // V(g) and K(g + 1) are freed together, by event g + 1 (K(0) by event 0); events alternate
                // between two barriers, and the issuer is never two events ahead of this wait (event g + 1
                // needs K(g + 1), which waited for event g)
                const int ev = (n - kTcSlots + 1) >> 1;
                if (n >= kTcSlots && !(ok = attn_wait(&freed[ev & 1], (ev >> 1) & 1, abort_flag))) break;
                const uint8_t *src = sm + L::raw_off + rs * L::raw;
                uint8_t *dst = sm + L::slot_off + cs * L::slot;
                const float4 *gs = sc + (g & 3) * 8;
                const int left = it->kend - (it->t0 + (i >> 1)) * kTcKeys;
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
            __syncwarp();
            if (lane == 0) mbar_arrive(&item_empty[k & (kTcItems - 1)]);
        }
    } else if (warp == 20) {
        // ── MMA issuer ──
        const uint32_t id_s = idesc_f16(128, kTcKeys), id_o = idesc_f16(128, HD) | (1u << 16);  // V is MN-major
        const uint32_t base = smem_u32(sm);
        const uint64_t dq = sw128_desc(base + L::q_off), dk = sw128_desc(base + L::slot_off), dv = mn128_desc(base + L::slot_off, 16384);
        // An MMA takes 64 cycles and an instruction of this warp about ten (its scheduler has three busy
        // warps): the warp stays whole (uniform registers), descriptors differ by constants, and the loop
        // over an item's tiles holds nothing but waits, MMAs and commits.
        bool ok = true;
        auto ready = [&](uint64_t *b, uint32_t ph) {
            ok = ok && attn_wait(b, ph, abort_flag);
            tc_fence_after();
        };
        // K(g) is in slot 2 g % 3, V(g) in slot (2 g + 1) % 3; MOD: g % 3
        static_assert(kTcSlots == 3, "slots");
        uint32_t ph_p[2] = {0, 0}, ph_q[2] = {0, 0}, ph_c[3] = {0, 0, 0};
        auto filled = [&](auto S) {
            ready(&conv_full[decltype(S)::value], ph_c[decltype(S)::value]);
            ph_c[decltype(S)::value] ^= 1;
        };
        // P V of row tile W from the values of a tile
        auto value = [&](auto W, auto MOD, bool first) {
            constexpr int w = decltype(W)::value;
            const uint64_t d = dv + (2 * decltype(MOD)::value + 1) % 3 * (L::slot >> 4);
            ready(&bar_pa[w], ph_p[w]);
            ready(&bar_pb[w], ph_p[w]);
            if (ok && elect_one())
                unrolled<kTcKeys / 16>([&](auto I) {
                    constexpr int i = decltype(I)::value;
                    mma1_f16_ts<256 + w * 128, w * 128 + 64 * (i >> 2) + 8 * (i & 3)>(d + (2048 >> 4) * i, id_o, i > 0 || !first);
                });
            ph_p[w] ^= 1;
        };
        auto score = [&](auto W, auto MOD) {
            constexpr int w = decltype(W)::value;
            const uint64_t d = dk + 2 * decltype(MOD)::value % 3 * (L::slot >> 4);
            if (ok && elect_one()) {
                unrolled<HD / 16>([&](auto K) {
                    constexpr int k = decltype(K)::value, off = ((k >> 2) * 16384 + (k & 3) * 32) >> 4;
                    mma1_f16_ss<w * 128, (k > 0)>(dq + w * (L::q >> 4) + off, d + off, id_s);
                });
                mma1_commit(&bar_s[w]);
            }
        };
        auto commit = [&](uint64_t *b) {
            if (ok && elect_one()) mma1_commit(b);
        };
        auto queries = [&](int w) {
            ready(&bar_q[w], ph_q[w]);
            ph_q[w] ^= 1;
        };
        int k = -1, g = 0, mod = 0, nt_next = 0;
        bool two_next = false;
        auto next = [&] {
            if (k >= 0 && lane == 0) mbar_arrive(&item_empty[k & (kTcItems - 1)]);
            k++;
            if (!(ok = attn_wait(&item_full[k & (kTcItems - 1)], (k / kTcItems) & 1, abort_flag))) return false;
            const volatile TcItem *it = items + (k & (kTcItems - 1));
            nt_next = it->nt;
            two_next = it->row0 + 128 < it->n_packed;
            __syncwarp();
            return nt_next > 0;
        };
        bool have = next();
        if (have) {
            filled(Int<0>());
            queries(0);
            score(Int<0>(), Int<0>());
            if (two_next) {
                queries(1);
                score(Int<1>(), Int<0>());
            }
            commit(&freed[0]);
        }
        while (have && ok) {
            const int nt = nt_next;
            const bool two = two_next;
            have = next();
            // tile t (MOD: its index g % 3) and the scores of the one after it
            auto tile = [&](auto MOD, int t) {
                using Next = Int<(decltype(MOD)::value + 1) % 3>;
                using KeySlot = Int<2 * Next::value % 3>;
                uint64_t *event = &freed[(g + 1) & 1];
                filled(Int<(2 * decltype(MOD)::value + 1) % 3>());
                value(Int<0>(), MOD, t == 0);
                if (t + 1 < nt) {
                    filled(KeySlot());
                    score(Int<0>(), Next());
                    if (two) {
                        value(Int<1>(), MOD, t == 0);
                        score(Int<1>(), Next());
                    }
                    commit(event);
                } else {  // the item's last tile, the next one's first
                    commit(&bar_o[0]);
                    if (have) {
                        filled(KeySlot());
                        queries(0);
                        score(Int<0>(), Next());
                    }
                    if (two) {
                        value(Int<1>(), MOD, t == 0);
                        commit(&bar_o[1]);
                    }
                    if (have) {
                        if (two_next) {
                            queries(1);
                            score(Int<1>(), Next());
                        }
                        commit(event);  // (the CTA's last commits are bar_o's, which the softmax warps wait for)
                    }
                }
            };
            for (int t = 0; t < nt && ok; t++, g++, mod = mod == 2 ? 0 : mod + 1) {
                if (mod == 0) tile(Int<0>(), t);
                else if (mod == 1) tile(Int<1>(), t);
                else tile(Int<2>(), t);
            }
        }
        if (!ok && elect_one()) {  // let what was issued end before TMEM is freed
            mma1_commit(bar_drain);
            spin_bounded(bar_drain, 0);
        }
        __syncwarp();
    } else if (warp == 21) {
        // ── loader ──
        const int box = min(c.page, kKeyTile), sh_box = __ffs(box) - 1, nb = kTcKeys >> sh_box, sh_page = __ffs(c.page) - 1;
        int n = 0, k = 0, idx = (int)blockIdx.x - (int)gridDim.x;
        bool ok = true;
        // The next item, published one ahead of its loads: the issuer looks at it while it works on the one before.
        auto publish = [&](TcItem &t) {
            do idx += gridDim.x;
            while (idx < grid.items && !(tc_item(c, a, parts, grid, rep, idx, status, t) && t.nt > 0));
            if (idx >= grid.items) t.nt = -1;
            if (k >= kTcItems && !(ok = attn_wait(&item_empty[k & (kTcItems - 1)], (k / kTcItems - 1) & 1, abort_flag))) return;
            if (lane == 0) {
                volatile TcItem *o = reinterpret_cast<volatile TcItem *>(sm + L::item_off) + (k & (kTcItems - 1));
                o->s = t.s; o->kvh = t.kvh; o->split = t.split; o->r0 = t.r0; o->len = t.len; o->row0 = t.row0;
                o->n_packed = t.n_packed; o->kend = t.kend; o->t0 = t.t0; o->nt = t.nt;
                mbar_arrive(&item_full[k & (kTcItems - 1)]);
            }
            __syncwarp();
            k++;
        };
        TcItem it, after;
        publish(it);
        while (ok && it.nt > 0) {
            publish(after);
            if (!ok) break;
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
            it = after;
        }
        if (*abort_flag)  // let the copies in flight land before the block goes
            for (int i = max(0, n - kTcRaw); i < n; i++) spin_bounded(&raw_full[i % kTcRaw], (i / kTcRaw) & 1);
    }
    if (warp == 22) {
        // ── rows of items without keys ──
        TcItem it;
        for (int idx = blockIdx.x; idx < grid.items; idx += gridDim.x) {
            if (!tc_item(c, a, parts, grid, rep, idx, status, it) || it.nt > 0) continue;
            for (int r = it.row0; r < min(it.row0 + kTcRows, it.n_packed); r++) {
                const int t = r / rep, tok = it.r0 + t, head = it.kvh * rep + r - t * rep;
                const size_t row = (size_t)tok * a.n_q + head;
                if (parts.o) {
                    if (lane == 0) parts.w[(size_t)it.split * a.n_rows * a.n_q + row] = -INFINITY;
                    continue;
                }
                if (a.lse && lane == 0) a.lse[row] = -INFINITY;
                for (int d = lane; d < HD; d += 32) reinterpret_cast<T *>(a.out)[tok * a.out_tok + head * a.out_head + d] = from_f32<T>(0.f);
            }
        }
    }
    __syncthreads();
    if (warp == 20) {
        tc_fence_after();
        tmem_dealloc1((uint32_t)shared_i[1], 512);
    }
}

}  // namespace dfb
