// Attention over the paged 8-bit K/V cache (dfb_kv_attention).
//   s_j = scale * q . k_j,  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  lse = m + log sum
// over the first min(vis, len) keys; k_j, v_j = code * scale of the page and KV head.
//
// The rows of one KV head are packed: row R of a sequence is its token R / rep, query head
// kvh * rep + R % rep, so all query heads of a group share one pass over the keys.
//
// Arithmetic.  E4M3 codes are exact in f16, and so is q (f16; bf16 rows are scaled by a power of
// two so that their largest value lies in [1, 2): what f16's subnormals cut off is below 2^-24 of
// it), so the scores' products are exact and summed in f32.  In base 2, with x = s log2(e) and the
// page's V scale sv:
//   t = x + log2 sv,  M = running max of t - kPOff,  p' = 2^(t - M) as f16,
//   O += p' . code_v,   l += p' / sv   (= 2^(x - M), in f32 before the rounding)
// so V's scale costs one addend of the exponent and 1 / sv one multiply-add per 16 keys, and p'
// keeps f16's precision down to 2^-(14 + kPOff) of the largest weight however far apart the pages'
// scales are.  out = O / l, lse = (M + log2 l) ln 2, with the rounding of f32 numbers of the size of
// |x| + |log2 sv| (scales of 2^-40: 2e-6).  Rounding p' to f16 (2^-11 relative, averaged
// over the keys) is the only rounding to 16 bits before the output's own.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cstdint>
#include <type_traits>

#include "../../../include/diffuse_b200.h"
#include "kv_append.cuh"
#include "ptx.cuh"
#include "simd.cuh"

namespace dfb {

constexpr float kPOff = 15.f;  // p' <= 2^15 stays below f16's largest value
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// One sequence's rows and keys, clamped to what the tensors hold.
struct AttnSeq {
    int r0, n_rows, len;
};
__device__ __forceinline__ AttnSeq attn_seq(const dfb_kv_cache &c, const dfb_kv_attn &a, int s, bool reporter, int32_t *status) {
    AttnSeq q;
    q.r0 = a.row_off[s];
    int r1 = a.row_off[s + 1];
    q.len = a.len[s];
    const int cap = (int)min((long long)a.max_keys, (long long)c.max_pages * c.page);
    int bad = 0;
    if (q.r0 < 0 || r1 < q.r0 || r1 > a.n_rows || r1 - q.r0 > a.max_rows) {
        bad |= DFB_STAT_ROWS;
        q.r0 = min(max(q.r0, 0), a.n_rows);
        r1 = min(max(r1, q.r0), a.n_rows);
        r1 = min(r1 - q.r0, a.max_rows) + q.r0;
    }
    if (q.len < 0 || q.len > cap) {
        bad |= DFB_STAT_POSITION;
        q.len = min(max(q.len, 0), cap);
    }
    q.n_rows = r1 - q.r0;
    if (bad && reporter && status) atomicOr(status, bad);
    return q;
}

__device__ __forceinline__ void tma_load_2d(void *dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}
// Bounded wait of one whole warp: false for all its lanes (and *abort set) after kWaitTimeoutNs, or
// when another warp of the CTA gave up.
__device__ __forceinline__ bool attn_wait(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
    bool ok = mbar_try_wait(bar, parity);
    if (!ok) {
        const uint64_t t0 = globaltimer();
        while (!(ok = mbar_try_wait_sleep(bar, parity, kWaitCheckNs))) {
            if (*abort_flag) break;
            if (globaltimer() - t0 > kWaitTimeoutNs) {
                *abort_flag = 1;
                break;
            }
        }
    }
    return __all_sync(0xffffffffu, ok);
}

// D += A (16 x 16, row) * B (16 x 8, col), f16 operands, f32 accumulators.
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two E4M3 codes (the low or high half of w) as an f16 pair, exact.
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t w, int half) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(half ? w >> 16 : w & 0xffff), __NV_E4M3);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

constexpr int kKeyTile = 64;    // keys of one stage
constexpr int kKvStages = 4;

constexpr int kMaxSplits = 128;

// Eight consecutive elements as f32; vec: 16-byte loads are aligned.
template <typename T>
__device__ __forceinline__ void load8(const T *p, bool vec, float (&v)[8]) {
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            const uint4 u = *reinterpret_cast<const uint4 *>(p);
            const T *t = reinterpret_cast<const T *>(&u);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = to_f32<T>(t[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = to_f32<T>(p[i]);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, bool vec, const float (&v)[8]) {
    T t[8];
#pragma unroll
    for (int i = 0; i < 8; i++) t[i] = from_f32<T>(v[i]);
    if (vec) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<float4 *>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(t);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = t[i];
    }
}

// Where a call's split parts go: normalised rows and their log2 weights, [split][row][query head].
struct AttnParts {
    float *o = nullptr;    // [splits][n_rows * n_q][head_dim]
    float *w = nullptr;    // [splits][n_rows * n_q]
    int splits = 1;
};

// Shared memory of one CTA: stages of K and V codes (swizzled by the tensor copy), reused for the
// rows' joining at the end; per stage and 16 keys the K scale, log2 of the V scale (-inf: no such
// keys) and 1 / V scale.
template <int HD, int MW, int KW>
struct KvSmem {
    static constexpr int tile = kKeyTile * HD;
    static constexpr int stages = kKvStages * 2 * tile;
    static constexpr int join = KW * MW * 16 * (HD + 4) * 4;
    static constexpr int data = stages > join ? stages : join;
    static constexpr int bytes = 1024 + data + kKvStages * 4 * 12 + KW * MW * 16 * 8 + 2 * kKvStages * 8 + 16;
};

// Eight dimensions of one finished row (or of one split part of it) and its log2 weight.
template <typename T, int HD>
__device__ __forceinline__ void attn_store(const dfb_kv_attn &a, const AttnParts &parts, int split, int tok, int head, int d0,
                                           const float (&v)[8], float lw, bool vec) {
    const size_t row = (size_t)tok * a.n_q + head;
    if (parts.o) {
        const size_t at = (size_t)split * a.n_rows * a.n_q + row;
        store8(parts.o + at * HD + d0, true, v);
        if (d0 == 0) parts.w[at] = lw;
    } else {
        store8(reinterpret_cast<T *>(a.out) + tok * a.out_tok + head * a.out_head + d0, vec, v);
        if (d0 == 0 && a.lse) a.lse[row] = lw * kLn2;
    }
}

// For few rows (dfb_kv_attention's plan): mma.sync on 16 to 64 packed rows x 64 keys.  Bound: for one
// token latency (28 / 4 heads over 4607 keys in 18 parts: 13 us with the join, 0.7 us of memory time), for
// 64-row tiles the conversion of codes to f16 fragments, which every warp does for its own 16 rows: a key
// tile takes 1.3 us of a CTA (256 rows of 32 heads over 320 keys: 13.4 us; tcgen05 tiles 19.9).
// MW warps of 16 rows each share a key tile; KW such groups take the tiles in turn; one more warp
// loads.  Grid: (splits x row tiles, KV heads, sequences).
template <typename T, int HD, int MW, int KW>
__global__ void __launch_bounds__((MW * KW + 1) * 32, MW * KW <= 4 ? 2 : 1)
    kv_attn_kernel(const dfb_kv_cache c, const dfb_kv_attn a, const __grid_constant__ CUtensorMap tm_k,
                   const __grid_constant__ CUtensorMap tm_v, const AttnParts parts, bool vec, int32_t *status) {
    using L = KvSmem<HD, MW, KW>;
    constexpr int TM = MW * 16, NT = (MW * KW + 1) * 32;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *sm = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    float *sc = reinterpret_cast<float *>(sm + L::data);                     // [stage][16 keys] ks, log2 vs, 1 / vs
    float2 *ml = reinterpret_cast<float2 *>(sc + kKvStages * 12);            // [KW][TM] M, l
    uint64_t *full = reinterpret_cast<uint64_t *>(ml + KW * TM), *empty = full + kKvStages;
    int *shared_i = reinterpret_cast<int *>(empty + kKvStages);              // abort flag, most and least keys of a row
    volatile int *abort_flag = shared_i;

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int s = blockIdx.z, kvh = blockIdx.y, split = blockIdx.x % parts.splits, tile = blockIdx.x / parts.splits;
    const int rep = a.n_q / c.n_kv;
    const AttnSeq sq = attn_seq(c, a, s, blockIdx.x == 0 && kvh == 0 && tid == 0, status);
    const int row0 = tile * TM;                     // first packed row of the tile
    const int n_packed = sq.n_rows * rep;
    if (row0 >= n_packed) return;
    auto keys_of = [&](int R) {
        if (R >= n_packed) return 0;
        return a.vis ? min(max(a.vis[sq.r0 + R / rep], 0), sq.len) : sq.len;
    };
    if (tid == 0) {
        shared_i[0] = 0;
        shared_i[1] = 0;
        shared_i[2] = 0x7fffffff;
        for (int i = 0; i < kKvStages; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], MW);
        }
        fence_barrier_init();
    }
    __syncthreads();
    for (int i = tid; i < TM; i += NT)
        if (row0 + i < n_packed) {
            const int n = keys_of(row0 + i);
            atomicMax(&shared_i[1], n);
            atomicMin(&shared_i[2], n);
        }
    __syncthreads();
    const int kend = shared_i[1], kmin = shared_i[2];
    const int n_tiles = (kend + kKeyTile - 1) / kKeyTile;
    const int t0 = (int)((long long)n_tiles * split / parts.splits), t1 = (int)((long long)n_tiles * (split + 1) / parts.splits);

    if (warp == MW * KW) {
        // ── loader: page ids and scales of 32 boxes at a time, one tensor copy per box ──
        const int box = min(c.page, kKeyTile), nb = kKeyTile / box;  // keys per copy, copies per tile
        int pid = 0;
        float ks = 0.f, vs = 1.f;
        int issued = 0;
        for (int t = t0; t < t1; t++) {
            const int i = t - t0, st = i % kKvStages;
            if ((i * nb) % 32 == 0) {
                const int key = (t0 * nb + i * nb + lane) * box;
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
                    vs = fmaxf(c.v_scale[(size_t)pid * c.n_kv + kvh], 5.421010862427522e-20f);
                }
            }
            if (i >= kKvStages && !attn_wait(&empty[st], ((i / kKvStages) - 1) & 1, abort_flag)) break;
            const int b0 = (i * nb) % 32;
            uint8_t *dk = sm + st * 2 * L::tile, *dv = dk + L::tile;
            int n_ok = 0;
            for (int b = 0; b < nb; b++) {
                const int p = __shfl_sync(0xffffffffu, pid, b0 + b);
                if (p < 0) continue;
                n_ok++;
                if (lane == 0) {
                    const int y = (p * c.n_kv + kvh) * c.page + ((t * nb + b) * box) % c.page;
                    tma_load_2d(dk + b * box * HD, &tm_k, 0, y, &full[st]);
                    tma_load_2d(dv + b * box * HD, &tm_v, 0, y, &full[st]);
                }
            }
            // the scales of the tile's four runs of 16 keys; the stage is complete once lane 0 has arrived
            // (after these writes) and the announced bytes have landed
            const int src = b0 + (lane & 3) * 16 / box;
            const int gp = __shfl_sync(0xffffffffu, pid, src);
            const float gk = __shfl_sync(0xffffffffu, ks, src), gv = __shfl_sync(0xffffffffu, vs, src);
            if (lane < 4) {
                float *d = sc + st * 12 + lane * 3;
                d[0] = gk;
                d[1] = gp < 0 ? -INFINITY : log2f(gv);
                d[2] = 1.f / gv;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive_expect_tx(&full[st], n_ok * 2 * box * HD);
            issued = i + 1;
        }
        if (*abort_flag)  // let the copies in flight land before the block goes
            for (int i = max(0, issued - kKvStages); i < issued; i++) spin_bounded(&full[i % kKvStages], (i / kKvStages) & 1);
        return;
    }

    // ── 16 rows of this warp: g and g + 8 of each thread ──
    constexpr int KS = HD / 16, KH = HD / 64;  // contraction steps of 16; 16-byte pieces of a key per thread
    const int wm = warp % MW, kg = warp / MW, g = lane >> 2, t4 = lane & 3;
    // column n of a tile of 8 keys is its row (n >> 1) + 4 (n & 1) (HD 128) or n (HD 64), and column
    // n of V's dimensions likewise: the eight threads of a shared-memory phase then read eight
    // different 16-byte columns of the swizzled rows
    const int kperm = HD == 128 ? (g >> 1) + 4 * (g & 1) : g;
    const int v0 = HD == 128 ? t4 : 2 * t4, v1 = HD == 128 ? t4 + 4 : 2 * t4 + 1;  // keys of columns 2 t4 and 2 t4 + 1
    uint32_t qf[KS][4];
    float cr[2];
    int nr[2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
        const int R = row0 + wm * 16 + g + 8 * r;
        nr[r] = keys_of(R);
        float x[KH][16];
        float mx = 0.f;
#pragma unroll
        for (int h = 0; h < KH; h++) {
            if (R < n_packed) {
                const T *q = reinterpret_cast<const T *>(a.q) + (sq.r0 + R / rep) * a.q_tok + (kvh * rep + R % rep) * a.q_head + 16 * (t4 + 4 * h);
                load8(q, vec, reinterpret_cast<float(&)[8]>(x[h][0]));
                load8(q + 8, vec, reinterpret_cast<float(&)[8]>(x[h][8]));
            } else {
#pragma unroll
                for (int e = 0; e < 16; e++) x[h][e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < 16; e++) mx = fmaxf(mx, fabsf(x[h][e]));
        }
        cr[r] = a.scale * kLog2e;
        if constexpr (!std::is_same<T, __half>::value) {
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const int e = (int)(__float_as_uint(mx) >> 23) - 127;  // mx = 1.x * 2^e
            if (mx > 0.f && mx < INFINITY) {
                const float up = exp2i(max(-e, -126));  // (|q| up to 2^128: e = 127 leaves 2 to 4)
#pragma unroll
                for (int h = 0; h < KH; h++)
#pragma unroll
                    for (int i = 0; i < 16; i++) x[h][i] *= up;
                cr[r] *= 1.f / up;
            }
        }
#pragma unroll
        for (int h = 0; h < KH; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                qf[4 * h + i][r] = pack_f16(x[h][4 * i], x[h][4 * i + 1]);
                qf[4 * h + i][2 + r] = pack_f16(x[h][4 * i + 2], x[h][4 * i + 3]);
            }
    }
    float o[KS][8], M[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    constexpr int NV = HD / 8;  // column tiles of the output
    float (&oa)[NV][4] = reinterpret_cast<float(&)[NV][4]>(o);
#pragma unroll
    for (int j = 0; j < NV; j++) oa[j][0] = oa[j][1] = oa[j][2] = oa[j][3] = 0.f;

    for (int t = t0 + kg; t < t1; t += KW) {
        const int i = t - t0, st = i % kKvStages;
        if (!attn_wait(&full[st], (i / kKvStages) & 1, abort_flag)) break;
        const uint8_t *K = sm + st * 2 * L::tile, *V = K + L::tile;
        const float *scl = sc + st * 12;
        // scores
        float x[8][4];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.f;
            const int kr = 8 * j + kperm;
#pragma unroll
            for (int h = 0; h < KH; h++) {
                const int ch = HD == 128 ? (t4 + 4 * h) ^ (kr & 7) : t4 ^ ((kr >> 1) & 3);
                const uint4 w = *reinterpret_cast<const uint4 *>(K + kr * HD + 16 * ch);
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t(&f)[4] = qf[4 * h + e];
                    mma16816(x[j], f[0], f[1], f[2], f[3], e4m3x2_f16x2(u[e], 0), e4m3x2_f16x2(u[e], 1));
                }
            }
        }
        // t = x + log2 sv of each key, -inf where there is none
        bool gone = false;
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const float f0 = cr[0] * scl[3 * p], f1 = cr[1] * scl[3 * p], lv = scl[3 * p + 1];
            gone |= lv == -INFINITY;
#pragma unroll
            for (int j = 2 * p; j < 2 * p + 2; j++) {
                x[j][0] = fmaf(x[j][0], f0, lv);
                x[j][1] = fmaf(x[j][1], f0, lv);
                x[j][2] = fmaf(x[j][2], f1, lv);
                x[j][3] = fmaf(x[j][3], f1, lv);
            }
        }
        const int key0 = t * kKeyTile;
        if (key0 + kKeyTile > kmin || gone) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const bool there = scl[3 * (j >> 1) + 1] != -INFINITY;
                const int c0 = key0 + 8 * j + v0, c1 = key0 + 8 * j + v1;
                if (!there || c0 >= nr[0]) x[j][0] = -INFINITY;
                if (!there || c1 >= nr[0]) x[j][1] = -INFINITY;
                if (!there || c0 >= nr[1]) x[j][2] = -INFINITY;
                if (!there || c1 >= nr[1]) x[j][3] = -INFINITY;
            }
        }
        float alpha[2], base[2];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; j++) mx = fmaxf(mx, fmaxf(x[j][2 * r], x[j][2 * r + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float mn = fmaxf(M[r], mx - kPOff);
            base[r] = mn == -INFINITY ? 0.f : mn;
            alpha[r] = ex2(M[r] - base[r]);
            M[r] = mn;
        }
#pragma unroll
        for (int r = 0; r < 2; r++) {
            l[r] *= alpha[r];
#pragma unroll
            for (int p = 0; p < 4; p++) {
                float sum = 0.f;
#pragma unroll
                for (int j = 2 * p; j < 2 * p + 2; j++) {
                    x[j][2 * r] = ex2(x[j][2 * r] - base[r]);
                    x[j][2 * r + 1] = ex2(x[j][2 * r + 1] - base[r]);
                    sum += x[j][2 * r] + x[j][2 * r + 1];
                }
                l[r] = fmaf(sum, scl[3 * p + 2], l[r]);
            }
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
            for (int j = 0; j < NV; j++) {
                oa[j][0] *= alpha[0]; oa[j][1] *= alpha[0];
                oa[j][2] *= alpha[1]; oa[j][3] *= alpha[1];
            }
        }
        // O += P V: 16 keys a step; codes of absent keys are not numbers to be multiplied, so they are 0
        const bool edge = key0 + kKeyTile > kend || gone;
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const uint32_t a0 = pack_f16(x[2 * p][0], x[2 * p][1]), a1 = pack_f16(x[2 * p][2], x[2 * p][3]);
            const uint32_t a2 = pack_f16(x[2 * p + 1][0], x[2 * p + 1][1]), a3 = pack_f16(x[2 * p + 1][2], x[2 * p + 1][3]);
            uint32_t u[4][HD / 32];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int kr = 16 * p + (e & 1 ? v1 : v0) + 8 * (e >> 1);
                if constexpr (HD == 128) {
                    const int ch = ((g >> 1) + 4 * (g & 1)) ^ (kr & 7);
                    const uint4 w = *reinterpret_cast<const uint4 *>(V + kr * HD + 16 * ch);
                    u[e][0] = w.x; u[e][1] = w.y; u[e][2] = w.z; u[e][3] = w.w;
                } else {
                    const int ch = (g >> 1) ^ ((kr >> 1) & 3);
                    const uint2 w = *reinterpret_cast<const uint2 *>(V + kr * HD + 16 * ch + 8 * (g & 1));
                    u[e][0] = w.x; u[e][1] = w.y;
                }
                if (edge && (key0 + kr >= kend || scl[3 * p + 1] == -INFINITY))
#pragma unroll
                    for (int q = 0; q < HD / 32; q++) u[e][q] = 0;
            }
#pragma unroll
            for (int q = 0; q < HD / 32; q++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++) {
                    const uint32_t sel = hf ? 0x7362 : 0x5140;
                    const uint32_t w0 = __byte_perm(u[0][q], u[1][q], sel), w1 = __byte_perm(u[2][q], u[3][q], sel);
                    mma16816(oa[4 * q + 2 * hf], a0, a1, a2, a3, e4m3x2_f16x2(w0, 0), e4m3x2_f16x2(w1, 0));
                    mma16816(oa[4 * q + 2 * hf + 1], a0, a1, a2, a3, e4m3x2_f16x2(w0, 1), e4m3x2_f16x2(w1, 1));
                }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[st]);
    }
#pragma unroll
    for (int r = 0; r < 2; r++) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    // ── join the key groups and write ──
    // (every stage's copies have been waited for by the group that took it: the stages are free)
    named_bar_sync(1, MW * KW * 32);
    if (*abort_flag && tid == 0 && status) atomicOr(status, DFB_STAT_TIMEOUT);
    float *J = reinterpret_cast<float *>(sm);
    constexpr int JP = HD + 4;
#pragma unroll
    for (int r = 0; r < 2; r++) {
        const int row = wm * 16 + g + 8 * r;
        float *d = J + (size_t)(kg * TM + row) * JP;
        if (t4 == 0) ml[kg * TM + row] = make_float2(M[r], l[r]);
#pragma unroll
        for (int n = 0; n < 2; n++) {
            // column n of the thread: HD / 8 consecutive dimensions
            const int d0 = HD == 128 ? 16 * (t4 + 4 * n) : 8 * (2 * t4 + n);
#pragma unroll
            for (int j = 0; j < NV; j += 4)
                *reinterpret_cast<float4 *>(d + d0 + j) = make_float4(oa[j][2 * r + n], oa[j + 1][2 * r + n], oa[j + 2][2 * r + n], oa[j + 3][2 * r + n]);
        }
    }
    named_bar_sync(1, MW * KW * 32);
    for (int it = tid; it < TM * (HD / 8); it += MW * KW * 32) {
        const int row = it / (HD / 8), d0 = it % (HD / 8) * 8, R = row0 + row;
        if (R >= n_packed) break;
        float mm = -INFINITY, ll = 0.f, v[8] = {};
#pragma unroll
        for (int k = 0; k < KW; k++) mm = fmaxf(mm, ml[k * TM + row].x);
        const float b = mm == -INFINITY ? 0.f : mm;
#pragma unroll
        for (int k = 0; k < KW; k++) {
            const float2 w = ml[k * TM + row];
            const float f = ex2(w.x - b);
            ll = fmaf(w.y, f, ll);
            const float *p = J + (size_t)(k * TM + row) * JP + d0;
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = fmaf(p[e], f, v[e]);
        }
        const float inv = ll == 0.f ? 0.f : 1.f / ll, lw = ll == 0.f ? -INFINITY : b + log2f(ll);  // (NaN stays NaN)
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] *= inv;
        attn_store<T, HD>(a, parts, split, sq.r0 + R / rep, kvh * rep + R % rep, d0, v, lw, vec);
    }
}

// Joins the split parts of one row and head per warp; rows of no sequence stay as they are.  The lanes
// share out the parts' weights, then each holds four (HD 64: two) dimensions with eight parts' loads in
// flight: the parts come from L2, and a thread that waited for one after the other took 20 us for 37 parts.
template <typename T, int HD>
__global__ void __launch_bounds__(128) kv_attn_join_kernel(const dfb_kv_cache c, const dfb_kv_attn a, const AttnParts parts) {
    constexpr int E = HD / 32;
    griddep_wait();
    const AttnSeq sq = attn_seq(c, a, blockIdx.y, false, nullptr);
    const int at = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (at >= sq.n_rows * a.n_q) return;
    const size_t stride = (size_t)a.n_rows * a.n_q, row = (size_t)sq.r0 * a.n_q + at;
    float w[kMaxSplits / 32], mx = -INFINITY, z = 0.f;
#pragma unroll
    for (int i = 0; i < kMaxSplits / 32; i++) {
        w[i] = 32 * i + lane < parts.splits ? parts.w[(32 * i + lane) * stride + row] : -INFINITY;
        mx = fmaxf(mx, w[i]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float base = mx == -INFINITY ? 0.f : mx;
#pragma unroll
    for (int i = 0; i < kMaxSplits / 32; i++) {
        w[i] = ex2(w[i] - base);
        z += w[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    float v[E] = {};
#pragma unroll
    for (int i = 0; i < kMaxSplits / 32; i++)
#pragma unroll 8
        for (int k = 32 * i; k < min(parts.splits, 32 * i + 32); k++) {
            const float f = __shfl_sync(0xffffffffu, w[i], k & 31);
            float u[E];
            const float *o = parts.o + (k * stride + row) * HD + lane * E;
            if constexpr (E == 4) *reinterpret_cast<float4 *>(u) = *reinterpret_cast<const float4 *>(o);
            else *reinterpret_cast<float2 *>(u) = *reinterpret_cast<const float2 *>(o);
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = f == 0.f ? v[e] : fmaf(u[e], f, v[e]);  // (a part without keys is not written)
        }
    const float inv = z == 0.f ? 0.f : 1.f / z;  // (NaN stays NaN)
    const int tok = sq.r0 + at / a.n_q, head = at % a.n_q;
    T *out = reinterpret_cast<T *>(a.out) + tok * a.out_tok + head * a.out_head + lane * E;
#pragma unroll
    for (int e = 0; e < E; e++) out[e] = from_f32<T>(v[e] * inv);
    if (a.lse && lane == 0) a.lse[row] = z == 0.f ? -INFINITY : (base + log2f(z)) * kLn2;
}

}  // namespace dfb
