// Rows of K and V into the paged 8-bit cache (dfb_kv_append), rotated on the way.
//
// For each touched page and KV head, with X the values the call writes there:
//   amax = max |X|,  need = min { e >= -64 : amax <= 448 * 2^e }  (448: E4M3's largest value),
//   e = need, or max(need, old e) while positions of the page keep their values,
//   code = E4M3(x * 2^-e), kept codes: E4M3(code * 2^(old e - e)) where e grew.
// A power-of-two scale costs E4M3 nothing (its relative step does not depend on the scale), makes
// x * 2^-e and the re-rounding of kept codes exact up to their one E4M3 rounding, and value =
// code * scale exact in f16 / bf16 arithmetic.
// Rotation: (a, b) -> (a c - b s, a s + b c) for NEOX pairs (i, i + hd / 2) with f32 c, s.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cstdint>
#include <type_traits>

#include "../../../include/diffuse_b200.h"
#include "simd.cuh"

namespace dfb {

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two consecutive elements as f32, and back.
template <typename T>
__device__ __forceinline__ float2 pair_at(const uint4 *v, int e) {
    if constexpr (sizeof(T) == 4) return reinterpret_cast<const float2 *>(v)[e];
    else if constexpr (std::is_same_v<T, __half>) return __half22float2(reinterpret_cast<const __half2 *>(v)[e]);
    else {
        const uint32_t u = reinterpret_cast<const uint32_t *>(v)[e];
        return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
    }
}
template <typename T>
__device__ __forceinline__ void set_pair(uint4 *v, int e, float2 x) {
    if constexpr (sizeof(T) == 4) reinterpret_cast<float2 *>(v)[e] = x;
    else if constexpr (std::is_same_v<T, __half>) reinterpret_cast<__half2 *>(v)[e] = __float22half2_rn(x);
    else reinterpret_cast<__nv_bfloat162 *>(v)[e] = __float22bfloat162_rn(x);
}

// x c + y s rounded to odd: the f32 next to the exact value towards zero, with its last bit set
// when the value lies between two f32.  One more rounding (to E4M3, f16, bf16 or f32's own
// nearest, which `near` receives) then gives what rounding the exact value gives: a value next
// to the border of two codes falls on its own side.  The products' and the sum's rounding
// errors come from fused multiply-adds and the two-sum identity.
__device__ __forceinline__ float rot_odd(float x, float c, float y, float s, float &near) {
    const float p = __fmul_rn(x, c), q = __fmul_rn(y, s);
    const float pe = __fmaf_rn(x, c, -p), qe = __fmaf_rn(y, s, -q);
    const float h = __fadd_rn(p, q), z = __fadd_rn(h, -p);
    const float e = __fadd_rn(__fadd_rn(p, -__fadd_rn(h, -z)), __fadd_rn(q, -z));
    const float lo = __fadd_rn(e, __fadd_rn(pe, qe));
    near = lo == 0.f ? h : __fadd_rn(h, lo);  // (keeps the sign of a zero)
    const float r = __fadd_rn(__fadd_rn(h, -near), lo);
    if (!(fabsf(near) < INFINITY) || r == 0.f) return near;
    uint32_t u = __float_as_uint(near);
    if ((r < 0.f) != (near < 0.f)) u -= 1;  // the exact value is nearer to zero
    return __uint_as_float(u | 1u);
}

// (a c - b s, a s + b c) of two pairs, each within 1.5 units in the last place: a product's rounding
// error is taken back (Kahan's difference of two products).  (A zero error is +0 here, so that taking it back keeps the sign of a zero.)
__device__ __forceinline__ void rot_near(float2 &a, float2 &b, float2 c, float2 s) {
    const float2 minus = make_float2(-1.f, -1.f), ns = mul2(s, minus);
    const float2 p = mul2(b, ns), q = mul2(a, s);
    const float2 x = fma2(fma2(b, s, p), minus, fma2(a, c, p));
    b = fma2(fma2(a, ns, q), minus, fma2(b, c, q));
    a = x;
}
// A value that rot_near gives lies within this of the exact one, relative to it (four times the bound).
constexpr float kRotTol = 4.76837158203125e-07f;  // 2^-21

// Smallest e >= -64 with amax <= 448 * 2^e = 0.875 * 2^(9 + e).
__device__ __forceinline__ int need_exp(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 126 - ((u & 0x7fffffu) > 0x600000u ? 8 : 9);
    return max(e, -64);
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// Exponent of a stored scale (a power of two; anything else counts as its power below).
__device__ __forceinline__ int scale_exp(float s) {
    const int e = (int)((__float_as_uint(s) >> 23) & 255) - 127;
    return min(max(e, -64), 120);
}
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float e4m3_value(uint32_t code) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3)));
}

// First index in [lo, hi) with pos[i] >= v (pos ascending).
__device__ __forceinline__ int lower_bound(const int32_t *pos, int lo, int hi, int v) {
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (pos[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// Eight elements and the eight that lie half a head further, as they are in memory.
template <typename T>
struct RawItem {
    static constexpr int NV = sizeof(T) / 2;  // 16-byte pieces of eight elements
    uint4 v[2 * NV];
    __device__ __forceinline__ void load(const T *p, int hd, bool vec) {
        if (vec) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                v[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
                v[NV + i] = __ldcs(reinterpret_cast<const uint4 *>(p + hd / 2) + i);
            }
        } else
#pragma unroll
            for (int e = 0; e < 8; e++) {
                reinterpret_cast<T *>(v)[e] = p[e];
                reinterpret_cast<T *>(v)[8 + e] = p[hd / 2 + e];
            }
    }
    __device__ __forceinline__ void store(T *p, int hd, bool vec) const {
        if (vec) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                reinterpret_cast<uint4 *>(p)[i] = v[i];
                reinterpret_cast<uint4 *>(p + hd / 2)[i] = v[NV + i];
            }
        } else
#pragma unroll
            for (int e = 0; e < 8; e++) {
                p[e] = reinterpret_cast<const T *>(v)[e];
                p[hd / 2 + e] = reinterpret_cast<const T *>(v)[8 + e];
            }
    }
    __device__ __forceinline__ float2 pair(int e) const { return pair_at<T>(v, e); }
    __device__ __forceinline__ void set(int e, float2 x) { set_pair<T>(v, e, x); }
};

// The codes of eight values times f.
__device__ __forceinline__ uint2 encode8(const float2 *v, float f) {
    const float2 g = make_float2(f, f);
    const float2 a = mul2(v[0], g), b = mul2(v[1], g), c = mul2(v[2], g), d = mul2(v[3], g);
    return make_uint2(e4m3_pair(a.x, a.y) | e4m3_pair(b.x, b.y) << 16, e4m3_pair(c.x, c.y) | e4m3_pair(d.x, d.y) << 16);
}

// One block: the rows that fall into one page of one sequence (the blockIdx.x-th touched page of
// sequence blockIdx.z), for `heads` K heads, V heads or query heads in turn (blockIdx.y).  A thread has
// one item, eight values and their rotation partners: it holds the item's cos and sin for all the heads,
// its values between the maximum and the conversion, and the next head's rows as they come, so rows are
// read once and the table's rows once for a group of heads.
//
// Bound: memory (rows in, codes out) as long as the rotation is cheap: rot_odd takes sixteen instructions
// a value.  rot_near's four, for two values at a time, decide every code but those whose value lies within
// kRotTol of a border of two codes (one in 10^5), and the scale unless the maximum lies that near to
// 448 * 2^e; those are worked out again with rot_odd, from memory, so that the usual path keeps its
// registers.  bf16, 32768 rows of 32 + 32 + 32 heads of 128, pages of 64: 322 us, 4.2 TB/s (520 us with
// scalar arithmetic and rows loaded when they are due); f32, 4096 rows: 77 us, 3.9 TB/s.  What is left is
// the wait for a head's rows and for its maximum (the barrier); half the issue slots are idle.  Rows
// three heads ahead through shared memory gave 314 us, and 95 us for f32: not worth their memory.
// 1024 threads of an SM with 64 registers each; f32 rows, twice as long, 512 with 128 where a page allows
// (4096 rows: 77 us, with 1024 and spills 82).
template <typename T, int N>
constexpr int kAppendCtas = (sizeof(T) == 2 || N == 1024 ? 1024 : 512) / N;

template <typename T, int HD, int kAppendThreads>
__global__ void __launch_bounds__(kAppendThreads, kAppendCtas<T, kAppendThreads>)
    kv_append_kernel(const dfb_kv_cache c, const dfb_kv_rows r, int heads, bool vec, int32_t *status) {
    constexpr int IPR = HD / 16;  // items per row
    __shared__ uint32_t red[3];
    __shared__ uint32_t written[4];
    __shared__ int first_of[128];  // at given positions: the first row of a slot (positions out of order may repeat one)
    const int s = blockIdx.z, P = c.page, tid = threadIdx.x;
    const int groups = (c.n_kv + heads - 1) / heads;  // blocks of the K heads
    const int sec = (int)blockIdx.y < groups ? 0 : (int)blockIdx.y < 2 * groups ? 1 : 2;
    const int head0 = (blockIdx.y - (sec == 0 ? 0 : sec == 1 ? groups : 2 * groups)) * heads, head1 = min(head0 + heads, sec == 2 ? r.n_q : c.n_kv);
    auto flag = [&](int bit) { if (status) atomicOr(status, bit); };
    const bool reporter = blockIdx.x == 0 && blockIdx.y == 0;  // one block per sequence reports on its rows
    // the sequence's rows
    int a = r.row_off[s], b = r.row_off[s + 1];
    const int len = r.len[s];
    if (a < 0 || b < a || b > r.n_rows || b - a > r.max_rows) {
        if (reporter && tid == 0) flag(DFB_STAT_ROWS);
        a = min(max(a, 0), r.n_rows);
        b = min(max(b, a), r.n_rows);
        b = a + min(b - a, r.max_rows);
    }
    if (a == b) return;
    const int cap = c.max_pages * P, limit = r.rope ? min(cap, r.n_rope) : cap;
    if (len < 0 || len > cap) {  // nothing of the sequence is stored
        if (reporter && tid == 0) flag(DFB_STAT_POSITION);
        return;
    }
    // positions of the rows: first + (row - a), or pos[row]
    const int first = r.pos ? r.pos[a] : len;
    const long long last = r.pos ? r.pos[b - 1] : (long long)len + (b - a - 1);
    if (reporter && (first < 0 || last >= limit) && tid == 0) flag(DFB_STAT_POSITION);
    if (reporter && r.pos)
        for (int i = a + 1 + tid; i < b; i += kAppendThreads)
            if (r.pos[i] <= r.pos[i - 1]) flag(DFB_STAT_POSITION);
    const long long pg = (long long)max(first, 0) / P + blockIdx.x;  // page of the sequence
    if (pg >= c.max_pages || pg * P > last || pg * P >= limit) return;
    const int p0 = (int)pg * P;
    int lo, hi;
    if (r.pos) {
        lo = lower_bound(r.pos, a, b, p0);
        hi = lower_bound(r.pos, lo, b, p0 + P);
    } else {
        lo = a + max(0, p0 - len);
        hi = min((long long)b, (long long)a + p0 + P - len);
    }
    hi = min(hi, lo + P);
    if (lo >= hi) return;
    const int pid = c.pages[(size_t)s * c.max_pages + pg];
    if (pid < 0 || pid >= c.n_pages) {
        if (tid == 0) flag(DFB_STAT_PAGE);
        return;
    }
    // slot of a row in the page, -1: left out (out of range, or not after the row before it)
    auto slot_of = [&](int row) {
        const int p = r.pos ? r.pos[row] : len + (row - a);
        const bool ok = p >= p0 && p < p0 + P && p < limit && !(r.pos && row > a && r.pos[row - 1] >= p);
        return ok ? p - p0 : -1;
    };
    const int64_t tok = sec == 0 ? r.k_tok : sec == 1 ? r.v_tok : r.q_tok, head_st = sec == 0 ? r.k_head : sec == 1 ? r.v_head : r.q_head;
    const T *src0 = reinterpret_cast<const T *>(sec == 0 ? r.k : sec == 1 ? r.v : r.q);
    const bool rotate = r.rope && sec != 1;

    if (tid < 4) written[tid] = 0;
    if (tid < 3) red[tid] = 0;
    if (r.pos && tid < P) first_of[tid] = 0x7fffffff;
    __syncthreads();
    const int row = lo + tid / IPR, i = (tid % IPR) * 8;
    int slot = row < hi ? slot_of(row) : -1;
    const T *src = src0 + row * tok + i;
    auto table = [&] { return r.rope + ((size_t)(p0 + slot) * (HD / 2) + i) * 2; };  // the item's cos and sin
    float2 cs[4], sn[4];
    RawItem<T> raw;
    if (slot >= 0) {
        raw.load(src + head0 * head_st, HD, vec);
        if (i == 0) {
            atomicOr(&written[slot >> 5], 1u << (slot & 31));
            if (r.pos) atomicMin(&first_of[slot], row);
        }
        if (rotate) {
            const float4 *t = reinterpret_cast<const float4 *>(table());
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float4 v = __ldg(t + e);
                cs[e] = make_float2(v.x, v.z);
                sn[e] = make_float2(v.y, v.w);
            }
        }
    }
    __syncthreads();
    if (r.pos) {
        if (!(written[0] | written[1] | written[2] | written[3])) return;
        if (slot >= 0 && first_of[slot] != row) slot = -1;
    }
    const int kept = min(max(len - p0, 0), P);  // filled positions of the page; those written now do not survive
    bool survive = false;
    for (int t = 0; t < kept; t += 32) {
        const uint32_t all = kept - t >= 32 ? 0xffffffffu : (1u << (kept - t)) - 1;
        survive |= (all & ~written[t >> 5]) != 0;
    }
    // value e of the item or its partner, rounded to odd; near: to the nearest f32
    auto exact = [&](int head, int e, bool second, float &near) {
        const T *p = src + head * head_st + e;
        const float u = to_f32<T>(p[0]), w = to_f32<T>(p[HD / 2]), cc = table()[2 * e], ss = table()[2 * e + 1];
        return second ? rot_odd(u, ss, w, cc, near) : rot_odd(u, cc, w, -ss, near);
    };
    // The block's maximum of values >= 0, for head n of the block: their bits, which have the same order.
    // Three words take turns, so that one barrier a head is enough: the one that head n - 1 has read is
    // cleared for head n + 2.
    auto block_max = [&](float v, int n) {
        const uint32_t u = __reduce_max_sync(0xffffffffu, __float_as_uint(v));
        if ((tid & 31) == 0) atomicMax(&red[n % 3], u);
        __syncthreads();
        if (tid == 0) red[(n + 2) % 3] = 0;
        return __uint_as_float(red[n % 3]);
    };
    bool bad = false;
    for (int head = head0; head < head1; head++) {
        float2 x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = raw.pair(e);
        if (slot >= 0 && head + 1 < head1) raw.load(src + (head + 1) * head_st, HD, vec);
        if (rotate) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (sizeof(T) == 4 && sec == 2) {  // f32 rows for the caller: the nearest f32
                    const float2 a = x[e], b = x[4 + e];
                    rot_odd(a.x, cs[e].x, b.x, -sn[e].x, x[e].x);
                    rot_odd(a.y, cs[e].y, b.y, -sn[e].y, x[e].y);
                    rot_odd(a.x, sn[e].x, b.x, cs[e].x, x[4 + e].x);
                    rot_odd(a.y, sn[e].y, b.y, cs[e].y, x[4 + e].y);
                } else rot_near(x[e], x[4 + e], cs[e], sn[e]);
            }
        }
        if (sec == 2) {
            if (slot < 0) continue;
            T *dst = reinterpret_cast<T *>(r.q_out) + row * r.q_out_tok + head * r.q_out_head + i;
            RawItem<T> y;
#pragma unroll
            for (int e = 0; e < 8; e++) y.set(e, x[e]);
            y.store(dst, HD, vec);
            continue;
        }
        const size_t blk = (size_t)pid * c.n_kv + head;
        float *scale = (sec == 0 ? c.k_scale : c.v_scale) + blk;
        uint8_t *codes = reinterpret_cast<uint8_t *>(sec == 0 ? c.k : c.v) + blk * P * HD;
        const int old = survive ? scale_exp(*scale) : 0;  // (every thread has it before block_max lets one write)
        float amax = 0.f;
        if (slot >= 0) {
#pragma unroll
            for (int e = 0; e < 8; e++) amax = max3_nan(amax, fabsf(x[e].x), fabsf(x[e].y));
            if (!(amax < INFINITY)) {  // the finite values' maximum; NaN is stored as 0, infinities as the largest code
                bad = true;
                amax = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    x[e].x = x[e].x != x[e].x ? 0.f : x[e].x;
                    x[e].y = x[e].y != x[e].y ? 0.f : x[e].y;
                    amax = fmaxf(amax, fmaxf(fabsf(x[e].x) < INFINITY ? fabsf(x[e].x) : 0.f, fabsf(x[e].y) < INFINITY ? fabsf(x[e].y) : 0.f));
                }
            }
        }
        amax = block_max(amax, head - head0);
        int e = need_exp(rotate ? amax * (1.f + kRotTol) : amax);
        if (rotate && e > -64 && amax * (1.f - kRotTol) <= 448.f * exp2i(e - 1)) {  // (the same for the whole block)
            amax = 0.f;
            if (slot >= 0) {
#pragma unroll 1
                for (int e = 0; e < 16; e++) {
                    float n;
                    const float v = fabsf(exact(head, e & 7, e & 8, n));
                    if (v < INFINITY) amax = fmaxf(amax, v);
                }
            }
            __syncthreads();
            if (tid == 0) red[(head - head0) % 3] = 0;
            __syncthreads();
            e = need_exp(block_max(amax, head - head0));
        }
        if (survive) {
            if (old >= e) e = old;
            else {  // grown: re-round the kept codes
                const float f = exp2i(max(old - e, -126));
                for (int it = tid; it < kept * (HD / 4); it += kAppendThreads) {
                    const int t = it / (HD / 4);
                    if (written[t >> 5] >> (t & 31) & 1) continue;
                    uint32_t *w = reinterpret_cast<uint32_t *>(codes + t * HD) + it % (HD / 4);
                    const uint32_t v = *w;
                    *w = e4m3_pair(e4m3_value(v & 255) * f, e4m3_value(v >> 8 & 255) * f) |
                         e4m3_pair(e4m3_value(v >> 16 & 255) * f, e4m3_value(v >> 24) * f) << 16;
                }
            }
        }
        if (tid == 0) *scale = exp2i(e);
        if (slot < 0) continue;
        const float inv = exp2i(-e);
        uint8_t *dst = codes + slot * HD + i;
        // rotated: a little more and a little less have the same code, or a border lies between
        const float up = rotate ? inv * (1.f + kRotTol) : inv, down = rotate ? inv * (1.f - kRotTol) : inv;
        const uint2 w0 = encode8(&x[0], up), w1 = encode8(&x[4], up);
        if (rotate) {
            const uint2 b0 = encode8(&x[0], down), b1 = encode8(&x[4], down);
            if ((w0.x ^ b0.x) | (w0.y ^ b0.y) | (w1.x ^ b1.x) | (w1.y ^ b1.y)) {
#pragma unroll 1
                for (int e = 0; e < 16; e++) {
                    float n;
                    const float v = exact(head, e & 7, e & 8, n);
                    dst[(e & 8) * (HD / 16) + (e & 7)] = (uint8_t)e4m3_pair(v != v ? 0.f : v * inv, 0.f);
                }
                continue;
            }
        }
        *reinterpret_cast<uint2 *>(dst) = w0;
        *reinterpret_cast<uint2 *>(dst + HD / 2) = w1;
    }
    if (bad) flag(DFB_STAT_NONFINITE);
}

}  // namespace dfb
