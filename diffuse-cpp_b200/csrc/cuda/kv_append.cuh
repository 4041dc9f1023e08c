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

#include "../../../include/diffuse_b200.h"

namespace dfb {

template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

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

constexpr int kAppendThreads = 256;

// One block: the rows that fall into one page of one sequence (the blockIdx.x-th touched page of
// sequence blockIdx.z), for one head: K heads, then V heads, then query heads (blockIdx.y).  An
// item is eight values and their rotation partners; a thread holds its items in registers
// between the maximum and the conversion, so the rows are read once.
template <typename T, int HD, int ITEMS>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const dfb_kv_cache c, const dfb_kv_rows r, bool vec,
                                                                   int32_t *status) {
    constexpr int IPR = HD / 16;  // items per row
    __shared__ float red[kAppendThreads / 32];
    __shared__ uint32_t written[4];
    const int s = blockIdx.z, P = c.page, tid = threadIdx.x;
    const int sec = (int)blockIdx.y < c.n_kv ? 0 : (int)blockIdx.y < 2 * c.n_kv ? 1 : 2;
    const int head = blockIdx.y - (sec == 0 ? 0 : sec == 1 ? c.n_kv : 2 * c.n_kv);
    auto flag = [&](int bit) { if (status) atomicOr(status, bit); };
    const bool reporter = blockIdx.x == 0 && blockIdx.y == 0;  // one block per sequence reports on its rows
    // the sequence's rows
    int a = r.row_off[s], b = r.row_off[s + 1];
    const int len = r.len[s];
    if (a < 0 || b < a || b > r.n_rows || b - a > r.max_rows) {
        if (reporter && tid == 0) flag(DFB_STAT_ROWS);
        a = min(max(a, 0), r.n_rows);
        b = min(min(max(b, a), r.n_rows), a + r.max_rows);
    }
    if (a == b) return;
    const int cap = c.max_pages * P, limit = r.rope ? min(cap, r.n_rope) : cap;
    if (len < 0 || len > cap) {  // nothing of the sequence is stored
        if (reporter && tid == 0) flag(DFB_STAT_POSITION);
        return;
    }
    // positions of the rows: first + (row - a), or pos[row]
    const int first = r.pos ? r.pos[a] : len, last = r.pos ? r.pos[b - 1] : len + (b - a - 1);
    if (reporter && (first < 0 || last >= limit) && tid == 0) flag(DFB_STAT_POSITION);
    if (reporter && r.pos)
        for (int i = a + 1 + tid; i < b; i += kAppendThreads)
            if (r.pos[i] <= r.pos[i - 1]) flag(DFB_STAT_POSITION);
    const long long pg = (long long)max(first, 0) / P + blockIdx.x;  // page of the sequence
    if (pg >= c.max_pages || pg * P > last) return;
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
    const T *src = reinterpret_cast<const T *>(sec == 0 ? r.k : sec == 1 ? r.v : r.q);
    const int64_t tok = sec == 0 ? r.k_tok : sec == 1 ? r.v_tok : r.q_tok;
    src += head * (sec == 0 ? r.k_head : sec == 1 ? r.v_head : r.q_head);
    const bool rotate = r.rope && sec != 1;

    if (tid < 4) written[tid] = 0;
    __syncthreads();
    float x[ITEMS][16], amax = 0.f;
    int slot[ITEMS];
    bool bad = false;
#pragma unroll
    for (int j = 0; j < ITEMS; j++) {
        const int it = tid + j * kAppendThreads, row = lo + it / IPR, i = (it % IPR) * 8;
        slot[j] = row < hi ? slot_of(row) : -1;
        if (slot[j] < 0) continue;
        float u[8], w[8];
        load8(src + row * tok + i, vec, u);
        load8(src + row * tok + i + HD / 2, vec, w);
        if (rotate) {
            const float4 *cs = reinterpret_cast<const float4 *>(r.rope + ((size_t)(p0 + slot[j]) * (HD / 2) + i) * 2);
            float nu[8], nw[8];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float4 t = cs[e];
                float x0 = rot_odd(u[2 * e], t.x, w[2 * e], -t.y, nu[2 * e]), x1 = rot_odd(u[2 * e], t.y, w[2 * e], t.x, nw[2 * e]);
                u[2 * e] = x0; w[2 * e] = x1;
                x0 = rot_odd(u[2 * e + 1], t.z, w[2 * e + 1], -t.w, nu[2 * e + 1]);
                x1 = rot_odd(u[2 * e + 1], t.w, w[2 * e + 1], t.z, nw[2 * e + 1]);
                u[2 * e + 1] = x0; w[2 * e + 1] = x1;
            }
            if (sec == 2 && sizeof(T) == 4) {
#pragma unroll
                for (int e = 0; e < 8; e++) { u[e] = nu[e]; w[e] = nw[e]; }
            }
        }
        if (sec == 2) {
            T *dst = reinterpret_cast<T *>(r.q_out) + row * r.q_out_tok + head * r.q_out_head + i;
            store8(dst, vec, u);
            store8(dst + HD / 2, vec, w);
            continue;
        }
        if (i == 0) atomicOr(&written[slot[j] >> 5], 1u << (slot[j] & 31));
#pragma unroll
        for (int e = 0; e < 8; e++) {
            x[j][e] = u[e];
            x[j][8 + e] = w[e];
        }
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const float m = fabsf(x[j][e]);
            if (m < INFINITY) amax = fmaxf(amax, m);
            else {
                bad = true;
                if (m != m) x[j][e] = 0.f;
            }
        }
    }
    if (sec == 2) return;
    if (bad) flag(DFB_STAT_NONFINITE);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if ((tid & 31) == 0) red[tid >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; w++) amax = fmaxf(amax, red[w]);

    const size_t blk = (size_t)pid * c.n_kv + head;
    float *scale = (sec == 0 ? c.k_scale : c.v_scale) + blk;
    uint8_t *codes = reinterpret_cast<uint8_t *>(sec == 0 ? c.k : c.v) + blk * P * HD;
    int e = need_exp(amax);
    const int kept = min(max(len - p0, 0), P);  // filled positions of the page; those written now do not survive
    bool survive = false;
    for (int t = 0; t < kept; t += 32) {
        const uint32_t all = kept - t >= 32 ? 0xffffffffu : (1u << (kept - t)) - 1;
        survive |= (all & ~written[t >> 5]) != 0;
    }
    if (survive) {
        const int old = scale_exp(*scale);
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
    __syncthreads();  // every thread has read the old scale
    if (tid == 0) *scale = exp2i(e);
    const float inv = exp2i(-e);
#pragma unroll
    for (int j = 0; j < ITEMS; j++) {
        if (slot[j] < 0) continue;
        const int i = ((tid + j * kAppendThreads) % IPR) * 8;
        uint8_t *dst = codes + slot[j] * HD + i;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float *v = &x[j][8 * h];
            uint2 w;
            w.x = e4m3_pair(v[0] * inv, v[1] * inv) | e4m3_pair(v[2] * inv, v[3] * inv) << 16;
            w.y = e4m3_pair(v[4] * inv, v[5] * inv) | e4m3_pair(v[6] * inv, v[7] * inv) << 16;
            *reinterpret_cast<uint2 *>(dst + h * (HD / 2)) = w;
        }
    }
}

}  // namespace dfb
