// Attention over the paged 8-bit K/V cache (dfb_kv_attention).
//   s_j = scale * q . k_j,  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  lse = m + log sum
// over the first min(vis, len) keys; k_j, v_j = code * scale of the page and KV head.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cstdint>

#include "../../../include/diffuse_b200.h"
#include "kv_append.cuh"

namespace dfb {

// The plain kernel: one warp per query row and head, one key at a time, f32 throughout.
template <typename T, int HD>
__global__ void __launch_bounds__(128) kv_attn_simple(const dfb_kv_cache c, const dfb_kv_attn a, int32_t *status) {
    constexpr int E = HD / 32;
    const int s = blockIdx.z, h = blockIdx.y, lane = threadIdx.x & 31, t = blockIdx.x * 4 + (threadIdx.x >> 5);
    int r0 = a.row_off[s], r1 = a.row_off[s + 1], len = a.len[s];
    if (r0 < 0 || r1 < r0 || r1 > a.n_rows || r1 - r0 > a.max_rows) {
        if (threadIdx.x == 0 && status) atomicOr(status, DFB_STAT_ROWS);
        r0 = min(max(r0, 0), a.n_rows);
        r1 = min(min(max(r1, r0), a.n_rows), r0 + a.max_rows);
    }
    if (len < 0 || len > min((long long)a.max_keys, (long long)c.max_pages * c.page)) {
        if (threadIdx.x == 0 && status) atomicOr(status, DFB_STAT_POSITION);
        len = min((long long)max(len, 0), min((long long)a.max_keys, (long long)c.max_pages * c.page));
    }
    if (t >= r1 - r0) return;
    const int row = r0 + t, kvh = h / (a.n_q / c.n_kv);
    const int n = a.vis ? min(max(a.vis[row], 0), len) : len;
    const T *q = reinterpret_cast<const T *>(a.q) + row * a.q_tok + h * a.q_head;
    float qv[E], o[E] = {}, m = -INFINITY, l = 0.f;
    for (int e = 0; e < E; e++) qv[e] = to_f32<T>(q[lane * E + e]);
    for (int j = 0; j < n; j++) {
        const int pid = c.pages[(size_t)s * c.max_pages + j / c.page];
        if (pid < 0 || pid >= c.n_pages) {
            if (lane == 0 && status) atomicOr(status, DFB_STAT_PAGE);
            continue;
        }
        const size_t blk = (size_t)pid * c.n_kv + kvh, at = (blk * c.page + j % c.page) * HD + lane * E;
        float d = 0.f;
        for (int e = 0; e < E; e++) d += qv[e] * e4m3_value(reinterpret_cast<const uint8_t *>(c.k)[at + e]);
        for (int x = 16; x > 0; x >>= 1) d += __shfl_xor_sync(0xffffffffu, d, x);
        d *= a.scale * c.k_scale[blk];
        const float mn = fmaxf(m, d), f = expf(m - mn), p = expf(d - mn);
        l = l * f + p;
        m = mn;
        const float pv = p * c.v_scale[blk];
        for (int e = 0; e < E; e++) o[e] = o[e] * f + pv * e4m3_value(reinterpret_cast<const uint8_t *>(c.v)[at + e]);
    }
    T *out = reinterpret_cast<T *>(a.out) + row * a.out_tok + h * a.out_head;
    for (int e = 0; e < E; e++) out[lane * E + e] = from_f32<T>(l > 0.f ? o[e] / l : 0.f);
    if (a.lse && lane == 0) a.lse[(size_t)row * a.n_q + h] = l > 0.f ? m + logf(l) : -INFINITY;
}

}  // namespace dfb
