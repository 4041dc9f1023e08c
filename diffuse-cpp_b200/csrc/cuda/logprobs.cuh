// Log probabilities of given tokens, entropy and top alternatives of logits rows
// (dfb_token_logprobs).  With m = max x and z = sum exp(x - m):
//   log p_t = (x_t - m) - log z,   H = log z + sum exp(x - m) (m - x) / z,
// both terms of H non-negative, so nothing cancels.
#pragma once
#include <cstdint>

#include "../../../include/diffuse_b200.h"
#include "kv_append.cuh"
#include "ptx.cuh"

namespace dfb {

constexpr int kLpThreads = 512;

// The plain kernel: one block per row, one pass for m, z and the entropy sum, then one pass per
// alternative (the largest key below the last one; a key orders by value, then lower id).
template <typename T>
__global__ void __launch_bounds__(kLpThreads) logprobs_simple(const dfb_logprob_args a, int32_t *status) {
    __shared__ float sm[16], sz[16], st[16];
    __shared__ unsigned long long sk[16];
    const int i = blockIdx.x, V = a.n_vocab, tid = threadIdx.x;
    auto flag = [&](int bit) { if (status && tid == 0) atomicOr(status, bit); };
    const int row = a.rows ? a.rows[i] : i;
    const bool there = row >= 0 && row < a.n_logits;
    if (!there) flag(DFB_STAT_TARGET);
    const T *x = reinterpret_cast<const T *>(a.logits) + (size_t)(there ? row : 0) * a.ld;
    float m = -INFINITY, z = 0.f, t = 0.f;
    bool bad = !there;
    auto join = [](float &m, float &z, float &t, float m2, float z2, float t2) {
        if (m2 == -INFINITY) return;
        if (m == -INFINITY) { m = m2; z = z2; t = t2; return; }
        const float mn = fmaxf(m, m2), d1 = fmaxf(m - mn, -1e30f), d2 = fmaxf(m2 - mn, -1e30f), f1 = expf(d1), f2 = expf(d2);
        t = f1 * (t - z * d1) + f2 * (t2 - z2 * d2);  // sum e^(x - mn) (mn - x)
        z = f1 * z + f2 * z2;
        m = mn;
    };
    if (there)
        for (int v = tid; v < V; v += kLpThreads) {
            const float f = to_f32<T>(x[v]);
            if (!(f < INFINITY)) bad = true;
            else join(m, z, t, f, 1.f, 0.f);
        }
    bad = __syncthreads_or(bad);
    for (int o = 16; o > 0; o >>= 1) {
        const float m2 = __shfl_xor_sync(0xffffffffu, m, o), z2 = __shfl_xor_sync(0xffffffffu, z, o), t2 = __shfl_xor_sync(0xffffffffu, t, o);
        join(m, z, t, m2, z2, t2);
    }
    if ((tid & 31) == 0) { sm[tid >> 5] = m; sz[tid >> 5] = z; st[tid >> 5] = t; }
    __syncthreads();
    m = -INFINITY; z = 0.f; t = 0.f;
    for (int w = 0; w < kLpThreads / 32; w++) join(m, z, t, sm[w], sz[w], st[w]);
    if (bad && there) flag(DFB_STAT_LOGITS);
    const float lz = logf(z);
    auto lp = [&](float f) { return bad ? NAN : m == -INFINITY ? -INFINITY : (f - m) - lz; };
    if (tid == 0) {
        if (a.entropy) a.entropy[i] = bad ? NAN : m == -INFINITY ? 0.f : lz + t / z;
        if (a.logprob) {
            const int tg = a.targets[i];
            if (tg >= V) flag(DFB_STAT_TARGET);
            a.logprob[i] = tg < 0 ? 0.f : tg >= V ? NAN : lp(to_f32<T>(x[tg]));
        }
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < a.top_k; k++) {
        unsigned long long best = 0;
        if (!bad)
            for (int v = tid; v < V; v += kLpThreads) {
                const uint32_t u = __float_as_uint(to_f32<T>(x[v]) + 0.f);
                const unsigned long long key = (unsigned long long)((u & 0x80000000u) ? ~u : u | 0x80000000u) << 32 | (0xffffffffu - v);
                if (key < last && key > best) best = key;
            }
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long b2 = __shfl_xor_sync(0xffffffffu, best, o);
            best = b2 > best ? b2 : best;
        }
        __syncthreads();
        if ((tid & 31) == 0) sk[tid >> 5] = best;
        __syncthreads();
        for (int w = 0; w < kLpThreads / 32; w++) best = sk[w] > best ? sk[w] : best;
        last = best;
        if (tid == 0) {
            const int id = bad ? -1 : (int)(0xffffffffu - (uint32_t)best);
            a.top_ids[(size_t)i * a.top_k + k] = id;
            a.top_logprob[(size_t)i * a.top_k + k] = bad ? NAN : lp(to_f32<T>(x[id]));
        }
    }
}

}  // namespace dfb
