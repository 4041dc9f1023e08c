// Log probabilities of given tokens, entropy and top alternatives of logits rows
// (dfb_token_logprobs), in one pass over the row.
//
// With m = max x, z = sum 2^y and t = sum -y 2^y over y = (x - m) log2(e):
//   log p_t = (x_t - m) - ln z,   H = ln z + ln 2 t / z,
// both terms of H non-negative, so nothing cancels.  A thread carries (m, z, t) of its elements and
// rescales when a batch of them raises m; the parts are joined in a fixed order.  y is held above -200,
// where 2^y is 0 in f32, so that logits of -inf add 0 to t; a NaN or +inf makes z NaN.
//
// Alternatives.  An element's key orders by value, then lower id.  The first batch, spread over the
// whole row, gives a threshold: the k-th largest of 32 groups' largest keys, no larger than the row's
// k-th key.  What passes it (some tens of elements; a batch's largest value tells whether it is worth a
// look) goes to a list in shared memory, whose members' ranks are counted in the end.  A row that
// overflows the list (ascending logits, say) is gone through again with a threshold that rises.
//
// Bound: the row read once from memory, and issue slots beside it: four instructions and one ex2 a value,
// one more for the batch's largest, two more where alternatives are wanted.  2048 rows of 152064 bf16:
// 176 us, 3.5 TB/s (138 us without alternatives); 256 rows of 126464 f32: 34 us, 3.8 TB/s (30).  A row is
// split over the CTAs of a cluster (joined through distributed shared memory) where rows alone would leave
// SMs without work: one row of 126464 in 8 CTAs takes 13 us (10 without alternatives).  Rows of one large
// value alone (2048 x 152064 of -1e10) overflow the list and take 1006 us.
#pragma once
#include <cstdint>
#include <type_traits>

#include "../../../include/diffuse_b200.h"
#include "kv_append.cuh"
#include "ptx.cuh"
#include "simd.cuh"

namespace dfb {

constexpr int kLpThreads = 256, kLpCtas = 4 /* of an SM */, kLpWarps = kLpThreads / 32, kLpMaxK = 32, kLpCap = 4096, kLpFew = 256;
constexpr float kLpLn2 = 0.6931471805599453f, kLpLog2e = 1.4426950408889634f, kLpFloor = -200.f;

struct LpSmem {
    unsigned long long list[kLpCap];
    unsigned long long top[kLpMaxK];      // this CTA's k largest keys, in order
    unsigned long long group[32];
    float m[kLpWarps], z[kLpWarps], t[kLpWarps];
    float part[3];                        // this CTA's m, z, t
    int count, n_top, kept;
};

__device__ __forceinline__ unsigned long long lp_key(float x, int id) {
    const uint32_t u = __float_as_uint(x + 0.f);  // (one zero)
    return (unsigned long long)((u & 0x80000000u) ? ~u : u | 0x80000000u) << 32 | (0xffffffffu - (uint32_t)id);
}
__device__ __forceinline__ float lp_value(unsigned long long key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int lp_id(unsigned long long key) { return (int)(0xffffffffu - (uint32_t)key); }
// A word of the same variable in CTA `rank` of the cluster.
__device__ __forceinline__ float ld_cluster_f32(const float *p, int rank) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ int ld_cluster_s32(const int *p, int rank) {
    int v;
    asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ unsigned long long ld_cluster_u64(const unsigned long long *p, int rank) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(p, rank)) : "memory");
    return v;
}

// Sums relative to 2^b, b = m log2(e) rounded: y = x log2(e) - b is one fused multiply-add.  With the
// offset d = m log2(e) - b the sum relative to m is z 2^-d, and b's rounding leaves ln z + ln 2 t / z as it
// is.  d is up to half a unit in the last place of b, so this holds up to kLpNarrow only, where |d| <= 2^-4;
// a larger m (a row or a part of one filled with -1e10, say) would send 2^d out of f32's range.  There
// y = (x - m) log2(e) and d = 0.
constexpr float kLpNarrow = 1048576.f;  // 2^20
struct LpSum {
    float m = -3.402823466e38f, z = 0.f, t = 0.f;  // (z = 0: nothing but -inf so far)
    __device__ __forceinline__ static bool wide(float m) { return fabsf(m) > kLpNarrow; }
    // (a product that the compiler may not fuse with the subtraction that follows it: b is a rounded value)
    __device__ __forceinline__ static float base(float m) { return __fmul_rn(m, kLpLog2e); }
    __device__ __forceinline__ static float offset(float m) { return wide(m) ? 0.f : fmaf(m, kLpLog2e, -base(m)); }
    // log2 of what a sum relative to `from` is worth relative to `to` (to >= from)
    __device__ __forceinline__ static float shift(float from, float to) {
        if (from == to) return 0.f;
        if (wide(from) || wide(to)) return max_nan(fmaf(from - to, kLpLog2e, offset(to) - offset(from)), kLpFloor);
        return max_nan(base(from) - base(to), kLpFloor);
    }
    __device__ __forceinline__ void raise(float mn) {  // mn >= m
        const float y = shift(m, mn), f = ex2(y);
        t = f * fmaf(-y, z, t);
        z *= f;
        m = mn;
    }
    __device__ __forceinline__ void join(LpSum o) {
        if (o.m > m) raise(o.m);
        else o.raise(m);
        z += o.z;
        t += o.t;
    }
    __device__ __forceinline__ float log_z() const {  // ln of the sum relative to m
        return fmaf(-offset(m), kLpLn2, logf(z));
    }
    __device__ __forceinline__ float entropy() const { return fmaf(t / z, kLpLn2, logf(z)); }
    __device__ __forceinline__ void add1(float f) {
        if (f > m) raise(f);
        const float y = max_nan(wide(m) ? (f - m) * kLpLog2e : fmaf(f, kLpLog2e, -base(m)), kLpFloor), p = ex2(y);
        z += p;
        t = fmaf(-y, p, t);
    }
};

// One batch: 16 values of a thread, in NV 16-byte pieces.
template <typename T>
struct LpBatch {
    static constexpr int PER = 16 / sizeof(T), N = 16, NV = N / PER;
    uint4 raw[NV];
    __device__ __forceinline__ uint32_t word(int i) const {
        const uint4 &u = raw[i / 4];
        return i % 4 == 0 ? u.x : i % 4 == 1 ? u.y : i % 4 == 2 ? u.z : u.w;
    }
    __device__ __forceinline__ static float half_of(uint32_t h, int e) {  // of two 16-bit values
        if constexpr (std::is_same<T, __nv_bfloat16>::value) return __uint_as_float(e ? h & 0xffff0000u : h << 16);
        const __half2 p = *reinterpret_cast<const __half2 *>(&h);
        return e ? __high2float(p) : __low2float(p);
    }
    __device__ __forceinline__ float at(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(word(i));
        return half_of(word(i / 2), i % 2);
    }
    // Values 2 i and 2 i + 1 where i is not known to the compiler.
    __device__ __forceinline__ float2 pair(int i) const {
        constexpr int W = sizeof(T) / 2;  // words of a pair
        uint32_t w[W];
#pragma unroll
        for (int e = 0; e < W; e++) {
            w[e] = word(e);
#pragma unroll
            for (int c = 1; c < N / 2; c++) w[e] = c == i ? word(W * c + e) : w[e];
        }
        if constexpr (W == 2) return make_float2(__uint_as_float(w[0]), __uint_as_float(w[1]));
        return make_float2(half_of(w[0], 0), half_of(w[0], 1));
    }
};

// A key above the threshold goes to the list; full: it is counted only.
__device__ __forceinline__ void lp_push(LpSmem &s, unsigned long long key) {
    const int at = atomicAdd(&s.count, 1);
    if (at < kLpCap) s.list[at] = key;
}
// With mine the largest key of group `lane` (32 groups of one set): the k-th largest of them, no larger
// than the set's k-th key (0: fewer than k groups have one).  first: the largest.
__device__ __forceinline__ unsigned long long lp_kth_group(const LpSmem &s, int k, unsigned long long *first = nullptr) {
    const int lane = threadIdx.x & 31;
    const unsigned long long mine = s.group[lane];
    int r = 0;
#pragma unroll
    for (int j = 0; j < 32; j++) {
        const unsigned long long c = s.group[j];
        r += c > mine || (c == mine && j < lane);
    }
    if (first) *first = __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, r == 0)) - 1);
    return k > 0 ? __shfl_sync(0xffffffffu, mine, __ffs(__ballot_sync(0xffffffffu, r == k - 1)) - 1) : 0;
}
// A group is eight threads: each gives its largest key.
__device__ __forceinline__ void lp_group_max(LpSmem &s, unsigned long long key) {
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        const unsigned long long c = __shfl_xor_sync(0xffffffffu, key, o);
        key = c > key ? c : key;
    }
    if ((threadIdx.x & 7) == 0) s.group[threadIdx.x >> 3] = key;
}
// The k largest of the list's n keys (n >= 0, all different) to s.top, in order; every thread of the block
// takes part, and the list is used up.  Counting each key's betters is n^2 steps (3151 keys: 300 us), so
// more than kLpFew of them are first held against the k-th of 32 groups' largest, which leaves some 4 k.
__device__ __forceinline__ void lp_rank(LpSmem &s, int n, int k) {
    const int tid = threadIdx.x;
    for (int pass = 0; n > kLpFew && pass < 4; pass++) {
        unsigned long long key = 0;
        for (int i = tid; i < n; i += kLpThreads) key = s.list[i] > key ? s.list[i] : key;
        lp_group_max(s, key);
        if (tid == 0) s.kept = 0;
        __syncthreads();
        const unsigned long long thr = lp_kth_group(s, k);
        for (int i0 = 0; i0 < n; i0 += kLpThreads) {
            key = i0 + tid < n ? s.list[i0 + tid] : 0;
            __syncthreads();  // (what is kept goes to places that have been read)
            if (key && key >= thr) s.list[atomicAdd(&s.kept, 1)] = key;
        }
        __syncthreads();
        n = s.kept;
        __syncthreads();
    }
    for (int i = tid; i < n; i += kLpThreads) {
        const unsigned long long key = s.list[i];
        int r = 0;
        for (int j = 0; j < n; j++) r += s.list[j] > key;
        if (r < k) s.top[r] = key;
    }
}

// Grid: rows x cluster size; CTA `rank` of a row's cluster takes an equal share of its 16-byte pieces.
template <typename T>
__global__ void __launch_bounds__(kLpThreads, kLpCtas) logprobs_kernel(const dfb_logprob_args a, int32_t *status) {
    using B = LpBatch<T>;
    __shared__ LpSmem s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, V = a.n_vocab, k = a.top_k;
    const int rank = (int)cluster_ctarank(), n_cta = (int)(gridDim.x / (unsigned)a.n_rows), i = blockIdx.x / n_cta;
    auto flag = [&](int bit) { if (status) atomicOr(status, bit); };
    const int row = a.rows ? a.rows[i] : i;
    const bool there = row >= 0 && row < a.n_logits;
    const T *x = reinterpret_cast<const T *>(a.logits) + (size_t)(there ? row : 0) * a.ld;
    // elements before the first 16-byte boundary and behind the last; pieces of this CTA [v0, v1)
    const int head = min(V, (int)((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T)));
    const int pieces = (V - head) / B::PER, tail = head + pieces * B::PER;
    const int v0 = (int)((long long)pieces * rank / n_cta), v1 = (int)((long long)pieces * (rank + 1) / n_cta);
    const uint4 *body = reinterpret_cast<const uint4 *>(x + head);
    const int tg = rank == 0 && a.logprob && there ? a.targets[i] : -1;
    const float xt = tg >= 0 && tg < V ? to_f32<T>(x[tg]) : 0.f;  // (under way beside the row)
    if (tid == 0) {
        s.count = 0;
        s.n_top = 0;
    }
    __syncthreads();
    LpSum sum;
    unsigned long long thr = 0;   // what passes goes to the list
    float thr_x = -INFINITY;      // its value

    // the pieces of a batch lie a quarter (16-bit logits: half) of the range apart
    const int quarter = ((v1 - v0 + B::NV - 1) / B::NV + kLpThreads - 1) / kLpThreads * kLpThreads;  // in pieces
    const int rounds = there ? quarter / kLpThreads : 0;
    const int full = max(0, (v1 - v0 - (B::NV - 1) * quarter) / kLpThreads);  // rounds that are whole in every part
    auto load = [&](B &b, int r) {
        const uint4 *p = body + (v0 + r * kLpThreads + tid);
        if (r < full) {
#pragma unroll
            for (int u = 0; u < B::NV; u++) b.raw[u] = __ldcs(p + u * quarter);
        } else if (r < rounds) {
#pragma unroll
            for (int u = 0; u < B::NV; u++) {
                const uint32_t none = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;  // -inf
                b.raw[u] = make_uint4(none, none, none, none);
                if (v0 + u * quarter + r * kLpThreads + tid < v1) b.raw[u] = __ldcs(p + u * quarter);
            }
        }
    };
    auto id_of = [&](int r, int e) { return head + (v0 + e / B::PER * quarter + r * kLpThreads + tid) * B::PER + e % B::PER; };
    // scalar elements (at most one of each kind a thread): head by the first CTA, tail by the last
    const bool has_head = there && rank == 0 && tid < head, has_tail = there && rank == n_cta - 1 && tid < V - tail;
    const float x_head = has_head ? to_f32<T>(x[tid]) : -INFINITY, x_tail = has_tail ? to_f32<T>(x[tail + tid]) : -INFINITY;
    auto add = [&](const B &b, float bm) {
        if (bm > sum.m) sum.raise(bm);
        float2 z = make_float2(0.f, 0.f), t = z;  // t: of y 2^y
        auto term = [&](float2 y) {
            y = make_float2(max_nan(y.x, kLpFloor), max_nan(y.y, kLpFloor));
            const float2 p = make_float2(ex2(y.x), ex2(y.y));
            z = add2(z, p);
            t = fma2(y, p, t);
        };
        const float2 l2e = make_float2(kLpLog2e, kLpLog2e);
        if (LpSum::wide(sum.m)) {
            const float2 nm = make_float2(-sum.m, -sum.m);
#pragma unroll 1  // (unrolled it costs the usual rows beside it 2 %)
            for (int e = 0; e < B::N / 2; e++) term(mul2(add2(b.pair(e), nm), l2e));
        } else {
            const float nb = -LpSum::base(sum.m);
#pragma unroll
            for (int e = 0; e < B::N; e += 2) term(fma2(make_float2(b.at(e), b.at(e + 1)), l2e, make_float2(nb, nb)));
        }
        sum.z += z.x + z.y;
        sum.t -= t.x + t.y;
    };
    auto largest = [&](const B &b) {
        float m = b.at(0);
#pragma unroll
        for (int e = 1; e + 1 < B::N; e += 2) m = max3(m, b.at(e), b.at(e + 1));
        return fmaxf(m, b.at(B::N - 1));
    };
    auto look = [&](const B &b, int r, float bm) {
        if (bm < thr_x || bm == -INFINITY) return;
        const float least = fmaxf(thr_x, -3.402823466e38f);  // (-inf is no alternative here: see the end)
        uint32_t pass = 0;
#pragma unroll
        for (int e = 0; e < B::N; e++) pass |= b.at(e) >= least ? 1u << e : 0u;
        if ((pass & (pass - 1)) == 0) {  // the usual case: it is the largest (2048 rows 176 us, with the loop alone 180)
            const unsigned long long key = lp_key(bm, id_of(r, __ffs(pass) - 1));
            if (pass && key >= thr) lp_push(s, key);
            return;
        }
        while (pass) {
            const int e = __ffs(pass) - 1;
            pass &= pass - 1;
            float f = b.at(0);
#pragma unroll
            for (int c = 1; c < B::N; c++) f = c == e ? b.at(c) : f;
            const unsigned long long key = lp_key(f, id_of(r, e));
            if (key >= thr) lp_push(s, key);
        }
    };
    auto look1 = [&](float f, int id) {
        if (f > -INFINITY && lp_key(f, id) >= thr) lp_push(s, lp_key(f, id));
    };
    // cuts the list to its k largest and takes the k-th for the threshold
    auto tighten = [&] {
        __syncthreads();
        const int n = s.count;
        __syncthreads();  // (no one adds to it before all have read it)
        if (n < k || n > kLpCap) return;
        lp_rank(s, n, k);
        __syncthreads();
        if (tid < k) s.list[tid] = s.top[tid];
        if (tid == 0) s.count = k;
        thr = s.top[k - 1];
        thr_x = lp_value(thr);
        __syncthreads();
    };
    B cur, nxt;
    load(cur, 0);
    load(nxt, 1);
    if (rounds > 0) {
        const float bm = largest(cur);
        // the 32 largest keys of groups of 8 threads: their k-th is the first threshold, the largest value
        // the m that all threads begin with (with an own one each, some lane of a warp rescales in nearly
        // every batch)
        unsigned long long key = 0;
#pragma unroll
        for (int e = 0; e < B::N; e++)
            if (cur.at(e) == bm && bm > -INFINITY) {
                const unsigned long long c = lp_key(bm, id_of(0, e));
                key = c > key ? c : key;
            }
        lp_group_max(s, key);
        __syncthreads();
        unsigned long long best;
        thr = lp_kth_group(s, k, &best);  // (every warp finds the same)
        if (best) sum.m = lp_value(best);
        if (thr) thr_x = lp_value(thr);
        add(cur, bm);
        if (k > 0) look(cur, 0, bm);
    }
    if (has_head) {
        sum.add1(x_head);
        if (k > 0) look1(x_head, tid);
    }
    if (has_tail) {
        sum.add1(x_tail);
        if (k > 0) look1(x_tail, tail + tid);
    }
    // a threshold from n of the row's elements lets some k (row / n - 1) more pass: it is taken again after
    // 1, 3, 7, ... batches (2048 rows of 152064 with k = 20: 180 us, after 1, 4, 13, ... 184, 1, 6, 31 208, once 332)
    int again = 1;
    auto batch = [&](const B &b, B &spare, int r) {
        load(spare, r + 1);
        if (k > 0 && r == again) {
            tighten();
            again = 2 * again + 1;
        }
        const float bm = largest(b);
        add(b, bm);
        if (k > 0) look(b, r, bm);
    };
    for (int r = 1; r < rounds; r += 2) {
        batch(nxt, cur, r);
        if (r + 1 < rounds) batch(cur, nxt, r + 1);
    }
    // ── the block's sums, its k largest keys ──
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        LpSum p;
        p.m = __shfl_xor_sync(0xffffffffu, sum.m, o);
        p.z = __shfl_xor_sync(0xffffffffu, sum.z, o);
        p.t = __shfl_xor_sync(0xffffffffu, sum.t, o);
        sum.join(p);
    }
    if (lane == 0) { s.m[warp] = sum.m; s.z[warp] = sum.z; s.t[warp] = sum.t; }
    __syncthreads();
    if (warp == 0) {
        sum = LpSum();
        if (lane < kLpWarps) { sum.m = s.m[lane]; sum.z = s.z[lane]; sum.t = s.t[lane]; }
#pragma unroll
        for (int o = kLpWarps / 2; o > 0; o >>= 1) {
            LpSum p;
            p.m = __shfl_xor_sync(0xffffffffu, sum.m, o);
            p.z = __shfl_xor_sync(0xffffffffu, sum.z, o);
            p.t = __shfl_xor_sync(0xffffffffu, sum.t, o);
            sum.join(p);
        }
        if (lane == 0) { s.part[0] = sum.m; s.part[1] = sum.z; s.part[2] = sum.t; }
    }
    if (k > 0) {
        if (s.count > kLpCap) {
            // again, two values a thread at a time, the list cut to its k largest whenever the next two might
            // not fit: the threshold rises to the k-th key so far
            __syncthreads();
            if (tid == 0) s.count = 0;
            __syncthreads();
            auto cut = [&] {
                __syncthreads();
                if (s.count + 2 * kLpThreads > kLpCap) tighten();
                else __syncthreads();
            };
            if (has_head) look1(x_head, tid);
            if (has_tail) look1(x_tail, tail + tid);
            for (int r = 0; r < rounds; r++) {
                load(cur, r);
                for (int e0 = 0; e0 < B::N; e0 += 2) {
                    cut();
#pragma unroll
                    for (int e = 0; e < B::N; e++)
                        if (e / 2 == e0 / 2) look1(cur.at(e), id_of(r, e));
                }
            }
        }
        __syncthreads();
        const int n = min(s.count, kLpCap);
        lp_rank(s, n, k);
        if (tid == 0) s.n_top = min(n, k);
    }
    // ── the cluster's: the first CTA takes the others' ──
    if (n_cta > 1) {
        cluster_sync();
        if (rank == 0) {
            if (tid == 0) {
                sum = LpSum();
                for (int c = 0; c < n_cta; c++) {
                    LpSum p;
                    p.m = ld_cluster_f32(&s.part[0], c);
                    p.z = ld_cluster_f32(&s.part[1], c);
                    p.t = ld_cluster_f32(&s.part[2], c);
                    sum.join(p);
                }
            }
            if (k > 0) {
                if (tid < kLpMaxK * n_cta && tid % kLpMaxK < ld_cluster_s32(&s.n_top, tid / kLpMaxK)) {
                    const unsigned long long key = ld_cluster_u64(&s.top[tid % kLpMaxK], tid / kLpMaxK);
                    s.list[tid] = key;
                } else if (tid < kLpMaxK * n_cta) {
                    s.list[tid] = 0;  // (no key is 0)
                }
            }
        }
        cluster_sync();  // the others' shared memory has been read
        if (rank != 0) return;
        if (k > 0) {
            if (tid == 0) s.count = 0;
            __syncthreads();
            // the keys that are there, to the front (their order does not matter)
            unsigned long long key = tid < kLpMaxK * n_cta ? s.list[tid] : 0;
            __syncthreads();
            if (key) s.list[atomicAdd(&s.count, 1)] = key;
            __syncthreads();
            lp_rank(s, s.count, k);
            if (tid == 0) s.n_top = min(s.count, k);
        }
    } else if (tid == 0) {
        sum.m = s.part[0]; sum.z = s.part[1]; sum.t = s.part[2];
    }
    __syncthreads();
    if (tid == 0) { s.part[0] = sum.m; s.part[1] = sum.z; s.part[2] = sum.t; }
    __syncthreads();
    sum.m = s.part[0]; sum.z = s.part[1]; sum.t = s.part[2];
    const float m = sum.m, z = sum.z, lz = sum.log_z();
    const bool bad = !there || z != z, none = z == 0.f;  // NaN or +inf; nothing but -inf
    auto lp = [&](float f) { return bad ? NAN : none ? -INFINITY : (f - m) - lz; };
    if (tid == 0) {
        if (!there) flag(DFB_STAT_TARGET);
        else if (bad) flag(DFB_STAT_LOGITS);
        if (a.entropy) a.entropy[i] = bad ? NAN : none ? 0.f : sum.entropy();
        if (a.logprob) {
            if (tg >= V) flag(DFB_STAT_TARGET);
            a.logprob[i] = !there ? NAN : tg < 0 ? 0.f : tg >= V ? NAN : lp(xt);
        }
    }
    if (tid < k) {
        const size_t at = (size_t)i * k + tid;
        if (bad) {
            a.top_ids[at] = -1;
            a.top_logprob[at] = NAN;
        } else if (tid < s.n_top) {
            a.top_ids[at] = lp_id(s.top[tid]);
            a.top_logprob[at] = lp(lp_value(s.top[tid]));
        } else {
            // fewer than k logits above -inf: the rest are the lowest ids whose logit is -inf, within the first 2 k
            int left = tid - s.n_top, id = 0;
            for (; id < V; id++)
                if (to_f32<T>(x[id]) == -INFINITY && left-- == 0) break;
            a.top_ids[at] = id;
            a.top_logprob[at] = -INFINITY;
        }
    }
}

}  // namespace dfb
