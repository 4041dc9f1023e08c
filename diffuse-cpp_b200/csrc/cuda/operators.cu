// Entry points of the operators on device tensors (include/diffuse_b200.h): argument checks, the
// choice of a kernel variant, launches.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>

#include "host_util.h"
#include "kv_append.cuh"
#include "kv_attention.cuh"
#include "kv_attention_tc.cuh"
#include "logprobs.cuh"

using namespace dfb;

namespace {

enum { T_F32 = 0, T_F16 = 1, T_BF16 = 30 };
int type_size(int t) { return t == T_F32 ? 4 : 2; }

// The calling thread's device while a call works on another one.
class DeviceGuard {
  public:
    // the device that holds p; false with an error recorded when p is no device memory
    int enter(const void *p, const char *what) {
        cudaPointerAttributes at{};
        const cudaError_t e = cudaPointerGetAttributes(&at, p);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return set_err(e == cudaErrorInvalidValue ? DFB_ERR_ARG : DFB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
        }
        if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
            return set_err(DFB_ERR_ARG, "%s is not device memory", what);
        dev_ = at.device;
        CK(cudaGetDevice(&old_));
        if (old_ != dev_) CK(cudaSetDevice(dev_));
        return DFB_OK;
    }
    ~DeviceGuard() {
        if (old_ >= 0 && old_ != dev_) cudaSetDevice(old_);
    }
    int device() const { return dev_; }

  private:
    int dev_ = -1, old_ = -1;
};

// Compute capability and SM count, looked up once per device.  (Calls of several threads may overlap: what they
// share is atomic, and whoever finds it unset sets it to the same value.)
int device_props(int dev, int *n_sm) {
    static std::atomic<int> sms[64];
    if (dev < 0 || dev >= 64) return set_err(DFB_ERR_UNSUPPORTED, "device %d", dev);
    int n = sms[dev];
    if (!n) {
        int major = 0;
        CK(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
        CK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
        if (major != 10) return set_err(DFB_ERR_UNSUPPORTED, "device %d is sm_%d; this build targets sm_100a", dev, 10 * major);
        sms[dev] = n;
    }
    *n_sm = n;
    return DFB_OK;
}

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check_cache(const dfb_kv_cache *c) {
    if (!c) return set_err(DFB_ERR_ARG, "null cache");
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->pages) return set_err(DFB_ERR_ARG, "null pointer in the cache");
    if (c->head_dim != 64 && c->head_dim != 128) return set_err(DFB_ERR_UNSUPPORTED, "head_dim %d not supported (64/128)", c->head_dim);
    if (c->page != 16 && c->page != 32 && c->page != 64 && c->page != 128)
        return set_err(DFB_ERR_UNSUPPORTED, "page of %d positions not supported (16/32/64/128)", c->page);
    if (c->n_pages <= 0 || c->n_kv <= 0 || c->n_seq <= 0 || c->max_pages <= 0)
        return set_err(DFB_ERR_ARG, "cache of %d pages, %d KV heads, %d sequences of %d pages", c->n_pages, c->n_kv, c->n_seq, c->max_pages);
    if (c->n_seq > 65535 || c->n_kv > 8192) return set_err(DFB_ERR_UNSUPPORTED, "%d sequences / %d KV heads", c->n_seq, c->n_kv);
    if ((int64_t)c->n_pages * c->n_kv * c->page > INT32_MAX) return set_err(DFB_ERR_UNSUPPORTED, "pool of %d pages of %d heads", c->n_pages, c->n_kv);
    if ((int64_t)c->max_pages * c->page > INT32_MAX) return set_err(DFB_ERR_UNSUPPORTED, "page table of %d pages", c->max_pages);
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) return set_err(DFB_ERR_ARG, "cache codes not 16-byte aligned");
    return DFB_OK;
}

// Strides of a [rows][heads][head_dim] tensor of caller memory: not negative (a row is the last one plus).
int check_rows(const char *what, const void *p, int type, int64_t tok, int64_t head) {
    if (!p) return set_err(DFB_ERR_ARG, "null %s", what);
    if (!aligned(p, type_size(type))) return set_err(DFB_ERR_ARG, "%s not aligned to its type", what);
    if (tok < 0 || head < 0) return set_err(DFB_ERR_ARG, "%s has a negative stride", what);
    return DFB_OK;
}
// Whether rows of an output [n][heads][head_dim] share elements (a broadcast view, say): blocks would write them
// at the same time.
bool rows_overlap(int64_t n, int64_t tok, int64_t heads, int64_t head, int hd) {
    if ((n > 1 && tok < hd) || (heads > 1 && head < hd)) return true;
    if (n == 1 || heads == 1) return false;
    const __int128 t = tok, h = head;
    if (t >= (heads - 1) * h + hd || h >= (n - 1) * t + hd) return false;  // one dimension within the other's steps
    for (int64_t i = 1; i < heads; i++) {  // neither: the tokens whose rows of head 0 lie next to token 0's row of head i
        const __int128 at = i * h, k = at / t;
        if ((k < n && at - k * t < hd) || (k + 1 < n && (k + 1) * t - at < hd)) return true;
    }
    return false;
}
int check_out(const char *what, const void *p, int type, int64_t n, int64_t tok, int64_t heads, int64_t head, int hd) {
    RET(check_rows(what, p, type, tok, head));
    if (rows_overlap(n, tok, heads, head, hd))
        return set_err(DFB_ERR_ARG, "%s: rows overlap (strides of %lld and %lld elements)", what, (long long)tok, (long long)head);
    return DFB_OK;
}
// Whether eight consecutive values of every row can be moved as 16-byte pieces.
bool vec_ok(const void *p, int type, int64_t tok, int64_t head) {
    const int64_t n = 16 / type_size(type);
    return aligned(p, 16) && tok % n == 0 && head % n == 0;
}

template <typename T, int HD>
int append_t(const dfb_kv_cache &c, const dfb_kv_rows &r, int64_t pages, int n_sm, bool vec, int32_t *status, cudaStream_t st) {
    // heads of one block: more of them read the table's rows less often, as long as there are four blocks
    // for every SM all the same
    int heads = 8;
    auto blocks_y = [&] { return 2 * ((c.n_kv + heads - 1) / heads) + (r.q ? (r.n_q + heads - 1) / heads : 0); };
    const int64_t filled = std::min<int64_t>(pages * c.n_seq, r.n_rows / c.page + c.n_seq);  // pages with rows, about
    while (heads > 1 && filled * blocks_y() < 4 * n_sm) heads /= 2;
    const dim3 grid((unsigned)pages, blocks_y(), c.n_seq);
    const int items = c.page * (HD / 16);  // of a page: one thread each
    if (items <= 256) kv_append_kernel<T, HD, 256><<<grid, 256, 0, st>>>(c, r, heads, vec, status);
    else if (items <= 512) kv_append_kernel<T, HD, 512><<<grid, 512, 0, st>>>(c, r, heads, vec, status);
    else if constexpr (HD == 128) kv_append_kernel<T, HD, 1024><<<grid, 1024, 0, st>>>(c, r, heads, vec, status);
    CK(cudaGetLastError());
    return DFB_OK;
}

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        cudaDriverEntryPointQueryResult q;
        void *p = nullptr;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}
// The cache's codes as a matrix of head_dim-byte rows, copied in boxes of at most kKeyTile
// positions of one page, swizzled over the row length.
int code_map(CUtensorMap *m, void *codes, const dfb_kv_cache &c) {
    const auto fn = tensor_map_encoder();
    if (!fn) return set_err(DFB_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    const cuuint64_t dims[2] = {(cuuint64_t)c.head_dim, (cuuint64_t)c.n_pages * c.n_kv * c.page};
    const cuuint64_t strides[1] = {(cuuint64_t)c.head_dim};
    const cuuint32_t box[2] = {(cuuint32_t)c.head_dim, (cuuint32_t)std::min(c.page, kKeyTile)}, es[2] = {1, 1};
    const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          c.head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_err(DFB_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return DFB_OK;
}

// How one call is cut up: rows per CTA, and parts of the key axis where the row tiles alone would
// leave SMs idle.
struct AttnPlan {
    int rows, tiles, splits;
};
// 16, 32 and 64 rows: mma.sync, two CTAs to an SM; 256: tcgen05, one.  Up to 64 packed rows take the
// smallest tile.  More take tcgen05 tiles, which pass four times the rows over a key tile in little more
// time, but start and finish slowly: where 64-row tiles, each with a part of the keys, give no SM more
// than one CTA and no CTA more than kShortTiles key tiles, they are faster (of one sequence of 256 rows
// and 32 heads, us: 320 keys 14.0 against 19.9, 768 keys 22.3 against 25.9, 2048 keys 47 against 32; of
// 32 rows of 28 / 4 heads: 2048 keys 15.7 against 22.4, 8192 keys 30.5 against 26.9).
// The key axis is split only as far as SMs would be idle, and to no fewer than four key tiles: a part
// costs its rows' sums a trip through memory (256 rows, 32 heads, 8192 keys in 1, 2, 4, 8 parts: 162,
// 95, 61, 75 us).
constexpr int kShortTiles = 12;
AttnPlan attn_plan(const dfb_kv_cache &c, const dfb_kv_attn &a, int n_sm) {
    const int64_t rep = a.n_q / c.n_kv, packed = a.max_rows * rep, key_tiles = ((int64_t)a.max_keys + kKeyTile - 1) / kKeyTile;
    auto plan = [&](int rows, int64_t ctas) {
        AttnPlan p;
        const int64_t tiles = (packed + rows - 1) / rows, base = tiles * c.n_kv * c.n_seq;
        p.rows = rows;
        // launched: no sequence has more rows than there are (the splits, and with them the workspace, go by max_rows alone)
        p.tiles = (int)std::min<int64_t>(tiles, (a.n_rows * rep + rows - 1) / rows);
        p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({ctas / std::max<int64_t>(base, 1), key_tiles / 4, kMaxSplits}));
        return p;
    };
    if (packed <= 64) return plan(packed <= 16 ? 16 : packed <= 32 ? 32 : 64, 2 * n_sm);
    const AttnPlan p = plan(64, n_sm);
    const bool alone = (packed + 63) / 64 * c.n_kv * c.n_seq <= n_sm;
    return alone && key_tiles <= (int64_t)kShortTiles * p.splits ? p : plan(kTcRows, n_sm);
}
size_t attn_ws_bytes(const dfb_kv_cache &c, const dfb_kv_attn &a, const AttnPlan &p) {
    return p.splits == 1 ? 0 : (size_t)p.splits * a.n_rows * a.n_q * (c.head_dim + 1) * sizeof(float);
}

template <typename T, int HD, int MW, int KW>
int attn_launch(const dfb_kv_cache &c, const dfb_kv_attn &a, const AttnPlan &p, const AttnParts &parts, const CUtensorMap &tk,
                const CUtensorMap &tv, bool vec, int dev, int32_t *status, cudaStream_t st) {
    const auto kern = kv_attn_kernel<T, HD, MW, KW>;
    constexpr int smem = KvSmem<HD, MW, KW>::bytes;
    static std::atomic<bool> attr_set[64];
    if (!attr_set[dev]) {
        CK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        attr_set[dev] = true;
    }
    kern<<<dim3(p.tiles * p.splits, c.n_kv, c.n_seq), (MW * KW + 1) * 32, smem, st>>>(c, a, tk, tv, parts, vec, status);
    CK(cudaGetLastError());
    return DFB_OK;
}

template <typename T, int HD>
int attn_tc_launch(const dfb_kv_cache &c, const dfb_kv_attn &a, const AttnPlan &p, const AttnParts &parts, const CUtensorMap &tk,
                   const CUtensorMap &tv, bool vec, int dev, int n_sm, int32_t *status, cudaStream_t st) {
    const auto kern = kv_attn_tc_kernel<T, HD>;
    constexpr int smem = TcSmem<HD>::bytes;
    static_assert(smem <= 232448, "shared memory of one CTA");
    static std::atomic<bool> attr_set[64];
    if (!attr_set[dev]) {
        CK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        attr_set[dev] = true;
    }
    const int64_t items = (int64_t)p.tiles * p.splits * c.n_kv * c.n_seq;
    if (items > INT32_MAX / 2) return set_err(DFB_ERR_UNSUPPORTED, "%lld work items", (long long)items);
    const TcGrid grid{p.tiles, (int)items};
    // 16-bit elements: the widest store that every row's start allows
    const int out_align = aligned(a.out, 32) && a.out_tok % 16 == 0 && a.out_head % 16 == 0 ? 32 : vec_ok(a.out, a.type, a.out_tok, a.out_head) ? 16 : 2;
    kern<<<(unsigned)std::min<int64_t>(items, n_sm), kTcThreads, smem, st>>>(c, a, tk, tv, parts, grid, vec, out_align, status);
    CK(cudaGetLastError());
    return DFB_OK;
}

template <typename T, int HD>
int attn_t(const dfb_kv_cache &c, const dfb_kv_attn &a, const AttnPlan &p, float *ws, int dev, int n_sm, int32_t *status, cudaStream_t st) {
    CUtensorMap tk, tv;
    RET(code_map(&tk, c.k, c));
    RET(code_map(&tv, c.v, c));
    const bool vec = vec_ok(a.q, a.type, a.q_tok, a.q_head) && vec_ok(a.out, a.type, a.out_tok, a.out_head);
    AttnParts parts;
    parts.splits = p.splits;
    if (p.splits > 1) {
        parts.o = ws;
        parts.w = ws + (size_t)p.splits * a.n_rows * a.n_q * HD;
    }
    switch (p.rows) {
        case 16: RET((attn_launch<T, HD, 1, 4>(c, a, p, parts, tk, tv, vec, dev, status, st))); break;
        case 32: RET((attn_launch<T, HD, 2, 4>(c, a, p, parts, tk, tv, vec, dev, status, st))); break;
        case 64: RET((attn_launch<T, HD, 4, 2>(c, a, p, parts, tk, tv, vec, dev, status, st))); break;
        default: RET((attn_tc_launch<T, HD>(c, a, p, parts, tk, tv, vec, dev, n_sm, status, st)));
    }
    if (p.splits > 1) {
        const int64_t per_seq = (int64_t)std::min(a.max_rows, a.n_rows) * a.n_q;
        CK(launch_k(kv_attn_join_kernel<T, HD>, dim3((unsigned)((per_seq + 3) / 4), c.n_seq), dim3(128), 0, st, true, c, a, parts));
    }
    return DFB_OK;
}

int check_attn(const dfb_kv_cache *c, const dfb_kv_attn *a) {
    RET(check_cache(c));
    if (!a) return set_err(DFB_ERR_ARG, "null arguments");
    if (a->type != T_F16 && a->type != T_BF16) return set_err(DFB_ERR_UNSUPPORTED, "query type %d not supported (F16 / BF16)", a->type);
    if (a->n_q <= 0 || a->n_q % c->n_kv) return set_err(DFB_ERR_ARG, "%d query heads over %d KV heads", a->n_q, c->n_kv);
    if (a->n_q > 65535 || (int64_t)a->max_rows * a->n_q > INT32_MAX) return set_err(DFB_ERR_UNSUPPORTED, "%d query heads of %d rows", a->n_q, a->max_rows);
    if (a->n_rows < 0 || a->max_rows < 0 || a->max_keys < 0) return set_err(DFB_ERR_ARG, "negative size");
    if (!std::isfinite(a->scale)) return set_err(DFB_ERR_ARG, "scale must be finite");
    return DFB_OK;
}

}  // namespace

extern "C" int dfb_kv_append(const dfb_kv_cache *c, const dfb_kv_rows *r, int32_t *status, void *stream) {
    RET(check_cache(c));
    if (!r) return set_err(DFB_ERR_ARG, "null arguments");
    if (r->type != T_F32 && r->type != T_F16 && r->type != T_BF16) return set_err(DFB_ERR_UNSUPPORTED, "row type %d not supported", r->type);
    if (r->n_rows < 0 || r->max_rows < 0) return set_err(DFB_ERR_ARG, "negative size");
    if (r->n_rows == 0 || r->max_rows == 0) return DFB_OK;
    RET(check_rows("k", r->k, r->type, r->k_tok, r->k_head));
    RET(check_rows("v", r->v, r->type, r->v_tok, r->v_head));
    if (!r->row_off || !r->len) return set_err(DFB_ERR_ARG, "null row offsets or lengths");
    if (r->rope && (r->n_rope <= 0 || !aligned(r->rope, 16))) return set_err(DFB_ERR_ARG, "rotation table empty or not 16-byte aligned");
    if (r->q) {
        if (r->n_q <= 0 || r->n_q > 8192) return set_err(DFB_ERR_ARG, "%d query heads", r->n_q);
        RET(check_rows("q", r->q, r->type, r->q_tok, r->q_head));
        RET(check_out("q_out", r->q_out, r->type, r->n_rows, r->q_out_tok, r->n_q, r->q_out_head, c->head_dim));
    }
    DeviceGuard g;
    RET(g.enter(c->k, "the cache"));
    int n_sm = 0;
    RET(device_props(g.device(), &n_sm));
    bool vec = vec_ok(r->k, r->type, r->k_tok, r->k_head) && vec_ok(r->v, r->type, r->v_tok, r->v_head);
    if (r->q) vec = vec && vec_ok(r->q, r->type, r->q_tok, r->q_head) && vec_ok(r->q_out, r->type, r->q_out_tok, r->q_out_head);
    // pages a sequence's rows can touch: consecutive positions n / page + 2 at most, given positions any of them
    const int64_t rows = std::min(r->max_rows, r->n_rows);
    const int64_t most = r->pos ? c->max_pages : std::min<int64_t>(c->max_pages, (rows + c->page - 2) / c->page + 1);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto go = [&](auto t) {
        using T = decltype(t);
        return c->head_dim == 64 ? append_t<T, 64>(*c, *r, most, n_sm, vec, status, st) : append_t<T, 128>(*c, *r, most, n_sm, vec, status, st);
    };
    return r->type == T_F32 ? go(float()) : r->type == T_F16 ? go(__half()) : go(__nv_bfloat16());
}

extern "C" int dfb_kv_attention_workspace(const dfb_kv_cache *c, const dfb_kv_attn *a, size_t *bytes) {
    if (!bytes) return set_err(DFB_ERR_ARG, "null pointer");
    *bytes = 0;
    RET(check_attn(c, a));
    if (a->n_rows == 0 || a->max_rows == 0) return DFB_OK;
    DeviceGuard g;
    RET(g.enter(c->k, "the cache"));
    int n_sm = 0;
    RET(device_props(g.device(), &n_sm));
    *bytes = attn_ws_bytes(*c, *a, attn_plan(*c, *a, n_sm));
    return DFB_OK;
}

extern "C" int dfb_kv_attention(const dfb_kv_cache *c, const dfb_kv_attn *a, void *workspace, size_t ws_bytes, int32_t *status,
                                void *stream) {
    RET(check_attn(c, a));
    if (a->n_rows == 0 || a->max_rows == 0) return DFB_OK;
    RET(check_rows("q", a->q, a->type, a->q_tok, a->q_head));
    RET(check_out("out", a->out, a->type, a->n_rows, a->out_tok, a->n_q, a->out_head, c->head_dim));
    if (!a->row_off || !a->len) return set_err(DFB_ERR_ARG, "null row offsets or lengths");
    DeviceGuard g;
    RET(g.enter(c->k, "the cache"));
    int n_sm = 0;
    RET(device_props(g.device(), &n_sm));
    const AttnPlan p = attn_plan(*c, *a, n_sm);
    const size_t need = attn_ws_bytes(*c, *a, p);
    if (need && (!workspace || ws_bytes < need || !aligned(workspace, 16)))
        return set_err(DFB_ERR_ARG, "workspace of %zu bytes at %p, need %zu 16-byte aligned", ws_bytes, workspace, need);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    float *ws = static_cast<float *>(workspace);
    auto go = [&](auto t) {
        using T = decltype(t);
        return c->head_dim == 64 ? attn_t<T, 64>(*c, *a, p, ws, g.device(), n_sm, status, st) : attn_t<T, 128>(*c, *a, p, ws, g.device(), n_sm, status, st);
    };
    return a->type == T_F16 ? go(__half()) : go(__nv_bfloat16());
}

extern "C" int dfb_token_logprobs(const dfb_logprob_args *a, int32_t *status, void *stream) {
    if (!a) return set_err(DFB_ERR_ARG, "null arguments");
    if (a->type != T_F32 && a->type != T_F16 && a->type != T_BF16) return set_err(DFB_ERR_UNSUPPORTED, "logits type %d not supported", a->type);
    if (a->n_rows < 0 || a->n_logits < 0) return set_err(DFB_ERR_ARG, "negative size");
    if (a->n_vocab <= 0) return set_err(DFB_ERR_ARG, "vocabulary of %d", a->n_vocab);
    if (a->ld < a->n_vocab && a->n_logits > 1) return set_err(DFB_ERR_ARG, "row stride %lld < %d", (long long)a->ld, a->n_vocab);
    if (a->top_k < 0 || a->top_k > 32 || a->top_k > a->n_vocab) return set_err(DFB_ERR_ARG, "top_k %d outside [0, min(32, %d)]", a->top_k, a->n_vocab);
    if (a->top_k > 0 && (!a->top_ids || !a->top_logprob)) return set_err(DFB_ERR_ARG, "null alternatives");
    if ((a->logprob != nullptr) != (a->targets != nullptr)) return set_err(DFB_ERR_ARG, "targets and logprob go together");
    if (!a->rows && a->n_rows > a->n_logits) return set_err(DFB_ERR_ARG, "%d rows of a matrix of %d", a->n_rows, a->n_logits);
    if (a->n_rows == 0) return DFB_OK;
    if (!a->logits || !aligned(a->logits, type_size(a->type))) return set_err(DFB_ERR_ARG, "logits null or not aligned to their type");
    DeviceGuard g;
    RET(g.enter(a->logits, "logits"));
    int n_sm = 0;
    RET(device_props(g.device(), &n_sm));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    // CTAs of a row (a cluster of up to 8): as many as still run all at once, with 8 KB of the
    // row to each at least.  More of them would share out the memory's bandwidth better, but each has a part of
    // its own (first batch, threshold, joining): 256 f32 rows of 126464 take 37, 34 and 43 us with one, two and
    // four, one row 30, 21, 15 and 13 with one, two, four and eight, 2048 bf16 rows of 152064 176 and 229 with
    // one and two.
    const int64_t row_bytes = (int64_t)a->n_vocab * type_size(a->type);
    int n_cta = 1;
    while (n_cta < 8 && (int64_t)a->n_rows * n_cta * 2 <= kLpCtas * n_sm && row_bytes / (2 * n_cta) >= 8192) n_cta *= 2;
    if ((int64_t)a->n_rows * n_cta > INT32_MAX) return set_err(DFB_ERR_UNSUPPORTED, "%d rows", a->n_rows);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(a->n_rows * n_cta));
    cfg.blockDim = dim3(kLpThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = n_cta;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    switch (a->type) {
        case T_F32: CK(cudaLaunchKernelEx(&cfg, logprobs_kernel<float>, *a, status)); break;
        case T_F16: CK(cudaLaunchKernelEx(&cfg, logprobs_kernel<__half>, *a, status)); break;
        default: CK(cudaLaunchKernelEx(&cfg, logprobs_kernel<__nv_bfloat16>, *a, status));
    }
    return DFB_OK;
}
