// obs_paged.cu -- C ABI of the paged key/value cache's operators: argument checks,
// the context's workspace, launches.
#include <cstddef>
#include <cstdio>
#include <new>
#include <string>

#include "obs_moe.h"
#include "paged.cuh"

namespace obs {

int ctx_fail(obs_ctx* ctx, int code, const char* msg);  // obs_api.cu

struct PagedState {
    obs_paged_config cfg{};
    uint8_t* mem = nullptr;
    float* part = nullptr;      // parts of items that several CTAs share
    uint32_t* count = nullptr;  // their arrivals
    float* scores = nullptr;    // with cfg.weights: [max_seqs][n_kv_heads][max_kv_len][group, even]
    float* pf_part = nullptr;   // parts of a prefill's rows that several CTAs share
    float2* ml = nullptr;       // with cfg.weights: [max_seqs][n_heads]
};

void paged_free(PagedState* p) {
    if (p->mem) cudaFree(p->mem);
    delete p;
}

const char* paged_mismatch(const PagedState* p, int nq, int nkv, int hd) {
    if (!p) return "paged cache not initialised (obs_paged_init)";
    const obs_paged_config& c = p->cfg;
    if (c.n_heads != nq || c.n_kv_heads != nkv || c.head_dim != hd || c.dtype != OBS_DTYPE_BF16)
        return "the paged cache's heads, head_dim or dtype are not the attention block's";
    return nullptr;
}

}  // namespace obs

using namespace obs;

namespace {

constexpr float kLog2e = 1.4426950408889634f;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// The caller's cache against the context's configuration; fills *a or returns a message.
const char* paged_args(const PagedState* p, const obs_paged_kv* kv, int* err, PagedArgs* a) {
    // (no sequences: a table and lengths of no elements have no address)
    if (!kv || !kv->k || !kv->v || (kv->n_seqs != 0 && (!kv->block_table || !kv->kv_len))) return "null cache pointer";
    const obs_paged_config& c = p->cfg;
    if (!aligned16(kv->k) || !aligned16(kv->v)) return "k and v must be 16-byte aligned";
    if (kv->page_stride % 8 || kv->slot_stride % 8 || kv->head_stride % 8)
        return "cache strides must be multiples of 8 elements (16 bytes)";
    if (kv->page_stride < 0 || kv->slot_stride < 0 || kv->head_stride < 0) return "cache strides must not be negative";
    if (kv->n_seqs < 0 || kv->n_seqs > c.max_seqs) return "n_seqs out of range (0..max_seqs)";
    if (kv->n_pages <= 0 || kv->table_pages < 0 || (kv->n_seqs > 0 && kv->table_pages == 0)) return "n_pages and table_pages must be positive";
    if (kv->n_seqs > 1 && kv->table_stride < kv->table_pages) return "table_stride is smaller than table_pages";
    const int64_t room = (int64_t)kv->table_pages * c.page_size;
    a->k = reinterpret_cast<const uint16_t*>(kv->k);
    a->v = reinterpret_cast<const uint16_t*>(kv->v);
    a->table = kv->block_table, a->len = kv->kv_len;
    a->page_stride = kv->page_stride, a->slot_stride = kv->slot_stride, a->head_stride = kv->head_stride;
    a->n_seqs = kv->n_seqs, a->n_pages = kv->n_pages, a->table_stride = kv->table_stride;
    a->page_size = c.page_size;
    a->page_magic = c.page_size == 1 ? 0u : (uint32_t)((1ull << 32) / (uint32_t)c.page_size + 1);
    a->cap = (int)(room < c.max_kv_len ? room : c.max_kv_len);
    a->nkv = c.n_kv_heads, a->group = c.n_heads / c.n_kv_heads, a->hd = c.head_dim;
    a->err = err;
    return nullptr;
}

const char* query_args(const PagedArgs& a, const void* q, int64_t q_stride, const void* out, int rows, int window,
                       int n_sink, float scale) {
    if (!q || !out) return "null pointer";
    if (!aligned16(q) || !aligned16(out) || q_stride % 8) return "q and out must be 16-byte aligned, q_stride a multiple of 8";
    const int64_t row = (int64_t)a.nkv * a.group * a.hd;
    if (q_stride < row) return "q_stride is smaller than a row";
    // (rows that come out not finite are computed again, from q)
    const char *qb = static_cast<const char*>(q), *ob = static_cast<const char*>(out);
    if (ob < qb + 2 * ((rows - 1) * q_stride + row) && qb < ob + 2 * rows * row) return "out may not overlap q";
    if (window < 0 || n_sink < 0) return "window and n_sink must not be negative";
    if (!(scale >= 0.0f) || scale > 3.0e38f) return "scale must be finite and not negative (0: 1/sqrt(head_dim))";
    return nullptr;
}

const char* decode_args(const PagedState* ps, const PagedArgs& a, const float* weights, int w_stride, int* code) {
    *code = OBS_ERR_INVALID;
    if ((int64_t)a.n_seqs * a.nkv * (a.cap / 64 + 2) > 0x7fffffff)
        return "n_seqs * n_kv_heads * positions is too large for one call";
    if (weights && !ps->cfg.weights) {
        *code = OBS_ERR_STATE;
        return "the paged cache was initialised without room for weights";
    }
    if (weights && w_stride <= 0) return "w_stride must be positive";
    return nullptr;
}

#define PAGED_BEGIN()                                                                                             \
    if (!ctx) return OBS_ERR_INVALID;                                                                             \
    const CtxParts parts = ctx_parts(ctx);                                                                        \
    PagedState* ps = *parts.paged;                                                                                \
    if (!ps) return ctx_fail(ctx, OBS_ERR_STATE, "paged cache not initialised (obs_paged_init)");                 \
    PagedArgs a{};                                                                                                \
    if (const char* m = paged_args(ps, kv, parts.err, &a)) return ctx_fail(ctx, OBS_ERR_INVALID, m)

int launched(obs_ctx* ctx, cudaError_t e, const char* what) {
    if (e == cudaSuccess) return OBS_OK;
    char msg[160];
    snprintf(msg, sizeof msg, "%s: %s", what, cudaGetErrorString(e));
    return ctx_fail(ctx, OBS_ERR_CUDA, msg);
}

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }

}  // namespace

int obs::paged_check(obs_ctx* ctx, const obs_paged_kv* kv, bool decode, int window, int n_sink, const float* weights,
                     int w_stride) {
    PAGED_BEGIN();
    if (window < 0 || n_sink < 0) return ctx_fail(ctx, OBS_ERR_INVALID, "window and n_sink must not be negative");
    if (a.n_seqs == 0) return ctx_fail(ctx, OBS_ERR_INVALID, "rows without sequences");
    int code;
    if (decode)
        if (const char* m = decode_args(ps, a, weights, w_stride, &code)) return ctx_fail(ctx, code, m);
    return OBS_OK;
}

extern "C" int obs_paged_init(obs_ctx* ctx, const obs_paged_config* cfg) {
    if (!ctx) return OBS_ERR_INVALID;
    if (!cfg) return ctx_fail(ctx, OBS_ERR_INVALID, "null paged config");
    const CtxParts parts = ctx_parts(ctx);
    if (*parts.paged) return ctx_fail(ctx, OBS_ERR_STATE, "paged cache already initialised");
    const int nq = cfg->n_heads, nkv = cfg->n_kv_heads, hd = cfg->head_dim;
    if (nq <= 0 || nkv <= 0 || nkv > 65535 || nq % nkv || nq / nkv > kPagedMaxGroup || hd <= 0 || hd > 128 || hd % 8 ||
        cfg->page_size <= 0 || cfg->page_size > kPagedMaxPage || cfg->max_seqs <= 0 || cfg->max_seqs > 65535 ||
        cfg->max_kv_len <= 0 || cfg->max_kv_len > kPagedMaxLen ||
        (cfg->dtype != OBS_DTYPE_BF16 && cfg->dtype != OBS_DTYPE_F16))
        return ctx_fail(ctx, OBS_ERR_INVALID,
                        "bad paged config (heads a multiple of kv heads, at most 16 per kv head, head_dim <= 128 a "
                        "multiple of 8, 0 < page_size <= 1024, 0 < max_seqs <= 65535, 0 < max_kv_len <= 1048576, dtype "
                        "OBS_DTYPE_BF16 or OBS_DTYPE_F16)");
    PagedState* ps = new (std::nothrow) PagedState();
    if (!ps) return ctx_fail(ctx, OBS_ERR_NOMEM, "paged cache state");
    ps->cfg = *cfg;
    const size_t n = (size_t)cfg->max_seqs * nq;
    const size_t sizes[] = {paged_decode_part_floats(nq / nkv, parts.num_sms) * 4, (size_t)kPagedCtas * parts.num_sms * 4,
                            cfg->weights ? (size_t)cfg->max_seqs * nkv * ((nq / nkv + 1) & ~1) * cfg->max_kv_len * 4 : 0, cfg->weights ? n * 8 : 0,
                            paged_prefill_part_floats(parts.num_sms) * 4};
    void** ptrs[] = {(void**)&ps->part, (void**)&ps->count, (void**)&ps->scores, (void**)&ps->ml, (void**)&ps->pf_part};
    size_t total = 0;
    for (size_t sz : sizes) total += (sz + 255) / 256 * 256;
    cudaError_t e = cudaSetDevice(parts.device);
    if (e == cudaSuccess) e = cudaMalloc(&ps->mem, total);
    if (e != cudaSuccess) {
        cudaGetLastError();  // the failed allocation is reported here, not by a later call
        delete ps;
        return ctx_fail(ctx, e == cudaErrorMemoryAllocation ? OBS_ERR_NOMEM : OBS_ERR_CUDA,
                        (std::string("paged workspace: ") + cudaGetErrorString(e)).c_str());
    }
    uint8_t* at = ps->mem;
    for (int i = 0; i < 5; ++i) *ptrs[i] = sizes[i] ? at : nullptr, at += (sizes[i] + 255) / 256 * 256;
    e = cudaMemset(ps->count, 0, sizes[1]);
    if (e == cudaSuccess) e = cudaDeviceSynchronize();  // the calls may come on any stream
    if (e != cudaSuccess) {
        paged_free(ps);
        return ctx_fail(ctx, OBS_ERR_CUDA, (std::string("paged workspace: ") + cudaGetErrorString(e)).c_str());
    }
    *parts.paged = ps;
    return OBS_OK;
}

int obs::paged_append(obs_ctx* ctx, const obs_paged_kv* kv, const void* k, const void* v, int64_t row_stride,
                      const int32_t* seq, const int32_t* slot, int T, const int32_t* pos, int max_pos, void* stream) {
    PAGED_BEGIN();
    if (T < 0) return ctx_fail(ctx, OBS_ERR_INVALID, "T < 0");
    if (T == 0) return OBS_OK;
    if (!k || !v || !seq || !slot) return ctx_fail(ctx, OBS_ERR_INVALID, "null pointer");
    if (!aligned16(k) || !aligned16(v) || row_stride % 8)
        return ctx_fail(ctx, OBS_ERR_INVALID, "rows must be 16-byte aligned, row_stride a multiple of 8");
    if (row_stride < (int64_t)a.nkv * a.hd) return ctx_fail(ctx, OBS_ERR_INVALID, "row_stride is smaller than a row");
    return launched(ctx,
                    launch_paged_append(a, reinterpret_cast<const uint16_t*>(k), reinterpret_cast<const uint16_t*>(v),
                                        row_stride, seq, slot, T, pos, max_pos, parts.num_sms, as_stream(stream)),
                    "paged append");
}

extern "C" int obs_paged_append(obs_ctx* ctx, const obs_paged_kv* kv, const void* k, const void* v, int64_t row_stride,
                                const int32_t* seq, const int32_t* slot, int T, void* stream) {
    return paged_append(ctx, kv, k, v, row_stride, seq, slot, T, nullptr, 0, stream);
}

extern "C" int obs_paged_decode(obs_ctx* ctx, const obs_paged_kv* kv, const void* q, int64_t q_stride, void* out,
                                int window, int n_sink, float scale, float* weights, int w_stride, void* stream) {
    PAGED_BEGIN();
    if (a.n_seqs == 0) return OBS_OK;
    if (const char* m = query_args(a, q, q_stride, out, a.n_seqs, window, n_sink, scale)) return ctx_fail(ctx, OBS_ERR_INVALID, m);
    int code;
    if (const char* m = decode_args(ps, a, weights, w_stride, &code)) return ctx_fail(ctx, code, m);
    if (weights && w_stride < a.cap) a.cap = w_stride;  // a longer sequence is refused on the device
    const float sc = scale > 0.0f ? scale : 1.0f / sqrtf((float)a.hd);
    DecodeArgs p{a, reinterpret_cast<const uint16_t*>(q), q_stride, reinterpret_cast<uint16_t*>(out), window, n_sink,
                 sc, sc * kLog2e, ps->part, ps->count, weights ? ps->scores : nullptr, ps->cfg.max_kv_len,
                 (a.group + 1) & ~1,
                 weights ? ps->ml : nullptr, weights, w_stride};
    return launched(ctx, launch_paged_decode(p, ps->cfg.dtype, parts.num_sms, as_stream(stream)), "paged decode");
}

extern "C" int obs_paged_prefill(obs_ctx* ctx, const obs_paged_kv* kv, const void* q, int64_t q_stride, void* out,
                                 const int32_t* q_start, int T, int window, int n_sink, float scale, void* stream) {
    PAGED_BEGIN();
    if (T < 0 || T > kPagedMaxLen) return ctx_fail(ctx, OBS_ERR_INVALID, "T out of range (0..1048576)");
    if (T == 0) return OBS_OK;
    if (a.n_seqs == 0) return ctx_fail(ctx, OBS_ERR_INVALID, "rows without sequences");
    if (!q_start) return ctx_fail(ctx, OBS_ERR_INVALID, "null pointer");
    if (const char* m = query_args(a, q, q_stride, out, T, window, n_sink, scale)) return ctx_fail(ctx, OBS_ERR_INVALID, m);
    const float sc = scale > 0.0f ? scale : 1.0f / sqrtf((float)a.hd);
    PrefillArgs p{a, reinterpret_cast<const uint16_t*>(q), q_stride, reinterpret_cast<uint16_t*>(out), q_start, T, window,
                  n_sink, sc, sc * kLog2e, parts.wait_ns, 1, nullptr, nullptr};
    return launched(ctx, launch_paged_prefill(p, ps->pf_part, ps->cfg.dtype, parts.num_sms, as_stream(stream)),
                    "paged prefill");
}

extern "C" int obs_paged_evict(obs_ctx* ctx, const obs_paged_kv* kv, const obs_paged_kv* dst, const float* weights,
                               float* weights_dst, int w_stride, int budget, int n_sink, int n_recent, int32_t* kept,
                               int32_t* new_len, void* stream) {
    PAGED_BEGIN();
    PagedArgs d{};
    if (const char* m = paged_args(ps, dst, parts.err, &d)) return ctx_fail(ctx, OBS_ERR_INVALID, m);
    if (d.n_seqs != a.n_seqs) return ctx_fail(ctx, OBS_ERR_INVALID, "dst has another number of sequences");
    if (a.n_seqs == 0) return OBS_OK;
    if (!weights || !kept || !new_len) return ctx_fail(ctx, OBS_ERR_INVALID, "null pointer");
    if (budget <= 0 || n_sink < 0 || n_recent < 0 || (int64_t)n_sink + n_recent > budget)
        return ctx_fail(ctx, OBS_ERR_INVALID, "need 0 <= n_sink + n_recent <= budget and budget > 0");
    if (budget > d.cap) return ctx_fail(ctx, OBS_ERR_INVALID, "dst has no room for budget positions");
    if (w_stride <= 0 || (weights_dst && w_stride < budget))
        return ctx_fail(ctx, OBS_ERR_INVALID, "w_stride must be positive (and at least budget with weights_dst)");
    if (new_len == kv->kv_len) return ctx_fail(ctx, OBS_ERR_INVALID, "new_len may not alias kv_len");
    if (w_stride < a.cap) a.cap = w_stride;  // a longer sequence is refused on the device
    return launched(ctx,
                    launch_paged_evict(a, d, weights, weights_dst, w_stride, budget, n_sink, n_recent, kept, new_len,
                                       as_stream(stream)),
                    "paged evict");
}

#define OBS_OFF(T, f) (int32_t) offsetof(T, f)
extern "C" int obs_paged_struct_layout(int32_t* out, int n) {
    const int32_t v[] = {
        (int32_t)sizeof(obs_paged_config),
        OBS_OFF(obs_paged_config, n_heads), OBS_OFF(obs_paged_config, n_kv_heads), OBS_OFF(obs_paged_config, head_dim),
        OBS_OFF(obs_paged_config, page_size), OBS_OFF(obs_paged_config, max_seqs), OBS_OFF(obs_paged_config, max_kv_len),
        OBS_OFF(obs_paged_config, dtype), OBS_OFF(obs_paged_config, weights),
        (int32_t)sizeof(obs_paged_kv),
        OBS_OFF(obs_paged_kv, k), OBS_OFF(obs_paged_kv, v), OBS_OFF(obs_paged_kv, block_table),
        OBS_OFF(obs_paged_kv, kv_len), OBS_OFF(obs_paged_kv, page_stride), OBS_OFF(obs_paged_kv, slot_stride),
        OBS_OFF(obs_paged_kv, head_stride), OBS_OFF(obs_paged_kv, n_seqs), OBS_OFF(obs_paged_kv, n_pages),
        OBS_OFF(obs_paged_kv, table_stride), OBS_OFF(obs_paged_kv, table_pages),
    };
    const int total = (int)(sizeof v / sizeof v[0]);
    for (int i = 0; i < total && i < n && out; ++i) out[i] = v[i];
    return total;
}
