// k_paged.cu -- the paged key/value cache: rows into their pages, and eviction by
// accumulated attention weight.  The reference keeps one dense cache per layer
// (kv_cache.rs:15-24, ops.metal:32-37) and has no counterpart of either.
#include <cooperative_groups.h>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace obs {
namespace {

// Row t of k and v ([T] rows of n_kv * head_dim elements, row_stride apart) to
// position slot[t] of sequence seq[t]; with `pos`, a row whose pos[t] lies outside
// [0, max_pos) is refused like one outside the cache.  One 16-byte piece per thread: neighbouring
// threads write neighbouring pieces of a row, so whole sectors move whatever the
// strides.  Bound by the launch for a decode step (16 rows of 4 x 128: 1.7 us) and by
// memory for a prompt (4096 such rows, 17 MB: 4.7 us, 3.6 TB/s).
__global__ void __launch_bounds__(256) k_paged_append(PagedArgs a, const uint16_t* k, const uint16_t* v,
                                                      int64_t row_stride, const int32_t* seq, const int32_t* slot,
                                                      int T, const int32_t* pos, int max_pos) {
    pdl_begin();
    const int per_head = a.hd / 8, per_row = a.nkv * per_head;  // 16-byte pieces
    const int64_t n = (int64_t)T * per_row * 2;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int t = (int)(i / (2 * per_row)), r = (int)(i - (int64_t)t * 2 * per_row);
        const bool isv = r >= per_row;
        const int c = isv ? r - per_row : r, head = c / per_head, piece = c - head * per_head;
        const int s = seq[t], j = slot[t];
        if ((unsigned)s >= (unsigned)a.n_seqs || (unsigned)j >= (unsigned)a.cap ||
            (pos && (unsigned)pos[t] >= (unsigned)max_pos)) {
            atomicExch(a.err, kDevBadPos);
            continue;
        }
        const int64_t off = row_offset(a, s, j, head);
        if (off < 0) continue;
        const uint4 x = *reinterpret_cast<const uint4*>((isv ? v : k) + t * row_stride + c * 8);
        *reinterpret_cast<uint4*>(const_cast<uint16_t*>(isv ? a.v : a.k) + off + piece * 8) = x;
    }
}

// ------------------------------------------------------------------ eviction
// Which positions of (sequence s, KV head h) stay: all n if n <= budget, else the
// first n_sink, the last n_recent and, of the rest, the `need` = budget - n_sink -
// n_recent with the largest weights (equal weights: the lowest position; NaN lowest
// of all), in two launches.
//   select   radix selection over the weights as ordered 32-bit keys, 11 + 11 + 10
//            bits from the top: a histogram in shared memory gives the digit of the
//            threshold key.  One CTA holds up to kEvChunk positions in shared memory; for
//            longer caches a cluster of kEvC shares them and adds its histograms up
//            through distributed shared memory.  Ballots then give every kept position
//            its place, in order.  Bound by the latency of its passes (12 us for 8192
//            positions; comparing the keys with three candidates a round, two bits at a
//            time, needs no histogram, but sixteen rounds took 20 us for 4096).
//   move     the kept rows to places 0, 1, ... of dst by CTAs of a few rows: with the
//            selection 42 us for 16 sequences of up to 8192 cut to 2048 (131 MB).  Moved by the selecting CTAs instead,
//            the same took 95 us: too few bytes in flight.
constexpr int kEvC = 8, kEvThreads = 1024, kEvWarps = kEvThreads / 32;
constexpr int kEvBins = 2048;
constexpr int kEvRows = 8, kEvChunk = kEvRows * kEvThreads;  // positions a CTA holds at a time
static_assert(2 * kEvRows * kEvWarps <= kEvThreads, "one thread per entry of s_at");

// larger weight <=> larger key; -0 and +0 equal; NaN the smallest (0)
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t b = __float_as_uint(w + 0.0f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

struct EvictArgs {
    PagedArgs src, dst;
    const float* w;
    float* w_dst;
    int w_stride;
    int budget, n_sink, n_recent;
    int32_t* kept;      // [n_seqs][nkv][budget]
    int32_t* new_len;   // [n_seqs]
    int in_place;
};

// exclusive prefix sum over the CTA of one value per thread (two barriers)
__device__ __forceinline__ int block_excl(int v, int* s_warp) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) s_warp[warp] = x;
    __syncthreads();
    return x - v + __reduce_add_sync(0xffffffffu, lane < warp ? s_warp[lane] : 0);
}

__global__ void __launch_bounds__(kEvThreads) k_paged_select(EvictArgs e) {
    pdl_begin();
    cg::cluster_group cl = cg::this_cluster();
    __shared__ uint32_t s_key[kEvChunk];
    __shared__ uint32_t s_hist[kEvBins];
    __shared__ int s_at[2][kEvRows * kEvWarps];  // kept above the threshold / equal to it, by row of 32
    __shared__ int s_warp[kEvWarps], s_tot[2];
    const PagedArgs& a = e.src;
    const int rank = (int)cl.block_rank(), size = (int)cl.num_blocks(), h = blockIdx.y, s = blockIdx.z;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = seq_len(a, s), m = n < e.budget ? n : e.budget;
    const int64_t row = (int64_t)s * a.nkv + h;
    const float* w = e.w + row * e.w_stride;
    int32_t* kept = e.kept + row * e.budget;
    if (rank == 0 && h == 0 && tid == 0) e.new_len[s] = m;

    const int all = n <= e.budget;
    const int lo = all ? n : e.n_sink, hi = all ? n : n - e.n_recent;  // the positions that are chosen from
    for (int j = rank * kEvThreads + tid; j < e.budget; j += size * kEvThreads) {
        if (all) kept[j] = j < n ? j : -1;
        else if (j < lo) kept[j] = j;
        else if (j >= e.budget - e.n_recent) kept[j] = n - e.budget + j;
    }
    const int need = e.budget - e.n_sink - e.n_recent;
    const int parts = hi - lo <= kEvChunk ? 1 : size;  // CTAs that share them
    if (!all && need > 0 && rank < parts) {
        const int per = (hi - lo + parts - 1) / parts;
        const int b0 = min(hi, lo + rank * per), len = min(hi, b0 + per) - b0;
        const bool held = len <= kEvChunk;
        if (held) {  // (each thread reads its own)
            float v[kEvRows];
#pragma unroll
            for (int i = 0; i < kEvRows; ++i) v[i] = i * kEvThreads + tid < len ? w[b0 + i * kEvThreads + tid] : 0.0f;
#pragma unroll
            for (int i = 0; i < kEvRows; ++i) s_key[i * kEvThreads + tid] = weight_key(v[i]);
        }
        auto key_at = [&](int j) { return j >= len ? 0u : held ? s_key[j] : weight_key(w[b0 + j]); };
        // (the loops are kept rolled: most of this code runs once, and unrolled it was
        // waiting for its instructions)
        // the threshold key t, digit by digit from the top; `left`: how many of the keys
        // that share the digits found so far are kept
        uint32_t t = 0;
        int left = need;
#pragma unroll 1
        for (int sh = 21, bits = 11; bits > 0; bits = sh ? (sh == 10 ? 10 : 11) : 0, sh = sh == 21 ? 10 : 0) {
            const int bins = 1 << bits;
            for (int i = tid; i < bins; i += kEvThreads) s_hist[i] = 0;
            __syncthreads();
#pragma unroll 2
            for (int base = 0; base < len; base += kEvThreads) {
                const uint32_t key = key_at(base + tid);
                const bool in = base + tid < len && (sh == 21 || key >> (sh + bits) == t);
                const uint32_t digit = key >> sh & (bins - 1);
                // (equal weights, a fresh cache's zeros, would all meet in one bin: then one lane adds)
                int one;
                __match_all_sync(0xffffffffu, in ? digit : 0xffffffffu, &one);
                if (in && (!one || lane == 0)) atomicAdd(&s_hist[digit], one ? 32u : 1u);
            }
            if (parts > 1) cl.sync();
            else __syncthreads();
            // bins from the top, a run of them per thread; the one in which the left-th
            // largest key lies
            const int run = max(1, bins / kEvThreads), top = tid < bins ? bins - 1 - tid * run : -1;
            int cnt[kEvBins / kEvThreads], mine = 0;
#pragma unroll
            for (int i = 0; i < kEvBins / kEvThreads; ++i) {
                cnt[i] = 0;
                if (i < run && top >= 0) {
                    if (parts == 1) cnt[i] = (int)s_hist[top - i];
                    else
                        for (int r = 0; r < parts; ++r) cnt[i] += (int)cl.map_shared_rank(s_hist, r)[top - i];
                }
                mine += cnt[i];
            }
            int before = block_excl(mine, s_warp);
            if (before < left && before + mine >= left) {
                int i = 0;
#pragma unroll
                for (int q = 0; q < kEvBins / kEvThreads - 1; ++q)
                    if (i == q && before + cnt[q] < left) before += cnt[q], ++i;
                s_tot[0] = top - i, s_tot[1] = before;
            }
            if (parts > 1) cl.sync();  // (also: the histograms have been read)
            else __syncthreads();
            t = t << bits | (uint32_t)s_tot[0];
            left -= s_tot[1];
            __syncthreads();
        }
        // above the threshold: kept; equal to it: the first `left` of them
        int gt0 = 0, eq0 = 0;  // in the CTAs and the chunks before
        if (parts > 1) {
            int g = 0, q = 0;
            for (int j = tid; j < len; j += kEvThreads) {
                const uint32_t key = key_at(j);
                g += key > t, q += key == t;
            }
            const int pg = block_excl(g, s_warp), pq = block_excl(q, s_warp);
            if (tid == kEvThreads - 1) s_tot[0] = pg + g, s_tot[1] = pq + q;
            cl.sync();
            gt0 = __reduce_add_sync(0xffffffffu, lane < rank ? cl.map_shared_rank(s_tot, lane)[0] : 0);
            eq0 = __reduce_add_sync(0xffffffffu, lane < rank ? cl.map_shared_rank(s_tot, lane)[1] : 0);
            cl.sync();
        }
#pragma unroll 1
        for (int c0 = 0; c0 < len; c0 += kEvChunk) {
            const int rows = min(kEvRows, (len - c0 + kEvThreads - 1) / kEvThreads);  // of kEvThreads positions
#pragma unroll 1
            for (int i = 0; i < kEvRows; ++i) {
                const int j = c0 + i * kEvThreads + tid;
                const uint32_t key = key_at(j);
                const uint32_t bg = __ballot_sync(0xffffffffu, j < len && key > t), bq = __ballot_sync(0xffffffffu, j < len && key == t);
                if (lane == 0) s_at[0][i * kEvWarps + warp] = __popc(bg), s_at[1][i * kEvWarps + warp] = __popc(bq);
            }
            __syncthreads();
            // exclusive sums in the order of the positions, both kinds at once: 256 each
            {
                constexpr int kN = kEvRows * kEvWarps;
                const int kind = tid / kN, at = tid % kN, v = tid < 2 * kN ? s_at[kind][at] : 0;
                const int x = block_excl(v, s_warp);
                if (tid == kN - 1) s_tot[0] = x + v;
                __syncthreads();
                if (tid == 2 * kN - 1) s_tot[1] = x + v - s_tot[0];
                if (tid < 2 * kN) s_at[kind][at] = x - (kind ? s_tot[0] : 0);
            }
            __syncthreads();
            const uint32_t below = (1u << lane) - 1u;
#pragma unroll 1
            for (int i = 0; i < rows; ++i) {
                const int j = c0 + i * kEvThreads + tid;
                const uint32_t key = key_at(j);
                const bool g = j < len && key > t, q = j < len && key == t;
                const uint32_t bg = __ballot_sync(0xffffffffu, g), bq = __ballot_sync(0xffffffffu, q);
                const int pg = gt0 + s_at[0][i * kEvWarps + warp] + __popc(bg & below);
                const int pq = eq0 + s_at[1][i * kEvWarps + warp] + __popc(bq & below);
                if (g || (q && pq < left)) kept[e.n_sink + pg + min(pq, left)] = b0 + j;
            }
            gt0 += s_tot[0], eq0 += s_tot[1];
            __syncthreads();  // the counts are written again by the next chunk
        }
    }
    cl.sync();  // no CTA ends while another may read its shared memory
}

// ---- move, to pages that the source does not hold: one warp (or two half ones) per
// kept row, a 16-byte piece of K or V per lane, kMoveU rows each; enough in flight
// for the memory's rate.  The weights move along, the rest of their row is cleared.
constexpr int kMoveU = 2, kMoveThreads = 128;          // (4 rows by 256 threads: 51 us instead of 42 us for the whole eviction)
constexpr int kInPlaceU = 4, kInPlaceThreads = 512;

__global__ void __launch_bounds__(kMoveThreads) k_paged_move(EvictArgs e) {
    pdl_begin();
    const PagedArgs& a = e.src;
    const int h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
    const int n = seq_len(a, s), m = n < e.budget ? n : e.budget;
    const int64_t row = (int64_t)s * a.nkv + h;
    const int32_t* kept = e.kept + row * e.budget;
    const int pieces = a.hd / 8, per_row = 2 * pieces, rows_cta = kMoveThreads / per_row;
    const int lr = tid / per_row, c = tid - lr * per_row, piece = (c >= pieces ? c - pieces : c) * 8;
    const uint16_t* from = c >= pieces ? a.v : a.k;
    uint16_t* to = const_cast<uint16_t*>(c >= pieces ? e.dst.v : e.dst.k);
    const int j0 = blockIdx.x * (rows_cta * kMoveU);
    if (lr < rows_cta) {
        int64_t src[kMoveU], dst[kMoveU];
        uint4 x[kMoveU];
#pragma unroll
        for (int u = 0; u < kMoveU; ++u) {
            const int j = j0 + u * rows_cta + lr;
            src[u] = dst[u] = -1;
            if (j < m) src[u] = row_offset(a, s, kept[j], h), dst[u] = row_offset(e.dst, s, j, h);
        }
#pragma unroll
        for (int u = 0; u < kMoveU; ++u)
            if (src[u] >= 0) x[u] = *reinterpret_cast<const uint4*>(from + src[u] + piece);
#pragma unroll
        for (int u = 0; u < kMoveU; ++u)
            if (src[u] >= 0 && dst[u] >= 0) *reinterpret_cast<uint4*>(to + dst[u] + piece) = x[u];
    }
    if (!e.w_dst) return;
    const float* w = e.w + row * e.w_stride;
    float* wd = e.w_dst + row * e.w_stride;
    for (int j = blockIdx.x * kMoveThreads + tid; j < e.w_stride; j += gridDim.x * kMoveThreads) wd[j] = j < m ? w[kept[j]] : 0.0f;
}

// ---- move in place: places [c0, c1) come from positions >= c0, so with a cluster
// barrier between a step's reads and its writes a later step finds its rows (at
// positions >= c1) as they were
__global__ void __cluster_dims__(kEvC, 1, 1) __launch_bounds__(kInPlaceThreads, 2) k_paged_move_in_place(EvictArgs e) {
    pdl_begin();
    cg::cluster_group cl = cg::this_cluster();
    const PagedArgs& a = e.src;
    const int rank = (int)cl.block_rank(), h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
    const int n = seq_len(a, s), m = n < e.budget ? n : e.budget;
    const int64_t row = (int64_t)s * a.nkv + h;
    const int32_t* kept = e.kept + row * e.budget;
    const float* w = e.w + row * e.w_stride;
    float* wd = e.w_dst ? e.w_dst + row * e.w_stride : nullptr;
    const int pieces = a.hd / 8, per_row = 2 * pieces, rows_cta = kInPlaceThreads / per_row;
    const int lr = tid / per_row, c = tid - lr * per_row, piece = (c >= pieces ? c - pieces : c) * 8;
    const uint16_t* from = c >= pieces ? a.v : a.k;
    uint16_t* to = const_cast<uint16_t*>(c >= pieces ? e.dst.v : e.dst.k);
    const int step = kEvC * rows_cta * kInPlaceU;
    for (int c0 = 0; c0 < m; c0 += step) {
        int64_t dst[kInPlaceU];
        uint4 x[kInPlaceU];
        float wv[kInPlaceU];
#pragma unroll
        for (int u = 0; u < kInPlaceU; ++u) {
            const int j = c0 + (u * kEvC + rank) * rows_cta + lr;
            dst[u] = -1, wv[u] = 0.0f;
            if (lr < rows_cta && j < m) {
                const int i = kept[j];
                const int64_t src = row_offset(a, s, i, h);
                if (c == 0) wv[u] = w[i];
                if (src >= 0) dst[u] = row_offset(e.dst, s, j, h), x[u] = *reinterpret_cast<const uint4*>(from + src + piece);
            }
        }
        cl.sync();
#pragma unroll
        for (int u = 0; u < kInPlaceU; ++u) {
            const int j = c0 + (u * kEvC + rank) * rows_cta + lr;
            if (dst[u] >= 0) *reinterpret_cast<uint4*>(to + dst[u] + piece) = x[u];
            if (wd && lr < rows_cta && j < m && c == 0) wd[j] = wv[u];
        }
    }
    cl.sync();
    if (wd)
        for (int j = m + rank * kInPlaceThreads + tid; j < e.w_stride; j += kEvC * kInPlaceThreads) wd[j] = 0.0f;
}

}  // namespace

cudaError_t launch_paged_append(const PagedArgs& a, const uint16_t* k, const uint16_t* v, int64_t row_stride,
                                const int32_t* seq, const int32_t* slot, int T, const int32_t* pos, int max_pos,
                                int num_sms, cudaStream_t st) {
    if (T <= 0) return cudaSuccess;
    const int64_t n = (int64_t)T * a.nkv * (a.hd / 8) * 2, want = (n + 255) / 256, most = (int64_t)num_sms * 8;
    const cudaError_t e = launch_pdl(k_paged_append, dim3((unsigned)(want < most ? want : most)), dim3(256), 0, st, a,
                                     k, v, row_stride, seq, slot, T, pos, max_pos);
    return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_paged_evict(const PagedArgs& src, const PagedArgs& dst, const float* w, float* w_dst, int w_stride,
                               int budget, int n_sink, int n_recent, int32_t* kept, int32_t* new_len, cudaStream_t st) {
    EvictArgs e{src, dst, w, w_dst, w_stride, budget, n_sink, n_recent, kept, new_len,
                src.k == dst.k || src.v == dst.v || w == w_dst};
    // more positions than one CTA holds: a cluster for each (sequence, KV head)
    const int size = src.cap > kEvChunk ? kEvC : 1;
    cudaError_t r = launch_pdl_cluster(k_paged_select, dim3(size, src.nkv, src.n_seqs), dim3(kEvThreads), size, st, e);
    if (r != cudaSuccess) return r;
    if (e.in_place) {
        r = launch_pdl(k_paged_move_in_place, dim3(kEvC, src.nkv, src.n_seqs), dim3(kInPlaceThreads), 0, st, e);
    } else {
        const int rows = kMoveThreads / (src.hd / 4) * kMoveU, most = budget < src.cap ? budget : src.cap;
        r = launch_pdl(k_paged_move, dim3((most + rows - 1) / rows, src.nkv, src.n_seqs), dim3(kMoveThreads), 0, st, e);
    }
    return r != cudaSuccess ? r : cudaGetLastError();
}

}  // namespace obs
