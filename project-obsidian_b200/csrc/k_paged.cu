// k_paged.cu -- the paged key/value cache: rows into their pages, and eviction by
// accumulated attention weight.  The reference keeps one dense cache per layer
// (kv_cache.rs:15-24, ops.metal:32-37) and has no counterpart of either.
#include <cooperative_groups.h>

#include "paged.cuh"

namespace cg = cooperative_groups;

namespace obs {
namespace {

// Row t of k and v ([T] rows of n_kv * head_dim elements, row_stride apart) to
// position slot[t] of sequence seq[t].  One 16-byte piece per thread; bound by
// the launch for a decode step and by memory for a prompt.
__global__ void __launch_bounds__(256) k_paged_append(PagedArgs a, const uint16_t* k, const uint16_t* v,
                                                      int64_t row_stride, const int32_t* seq, const int32_t* slot,
                                                      int T) {
    pdl_begin();
    const int per_head = a.hd / 8, per_row = a.nkv * per_head;  // 16-byte pieces
    const int64_t n = (int64_t)T * per_row * 2;
    for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int t = (int)(i / (2 * per_row)), r = (int)(i - (int64_t)t * 2 * per_row);
        const bool isv = r >= per_row;
        const int c = isv ? r - per_row : r, head = c / per_head, piece = c - head * per_head;
        const int s = seq[t], j = slot[t];
        if ((unsigned)s >= (unsigned)a.n_seqs || (unsigned)j >= (unsigned)a.cap) {
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
// first n_sink, the last n_recent and, of the rest, the budget - n_sink - n_recent
// with the largest weights (equal weights: the lowest position; NaN lowest of all).
// A cluster of kEvC CTAs per (s, h):
//   select   radix selection over the weights as ordered 32-bit keys, 11 + 11 + 10
//            bits from the top: a histogram per CTA in shared memory, summed over
//            the cluster through distributed shared memory, gives the digit of the
//            threshold key; then each CTA's part of the positions is counted and
//            walked in order, which gives every kept position its place.
//   move     the kept rows to places 0, 1, ... of dst in steps of rows that the
//            cluster holds in registers: places [c0, c1) come from positions >= c0,
//            so with a cluster barrier between a step's reads and its writes the
//            move may be in place (a later step reads positions >= c1 only).
constexpr int kEvC = 8, kEvThreads = 512, kEvBins = 2048;

// larger weight <=> larger key; -0 and +0 equal; NaN the smallest
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

// inclusive prefix sum of one value per thread over the CTA; returns the sum over
// the threads before this one, total in *sum
__device__ __forceinline__ int block_excl(int v, int* s_warp, int* sum) {
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
    if (warp == 0) {
        int t = lane < kEvThreads / 32 ? s_warp[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, t, o);
            if (lane >= o) t += y;
        }
        s_warp[lane] = t;
    }
    __syncthreads();
    *sum = s_warp[kEvThreads / 32 - 1];
    return x - v + (warp ? s_warp[warp - 1] : 0);
}

__global__ void __cluster_dims__(kEvC, 1, 1) __launch_bounds__(kEvThreads) k_paged_evict(EvictArgs e) {
    pdl_begin();
    cg::cluster_group cl = cg::this_cluster();
    __shared__ uint32_t s_hist[2][kEvBins];
    __shared__ int s_warp[32];
    __shared__ int s_cnt[2];
    __shared__ uint32_t s_digit, s_above;
    const PagedArgs& a = e.src;
    const int rank = (int)cl.block_rank(), h = blockIdx.y, s = blockIdx.z, tid = threadIdx.x;
    const int n = seq_len(a, s), m = n < e.budget ? n : e.budget;
    const int64_t row = (int64_t)s * a.nkv + h;
    const float* w = e.w + row * e.w_stride;
    int32_t* kept = e.kept + row * e.budget;
    if (rank == 0 && h == 0 && tid == 0) e.new_len[s] = m;

    if (n <= e.budget) {
        for (int j = rank * kEvThreads + tid; j < e.budget; j += kEvC * kEvThreads) kept[j] = j < n ? j : -1;
    } else {
        const int lo = e.n_sink, hi = n - e.n_recent, need = e.budget - e.n_sink - e.n_recent;
        const int per = (hi - lo + kEvC - 1) / kEvC;
        const int b0 = min(hi, lo + rank * per), b1 = min(hi, b0 + per);
        // the threshold key, digit by digit from the top; `left`: how many of the keys
        // that share the digits found so far are kept
        uint32_t prefix = 0;
        int left = need;
        const int shift[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            uint32_t* hist = s_hist[pass & 1];
            const int bins = 1 << bits[pass], sh = shift[pass];
            for (int i = tid; i < bins; i += kEvThreads) hist[i] = 0;
            __syncthreads();
            for (int j = b0 + tid; j < b1; j += kEvThreads) {
                const uint32_t key = weight_key(w[j]);
                if (pass == 0 || (key >> (sh + bits[pass])) == prefix) atomicAdd(&hist[(key >> sh) & (bins - 1)], 1u);
            }
            cl.sync();
            // bins from the top, a run of them per thread
            const int run = bins / kEvThreads;
            uint32_t c[kEvBins / kEvThreads];
            int mine = 0;
#pragma unroll
            for (int i = 0; i < kEvBins / kEvThreads; ++i) {
                c[i] = 0;
                if (i < run) {
                    const int b = bins - 1 - (tid * run + i);
#pragma unroll
                    for (int r = 0; r < kEvC; ++r) c[i] += cl.map_shared_rank(hist, r)[b];
                    mine += (int)c[i];
                }
            }
            int total;
            int before = block_excl(mine, s_warp, &total);
            // the bin in which the left-th largest key lies (left == 0: no key is kept)
#pragma unroll
            for (int i = 0; i < kEvBins / kEvThreads; ++i) {
                if (i < run) {
                    if (before < left && before + (int)c[i] >= left)
                        s_digit = bins - 1 - (tid * run + i), s_above = before;
                    before += (int)c[i];
                }
            }
            if (left == 0 && tid == 0) s_digit = bins - 1, s_above = 0;
            __syncthreads();
            prefix = (prefix << bits[pass]) | s_digit;
            left -= (int)s_above;
            __syncthreads();
        }
        // above the threshold: kept; equal to it: the first `left` of them
        int ngt = 0, neq = 0;
        for (int j = b0 + tid; j < b1; j += kEvThreads) {
            const uint32_t key = weight_key(w[j]);
            ngt += key > prefix, neq += key == prefix;
        }
        if (need == 0) ngt = 0;
        int tgt, teq;
        block_excl(ngt, s_warp, &tgt);
        block_excl(neq, s_warp, &teq);
        if (tid == 0) s_cnt[0] = tgt, s_cnt[1] = teq;
        cl.sync();
        int gt0 = 0, eq0 = 0;
        for (int r = 0; r < rank; ++r) {
            const int* c = cl.map_shared_rank(s_cnt, r);
            gt0 += c[0], eq0 += c[1];
        }
        for (int j = rank * kEvThreads + tid; j < e.n_sink; j += kEvC * kEvThreads) kept[j] = j;
        for (int j = rank * kEvThreads + tid; j < e.n_recent; j += kEvC * kEvThreads)
            kept[e.budget - e.n_recent + j] = n - e.n_recent + j;
        for (int base = b0; base < b1 && need > 0; base += kEvThreads) {
            const int j = base + tid;
            const uint32_t key = j < b1 ? weight_key(w[j]) : 0u;
            const bool gt = j < b1 && key > prefix, eq = j < b1 && key == prefix;
            int ng, ne;
            const int g = gt0 + block_excl(gt, s_warp, &ng);
            const int q = eq0 + block_excl(eq, s_warp, &ne);
            if (gt || (eq && q < left)) kept[e.n_sink + g + min(q, left)] = j;
            gt0 += ng, eq0 += ne;
        }
    }
    cl.sync();  // kept is complete (and no CTA reads another's shared memory any more)

    // ---- move
    const int pieces = a.hd / 8;                 // 16-byte pieces of one row of K (or V)
    const int per_row = 2 * pieces;
    const int rows_cta = kEvThreads / per_row;   // rows of one register step of a CTA
    const int lr = tid / per_row, c = tid - lr * per_row;
    const bool isv = c >= pieces;
    const int piece = (isv ? c - pieces : c) * 8;
    constexpr int U = 4;
    const int step = kEvC * rows_cta * U;
    const float* wsrc = w;
    float* wdst = e.w_dst ? e.w_dst + row * e.w_stride : nullptr;
    for (int c0 = 0; c0 < m; c0 += step) {
        uint4 x[U];
        int64_t to[U];
        float wv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = c0 + (u * kEvC + rank) * rows_cta + lr;
            to[u] = -1;
            if (lr < rows_cta && j < m) {
                const int from = kept[j];
                if (c == 0) wv[u] = wsrc[from];
                const int64_t src = row_offset(a, s, from, h);
                to[u] = row_offset(e.dst, s, j, h);
                if (src < 0) to[u] = -1;
                if (to[u] >= 0) x[u] = *reinterpret_cast<const uint4*>((isv ? a.v : a.k) + src + piece);
            }
        }
        if (e.in_place) cl.sync();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = c0 + (u * kEvC + rank) * rows_cta + lr;
            if (to[u] >= 0) {
                *reinterpret_cast<uint4*>(const_cast<uint16_t*>(isv ? e.dst.v : e.dst.k) + to[u] + piece) = x[u];
            }
            if (wdst && lr < rows_cta && j < m && c == 0) wdst[j] = wv[u];
        }
    }
    // the rest of the weights' row is cleared for the positions to come
    if (e.in_place) cl.sync();
    if (wdst)
        for (int j = m + rank * kEvThreads + tid; j < e.w_stride; j += kEvC * kEvThreads) wdst[j] = 0.0f;
}

// ------------------------------------------------- attention, the plain kernel
// One CTA per (query row, KV head), one warp per query head of the group: every
// visible position in order.  weights (decode): the probabilities in a second
// walk, the group's heads summed in order.
template <int DT>
__global__ void __launch_bounds__(kPagedMaxGroup * 32) k_paged_attn_rows(AttnRowsArgs p) {
    pdl_begin();
    using X = Elem<DT>;
    __shared__ float s_m[kPagedMaxGroup], s_l[kPagedMaxGroup];
    const PagedArgs& a = p.c;
    const int t = blockIdx.x, h = blockIdx.y, g = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int s = t, i;
    if (p.q_start) {
        if (!find_row(a, p.q_start, t, p.T, &s, &i)) return;
    } else {
        i = seq_len(a, s) - 1;
    }
    const int nq = a.nkv * a.group, head = h * a.group + g;
    const int hi = i + 1, lo = window_lo(i, p.window), sink_end = min(p.n_sink, lo);
    const uint16_t* q = p.q + t * p.q_stride + head * a.hd;
    float qf[4] = {0.0f, 0.0f, 0.0f, 0.0f}, acc[4], m, l;
    if (4 * lane < a.hd) {
        const uint2 w = *reinterpret_cast<const uint2*>(q + 4 * lane);
        qf[0] = X::lo(w.x), qf[1] = X::hi(w.x), qf[2] = X::lo(w.y), qf[3] = X::hi(w.y);
    }
    attend_row<DT>(a, s, h, qf, p.scale, sink_end, lo, hi, acc, m, l);
    if (4 * lane < a.hd) {
        uint2 o = make_uint2(0, 0);  // nothing visible: zeros
        if (hi > 0) o = make_uint2(X::pack(acc[0] / l, acc[1] / l), X::pack(acc[2] / l, acc[3] / l));
        *reinterpret_cast<uint2*>(p.out + ((int64_t)t * nq + head) * a.hd + 4 * lane) = o;
    }
    if (!p.weights) return;
    if (lane == 0) s_m[g] = m, s_l[g] = l;
    __syncthreads();
    float* w = p.weights + ((int64_t)s * a.nkv + h) * p.w_stride;
    for (int j = g; j < hi; j += a.group) {
        if (j >= sink_end && j < lo) continue;
        const int64_t off = row_offset(a, s, j, h);
        if (off < 0) continue;
        float sum = 0.0f;
        for (int gg = 0; gg < a.group; ++gg) {
            float x = 0.0f;
            for (int d = lane; d < a.hd; d += 32)
                x += X::f(p.q[t * p.q_stride + (h * a.group + gg) * a.hd + d]) * X::f(a.k[off + d]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
            sum += expf(x * p.scale - s_m[gg]) / s_l[gg];
        }
        if (lane == 0) w[j] += sum;
    }
}

}  // namespace

cudaError_t launch_paged_append(const PagedArgs& a, const uint16_t* k, const uint16_t* v, int64_t row_stride,
                                const int32_t* seq, const int32_t* slot, int T, int num_sms, cudaStream_t st) {
    if (T <= 0) return cudaSuccess;
    const int64_t n = (int64_t)T * a.nkv * (a.hd / 8) * 2, want = (n + 255) / 256, most = (int64_t)num_sms * 8;
    const cudaError_t e = launch_pdl(k_paged_append, dim3((unsigned)(want < most ? want : most)), dim3(256), 0, st, a,
                                     k, v, row_stride, seq, slot, T);
    return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_paged_evict(const PagedArgs& src, const PagedArgs& dst, const float* w, float* w_dst, int w_stride,
                               int budget, int n_sink, int n_recent, int32_t* kept, int32_t* new_len, cudaStream_t st) {
    EvictArgs e{src, dst, w, w_dst, w_stride, budget, n_sink, n_recent, kept, new_len,
                src.k == dst.k || src.v == dst.v || w == w_dst};
    const cudaError_t r = launch_pdl(k_paged_evict, dim3(kEvC, src.nkv, src.n_seqs), dim3(kEvThreads), 0, st, e);
    return r != cudaSuccess ? r : cudaGetLastError();
}

cudaError_t launch_paged_attn_rows(const AttnRowsArgs& p, int dtype, cudaStream_t st) {
    const int rows = p.q_start ? p.T : p.c.n_seqs;
    if (rows <= 0) return cudaSuccess;
    const cudaError_t e = launch_pdl(dtype ? k_paged_attn_rows<1> : k_paged_attn_rows<0>, dim3(rows, p.c.nkv),
                                     dim3(32 * p.c.group), 0, st, p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace obs
