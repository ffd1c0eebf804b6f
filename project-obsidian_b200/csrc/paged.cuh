// paged.cuh -- the paged key/value cache as the kernels see it, and what they
// share: page lookup, element types, the visible range of a query.
#pragma once
#include <cuda_fp16.h>

#include "obs_internal.cuh"

namespace obs {

constexpr int kPagedMaxGroup = 16;         // query heads per KV head
constexpr int kPagedMaxLen = 1 << 20;      // positions of one sequence
constexpr int kPagedMaxPage = 1024;        // positions of one page

// One cache: row (position) j of sequence s lies in page table[s][j / page_size]
// of the pool, at k + page * page_stride + (j % page_size) * slot_stride + head *
// head_stride (elements; head_dim consecutive ones).
struct PagedArgs {
    const uint16_t* k;
    const uint16_t* v;
    const int32_t* table;   // [n_seqs][table_stride]
    const int32_t* len;     // [n_seqs] positions held
    int64_t page_stride, slot_stride, head_stride;
    int n_seqs, n_pages, table_stride;
    int page_size;
    uint32_t page_magic;    // floor(2^32 / page_size) + 1 (0 for page_size 1), see page_of
    int cap;                // positions the table (and the context) has room for
    int nkv, group, hd;
    int* err;
};

// j / page_size for 0 <= j < 2^32 / page_size (here j <= 2^20 + a tile and page_size
// <= 2^10): with m = floor(2^32 / p) + 1, j * m / 2^32 exceeds j / p by at most
// j / 2^32 < 1 / p, less than what separates j / p from the next whole number.
__host__ __device__ __forceinline__ int page_of(const PagedArgs& a, int j) {
#ifdef __CUDA_ARCH__
    return a.page_magic ? (int)__umulhi((uint32_t)j, a.page_magic) : j;
#else
    return a.page_magic ? (int)(((uint64_t)(uint32_t)j * a.page_magic) >> 32) : j;
#endif
}

// Element offset of a row in the pools, or -1 (recorded) where the table names a
// page outside the pool.  j lies in [0, cap).
__device__ __forceinline__ int64_t row_offset(const PagedArgs& a, int s, int j, int head) {
    const int pi = page_of(a, j);
    const int page = a.table[(int64_t)s * a.table_stride + pi];
    if ((unsigned)page >= (unsigned)a.n_pages) {
        atomicExch(a.err, kDevBadPage);
        return -1;
    }
    return page * a.page_stride + (j - pi * a.page_size) * a.slot_stride + head * a.head_stride;
}

// Positions the sequence holds; one outside [0, cap] is refused and recorded.
__device__ __forceinline__ int seq_len(const PagedArgs& a, int s) {
    const int n = a.len[s];
    if (n < 0 || n > a.cap) {
        atomicExch(a.err, kDevBadPage);
        return n < 0 ? 0 : a.cap;
    }
    return n;
}

// The query at position i sees position j <= i where j < n_sink or i - j < window
// (window 0: all of them): the two ranges [0, sink_end) and [win_lo, i + 1).
__device__ __forceinline__ int window_lo(int i, int window) { return window > 0 && i + 1 > window ? i + 1 - window : 0; }

// The sequence and the position of query row t of a prefill: rows q_start[s] ..
// q_start[s + 1] are the sequence's last ones, the last at position len[s] - 1 (a
// sequence with more new rows than positions starts at a negative position: such
// rows see nothing).  False (and recorded) for a row of no sequence.
__device__ __forceinline__ bool find_row(const PagedArgs& a, const int32_t* q_start, int t, int T, int* seq, int* pos) {
    int lo = 0, hi = a.n_seqs;  // q_start[lo] <= t, q_start[hi] > t for some hi > lo
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (q_start[mid] <= t) lo = mid;
        else hi = mid;
    }
    const int q0 = q_start[lo], q1 = q_start[lo + 1];
    if (q0 < 0 || t < q0 || t >= q1 || q1 > T) {
        atomicExch(a.err, kDevBadPos);
        return false;
    }
    *seq = lo;
    *pos = seq_len(a, lo) - (q1 - q0) + (t - q0);
    return true;
}

constexpr int kPagedCtas = 2;  // CTAs per SM of the decode kernel
struct DecodeArgs {
    PagedArgs c;
    const uint16_t* q;        // [n_seqs][nq][hd], rows q_stride elements apart
    int64_t q_stride;
    uint16_t* out;            // [n_seqs][nq][hd]
    int window, n_sink;
    float scale, scale_log2;  // scale_log2 = scale * log2(e)
    float* part;              // 2 per CTA: its parts of (sequence, head)s it shares
    uint32_t* count;          // [CTAs] arrivals, zero between launches
    float* scores;            // with weights: [n_seqs][nkv][score_ld][score_heads] x_j
    int64_t score_ld;
    int score_heads;          // the group, rounded up to even
    float2* ml;               // with weights: [n_seqs][nq] maximum and sum
    float* weights;           // optional: [n_seqs][nkv][w_stride]
    int w_stride;
};
cudaError_t launch_paged_decode(const DecodeArgs& p, int dtype, int num_sms, cudaStream_t st);
size_t paged_decode_part_floats(int group, int num_sms);
struct PrefillArgs {
    PagedArgs c;
    const uint16_t* q;        // [T][nq][hd], rows q_stride elements apart
    int64_t q_stride;
    uint16_t* out;            // [T][nq][hd]
    const int32_t* q_start;   // [n_seqs + 1]
    int T;
    int window, n_sink;
    float scale, scale_log2;  // scale_log2 = scale * log2(e)
    uint64_t wait_ns;
    // set by the launcher
    int splits;
    float* part_acc;          // [splits][T][nq][64 or 128]
    float2* part_ml;          // [splits][T][nq]
    uint32_t group_magic;     // for row_of
};
cudaError_t launch_paged_prefill(PrefillArgs p, float* part, int dtype, int num_sms, cudaStream_t st);
size_t paged_prefill_part_floats(int num_sms);
cudaError_t launch_paged_append(const PagedArgs& a, const uint16_t* k, const uint16_t* v, int64_t row_stride,
                                const int32_t* seq, const int32_t* slot, int T, const int32_t* pos, int max_pos,
                                int num_sms, cudaStream_t st);
cudaError_t launch_paged_evict(const PagedArgs& src, const PagedArgs& dst, const float* w, float* w_dst, int w_stride,
                               int budget, int n_sink, int n_recent, int32_t* kept, int32_t* new_len, cudaStream_t st);

// 16-bit element types: bf16 (0) and f16 (1)
template <int DT>
struct Elem;
template <>
struct Elem<0> {
    static __device__ __forceinline__ float f(uint16_t h) { return bf2f(h); }
    static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
    static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
    static __device__ __forceinline__ uint16_t h(float f) { return f2bf(f); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf2(a, b); }
};
template <>
struct Elem<1> {
    static __device__ __forceinline__ float f(uint16_t h) { return __half2float(__ushort_as_half(h)); }
    static __device__ __forceinline__ float lo(uint32_t w) { return f((uint16_t)w); }
    static __device__ __forceinline__ float hi(uint32_t w) { return f((uint16_t)(w >> 16)); }
    static __device__ __forceinline__ uint16_t h(float f) { return __half_as_ushort(__float2half_rn(f)); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 16 bytes to shared memory without passing the registers, or zeros
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}

// One query row against its visible positions, one warp, scalar (lane l holds the
// four dimensions 4l .. 4l+3): the online softmax in the order of the positions.
// qf: the lane's four query values; acc, m, l: the lane's four output sums, the
// maximum and the sum.  Positions are visited as [0, sink_end) then [lo, hi).
template <int DT>
__device__ __forceinline__ void attend_row(const PagedArgs& a, int s, int head, const float (&qf)[4], float scale,
                                           int sink_end, int lo, int hi, float (&acc)[4], float& m, float& l) {
    using X = Elem<DT>;
    const int lane = threadIdx.x & 31;
    const bool mine = 4 * lane < a.hd;
    m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = 0.0f;
    for (int j = sink_end > 0 ? 0 : lo; j < hi; j = (j + 1 == sink_end && lo > sink_end) ? lo : j + 1) {
        const int64_t off = row_offset(a, s, j, head);
        uint2 kw = make_uint2(0, 0), vw = make_uint2(0, 0);
        if (mine && off >= 0) {
            kw = *reinterpret_cast<const uint2*>(a.k + off + 4 * lane);
            vw = *reinterpret_cast<const uint2*>(a.v + off + 4 * lane);
        }
        float x = qf[0] * X::lo(kw.x) + qf[1] * X::hi(kw.x) + qf[2] * X::lo(kw.y) + qf[3] * X::hi(kw.y);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        x *= scale;
        const float mn = fmaxf(m, x), ref = mn == -INFINITY ? 0.0f : mn;
        const float corr = expf(m - ref), p = expf(x - ref);
        l = l * corr + p;
        acc[0] = acc[0] * corr + p * X::lo(vw.x), acc[1] = acc[1] * corr + p * X::hi(vw.x);
        acc[2] = acc[2] * corr + p * X::lo(vw.y), acc[3] = acc[3] * corr + p * X::hi(vw.y);
        m = mn;
    }
}

}  // namespace obs
