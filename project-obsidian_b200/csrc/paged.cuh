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
    static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
    static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
    static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf2(a, b); }
};
template <>
struct Elem<1> {
    static __device__ __forceinline__ float lo(uint32_t w) { return __half2float(__ushort_as_half((uint16_t)w)); }
    static __device__ __forceinline__ float hi(uint32_t w) { return __half2float(__ushort_as_half((uint16_t)(w >> 16))); }
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

template <int DT>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (DT == 0)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// ---- rows whose result is not finite although the sum of their exponentials is: a NaN
// or an infinity in V, which the products spread to rows that do not see it (0 * NaN) and
// turn into NaN (infinity times what rounding left of p).  Their dimensions that are not
// finite are computed again, 16 rows by a warp: p from the known maximum and sum (divided
// by the sum before the products: finite values that only added up past fp32 do not here),
// the products on mma.sync with the positions that hold anything not finite taken out, and
// those, for the rows that see them, by fp32 FMAs, where IEEE arithmetic does what the
// formula says.
//
// Bounded: every position that the rows see is read once more per 16 rows, whatever V
// holds.  One prompt of 4096 (32 / 4 heads of 128, bf16) with one infinity at its front,
// which every row sees: 1.9 ms; with nothing but infinities in V 8.9 ms; 155 us without.
// A row by a warp, one position at a time, took 25 ms for a prompt of 2048.
// A part's sums and its l are kept times 2^-28: l is at most 2^20 positions times 2^8 (a
// maximum in use that the scores have outgrown), so no join of finite values passes fp32.
constexpr float kJoinScale = 1.0f / (1 << 28);
static_assert(kPagedMaxLen <= 1 << 20, "l");

struct AgainRows {              // a lane's two rows: g and g + 8 of 16, g = lane / 4
    const uint16_t* q[2];       // null: no such row
    void* out[2];               // 16-bit values, or a part's fp32 sums
    int i[2], lo[2];            // its position and its window's first
    float ref[2], l[2];         // p = 2^(scale log2 e q . k - ref) / l
};
// Positions: tiles x0 .. x0 + nt of 64 (x < ts: tile x, else x - ts + wt).  Dimensions 64 v .. 64 v + 63.
template <int DT>
__device__ __forceinline__ void attend_again(const PagedArgs& a, int s, int h, const AgainRows& rows, bool f32, int x0, int nt,
                                          int ts, int wt, int n_sink, float scale_log2, int v) {
    using X = Elem<DT>;
    constexpr uint32_t kExp = DT == 0 ? 0x7F80u : 0x7C00u;
    constexpr float kScaleP = DT == 0 ? 1.0f : 32768.0f;  // f16 holds nothing below 2^-25
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int hd = a.hd;
    float wl[2];
    int i_max = -1, lo_min = 0x7fffffff;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const bool row = rows.q[r] != nullptr;
        wl[r] = kScaleP / rows.l[r];
        if (row) i_max = max(i_max, rows.i[r]), lo_min = min(lo_min, rows.lo[r]);
    }
    i_max = __reduce_max_sync(0xffffffffu, i_max), lo_min = __reduce_min_sync(0xffffffffu, lo_min);
    auto sees = [&](int r, int j) {
        return rows.q[r] != nullptr && j <= rows.i[r] && (j >= rows.lo[r] || j < n_sink);
    };
    // acc[e][2 r + b]: row r of the lane's, dimension 64 v + 16 t + 8 b + e
    float acc[8][4];
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[e][c] = 0.0f;

#pragma unroll 1
    for (int n = 0; n < 4 * nt; ++n) {
        const int x = x0 + n / 4, j0 = (x < ts ? x : x - ts + wt) * 64 + (n & 3) * 16;
        int64_t off = -1;
        const int jl = j0 + (lane & 15);
        if (jl <= i_max && (jl >= lo_min || jl < n_sink)) off = row_offset(a, s, jl, h);
        if (!__any_sync(0xffffffffu, off >= 0)) continue;
        float x8[2][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int64_t o = __shfl_sync(0xffffffffu, off, 8 * half + g);
            float (&c)[4] = x8[half];
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] = 0.0f;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                // any order of the dimensions will do in q . k, the same for both: lane t takes 16
                // bytes, dimensions 32 u + 8 t .. + 7, for two steps of 16 (q again for every 8
                // positions: held, it would cost the calling kernel's loop registers)
                uint4 k = make_uint4(0, 0, 0, 0), q0 = k, q1 = k;
                const int d = 32 * u + 8 * t;
                if (d < hd) {
                    if (o >= 0) k = *reinterpret_cast<const uint4*>(a.k + o + d);
                    if (rows.q[0]) q0 = *reinterpret_cast<const uint4*>(rows.q[0] + d);
                    if (rows.q[1]) q1 = *reinterpret_cast<const uint4*>(rows.q[1] + d);
                }
                const uint32_t a0[4] = {q0.x, q1.x, q0.y, q1.y}, a1[4] = {q0.z, q1.z, q0.w, q1.w};
                mma16816<DT>(c, a0, k.x, k.y);
                mma16816<DT>(c, a1, k.z, k.w);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {  // row e / 2 of the lane's, position 2 t + e % 2
                c[e] = sees(e >> 1, j0 + 8 * half + 2 * t + (e & 1)) ? ex2(c[e] * scale_log2 - rows.ref[e >> 1]) * wl[e >> 1] : 0.0f;
            }
        }
        // p and what its rounding left, as the A operand of 16 positions
        uint32_t p[4], rest[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float p0 = x8[e >> 1][2 * (e & 1)], p1 = x8[e >> 1][2 * (e & 1) + 1];
            p[e] = X::pack(p0, p1);
            rest[e] = X::pack(p0 - X::lo(p[e]), p1 - X::hi(p[e]));
        }
        // rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of V, dimensions 64 v + 8 g .. + 7
        uint4 w[4];
        uint32_t odd = 0;  // bit r: the lane's piece of row r holds something not finite
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t o = __shfl_sync(0xffffffffu, off, 2 * t + (r & 1) + 8 * (r >> 1));
            w[r] = make_uint4(0, 0, 0, 0);
            if (o >= 0 && 64 * v + 8 * g < hd) w[r] = *reinterpret_cast<const uint4*>(a.v + o + 64 * v + 8 * g);
            const uint32_t z[4] = {w[r].x, w[r].y, w[r].z, w[r].w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if ((z[e] & kExp) == kExp || (z[e] >> 16 & kExp) == kExp) odd |= 1u << r;
        }
        uint32_t taken = 0;  // positions of the 16 that hold something not finite
        if (__any_sync(0xffffffffu, odd != 0)) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t who = __ballot_sync(0xffffffffu, odd >> r & 1u);  // lanes 4 g + t
#pragma unroll
                for (int tt = 0; tt < 4; ++tt)
                    if (who >> tt & 0x11111111u) taken |= 1u << (2 * tt + (r & 1) + 8 * (r >> 1));
                if (taken >> (2 * t + (r & 1) + 8 * (r >> 1)) & 1u) w[r] = make_uint4(0, 0, 0, 0);
            }
        }
        // column g of the product e is dimension 64 v + 8 g + e
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int sel = e & 1 ? 0x7632 : 0x5410;
            const uint32_t lo4[4] = {w[0].x, w[0].y, w[0].z, w[0].w}, lo5[4] = {w[1].x, w[1].y, w[1].z, w[1].w};
            const uint32_t hi4[4] = {w[2].x, w[2].y, w[2].z, w[2].w}, hi5[4] = {w[3].x, w[3].y, w[3].z, w[3].w};
            const uint32_t b0 = __byte_perm(lo4[e >> 1], lo5[e >> 1], sel), b1 = __byte_perm(hi4[e >> 1], hi5[e >> 1], sel);
            mma16816<DT>(acc[e], rest, b0, b1);
            mma16816<DT>(acc[e], p, b0, b1);
        }
        while (taken) {
            const int c = __ffs(taken) - 1;
            taken &= taken - 1;
            const int64_t o = __shfl_sync(0xffffffffu, off, c);
            const int half = c >> 3, from = (lane & ~3) | ((c & 7) >> 1);  // the lane that holds the rows' p at c
            float pc[2];
            bool see[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float p0 = __shfl_sync(0xffffffffu, half ? x8[1][2 * r] : x8[0][2 * r], from);
                const float p1 = __shfl_sync(0xffffffffu, half ? x8[1][2 * r + 1] : x8[0][2 * r + 1], from);
                pc[r] = c & 1 ? p1 : p0, see[r] = sees(r, j0 + c);
            }
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int d = 64 * v + 16 * t + 8 * b;
                if (o < 0 || d >= hd) continue;
                const uint4 y = *reinterpret_cast<const uint4*>(a.v + o + d);
                const uint32_t z[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float f = e & 1 ? X::hi(z[e >> 1]) : X::lo(z[e >> 1]);
#pragma unroll
                    for (int r = 0; r < 2; ++r)
                        if (see[r]) acc[e][2 * r + b] += pc[r] * f;
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int d = 64 * v + 16 * t + 8 * b;
            if (rows.q[r] == nullptr || d >= hd) continue;
            if (f32) {
                float* dst = static_cast<float*>(rows.out[r]) + d;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (!(fabsf(dst[e]) <= 3.4e38f)) dst[e] = acc[e][2 * r + b] * kJoinScale / wl[r];
            } else {
                uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(rows.out[r]) + d);
                const uint4 y = *dst;
                uint32_t z[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t n = X::pack(acc[2 * e][2 * r + b] * (1.0f / kScaleP), acc[2 * e + 1][2 * r + b] * (1.0f / kScaleP));
                    if ((z[e] & kExp) == kExp) z[e] = (z[e] & 0xFFFF0000u) | (n & 0xFFFFu);
                    if ((z[e] >> 16 & kExp) == kExp) z[e] = (z[e] & 0xFFFFu) | (n & 0xFFFF0000u);
                }
                *dst = make_uint4(z[0], z[1], z[2], z[3]);
            }
        }
}

}  // namespace obs
