// k_paged_decode.cu -- attention of one new token per sequence over its pages,
// split over the length and joined, in one launch.
//
//   out[s][h] = sum_j p_j v_j,  p = softmax over the visible j of scale * q[s][h] . k_j
//
// What bounds it: every visible row of K and V is read once from memory for the
// group of query heads that share it, 2 * head_dim * 2 bytes against 4 * head_dim *
// group operations, 8 operations a byte at a group of 8: far below what the tensor
// cores want and, with the conversions to fp32, above what the FMA units give, so
// the two products run on mma.sync tiles whose N is the group (tcgen05's M = 128
// would be seven eighths padding) and the loads decide.
//
// Work: the visible positions of every (sequence, KV head) in tiles of 64, all the
// tiles in one line, cut into equal runs, one per CTA, however ragged the lengths.
// A CTA has four warps; warp w owns positions 16w .. 16w + 15 of each tile, its own
// ring of cp.async stages (16 K rows and 16 V rows each, 16-byte pieces swizzled by
// row so that ldmatrix meets no bank twice) and its own running maximum, sum and
// accumulator, so nothing in the loop waits for another warp:
//   S^T [16 positions x 8 heads] = K . Q^T       A = K rows, B = q held in registers
//   p = 2^(x - m) with x = S scale log2 e, m the running maximum per head
//   O^T [head_dim x 8 heads] += V^T . P^T         A = V rows transposed by ldmatrix,
//                                                 B = the P tile transposed in registers
// Positions a query does not see are not loaded (zeros stand in) and get x = -inf,
// so what lies there does not matter.  The four warps meet at the end of a run of
// one (sequence, KV head); a run that is not all of it leaves (m, l, O) in fp32 and
// the last of its CTAs to arrive joins the parts in their order, so the result does
// not depend on which one that is.
//
// p enters the second product as two 16-bit values, its rounding and what the
// rounding left: the tensor cores multiply 16-bit values, one rounding of p would add
// as much error as the output's own (k_paged_prefill.cu has the figures), and the
// second set of products is hidden behind the loads.
//
// f16 holds nothing below 2^-25, and a first position that many scores fall 2^25 behind
// is common: p <= 1 is multiplied by 2^15 there, and the sums by 2^-15 at their end.
//
// An infinity in V times what rounding left of its p, zero or negative, would be NaN: a
// CTA whose sums of a run are not finite although l is computes those of its run again
// (attend_again), before the join.  When nothing is wrong this costs a comparison.
//
// Measured, 32 / 4 heads of 128: 32 sequences of 61 to 32768 positions in f16, pages of
// 16: 173 to 190 us on different GPUs, 6.4 to 5.9 TB/s, 98% to 89% of the measured copy
// rate; 128 sequences with a window of 1024 and 4 sinks 52 to 57 us (79% to 72%: each CTA
// starts and ends inside some item, and joining takes it from loading); one of 2049 9.4 us, where the launch, four dependent accesses
// to the first rows and the join are nearly all of it.
#include "paged.cuh"

namespace obs {
namespace {

constexpr int kTile = 64;                       // positions per tile: 16 per warp
constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kStages = 3;                      // per warp
constexpr int kMinTiles = 3;                    // of a CTA's run: fewer parts to join (one sequence of 2049: 9.3 us,
                                                // with 1 or 2 tiles 9.9 and 10.1, with 4 or 6 11.2 and 12.6)

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t movm(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// The visible tiles of one sequence: tiles 0 .. ts-1 (sinks), then wt .. (window).
struct Span {
    int n, lo, sink_end;  // positions held, the window's first, the sinks' end
    int ts, wt, nt;       // sink tiles, the window's first tile, tiles in all
};
__device__ __forceinline__ Span span_of(int n, int window, int n_sink) {
    Span p;
    p.n = n;
    p.lo = n > 0 ? window_lo(n - 1, window) : 0;
    p.sink_end = min(n_sink, p.lo);
    p.ts = (p.sink_end + kTile - 1) / kTile;
    p.wt = max(p.ts, p.lo / kTile);
    p.nt = p.ts + max(0, (n + kTile - 1) / kTile - p.wt);
    return p;
}

// A place in the line of tiles: tile x of (sequence s, KV head h).
struct Place {
    int s, h, x;
    Span sp;
};
// to the next tile (the caller knows that there is one)
__device__ __forceinline__ void advance(const PagedArgs& a, int window, int n_sink, Place& p) {
    if (++p.x < p.sp.nt) return;
    p.x = 0;
    if (++p.h < a.nkv) return;
    p.h = 0;
    do {
        ++p.s;
        p.sp = span_of(seq_len(a, p.s), window, n_sink);
    } while (p.sp.nt == 0 && p.s + 1 < a.n_seqs);
}

// one part: group rows of HD sums, then group (maximum, sum) pairs; 16-byte aligned
__host__ __device__ constexpr int part_floats(int group, int hd) { return group * hd + (2 * group + 3) / 4 * 4; }

__device__ __forceinline__ bool needs_again(const float (&o)[4], float l) {
    const float z = o[0] * 0.0f + o[1] * 0.0f + (o[2] * 0.0f + o[3] * 0.0f);  // NaN unless all are finite
    return z != 0.0f && l > 0.0f && l <= 3.4e38f;
}
// The group's rows of one run again, by a warp for 64 dimensions: tiles x0 .. x1 of (s, h),
// `part` null where the run is all of it.  run: each head's maximum and sum.
template <int DT, int HD>
__device__ __noinline__ void run_again(const DecodeArgs& p, int s, int h, int x0, int x1, float* part, const float2* run) {
    const PagedArgs& a = p.c;
    const int g = (threadIdx.x & 31) >> 2, warp = threadIdx.x >> 5, nq = a.nkv * a.group;
    if (warp >= HD / 64) return;
    const Span sp = span_of(seq_len(a, s), p.window, p.n_sink);
    AgainRows rows;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int head = g + 8 * r;
        const bool in = head < a.group;
        rows.q[r] = in ? p.q + s * p.q_stride + (h * a.group + head) * a.hd : nullptr;
        rows.out[r] = part ? static_cast<void*>(part + head * HD)
                           : static_cast<void*>(p.out + ((int64_t)s * nq + h * a.group + head) * a.hd);
        rows.i[r] = sp.n - 1, rows.lo[r] = sp.lo;
        rows.ref[r] = in ? run[head].x : 0.0f, rows.l[r] = in ? run[head].y : 1.0f;
    }
    attend_again<DT>(a, s, h, rows, part != nullptr, x0, x1 - x0 + 1, sp.ts, sp.wt, p.n_sink, p.scale_log2, warp);
}

template <int HD>
struct DecodeSmem {
    static constexpr int ROW = HD * 2, HALF = 16 * ROW;      // a stage: 16 K rows, 16 V rows
    static constexpr int STAGE = 2 * HALF;
    static constexpr int RING = kWarps * kStages * STAGE;
    static constexpr int MRG_LD = 64 + 4;                    // a head's row in the joining buffer
    static constexpr int MRG = kWarps * 8 * MRG_LD * 4;      // one half of the dimensions of 8 heads
    static constexpr int BYTES = RING + MRG;
};

template <int DT, int HD, int NT>
__global__ void __launch_bounds__(kThreads, 2) k_paged_decode(const __grid_constant__ DecodeArgs p) {
    pdl_begin();
    using X = Elem<DT>;
    using M = DecodeSmem<HD>;
    constexpr float kScaleP = DT == 0 ? 1.0f : 32768.0f;
    extern __shared__ __align__(1024) uint8_t smem[];
    float* s_mrg = reinterpret_cast<float*>(smem + M::RING);
    __shared__ float s_m[kWarps][16], s_l[kWarps][16];
    __shared__ float2 s_run[16];  // the run's maximum (0 for -inf) and sum
    __shared__ uint32_t s_scan[kWarps], s_first;
    __shared__ int s_seq;
    __shared__ int s_last;
    const PagedArgs& a = p.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int nq = a.nkv * a.group, G = a.group;

    // ---- this CTA's run of the line: N tiles in `grid` runs, the first `more` of them
    // one longer than the others
    uint32_t N, first = 0;
    int seq = 0;
    auto cut = [&](uint32_t total, uint32_t* grid, uint32_t* each, uint32_t* more) {
        *grid = min((uint32_t)gridDim.x, max(1u, total / kMinTiles));
        *each = total / *grid, *more = total - *each * *grid;
    };
    uint32_t grid, each, more, u0;
    auto start_of = [&](uint32_t c) { return c * each + min(c, more); };
    auto owner_of = [&](uint32_t u) {
        const uint32_t longer = more * (each + 1);
        return u < longer ? u / (each + 1) : more + (u - longer) / each;
    };
    if (a.n_seqs <= 32) {
        // every warp for itself, a sequence per lane
        const uint32_t mine = lane < a.n_seqs ? span_of(seq_len(a, lane), p.window, p.n_sink).nt * a.nkv : 0;
        uint32_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        N = __shfl_sync(0xffffffffu, incl, 31);
        cut(N, &grid, &each, &more);
        u0 = start_of(min((uint32_t)blockIdx.x, grid));
        const uint32_t who = __ballot_sync(0xffffffffu, u0 >= incl - mine && u0 < incl);
        seq = who ? __ffs(who) - 1 : 0;
        first = __shfl_sync(0xffffffffu, incl - mine, seq);
    } else {
        const int per = (a.n_seqs + kThreads - 1) / kThreads;
        const int sb = min(a.n_seqs, tid * per), se = min(a.n_seqs, sb + per);
        uint32_t mine = 0;
        for (int s = sb; s < se; ++s) mine += span_of(seq_len(a, s), p.window, p.n_sink).nt * a.nkv;
        uint32_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) s_scan[warp] = incl;
        __syncthreads();
        uint32_t before = incl - mine;
        N = 0;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            if (w < warp) before += s_scan[w];
            N += s_scan[w];
        }
        cut(N, &grid, &each, &more);
        u0 = start_of(min((uint32_t)blockIdx.x, grid));
        if (u0 >= before && u0 < before + mine) {
            uint32_t b = before;
            for (int s = sb; s < se; ++s) {
                const uint32_t c = span_of(seq_len(a, s), p.window, p.n_sink).nt * a.nkv;
                if (u0 < b + c) {
                    s_seq = s, s_first = b;
                    break;
                }
                b += c;
            }
        }
        __syncthreads();
        seq = s_seq, first = s_first;
    }
    // a sequence without positions gives zeros
    for (int s = blockIdx.x; s < a.n_seqs; s += gridDim.x)
        if (seq_len(a, s) == 0)
            for (int i = tid; i < nq * a.hd; i += kThreads) p.out[(int64_t)s * nq * a.hd + i] = 0;
    if (blockIdx.x >= grid || N == 0) return;
    const int count = (int)(start_of(blockIdx.x + 1) - u0);
    Place ld;
    ld.s = seq;
    ld.sp = span_of(seq_len(a, seq), p.window, p.n_sink);
    ld.h = (int)((u0 - first) / (uint32_t)ld.sp.nt);
    ld.x = (int)(u0 - first) - ld.h * ld.sp.nt;
    Place cs = ld;  // the consumer's place; ld runs ahead

    // ---- loads: this warp's 16 rows of the tile at `ld` into stage st
    const uint32_t ring = smem_u32(smem) + warp * (kStages * M::STAGE);
    constexpr int CH = HD / 8;           // 16-byte pieces per row
    constexpr int RPI = 32 / CH;         // rows per instruction
    const int ch = lane % CH, rsub = lane / CH, chunks = a.hd / 8;
    // the row that lane l < 16 looks up: -1 where it is not visible (or refused)
    auto lookup = [&](const Place& q) -> int64_t {
        const int tile = q.x < q.sp.ts ? q.x : q.x - q.sp.ts + q.sp.wt;
        const int j = tile * kTile + warp * 16 + (lane & 15);
        if (j >= q.sp.n || (j >= q.sp.sink_end && j < q.sp.lo)) return -1;
        return row_offset(a, q.s, j, q.h);
    };
    auto issue = [&](int64_t off, int st) {
        const uint32_t base = ring + st * M::STAGE;
#pragma unroll
        for (int i = 0; i < 16 / RPI; ++i) {
            const int row = i * RPI + rsub;
            const int64_t o = __shfl_sync(0xffffffffu, off, row);
            const bool take = o >= 0 && ch < chunks;
            const int64_t src = take ? o + ch * 8 : 0;
            const uint32_t dst = base + row * M::ROW + ((ch ^ (row & 7)) << 4);
            cp16(dst, a.k + src, take);
            cp16(dst + M::HALF, a.v + src, take);
        }
    };
    // B fragments of q: head 8 nt + g, dimensions 16 kk + 2t, + 8
    uint32_t qf[NT][HD / 16][2];
    auto load_q = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int head = nt * 8 + g;
            const uint16_t* q = p.q + cs.s * p.q_stride + (cs.h * G + head) * a.hd;
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int d = 16 * kk + 8 * b + 2 * t;
                    qf[nt][kk][b] = head < G && d < a.hd ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
                }
        }
    };
    int64_t off = lookup(ld);
    load_q();
    int loaded = 0;  // tiles issued
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
        if (loaded < count) {
            issue(off, i);
            if (++loaded < count) advance(a, p.window, p.n_sink, ld), off = lookup(ld);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // ---- the loop
    float acc[NT][HD / 16][4], m[NT][2], l[NT][2];
    bool fresh = true;
    int x_first = 0;
    for (int u = 0; u < count; ++u) {
        if (fresh) {
            fresh = false;
            x_first = cs.x;
            if (u) load_q();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int i = 0; i < HD / 16; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[nt][i][e] = 0.0f;
                m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.0f;
            }
        }
        if (loaded < count) {
            issue(off, (u + kStages - 1) % kStages);
            if (++loaded < count) advance(a, p.window, p.n_sink, ld), off = lookup(ld);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        __syncwarp();
        const uint32_t kb = ring + (u % kStages) * M::STAGE, vb = kb + M::HALF;
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[nt][e] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk) {
            uint32_t ak[4];
            const int row = lane & 15, c = 2 * kk + (lane >> 4);
            ldsm4(kb + row * M::ROW + ((c ^ (row & 7)) << 4), ak);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816<DT>(s[nt], ak, qf[nt][kk][0], qf[nt][kk][1]);
        }
        const int tile = cs.x < cs.sp.ts ? cs.x : cs.x - cs.sp.ts + cs.sp.wt;
        const int j0 = tile * kTile + warp * 16 + g;
        uint32_t pb[NT][2], pr[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int j = j0 + (e >> 1) * 8;
                const bool vis = j < cs.sp.n && (j < cs.sp.sink_end || j >= cs.sp.lo);
                x[e] = vis ? s[nt][e] * p.scale_log2 : -INFINITY;
            }
            if (p.scores && nt * 8 + 2 * t < p.score_heads) {
                // [j][head of the group]: a warp's store is one run
                float* sc = p.scores + (((int64_t)cs.s * a.nkv + cs.h) * p.score_ld + j0) * p.score_heads + nt * 8 + 2 * t;
                if (j0 < cs.sp.n) *reinterpret_cast<float2*>(sc) = make_float2(x[0], x[1]);
                if (j0 + 8 < cs.sp.n) *reinterpret_cast<float2*>(sc + 8 * p.score_heads) = make_float2(x[2], x[3]);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {  // head 2t + c of the eight
                float mx = fmaxf(x[c], x[c + 2]);
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float mn = fmaxf(m[nt][c], mx), ref = mn == -INFINITY ? 0.0f : mn;
                const float corr = ex2(m[nt][c] - ref);
                m[nt][c] = mn;
                x[c] = ex2(x[c] - ref), x[c + 2] = ex2(x[c + 2] - ref);
                l[nt][c] = l[nt][c] * corr + x[c] + x[c + 2];
                if (corr != 1.0f) {
#pragma unroll
                    for (int i = 0; i < HD / 16; ++i) acc[nt][i][c] *= corr, acc[nt][i][c + 2] *= corr;
                }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float x0 = x[2 * r] * kScaleP, x1 = x[2 * r + 1] * kScaleP;
                const uint32_t hi = X::pack(x0, x1);
                pb[nt][r] = movm(hi);
                pr[nt][r] = movm(X::pack(x0 - X::lo(hi), x1 - X::hi(hi)));
            }
        }
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) {
            uint32_t av[4];
            const int row = (lane & 7) + ((lane >> 4) << 3), c = 2 * i + ((lane >> 3) & 1);
            ldsm4t(vb + row * M::ROW + ((c ^ (row & 7)) << 4), av);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                mma16816<DT>(acc[nt][i], av, pr[nt][0], pr[nt][1]);
                mma16816<DT>(acc[nt][i], av, pb[nt][0], pb[nt][1]);
            }
        }
        __syncwarp();  // the stage may be loaded again

        const bool item_end = cs.x + 1 == cs.sp.nt;
        if (!item_end && u + 1 < count) {
            ++cs.x;
            continue;
        }
        // ---- the end of a run of (s, h): the four warps' parts at a common maximum
        const bool whole = item_end && x_first == 0;
        const uint32_t first_u = u0 + u - cs.x, last_u = first_u + cs.sp.nt - 1;
        const int slot = 2 * blockIdx.x + (x_first == 0 ? 1 : 0);
        float* part = p.part + (int64_t)slot * part_floats(G, HD);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float ls = l[nt][c];
                ls += __shfl_xor_sync(0xffffffffu, ls, 4);
                ls += __shfl_xor_sync(0xffffffffu, ls, 8);
                ls += __shfl_xor_sync(0xffffffffu, ls, 16);
                if (g == 0) s_m[warp][nt * 8 + 2 * t + c] = m[nt][c], s_l[warp][nt * 8 + 2 * t + c] = ls;
            }
        __syncthreads();
        const int hsub = tid >> 4, dsub = (tid & 15) * 4;  // of 8 heads x 64 dimensions
        bool bad = false;  // a sum of this thread's is not finite, with l > 0 that is
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int head = nt * 8 + hsub;
            float mw[kWarps], mx = -INFINITY, ls = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, s_m[w][head]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                mw[w] = ex2(s_m[w][head] - ref), ls += mw[w] * s_l[w][head];
                mw[w] *= whole ? 1.0f / kScaleP : kJoinScale / kScaleP;  // of the sums of p v
            }
#pragma unroll
            for (int half = 0; half < HD / 64; ++half) {
                if (nt || half) __syncthreads();
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        s_mrg[(warp * 8 + 2 * t + (e & 1)) * M::MRG_LD + 16 * i + g + (e >> 1) * 8] =
                            acc[nt][half * 4 + i][e];
                __syncthreads();
                if (head < G) {
                    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int w = 0; w < kWarps; ++w) {
                        const float4 v = *reinterpret_cast<const float4*>(s_mrg + (w * 8 + hsub) * M::MRG_LD + dsub);
                        o[0] += mw[w] * v.x, o[1] += mw[w] * v.y, o[2] += mw[w] * v.z, o[3] += mw[w] * v.w;
                    }
                    const int d = half * 64 + dsub;
                    bad |= needs_again(o, ls);
                    if (whole) {
                        if (d < a.hd) {
                            uint16_t* dst = p.out + ((int64_t)cs.s * nq + cs.h * G + head) * a.hd + d;
                            *reinterpret_cast<uint2*>(dst) =
                                make_uint2(X::pack(o[0] / ls, o[1] / ls), X::pack(o[2] / ls, o[3] / ls));
                        }
                    } else {
                        *reinterpret_cast<float4*>(part + head * HD + d) = make_float4(o[0], o[1], o[2], o[3]);
                    }
                }
            }
            if (head < G && (tid & 15) == 0) {
                s_run[head] = make_float2(ref, ls);
                if (whole) {
                    if (p.ml) p.ml[(int64_t)cs.s * nq + cs.h * G + head] = make_float2(ref, ls);
                } else {
                    reinterpret_cast<float2*>(part + G * HD)[head] = make_float2(mx, ls * kJoinScale);
                }
            }
        }
        if (__syncthreads_or(bad)) {
            run_again<DT, HD>(p, cs.s, cs.h, x_first, cs.x, whole ? nullptr : part, s_run);
            __syncthreads();
        }
        if (!whole) {
            // ---- the last CTA of the item joins its parts, in their order
            const int c0 = (int)owner_of(first_u), c1 = (int)owner_of(last_u);
            const int parts = c1 - c0 + 1;
            if (tid == 0) {
                __threadfence();
                s_last = atomicInc(p.count + c0, parts - 1) == (unsigned)(parts - 1);
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                constexpr int V4 = HD / 4;                                  // float4 per head
                constexpr int PER = (NT * 8 * V4 + kThreads - 1) / kThreads;  // of each thread
                constexpr int B = 8 / NT;                                   // parts in flight
                const int pf = part_floats(G, HD);
                float o[PER][4], M[PER], L[PER];
#pragma unroll
                for (int r = 0; r < PER; ++r) {
                    M[r] = -INFINITY, L[r] = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[r][e] = 0.0f;
                }
                for (int p0 = 0; p0 < parts; p0 += B) {
                    float4 x[PER][B];
                    float2 ml[PER][B];
#pragma unroll
                    for (int k = 0; k < B; ++k) {
                        const int i = p0 + k;
                        const float* base = p.part + (int64_t)(2 * (c0 + i) + (i == 0 ? 1 : 0)) * pf;
#pragma unroll
                        for (int r = 0; r < PER; ++r) {
                            const int v = r * kThreads + tid, head = v / V4;
                            ml[r][k] = make_float2(-INFINITY, 0.0f), x[r][k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            if (i < parts && head < G) {
                                ml[r][k] = __ldcg(reinterpret_cast<const float2*>(base + G * HD) + head);
                                x[r][k] = __ldcg(reinterpret_cast<const float4*>(base) + v);
                            }
                        }
                    }
#pragma unroll
                    for (int r = 0; r < PER; ++r) {
                        float mx = M[r];
#pragma unroll
                        for (int k = 0; k < B; ++k) mx = fmaxf(mx, ml[r][k].x);
                        const float ref = mx == -INFINITY ? 0.0f : mx, old = ex2(M[r] - ref);
                        M[r] = mx, L[r] *= old;
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[r][e] *= old;
#pragma unroll
                        for (int k = 0; k < B; ++k) {
                            const float f = ex2(ml[r][k].x - ref);
                            L[r] += f * ml[r][k].y;
                            o[r][0] += f * x[r][k].x, o[r][1] += f * x[r][k].y;
                            o[r][2] += f * x[r][k].z, o[r][3] += f * x[r][k].w;
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < PER; ++r) {
                    const int v = r * kThreads + tid, head = v / V4, d = (v - head * V4) * 4;
                    if (head < G && d < a.hd) {
                        uint16_t* dst = p.out + ((int64_t)cs.s * nq + cs.h * G + head) * a.hd + d;
                        *reinterpret_cast<uint2*>(dst) = make_uint2(X::pack(o[r][0] / L[r], o[r][1] / L[r]),
                                                                    X::pack(o[r][2] / L[r], o[r][3] / L[r]));
                        if (p.ml && d == 0)
                            p.ml[(int64_t)cs.s * nq + cs.h * G + head] = make_float2(M[r] == -INFINITY ? 0.0f : M[r], L[r] / kJoinScale);
                    }
                }
            }
        }
        __syncthreads();  // s_m, s_l and s_mrg are written again by the next run
        fresh = true;
        if (u + 1 < count) advance(a, p.window, p.n_sink, cs);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// weights[s][h][j] += sum over the group of 2^(x_j - M) / L, from the decode's scores:
// one position per thread, its scores side by side.
__global__ void __launch_bounds__(256) k_paged_add_weights(DecodeArgs p) {
    pdl_begin();
    __shared__ float2 s_ml[kPagedMaxGroup];
    const PagedArgs& a = p.c;
    const int h = blockIdx.y, s = blockIdx.z, nq = a.nkv * a.group;
    const Span sp = span_of(seq_len(a, s), p.window, p.n_sink);
    if ((int)threadIdx.x < kPagedMaxGroup) {
        float2 ml = make_float2(0.0f, 0.0f);
        if ((int)threadIdx.x < a.group) ml = p.ml[(int64_t)s * nq + h * a.group + threadIdx.x], ml.y = 1.0f / ml.y;
        s_ml[threadIdx.x] = ml;
    }
    __syncthreads();
    float* w = p.weights + ((int64_t)s * a.nkv + h) * p.w_stride;
    const float* sc = p.scores + ((int64_t)s * a.nkv + h) * p.score_ld * p.score_heads;
    for (int j = blockIdx.x * blockDim.x + threadIdx.x; j < sp.n; j += gridDim.x * blockDim.x) {
        if (j >= sp.sink_end && j < sp.lo) continue;
        float sum = 0.0f;
        const float old = w[j];
#pragma unroll
        for (int g = 0; g < kPagedMaxGroup; g += 2)
            if (g < p.score_heads) {
                const float2 x = *reinterpret_cast<const float2*>(sc + (int64_t)j * p.score_heads + g);
                sum += ex2(x.x - s_ml[g].x) * s_ml[g].y;
                if (g + 1 < a.group) sum += ex2(x.y - s_ml[g + 1].x) * s_ml[g + 1].y;
            }
        w[j] = old + sum;
    }
}

template <int DT, int HD, int NT>
cudaError_t launch_t(const DecodeArgs& p, int num_sms, cudaStream_t st) {
    constexpr int smem = DecodeSmem<HD>::BYTES;
    auto kern = k_paged_decode<DT, HD, NT>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    e = launch_pdl(kern, dim3(kPagedCtas * num_sms), dim3(kThreads), smem, st, p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

size_t paged_decode_part_floats(int group, int num_sms) {
    return (size_t)2 * kPagedCtas * num_sms * part_floats(group, 128);
}

cudaError_t launch_paged_decode(const DecodeArgs& p, int dtype, int num_sms, cudaStream_t st) {
    if (p.c.n_seqs <= 0) return cudaSuccess;
    if (p.c.hd > 128 || p.c.hd % 8 || p.c.group > kPagedMaxGroup) return cudaErrorInvalidValue;
    if ((int64_t)p.c.n_seqs * p.c.nkv * (p.c.cap / kTile + 2) > 0x7fffffff) return cudaErrorInvalidValue;  // tiles are counted in 32 bits
    const int sel = (dtype ? 4 : 0) + (p.c.hd > 64 ? 2 : 0) + (p.c.group > 8 ? 1 : 0);
    cudaError_t e = cudaErrorInvalidValue;
    switch (sel) {
        case 0: e = launch_t<0, 64, 1>(p, num_sms, st); break;
        case 1: e = launch_t<0, 64, 2>(p, num_sms, st); break;
        case 2: e = launch_t<0, 128, 1>(p, num_sms, st); break;
        case 3: e = launch_t<0, 128, 2>(p, num_sms, st); break;
        case 4: e = launch_t<1, 64, 1>(p, num_sms, st); break;
        case 5: e = launch_t<1, 64, 2>(p, num_sms, st); break;
        case 6: e = launch_t<1, 128, 1>(p, num_sms, st); break;
        case 7: e = launch_t<1, 128, 2>(p, num_sms, st); break;
    }
    if (e != cudaSuccess || !p.weights) return e;
    const int chunks = (p.c.cap + 255) / 256;
    e = launch_pdl(k_paged_add_weights, dim3(chunks < 64 ? chunks : 64, p.c.nkv, p.c.n_seqs), dim3(256), 0, st, p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace obs
