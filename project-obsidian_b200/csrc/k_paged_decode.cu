// k_paged_decode.cu -- attention of one new token per sequence over its pages,
// split over the length and joined, in one launch.
//
//   out[s][h] = sum_j p_j v_j,  p = softmax over the visible j of scale * q[s][h] . k_j
//
// What bounds it: every visible row of K and V is read once from memory for the
// group of query heads that share it, 4 * head_dim * 2 bytes against 4 * head_dim *
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
// rounding left: the tensor cores multiply 16-bit values, one rounding of p would
// cost a short sequence (few p to average over) as much as the output's own, and
// the second set of products is hidden behind the loads.
#include "paged.cuh"

namespace obs {
namespace {

constexpr int kTile = 64;                       // positions per tile: 16 per warp
constexpr int kWarps = 4, kThreads = 32 * kWarps;
constexpr int kStages = 3;                      // per warp
constexpr int kMaxParts = 128;                  // parts whose factors are held at once

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
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
// 16 bytes to shared memory, or zeros
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
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

template <int HD>
struct DecodeSmem {
    static constexpr int ROW = HD * 2, HALF = 16 * ROW;      // a stage: 16 K rows, 16 V rows
    static constexpr int STAGE = 2 * HALF;
    static constexpr int RING = kWarps * kStages * STAGE;
    static constexpr int MRG_LD = 64 + 4;                    // a head's row in the joining buffer
    static constexpr int MRG = kWarps * 8 * MRG_LD * 4;      // one half of the dimensions of 8 heads
    static constexpr int W = kMaxParts * kPagedMaxGroup * 4; // factors of the parts
    static constexpr int BYTES = RING + (MRG > W ? MRG : W);
};

template <int DT, int HD, int NT>
__global__ void __launch_bounds__(kThreads, 2) k_paged_decode(DecodeArgs p) {
    pdl_begin();
    using X = Elem<DT>;
    using M = DecodeSmem<HD>;
    extern __shared__ __align__(1024) uint8_t smem[];
    float* s_mrg = reinterpret_cast<float*>(smem + M::RING);
    __shared__ float s_m[kWarps][16], s_l[kWarps][16];
    __shared__ float s_M[16], s_L[16];
    __shared__ long long s_scan[kWarps];
    __shared__ long long s_first;
    __shared__ int s_seq;
    __shared__ int s_last;
    const PagedArgs& a = p.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int nq = a.nkv * a.group, G = a.group;

    // ---- this CTA's run of the line
    const int per = (a.n_seqs + kThreads - 1) / kThreads;
    const int sb = min(a.n_seqs, tid * per), se = min(a.n_seqs, sb + per);
    long long mine = 0;
    for (int s = sb; s < se; ++s) mine += span_of(seq_len(a, s), p.window, p.n_sink).nt;
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    long long total = 0, before = incl - mine;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) before += s_scan[w];
        total += s_scan[w];
    }
    const long long N = total * a.nkv;
    const long long grid = N < (long long)gridDim.x ? N : (long long)gridDim.x;
    // a sequence without positions gives zeros
    for (int s = blockIdx.x; s < a.n_seqs; s += gridDim.x)
        if (seq_len(a, s) == 0)
            for (int i = tid; i < nq * a.hd; i += kThreads) p.out[(int64_t)s * nq * a.hd + i] = 0;
    if ((long long)blockIdx.x >= grid) return;
    const long long u0 = N * blockIdx.x / grid, u1 = N * (blockIdx.x + 1) / grid;
    {
        long long b = before * a.nkv;
        for (int s = sb; s < se; ++s) {
            const long long c = (long long)span_of(seq_len(a, s), p.window, p.n_sink).nt * a.nkv;
            if (u0 >= b && u0 < b + c) s_seq = s, s_first = b;
            b += c;
        }
    }
    __syncthreads();
    Place ld;
    ld.s = s_seq;
    ld.sp = span_of(seq_len(a, ld.s), p.window, p.n_sink);
    {
        const long long r = u0 - s_first;
        ld.h = (int)(r / ld.sp.nt);
        ld.x = (int)(r - (long long)ld.h * ld.sp.nt);
    }
    Place cs = ld;  // the consumer's place; ld runs ahead
    const int count = (int)(u1 - u0);

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
    int64_t off = lookup(ld);
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
    uint32_t qf[NT][HD / 16][2];
    float acc[NT][HD / 16][4], m[NT][2], l[NT][2];
    bool fresh = true;
    int x_first = 0;
    for (int u = 0; u < count; ++u) {
        if (fresh) {
            fresh = false;
            x_first = cs.x;
            // B fragments of q: head 8 nt + g, dimensions 16 kk + 2t, + 8
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
                if (p.scores && vis) {
                    const int head = nt * 8 + 2 * t + (e & 1);
                    if (head < G) p.scores[((int64_t)cs.s * nq + cs.h * G + head) * p.score_ld + j] = x[e];
                }
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
                const uint32_t hi = X::pack(x[2 * r], x[2 * r + 1]);
                pb[nt][r] = movm(hi);
                pr[nt][r] = movm(X::pack(x[2 * r] - X::lo(hi), x[2 * r + 1] - X::hi(hi)));
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
        const long long first_u = u0 + u - cs.x, last_u = first_u + cs.sp.nt - 1;
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
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int head = nt * 8 + hsub;
            float mw[kWarps], mx = -INFINITY, ls = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, s_m[w][head]);
            const float ref = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) mw[w] = ex2(s_m[w][head] - ref), ls += mw[w] * s_l[w][head];
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
                if (whole) {
                    if (p.ml) p.ml[(int64_t)cs.s * nq + cs.h * G + head] = make_float2(ref, ls);
                } else {
                    reinterpret_cast<float2*>(part + G * HD)[head] = make_float2(mx, ls);
                }
            }
        }
        if (!whole) {
            // ---- the last CTA of the item joins its parts, in their order
            const int c0 = (int)(((first_u + 1) * grid - 1) / N), c1 = (int)(((last_u + 1) * grid - 1) / N);
            const int parts = c1 - c0 + 1;
            __threadfence();
            __syncthreads();
            if (tid == 0) s_last = atomicInc(p.count + c0, parts - 1) == (unsigned)(parts - 1);
            __syncthreads();
            if (s_last) {
                __threadfence();
                auto base = [&](int i) { return p.part + (int64_t)(2 * (c0 + i) + (i == 0 ? 1 : 0)) * part_floats(G, HD); };
                for (int head = warp; head < G; head += kWarps) {
                    float mx = -INFINITY, ls = 0.0f;
                    for (int i = lane; i < parts; i += 32)
                        mx = fmaxf(mx, __ldcg(reinterpret_cast<const float2*>(base(i) + G * HD) + head).x);
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                    const float ref = mx == -INFINITY ? 0.0f : mx;
                    for (int i = lane; i < parts; i += 32) {
                        const float2 v = __ldcg(reinterpret_cast<const float2*>(base(i) + G * HD) + head);
                        ls += ex2(v.x - ref) * v.y;
                    }
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) ls += __shfl_xor_sync(0xffffffffu, ls, o);
                    if (lane == 0) {
                        s_M[head] = ref, s_L[head] = ls;
                        if (p.ml) p.ml[(int64_t)cs.s * nq + cs.h * G + head] = make_float2(ref, ls);
                    }
                }
                constexpr int V4 = HD / 4;
                constexpr int PER = (NT * 8 * V4 + kThreads - 1) / kThreads;
                float o[PER][4];
#pragma unroll
                for (int r = 0; r < PER; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[r][e] = 0.0f;
                for (int p0 = 0; p0 < parts; p0 += kMaxParts) {
                    const int np = min(kMaxParts, parts - p0);
                    __syncthreads();
                    for (int i = tid; i < np * G; i += kThreads) {
                        const int pi = i / G, head = i - pi * G;
                        s_mrg[pi * G + head] =
                            ex2(__ldcg(reinterpret_cast<const float2*>(base(p0 + pi) + G * HD) + head).x - s_M[head]);
                    }
                    __syncthreads();
#pragma unroll
                    for (int r = 0; r < PER; ++r) {
                        const int v = r * kThreads + tid, head = v / V4;
                        if (head >= G) continue;
#pragma unroll 8
                        for (int pi = 0; pi < np; ++pi) {
                            const float4 x = __ldcg(reinterpret_cast<const float4*>(base(p0 + pi)) + v);
                            const float f = s_mrg[pi * G + head];
                            o[r][0] += f * x.x, o[r][1] += f * x.y, o[r][2] += f * x.z, o[r][3] += f * x.w;
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < PER; ++r) {
                    const int v = r * kThreads + tid, head = v / V4, d = (v - head * V4) * 4;
                    if (head < G && d < a.hd) {
                        const float ls = s_L[head];
                        uint16_t* dst = p.out + ((int64_t)cs.s * nq + cs.h * G + head) * a.hd + d;
                        *reinterpret_cast<uint2*>(dst) =
                            make_uint2(X::pack(o[r][0] / ls, o[r][1] / ls), X::pack(o[r][2] / ls, o[r][3] / ls));
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

// weights[s][h][j] += sum over the group of 2^(x_j - M) / L, from the decode's scores.
__global__ void __launch_bounds__(256) k_paged_add_weights(DecodeArgs p) {
    pdl_begin();
    const PagedArgs& a = p.c;
    const int h = blockIdx.y, s = blockIdx.z, nq = a.nkv * a.group;
    const Span sp = span_of(seq_len(a, s), p.window, p.n_sink);
    float* w = p.weights + ((int64_t)s * a.nkv + h) * p.w_stride;
    for (int j = blockIdx.x * blockDim.x + threadIdx.x; j < sp.n; j += gridDim.x * blockDim.x) {
        if (j >= sp.sink_end && j < sp.lo) continue;
        float sum = 0.0f;
        for (int g = 0; g < a.group; ++g) {
            const int64_t row = (int64_t)s * nq + h * a.group + g;
            const float2 ml = p.ml[row];
            sum += ex2(p.scores[row * p.score_ld + j] - ml.x) / ml.y;
        }
        w[j] += sum;
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
