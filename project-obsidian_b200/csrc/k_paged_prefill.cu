// k_paged_prefill.cu -- causal attention of prompts (or chunks of them) over their
// pages, with a sliding window and a few first positions that stay visible, on
// tcgen05.
//
//   out[t][h] = sum_j p_j v_j,  p = softmax over the visible j of scale * q[t][h] . k_j
//
// Rows: the query heads of one KV head and the new tokens of one sequence are one
// line of rows, row R = token * group + head of the group, so the heads share the
// tiles of K and V and a block of 256 rows spans only 256 / group tokens: few tiles
// lie across the causal diagonal or the window's edge, and a chunk of a few tokens
// still fills the tensor cores' 128 rows.
//
// One CTA takes one block of 256 rows, two row tiles of 128 (A and B), against the tiles
// of 64 positions that any of its rows sees (sinks, then the window):
//   S = Q . K^T     128 x 64 fp32 in TMEM; Q and K in shared memory, K-major
//   P = 2^(S scale log2 e - m)   in registers, one row per thread, written back over
//                   S as 16-bit values, the A operand of
//   O += P . V      128 x head_dim fp32 in TMEM; V as it lies (its rows are the
//                   reduction: the N-major form of the B operand)
// O takes half of TMEM, the other half is two buffers of S for each row tile: S of the
// next tile of positions is there when the softmax of one is done.  Tiles of 128
// positions leave no second buffer, and the way from P through two products to the
// next S is waited for (169 us instead of 157 us for one prompt of 4096).
// Sixteen warps:
//   0-3, 4-7   softmax of row tile A, of B: running maximum m and sum l of the thread's
//              row.  O is rescaled only when the maximum has grown by more than 2^8 (p
//              stays below 2^8, in f16 below 2^15), by the same threads, between a
//              tile's S and its P, when no product touches O.  The two row tiles' warps
//              of one scheduler take turns at the exponentials: in step they would share
//              the exponential unit and then leave it idle, and both row tiles' products
//              would queue up behind one another (157 -> 145 us)
//   8, 9       issue the products of A, of B: PV of a tile of positions, then QK of the
//              tile after the next into the columns that this P leaves
//   12-15      loads: rows of K and V by page, 16 bytes per cp.async, into the
//              128-byte-swizzled tiles (rows that no query of the block sees as zeros);
//              a stage's barrier counts the pieces as they land, and the fence that lets
//              the tensor cores see them is the issuing warp's (in the loading warps it
//              would wait for every load in flight)
// Measured for 32 / 4 heads of 128 in bf16: one prompt of 4096 137 us, 1.0 PFLOP/s, 60% of
// the measured bf16 rate (up to 158 us, 52%, with the clock under its power limit); one
// of 8192 with a window of 1024 and 4 sinks 173 to 184 us, 750 to 703 TFLOP/s.  What bounds it: a tile
// takes 1770 cycles a block, of which the exponentials (64 a row at 16 a clock and SM)
// need 1024 and the products 1370 (390 for a 128 x 64 x 128 QK, whose operands come from
// shared memory at its full rate, 294 for a PV); half the products left out saves 5%,
// no loads at all nothing, so the rest is the softmax warps' own latency from S to P.
// A block's start (finding it, Q, the first tiles) and end cost 9000 cycles, a fifth of
// a window of 1024.
//
// p is rounded to 16 bits once.  Against sum p |v| the roundings average out with the
// square root of the number of positions; against the output of values without a common
// mean, which shrinks the same way, they do not: rms error of unit normal inputs against
// 64 bits 2.2e-3 to 2.3e-3 in bf16 from 512 to 16,432 positions where the output's own
// rounding is 1.66e-3 (f16 2.9e-4 and 2.1e-4).  Multiplying what the rounding left too (the
// other half of S's columns holds it) brings the error down to the output's own and
// takes half the products again: a prompt of 4096 194 us instead of 156 us, 8192 with a
// window 224 instead of 184, 48 rows after 16384 36.4 instead of 33.0.  So only blocks do
// it of which a row sees fewer than kFewKeys positions, where one p can be most of the
// sum and its rounding of the order of sum p |v| itself: the first tiles of a prompt,
// which are few (9 prompts of 1 to 700: 30.5 us, 28.7 us without; 4096: no difference).
//
// f16 holds nothing below 2^-25, and a first position that many scores fall 2^25 behind
// is common: there p is 2^7 times as large (2^15 at most, with what the maximum may have
// grown by), and so are l and O.
//
// A NaN or infinity in V meets p = 0 of rows that do not see it, and 0 * NaN is NaN:
// a row whose sums are not finite has those computed again from its visible positions
// alone (attend_again), unless l says that its own scores are the reason (NaN or +inf
// among them, or all -inf: the whole row is NaN).  When nothing is wrong this costs a
// comparison.
//
// Few rows, long axis: where there are fewer blocks than SMs the tiles of a block
// are split over several CTAs, whose (m, l, O) k_paged_join puts together in order.
// Every wait is bounded as in k_gemm.cu.
#include "paged.cuh"

namespace obs {
namespace {

constexpr int kRows = 256, kM = 128, kKeys = 64;
constexpr int kFewKeys = 512;
constexpr int kThreads = 512;
constexpr int kWarpMma = 8, kWarpLd = 12, kLdWarps = 4;
constexpr float kRescale = 8.0f;  // log2 of the growth of the maximum that O tolerates

template <int HD>
struct Pf {
    static constexpr int NH = HD / 64;                // 64-element halves of a row
    static constexpr int QHALF = kM * 128, QTILE = NH * QHALF;    // rows x 128 bytes, swizzled
    static constexpr int HALF = kKeys * 128, TILE = NH * HALF;
    static constexpr int STAGE = 2 * TILE;            // K of tiles 0 and 1, then V of tile j with K of tile j + 2
    static constexpr int NST = HD == 128 ? 4 : 8;
    static constexpr int RING = 2 * QTILE;
    static constexpr int BAR = RING + NST * STAGE;
    static constexpr int NBAR = 2 * NST + 1 + 2 * 7 + 1 + 8;
    static constexpr int SMEM = BAR + NBAR * 8 + 1024;
    static constexpr int O = 256;                     // TMEM: S of tile x, buffer b at 128 x + 64 b; O at 256 + 128 x
};

// (obs_check_device names the codes' kernel)
enum Wait : int { kWtEmpty = 31, kWtFull, kWtQ, kWtS, kWtP, kWtPv, kWtO, kWtTurn };

// mbar_wait without the suspend hint (waits here are shorter than waking up takes)
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile int* abort, int code,
                                         uint64_t limit_ns) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_ns();
    for (;;) {
#pragma unroll 1
        for (int i = 0; i < 64; ++i)
            if (mbar_try_wait(bar, parity)) return true;
        if (*abort) return false;
        if (global_ns() - t0 > limit_ns) {
            *abort = code;
            return false;
        }
    }
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// two at once: (a0, a1) * s + c
__device__ __forceinline__ void fma2(float& a0, float& a1, float s, float c) {
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\tmov.b64 c, {%3, %3};\n\t"
        "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "+f"(a0), "+f"(a1)
        : "f"(s), "f"(c));
}
// two at once: a * b + c
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ void add2(float& s0, float& s1, float a0, float a1) {
    asm("{\n\t.reg .b64 s, a;\n\tmov.b64 s, {%0, %1};\n\tmov.b64 a, {%2, %3};\n\tadd.rn.f32x2 s, s, a;\n\t"
        "mov.b64 {%0, %1}, s;\n\t}"
        : "+f"(s0), "+f"(s1)
        : "f"(a0), "f"(a1));
}
// 32 lanes x 32 consecutive fp32 columns (no wait)
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Instruction descriptor, kind::f16: fp32 sums, both operands of one 16-bit type;
// bnk: B is N-major (its rows are the reduction).
template <int DT>
__device__ __forceinline__ uint32_t idesc16(int M, int N, bool bnk) {
    const uint32_t f = DT == 0 ? 1u : 0u;  // bf16 : f16
    return (1u << 4) | (f << 7) | (f << 10) | (bnk ? 1u << 16 : 0u) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// N-major operand, 128-byte swizzle: 64 elements of N side by side in a row, 8 rows
// of the reduction per 1 KB; `next` bytes to the following 64 elements of N.
__device__ __forceinline__ uint64_t sw128_desc_n(uint32_t saddr, uint32_t next) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
    d |= (uint64_t)(next >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// The tiles that a block of rows at positions i_lo .. i_hi sees.
struct Tiles {
    int ts, wt, nt;        // sink tiles, the window's first tile, tiles in all
    int lo, hi, sink_end;  // positions some row sees: j < sink_end or lo <= j < hi
};
__device__ __forceinline__ Tiles tiles_of(int i_lo, int i_hi, int window, int n_sink) {
    Tiles t;
    t.hi = max(i_hi + 1, 0);
    t.lo = min(window_lo(max(i_lo, 0), window), t.hi);
    t.sink_end = min(n_sink, t.lo);
    t.ts = (t.sink_end + kKeys - 1) / kKeys;
    t.wt = max(t.ts, t.lo / kKeys);
    t.nt = t.ts + max(0, (t.hi + kKeys - 1) / kKeys - t.wt);
    return t;
}
// positions the query at i sees
__device__ __forceinline__ int seen(int i, int window, int n_sink) {
    const int lo = window_lo(i, window);
    return i + 1 - lo + min(n_sink, lo);
}

// the n lowest bits set (none for n <= 0, all from 32)
__device__ __forceinline__ uint32_t low_bits(int n) {
    return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
}

// The row of q (and out) that line row R of (sequence, KV head) stands for.  R / group
// as in page_of: R < 2^20 * 16 <= 2^32 / group.
__device__ __forceinline__ int row_of(const PagedArgs& a, uint32_t magic, int q0, int h, int R, int* token) {
    const int t = magic ? (int)__umulhi((uint32_t)R, magic) : R, g = R - t * a.group;
    *token = q0 + t;
    return h * a.group + g;
}

// A block's rows that are computed again: 16 w .. 16 w + 15 by warp w, against the CTA's tiles.
struct Again {
    int any, s, q0, base, R0, x0, nt, ts, wt;
    uint32_t rows[kRows / 32];  // which
};
// Each warp's rows: ref and l, p = 2^(x - ref) / l, at its staging place (stg).
template <int DT, int HD>
__device__ __forceinline__ void rows_again(const PrefillArgs& p, const Again& b, const uint8_t* smem) {
    const PagedArgs& a = p.c;
    const int lane = threadIdx.x & 31, r0 = (threadIdx.x >> 5) * 16, nq = a.nkv * a.group, h = blockIdx.x % a.nkv;
    const uint32_t which = b.rows[r0 / 32] >> (r0 & 16) & 0xFFFFu;
    if (!which) return;
    const float2* ref_l = reinterpret_cast<const float2*>(smem + r0 / kM * Pf<HD>::QTILE + (r0 / 32 & 3) * 4096) + (r0 & 16);
    const bool split = p.splits > 1;
    AgainRows rows;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int r = (lane >> 2) + 8 * k;
        int t;
        const int head = row_of(a, p.group_magic, b.q0, h, b.R0 + r0 + r, &t);
        const bool in = which >> r & 1u;
        const int64_t row = (int64_t)t * nq + head;
        rows.q[k] = in ? p.q + t * p.q_stride + head * a.hd : nullptr;
        rows.out[k] = split ? static_cast<void*>(p.part_acc + ((int64_t)blockIdx.y * p.T * nq + row) * HD)
                            : static_cast<void*>(p.out + row * a.hd);
        rows.i[k] = b.base + (t - b.q0), rows.lo[k] = window_lo(rows.i[k], p.window);
        rows.ref[k] = in ? ref_l[r].x : 0.0f, rows.l[k] = in ? ref_l[r].y : 1.0f;
    }
#pragma unroll 1
    for (int v = 0; v < HD / 64; ++v)
        attend_again<DT>(a, b.s, h, rows, split, b.x0, b.nt, b.ts, b.wt, p.n_sink, p.scale_log2, v);
}

template <int DT, int HD>
__global__ void __launch_bounds__(kThreads, 1) k_paged_prefill(const __grid_constant__ PrefillArgs p) {
    pdl_begin();
    using X = Elem<DT>;
    using C = Pf<HD>;
    constexpr float kShift = DT == 0 ? 0.0f : 7.0f;  // p is taken against m - kShift
    extern __shared__ uint8_t smem_raw[];
    __shared__ int s_scan[kThreads / 32];
    __shared__ Again s_again;
    __shared__ int s_blk[5];  // sequence, block of it, its rows' range, its length
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t sbase = smem_u32(smem), bars = sbase + C::BAR;
    auto full = [&](int s) { return bars + 8 * s; };
    auto empty = [&](int s) { return bars + 8 * (C::NST + s); };
    const uint32_t qfull = bars + 8 * (2 * C::NST);
    auto sfull = [&](int x, int b) { return qfull + 8 + 8 * (2 * x + b); };
    auto pfull = [&](int x, int b) { return qfull + 40 + 8 * (2 * x + b); };
    auto pvdone = [&](int x, int b) { return qfull + 72 + 8 * (2 * x + b); };
    auto ofull = [&](int x) { return qfull + 104 + 8 * x; };
    const uint32_t mma_done = qfull + 120;
    auto turn = [&](int x, int w) { return qfull + 128 + 8 * (4 * x + w); };
    const PagedArgs& a = p.c;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    volatile int* abort = &s_abort;

    if (warp == kWarpMma) {  // (under the loads of the search)
        tmem_alloc(smem_u32(&s_tmem), 512);
        tmem_relinquish();
    }
    // ---- which block of rows: blocks of all the sequences in one line, the last
    // (the longest of their sequence) first; the KV heads of a block side by side
    const int h = blockIdx.x % a.nkv, bi = blockIdx.x / a.nkv, z = blockIdx.y;
    int s = -1, blk = 0, q0 = 0, q1 = 0, len = 0;
    if (a.n_seqs <= 32) {
        // every warp for itself, a sequence per lane
        const bool in = lane < a.n_seqs;
        const int lq0 = in ? p.q_start[lane] : 0, lq1 = in ? p.q_start[lane + 1] : 0, ll = in ? seq_len(a, lane) : 0;
        const bool ok = lq0 >= 0 && lq1 >= lq0 && lq1 <= p.T && (lane > 0 || lq0 == 0) &&
                        (lane != a.n_seqs - 1 || lq1 == p.T);
        if (!ok && tid == lane) atomicExch(a.err, kDevBadPos);
        const int mine = ok ? ((lq1 - lq0) * a.group + kRows - 1) / kRows : 0;
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        const int want = __shfl_sync(0xffffffffu, incl, 31) - 1 - bi;
        const uint32_t who = __ballot_sync(0xffffffffu, want >= incl - mine && want < incl);
        if (who) {
            s = __ffs(who) - 1;
            blk = want - __shfl_sync(0xffffffffu, incl - mine, s);
            q0 = __shfl_sync(0xffffffffu, lq0, s), q1 = __shfl_sync(0xffffffffu, lq1, s);
            len = __shfl_sync(0xffffffffu, ll, s);
        }
    } else {
        const int per = (a.n_seqs + kThreads - 1) / kThreads;
        const int sb = min(a.n_seqs, tid * per), se = min(a.n_seqs, sb + per);
        int mine = 0;
        bool bad = tid == 0 && (p.q_start[0] != 0 || p.q_start[a.n_seqs] != p.T);
        for (int i = sb; i < se; ++i) {
            const int b0 = p.q_start[i], b1 = p.q_start[i + 1];
            if (b0 < 0 || b1 < b0 || b1 > p.T) bad = true;
            else mine += ((b1 - b0) * a.group + kRows - 1) / kRows;
        }
        if (bad) atomicExch(a.err, kDevBadPos);
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) s_scan[warp] = incl;
        if (tid == 0) s_blk[0] = -1;
        __syncthreads();
        int before = incl - mine, total = 0;
#pragma unroll
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) before += s_scan[w];
            total += s_scan[w];
        }
        const int want = total - 1 - bi;
        if (want >= before && want < before + mine) {
            int b = before;
            for (int i = sb; i < se; ++i) {
                const int b0 = p.q_start[i], b1 = p.q_start[i + 1];
                if (b0 < 0 || b1 < b0 || b1 > p.T) continue;
                const int c = ((b1 - b0) * a.group + kRows - 1) / kRows;
                if (want < b + c) {
                    s_blk[0] = i, s_blk[1] = want - b, s_blk[2] = b0, s_blk[3] = b1, s_blk[4] = seq_len(a, i);
                    break;
                }
                b += c;
            }
        }
        __syncthreads();
        s = s_blk[0], blk = s_blk[1], q0 = s_blk[2], q1 = s_blk[3], len = s_blk[4];
    }
    if (s < 0) {
        __syncthreads();
        if (warp == kWarpMma) tmem_dealloc(s_tmem, 512);
        return;
    }
    const int R0 = blk * kRows, rows = min(kRows, (q1 - q0) * a.group - R0);
    const int base = len - (q1 - q0);  // position of the sequence's first new token
    int t_lo, t_hi;
    row_of(a, p.group_magic, base, h, R0, &t_lo), row_of(a, p.group_magic, base, h, R0 + rows - 1, &t_hi);
    const int i_lo = t_lo, i_hi = t_hi;
    const bool hasB = rows > kM;
    const Tiles tl = tiles_of(i_lo, i_hi, p.window, p.n_sink);
    const bool split = p.splits > 1;
    const int ns = min(p.splits, tl.nt);
    const int nq = a.nkv * a.group;
    if (z >= ns) {  // nothing (or nothing more) to see
        for (int r = tid; r < rows; r += kThreads) {
            int t;
            const int head = row_of(a, p.group_magic, q0, h, R0 + r, &t);
            if (split) p.part_ml[((int64_t)z * p.T + t) * nq + head] = make_float2(-INFINITY, 0.0f);
            else
                for (int d = 0; d < a.hd; d += 8)
                    *reinterpret_cast<uint4*>(p.out + ((int64_t)t * nq + head) * a.hd + d) = make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
        if (warp == kWarpMma) tmem_dealloc(s_tmem, 512);
        return;
    }
    // (nt <= 2^14, splits <= the number of SMs)
    const int x0 = split ? tl.nt * z / ns : 0, nt = (split ? tl.nt * (z + 1) / ns : tl.nt) - x0;
    if (warp == kWarpMma + 2 && lane == 0) s_again = {0, s, q0, base, R0, x0, nt, tl.ts, tl.wt, {}};
    auto tile_key = [&](int x) { return (x < tl.ts ? x : x - tl.ts + tl.wt) * kKeys; };
    const bool precise = i_lo < 0 || seen(i_lo, p.window, p.n_sink) < kFewKeys;

    if (warp == kWarpMma + 1) {
        // the barriers in the order of their places; two of a kind for the two row tiles
        const int nx = hasB ? 2 : 1;
        for (int i = lane; i < C::NBAR; i += 32) {
            const int k = i - 2 * C::NST;
            const int count = i < C::NST ? 32 * kLdWarps                   // full
                              : k < 0 ? nx                                 // empty
                              : k == 0 ? 4 * nx                            // Q
                              : k >= 5 && k < 9 ? 4                        // P
                              : k == 15 ? nx                               // the last products
                                        : 1;                               // S, PV done, O, turns
            mbar_init(bars + 8 * i, count);
        }
        if (lane == 0) s_abort = 0;
        fence_mbar_init();
    }
    // ---- the first loads, then everybody's barriers and tensor memory
    constexpr int CH = HD / 8, RPI = 32 / CH;       // 16-byte pieces per row, rows per instruction
    constexpr int NI = kKeys / (kLdWarps * RPI);    // instructions per tile and loading warp
    static_assert(NI * RPI == 16, "a loading warp takes 16 rows of a tile");
    const int ch = lane % CH, rsub = lane / CH, chunks = a.hd / 8;
    int64_t off = -1;
    // lanes 0-15 look up the warp's rows of tile xa, lanes 16-31 those of tile xb
    auto lookup = [&](int xa, int xb) {
        const int x = lane < 16 ? xa : xb, r = lane & 15;
        off = -1;
        if (x < nt) {
            const int j = tile_key(x0 + x) + ((r / RPI) * kLdWarps + warp - kWarpLd) * RPI + r % RPI;
            if (j < tl.sink_end || (j >= tl.lo && j < tl.hi)) off = row_offset(a, s, j, h);
        }
    };
    auto load_stage = [&](int n) {
        const uint32_t dst = sbase + C::RING + (n % C::NST) * C::STAGE + (ch >> 3) * C::HALF;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (u && n + 1 >= nt) break;  // no tile n + 1
            const uint16_t* pool = n && !u ? a.v : a.k;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int r = (i * kLdWarps + warp - kWarpLd) * RPI + rsub;
                const int64_t o = __shfl_sync(0xffffffffu, off, u * 16 + i * RPI + rsub);
                const bool take = o >= 0 && ch < chunks;
                cp16(dst + u * C::TILE + r * 128 + (((ch & 7) ^ (r & 7)) << 4), pool + (take ? o + ch * 8 : 0), take);
            }
        }
    };
    if (warp >= kWarpLd) {
        lookup(0, 1);
        load_stage(0);
    } else if (warp < (hasB ? 8 : 4)) {
        // the warp's 32 rows of Q: piece ch of row r lies in half ch / 8 at (ch % 8) ^ (r % 8);
        // lane l knows where row l of them is
        const int r = warp * 32 + lane;
        int t;
        const int head = row_of(a, p.group_magic, q0, h, R0 + min(r, rows - 1), &t);
        const int64_t at = r < rows ? t * p.q_stride + (int64_t)head * a.hd : -1;
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            const int rr = k * RPI + rsub, rt = (warp & 3) * 32 + rr;
            const int64_t o = __shfl_sync(0xffffffffu, at, rr);
            const bool take = o >= 0 && ch < chunks;
            cp16(sbase + (warp >> 2) * C::QTILE + (ch >> 3) * C::QHALF + rt * 128 + (((ch & 7) ^ (rt & 7)) << 4),
                 p.q + (take ? o + ch * 8 : 0), take);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;

    if (warp >= kWarpLd) {
        // ------------------------------------------------------------- loads
        for (int n = 0; n <= nt; ++n) {
            const int st = n % C::NST;
            if (n) {
                if (!__all_sync(0xffffffffu, wait_bar(empty(st), ((n / C::NST) & 1) ^ 1, abort, kWtEmpty, p.wait_ns))) break;
                load_stage(n);
            }
            // the barrier counts this thread's pieces when they have landed
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full(st)) : "memory");
            lookup(n, n + 2);  // of the next stage: V of tile n, K of tile n + 2
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp >= kWarpMma) {
        // ---------------------------------------------------------- products
        const int x = warp - kWarpMma;
        if (x < (hasB ? 2 : 1)) {
            const uint32_t id_qk = idesc16<DT>(kM, kKeys, false), id_pv = idesc16<DT>(kM, HD, true);
            const uint64_t qd = sw128_desc(sbase + x * C::QTILE), kd0 = sw128_desc(sbase + C::RING),
                           vd0 = sw128_desc_n(sbase + C::RING, C::HALF);
            auto wait = [&](uint32_t bar, int par, int code) {
                return __all_sync(0xffffffffu, wait_bar(bar, par & 1, abort, code, p.wait_ns));
            };
            // S of buffer b from the K tile at `at` (in descriptor units from the ring's start)
            auto qk = [&](int b, int at) {
#pragma unroll
                for (int kk = 0; kk < HD / 16; ++kk)
                    tc_mma_f16(tmem + x * 128 + b * 64, qd + (uint64_t)((kk >> 2) * (C::QHALF >> 4) + 2 * (kk & 3)),
                               kd0 + at + (uint64_t)((kk >> 2) * (C::HALF >> 4) + 2 * (kk & 3)), id_qk, kk != 0);
                tc_commit(sfull(x, b));
            };
            bool ok = wait(qfull, 0, kWtQ) && wait(full(0), 0, kWtFull);
            fence_proxy_async_smem();
            tc_fence_after();
            if (ok && elect_one()) {
                qk(0, 0);
                if (nt > 1) qk(1, C::TILE >> 4);
                tc_commit(empty(0));
            }
            __syncwarp();
            for (int j = 0; j < nt && ok; ++j) {
                const int b = j & 1, par = (j >> 1) & 1, st = (j + 1) % C::NST;
                ok = wait(full(st), (j + 1) / C::NST, kWtFull) && wait(pfull(x, b), par, kWtP);
                if (!ok) break;
                fence_proxy_async_smem();
                tc_fence_after();
                const int at = st * (C::STAGE >> 4);
                if (elect_one()) {
                    const uint32_t o = tmem + C::O + x * 128, pp = tmem + x * 128 + b * 64;
#pragma unroll
                    for (int kk = 0; kk < kKeys / 16; ++kk)
                        tc_mma_f16_ts(o, pp + kk * 8, vd0 + at + kk * (2048 >> 4), id_pv, (j | kk) != 0);
                    if (precise) {
#pragma unroll
                        for (int kk = 0; kk < kKeys / 16; ++kk)
                            tc_mma_f16_ts(o, pp + 32 + kk * 8, vd0 + at + kk * (2048 >> 4), id_pv, 1);
                    }
                    tc_commit(pvdone(x, b));
                    if (j + 1 == nt) tc_commit(ofull(x));
                    if (j + 2 >= nt) tc_commit(empty(st));
                }
                __syncwarp();
                if (j + 2 >= nt) continue;
                // S of the tile after the next takes P's columns: the products that read them must be done
                ok = wait(pvdone(x, b), par, kWtPv);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    qk(b, at + (C::TILE >> 4));
                    tc_commit(empty(st));
                }
                __syncwarp();
            }
            // every product has finished before the CTA frees its tensor memory, also when a role gave up
            if (elect_one()) tc_commit(mma_done);
            __syncwarp();
            const uint64_t t0 = global_ns();
            while (!mbar_try_wait(mma_done, 0) && global_ns() - t0 < p.wait_ns) {
            }
        }
    } else if (warp < 4 || hasB) {
        // ----------------------------------------------------------- softmax
        const int x = warp >> 2, r = x * kM + (warp & 3) * 32 + lane;
        const uint32_t tq = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t to = tq + C::O + x * 128;
        const bool valid = r < rows;
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(qfull);
        int t;
        const int head = row_of(a, p.group_magic, q0, h, R0 + min(r, rows - 1), &t);
        const int i = base + (t - q0), lo = window_lo(i, p.window);
        int i_min = i, lo_max = lo;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            i_min = min(i_min, __shfl_xor_sync(0xffffffffu, i_min, o));
            lo_max = max(lo_max, __shfl_xor_sync(0xffffffffu, lo_max, o));
        }
        float m0 = -INFINITY, m = -INFINITY, l = 0.0f;  // running maximum of q . k; the one in use, scaled
        bool ok = true;
        for (int j = 0; j < nt; ++j) {
            const int b = j & 1;
            const uint32_t ts = tq + x * 128 + b * 64;
            if (!__all_sync(0xffffffffu, wait_bar(sfull(x, b), (j >> 1) & 1, abort, kWtS, p.wait_ns))) {
                ok = false;
                break;
            }
            tc_fence_after();
            float v[kKeys];
#pragma unroll
            for (int c = 0; c < kKeys; c += 32) tmem_ld32(ts + c, v + c);
            tc_wait_ld();
            const int k0 = tile_key(x0 + j);
            if (!(k0 + kKeys - 1 <= i_min && (k0 >= lo_max || k0 + kKeys <= p.n_sink))) {
                // bit c of word w: column 32 w + c is visible (below i + 1, and a sink or in the window)
#pragma unroll
                for (int w = 0; w < kKeys / 32; ++w) {
                    const int b = k0 + 32 * w;
                    const uint32_t vis = low_bits(i + 1 - b) & (~low_bits(lo - b) | low_bits(p.n_sink - b));
#pragma unroll
                    for (int c = 0; c < 32; ++c) v[32 * w + c] = (vis >> c) & 1u ? v[32 * w + c] : -INFINITY;
                }
            }
            float mx[4] = {m0, v[0], v[1], v[2]};
#pragma unroll
            for (int c = 3; c + 1 < kKeys; c += 2) mx[(c >> 1) & 3] = max3(mx[(c >> 1) & 3], v[c], v[c + 1]);
            m0 = max3(fmaxf(mx[0], v[kKeys - 1]), mx[1], fmaxf(mx[2], mx[3]));
            const float mn = m0 * p.scale_log2;
            if (__any_sync(0xffffffffu, mn > m + kRescale)) {
                const float corr = mn == -INFINITY ? 1.0f : ex2(m - mn);
                m = mn;
                l *= corr;
                if (j > 0) {
                    // the product of the tile before this one may still be adding to O
                    if (!__all_sync(0xffffffffu, wait_bar(pvdone(x, b ^ 1), ((j - 1) >> 1) & 1, abort, kWtPv, p.wait_ns))) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < HD; c += 16) {
                        float o[16];
                        tmem_ld16(to + c, o);
                        tc_wait_ld();
                        uint32_t w[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(o[e] * corr);
                        tmem_st16(to + c, w);
                    }
                }
            }
            // the two tiles' warps of one scheduler take turns at the exponentials
            if (hasB && !__all_sync(0xffffffffu, wait_bar(turn(x, warp & 3), (j & 1) ^ (x == 0), abort, kWtTurn, p.wait_ns))) {
                ok = false;
                break;
            }
            const float ref = m == -INFINITY ? 0.0f : m - kShift;
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c0 = 0; c0 < kKeys; c0 += 32) {
                uint32_t w[16];
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    float &a0 = v[c0 + c], &a1 = v[c0 + c + 1];
                    fma2(a0, a1, p.scale_log2, -ref);
                    a0 = ex2(a0), a1 = ex2(a1);
                    add2(sum[c & 2], sum[(c & 2) + 1], a0, a1);
                    w[c / 2] = X::pack(a0, a1);
                }
                tmem_st16(ts + c0 / 2, w);
                // (handing over takes as long as the second half)
                if (c0 == 0 && hasB && lane == 0) mbar_arrive(turn(x ^ 1, warp & 3));
                if (precise) {
#pragma unroll
                    for (int c = 0; c < 32; c += 2)
                        w[c / 2] = X::pack(v[c0 + c] - X::lo(w[c / 2]), v[c0 + c + 1] - X::hi(w[c / 2]));
                    tmem_st16(ts + 32 + c0 / 2, w);
                }
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(pfull(x, b));
        }
        // ------------------------------------------------------- the rows out
        ok = ok && __all_sync(0xffffffffu, wait_bar(ofull(x), 0, abort, kWtO, p.wait_ns));
        if (ok) {
            tc_fence_after();
            const int64_t row = (int64_t)t * nq + head;
            float2 fin = make_float2(0.0f, 0.0f);  // NaN once a sum is not finite
            uint8_t* stg = smem + x * C::QTILE + (warp & 3) * 4096;
            if (split && valid) p.part_ml[(int64_t)z * p.T * nq + row] = make_float2(m - kShift, l * kJoinScale);
            const float inv = split ? kJoinScale : i < 0 ? 1.0f : 1.0f / l;
#pragma unroll
            for (int c = 0; c < HD; c += 64) {
                float o[64];
                tmem_ld32(to + c, o);
                tmem_ld32(to + c + 32, o + 32);
                tc_wait_ld();
                if (i < 0) {  // nothing to see
#pragma unroll
                    for (int e = 0; e < 64; ++e) o[e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 64; e += 2)
                    fin = fma2(make_float2(o[e], o[e + 1]), make_float2(0.0f, 0.0f), fin);
                if (split) {
                    float4* dst = reinterpret_cast<float4*>(p.part_acc + ((int64_t)z * p.T * nq + row) * HD + c);
                    if (valid)
#pragma unroll
                        for (int e = 0; e < 16; ++e) dst[e] = make_float4(o[4 * e] * inv, o[4 * e + 1] * inv, o[4 * e + 2] * inv, o[4 * e + 3] * inv);
                } else {
                    // through shared memory (Q's rows of this warp, which no product needs any more), so
                    // that a store writes whole lines: piece e of row lane lies at e ^ (lane % 8)
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        float* y = o + 8 * e;
#pragma unroll
                        for (int d = 0; d < 8; d += 2) fma2(y[d], y[d + 1], inv, 0.0f);
                        *reinterpret_cast<uint4*>(stg + lane * 128 + ((e ^ (lane & 7)) << 4)) =
                            make_uint4(X::pack(y[0], y[1]), X::pack(y[2], y[3]), X::pack(y[4], y[5]), X::pack(y[6], y[7]));
                    }
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int rr = e * 4 + (lane >> 3), pc = lane & 7;
                        const int64_t out_row = __shfl_sync(0xffffffffu, row, rr);
                        if (x * kM + (warp & 3) * 32 + rr < rows && c + pc * 8 < a.hd)
                            *reinterpret_cast<uint4*>(p.out + out_row * a.hd + c + pc * 8) =
                                *reinterpret_cast<const uint4*>(stg + rr * 128 + ((pc ^ (rr & 7)) << 4));
                    }
                }
            }
            const uint32_t again =
                __ballot_sync(0xffffffffu, valid && i >= 0 && !(fin.x + fin.y == 0.0f) && l > 0.0f && l <= 3.4e38f);
            if (again) {
                reinterpret_cast<float2*>(stg)[lane] = make_float2(m - kShift, l);
                if (lane == 0) s_again.rows[warp] = again, s_again.any = 1;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kWarpMma) tmem_dealloc(tmem, 512);
    if (s_again.any) rows_again<DT, HD>(p, s_again, smem);
    if (tid == 0 && s_abort) {
        atomicExch(a.err + 1, s_abort);
        atomicExch(a.err, kDevTimeout);
    }
}

// The splits' parts of each row, in their order: one warp per (token, query head).
template <int DT, int HD>
__global__ void __launch_bounds__(256) k_paged_join(PrefillArgs p) {
    pdl_begin();
    using X = Elem<DT>;
    const PagedArgs& a = p.c;
    const int lane = threadIdx.x & 31, nq = a.nkv * a.group;
    const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= (int64_t)p.T * nq) return;
    const int t = (int)(row / nq), head = (int)(row - (int64_t)t * nq);
    int s, i;
    if (!find_row(a, p.q_start, t, p.T, &s, &i)) return;
    const int64_t step = (int64_t)p.T * nq;
    constexpr int PER = HD / 32;  // consecutive dimensions of a lane
    float M = -INFINITY, o[PER] = {}, l = 0.0f;
    // 32 splits at a time: a lane reads one split's maximum and sum, then all of them the
    // split's row
    for (int z0 = 0; z0 < p.splits; z0 += 32) {
        const float2 ml = z0 + lane < p.splits ? p.part_ml[(z0 + lane) * step + row] : make_float2(-INFINITY, 0.0f);
        float mx = ml.x;
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
        mx = fmaxf(mx, M);
        const float ref = mx == -INFINITY ? 0.0f : mx, old = ex2(M - ref);
        M = mx, l *= old;
#pragma unroll
        for (int e = 0; e < PER; ++e) o[e] *= old;
        // (an unused split, or one that saw only -inf, adds nothing: its row may be anything)
        const bool use = !(ml.x == -INFINITY && ml.y == 0.0f);
        const float f = use ? ex2(ml.x - ref) : 0.0f;
        float add = use ? f * ml.y : 0.0f;
#pragma unroll
        for (int k = 16; k > 0; k >>= 1) add += __shfl_xor_sync(0xffffffffu, add, k);
        l += add;
        const uint32_t used = __ballot_sync(0xffffffffu, use);
        const float* part = p.part_acc + (z0 * step + row) * HD + lane * PER;
#pragma unroll 8
        for (int z = 0; z < min(32, p.splits - z0); ++z) {
            const float fz = __shfl_sync(0xffffffffu, f, z);
            if (!(used >> z & 1u)) continue;
            if constexpr (PER == 4) {
                const float4 x = *reinterpret_cast<const float4*>(part + z * step * HD);
                o[0] += fz * x.x, o[1] += fz * x.y, o[2] += fz * x.z, o[3] += fz * x.w;
            } else {
                const float2 x = *reinterpret_cast<const float2*>(part + z * step * HD);
                o[0] += fz * x.x, o[1] += fz * x.y;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] = i < 0 ? 0.0f : o[e] / l;
    const int d = lane * PER;
    if (d < a.hd) {
        uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + row * a.hd + d);
        if constexpr (PER == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(X::pack(o[0], o[1]), X::pack(o[2], o[3]));
        else *dst = X::pack(o[0], o[1]);
    }
}

template <int DT, int HD>
cudaError_t launch_t(const PrefillArgs& p, int blocks, cudaStream_t st) {
    constexpr int smem = Pf<HD>::SMEM;
    static_assert(smem <= 232448 - 1024, "smem");
    auto kern = k_paged_prefill<DT, HD>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    e = launch_pdl(kern, dim3(blocks, p.splits), dim3(kThreads), smem, st, p);
    if (e == cudaSuccess && p.splits > 1)
        e = launch_pdl(k_paged_join<DT, HD>, dim3((unsigned)(((int64_t)p.T * p.c.nkv * p.c.group + 7) / 8)), dim3(256), 0, st, p);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

// (blocks of a call that splits) * splits <= num_sms, 256 rows each
size_t paged_prefill_part_floats(int num_sms) { return (size_t)num_sms * kRows * (128 + 2); }

cudaError_t launch_paged_prefill(PrefillArgs p, float* part, int dtype, int num_sms, cudaStream_t st) {
    const PagedArgs& a = p.c;
    if (p.T <= 0 || a.n_seqs <= 0) return cudaSuccess;
    if (a.hd > 128 || a.hd % 8 || a.group > kPagedMaxGroup) return cudaErrorInvalidValue;
    // at most this many blocks of rows: every sequence's last one may be ragged
    const int64_t blocks = ((int64_t)p.T * a.group / kRows + (a.n_seqs < p.T ? a.n_seqs : p.T)) * a.nkv;
    if (blocks > 0x7fffffff) return cudaErrorInvalidValue;
    int splits = (int)(num_sms / blocks);
    const int most = (a.cap + 2 * kKeys - 1) / (2 * kKeys);  // two tiles or more each
    if (splits > most) splits = most;
    p.splits = splits < 1 ? 1 : splits;
    p.group_magic = a.group == 1 ? 0u : (uint32_t)((1ull << 32) / (uint32_t)a.group + 1);
    const int64_t rows = (int64_t)p.T * a.nkv * a.group * p.splits;
    p.part_acc = part;
    p.part_ml = reinterpret_cast<float2*>(part + rows * (a.hd > 64 ? 128 : 64));
    const int b = (int)blocks;
    if (dtype) return a.hd > 64 ? launch_t<1, 128>(p, b, st) : launch_t<1, 64>(p, b, st);
    return a.hd > 64 ? launch_t<0, 128>(p, b, st) : launch_t<0, 64>(p, b, st);
}

}  // namespace obs
