// Attention of a few query rows per key head over the paged 4-bit cache (cora_kv4_attend).
//
//   score_t = (scale_t (q . c_t) + low_t sum(q)) * softmax scale
//   out     = sum_t p_t (scale'_t c'_t + low'_t),   p = softmax(score)
//
// so codes enter the matrix instructions as integers and a token's factors are applied once per
// (token, query), to fp32 sums. What bounds it: reading the cache once; instruction issue is
// next (4 bits arrive at 48 codes per clock and SM). Hence:
//  - tokens (then value dimensions) are the 16-row side of m16n8k16, query rows the 8-column
//    side: the query heads that share a key head fill one instruction;
//  - a code becomes an fp16 operand by one AND: nibble 0 of a 16-bit half is the subnormal
//    c 2^-24, nibble 1 is c 2^-20, both exact in the tensor core. The powers of two go into q
//    (a common power of two per block, so fp16 holds every bit of a bf16 or fp16 q that is
//    within 2^-24 of the largest) and into the final scaling of the output;
//  - w = fp16(p scale') is the operand of the second product (11 bits; scaled by a power of two
//    that follows the largest scale' met, so it uses the normal range). What the rounding of w
//    loses would be multiplied by codes of 0..15 although values spread around the middle of
//    their group's range; so the sum is taken as sum w (c' - 7.5) + sum p (low' + 7.5 scale'),
//    sum w by one more product with ones: the loss is then 2^-12 of |value - middle|.
//    Statistics, sums and accumulators are fp32;
//  - each warp streams its own tiles of kTile tokens through a private ring of bulk copies, and
//    keeps its own running maximum and sum; a block's warps join in shared memory;
//  - (sequence, key head, row tile, token tile) units are cut into equal runs, one per block,
//    so ragged batches balance; a job cut over several blocks is joined by the last to arrive.
#pragma once
#include <cuda_fp16.h>

#include "../../include/cora_b200.h"
#include "common.cuh"
#include "kernels_lowbit_append.cuh"
#include "kernels_lowbit_matvec.cuh"

namespace cora {

constexpr int kAtWarps = 8, kAtThreads = kAtWarps * 32, kAtTile = 32, kAtStages = 2;
constexpr int kAtMinRun = 4;       // units of a block, at least
constexpr int kAtMaxSeqs = 1024;   // sequences of one launch (their unit offsets are in smem)
constexpr float kLog2e = 1.4426950408889634f;

struct AttendParams {
    cora_kv4_cache c;
    cora_kv4_attend_args a;
    uint32_t seq0, seqs;      // this launch's sequences
    int64_t q_tokens;         // rows of q
    float *part;              // partial results: [2 * blocks][rows][D] then [2 * blocks][rows][2]
    uint32_t *arrived;        // per block, zero between launches
};

// The shared memory of a block, in order (each part a multiple of 16 bytes).
template <int D, int kNG, int kNT>
struct AttendSmem {
    static constexpr int kRows = 8 * kNT;
    static constexpr uint32_t kCodes = kAtTile * D / 2, kMeta = kAtTile * kNG * 4;
    static constexpr uint32_t kStage = 2 * kCodes + 2 * kMeta;
    static constexpr uint32_t ring = 0;
    static constexpr uint32_t qfrag = ring + kAtWarps * kAtStages * kStage;  // D / 32 * kNT * 512
    static constexpr uint32_t red = qfrag + (D / 32) * kNT * 512;            // [warp][row][64]
    static constexpr uint32_t qsum = red + kAtWarps * kRows * 64 * 4;        // [row][kNG]
    static constexpr uint32_t lim = qsum + kRows * kNG * 4;                  // [row] {lo, hi}
    static constexpr uint32_t stat = lim + kRows * 8;                        // [warp][row] {m, l}
    static constexpr uint32_t om = stat + kAtWarps * kRows * 8;              // [warp][row][kNG]
    static constexpr uint32_t fin = om + kAtWarps * kRows * kNG * 4;         // [row] {m, l}
    static constexpr uint32_t misc = fin + kRows * 8;                        // max |q|, last to arrive
    static constexpr uint32_t bars = misc + 32;
    static constexpr uint32_t base = bars + kAtWarps * kAtStages * 8;        // int64[seqs + 1]
    static constexpr size_t bytes(uint32_t seqs) { return base + 8 * (size_t)(seqs + 1); }
};

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// Largest and sum over the eight lanes of one column pair (lane = 4 g + t, over g).
__device__ __forceinline__ float max_over_g(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float sum_over_g(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 4);
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

// What a sequence asks for, from device memory.
struct SeqWork {
    int q0, n;        // first row of q and number of query tokens
    int len, first;   // cached tokens; first tile-aligned token that any query sees
    int tiles, row_tiles;
};
__device__ __forceinline__ SeqWork seq_work(const AttendParams &p, int b, int rows) {
    SeqWork s;
    const int seq = p.seq0 + b;
    int q0 = p.a.q_start ? __ldg(p.a.q_start + seq) : seq;
    int q1 = p.a.q_start ? __ldg(p.a.q_start + seq + 1) : seq + 1;
    int len = __ldg(p.a.lens + seq);
    const int64_t room = (int64_t)p.a.table_width * p.c.page_size;
    if (q0 < 0 || q1 < q0 || q1 > p.q_tokens || len < 0 || len > room) {
        atomicOr(p.c.status, kDevBadInput);
        q0 = max(0, min(q0, (int)p.q_tokens));
        q1 = max(q0, min(q1, (int)p.q_tokens));
        len = max(0, (int)min((int64_t)len, room));
    }
    s.q0 = q0;
    s.n = q1 - q0;
    s.len = len;
    const int w = (int)p.a.window;
    s.first = w ? max(0, len - s.n - w + 1) / kAtTile * kAtTile : 0;
    if (s.first > len) s.first = len / kAtTile * kAtTile;
    s.tiles = max(1, (len - s.first + kAtTile - 1) / kAtTile);  // an empty one still writes zeros
    s.row_tiles = (s.n * (int)(p.a.q_heads / p.c.kv_heads) + rows - 1) / rows;
    return s;
}

template <typename T, int D, int kNG, int kNT>
__global__ void __launch_bounds__(kAtThreads, kNT * D <= 128 ? 2 : 1) kv4_attend_kernel(const AttendParams p) {
    using S = AttendSmem<D, kNG, kNT>;
    constexpr int kRows = 8 * kNT, kG = D / kNG;
    constexpr int kWords = kG / 32;         // words of one lane and group
    constexpr int kVB = D / 64;             // 64-dimension blocks of the values
    extern __shared__ __align__(128) unsigned char at_smem[];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    unsigned char *ring = at_smem + S::ring + warp * kAtStages * S::kStage;
    uint4 *qfrag = reinterpret_cast<uint4 *>(at_smem + S::qfrag);
    float *red = reinterpret_cast<float *>(at_smem + S::red);
    float *qsum = reinterpret_cast<float *>(at_smem + S::qsum);
    int2 *lim = reinterpret_cast<int2 *>(at_smem + S::lim);
    float2 *stat = reinterpret_cast<float2 *>(at_smem + S::stat);
    float *omw = reinterpret_cast<float *>(at_smem + S::om);
    float2 *fin = reinterpret_cast<float2 *>(at_smem + S::fin);
    volatile int *misc = reinterpret_cast<volatile int *>(at_smem + S::misc);
    uint64_t *bars = reinterpret_cast<uint64_t *>(at_smem + S::bars) + warp * kAtStages;
    int64_t *base = reinterpret_cast<int64_t *>(at_smem + S::base);

    const int H = p.c.kv_heads, heads = p.a.q_heads / H, P = p.c.page_size;
    const Kv4Block blk(P, D, kG);

    if (lane == 0) {
        for (int s = 0; s < kAtStages; ++s) mbar_init(bars + s, 1);
        fence_barrier_init();
    }
    // unit offsets of the sequences: inclusive sums by warp 0, 32 sequences at a time
    if (warp == 0) {
        int64_t run = 0;
        if (lane == 0) base[0] = 0;
        for (int b0 = 0; b0 < (int)p.seqs; b0 += 32) {
            int64_t v = 0;
            if (b0 + lane < (int)p.seqs) {
                const SeqWork s = seq_work(p, b0 + lane, kRows);
                v = (int64_t)s.tiles * s.row_tiles * H;
            }
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int64_t o = __shfl_up_sync(0xffffffffu, v, off);
                if (lane >= off) v += o;
            }
            if (b0 + lane < (int)p.seqs) base[b0 + lane + 1] = run + v;
            run += __shfl_sync(0xffffffffu, v, 31);
        }
    }
    __syncthreads();
    // Equal runs of at least kAtMinRun units: block i holds units [i U / B, (i + 1) U / B).
    const int64_t units = base[p.seqs], blocks = max((int64_t)1, min((int64_t)gridDim.x, units / kAtMinRun));
    if (blockIdx.x >= blocks) return;
    auto cut = [&](int64_t i) { return i * units / blocks; };
    const int64_t u0 = cut(blockIdx.x), u1 = cut(blockIdx.x + 1);
    if (u0 >= u1) return;

    // The sequence that holds unit u (base is ascending; units of one sequence fit 32 bits).
    auto find = [&](int64_t u) {
        int lo = 0, hi = (int)p.seqs - 1;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (base[mid + 1] > u) hi = mid;
            else lo = mid + 1;
        }
        return lo;
    };

    // ---- the warp's stream of tiles: units u0 + warp, + kAtWarps, ... ----
    // Copies of one tile: lane 4 i + k copies section k of the tile's i-th page piece.
    const int per = min(P, kAtTile), shift = 31 - __clz(P);  // tokens of a piece
    const int piece = lane >> 2, kind = lane & 3;
    const uint32_t rowb = kind < 2 ? D / 2 : kNG * 4;
    const uint32_t src_at = (kind & 1 ? (kind < 2 ? blk.codes : blk.metas) : 0) + (kind < 2 ? 0 : 2 * blk.codes);
    const uint32_t dst_at = (kind & 1 ? (kind < 2 ? S::kCodes : S::kMeta) : 0) + (kind < 2 ? 0 : 2 * S::kCodes) +
                            piece * per * rowb;
    int fb = -1, ftile = 0, frt = 0, fhead = 0, fpage = 0;  // the next tile to fetch
    SeqWork fs{};
    const int *ftable = nullptr;
    auto fetch_page = [&]() {  // its page's number, early: the copy needs it one tile later
        const int tok = fs.first + ftile * kAtTile + piece * per;
        fpage = piece * per < kAtTile && tok < fs.len ? __ldg(ftable + (tok >> shift)) : -2;
    };
    auto fetch_seek = [&](int64_t u) {  // warp-uniform
        fb = find(u);
        fs = seq_work(p, fb, kRows);
        ftable = p.a.page_table + (int64_t)(p.seq0 + fb) * p.a.table_stride;
        const uint32_t r = (uint32_t)(u - base[fb]), job = r / (uint32_t)fs.tiles;
        ftile = (int)(r - job * fs.tiles);
        fhead = (int)(job / fs.row_tiles);
        frt = (int)(job - fhead * fs.row_tiles);
        fetch_page();
    };
    auto fetch = [&](int64_t u, int stage) {
        const bool got = fpage != -2, ok = got && fpage >= 0 && (uint32_t)fpage < p.c.num_pages;
        const uint32_t lanes = __ballot_sync(0xffffffffu, ok);
        if (got && !ok) atomicOr(p.c.status, kDevBadInput);
        const uint32_t bytes = per * rowb;
        // sections of a piece are copied by four neighbouring lanes, all or none
        if (lane == 0) mbar_arrive_expect_tx(bars + stage, __popc(lanes) / 4 * per * (D + 8 * kNG));
        __syncwarp();
        if (ok) {
            const int tok = fs.first + ftile * kAtTile + piece * per;
            bulk_g2s(ring + stage * S::kStage + dst_at,
                     p.c.pool + ((uint64_t)fpage * H + fhead) * blk.bytes + src_at + (uint32_t)(tok & (P - 1)) * rowb, bytes,
                     bars + stage);
        }
        // on to the tile after next of this block
        u += kAtWarps;
        if (u >= u1) return;
        if (u >= base[fb + 1]) return fetch_seek(u);
        ftile += kAtWarps;
        while (ftile >= fs.tiles) {
            ftile -= fs.tiles;
            if (++frt == fs.row_tiles) frt = 0, ++fhead;
        }
        fetch_page();
    };

    int64_t ahead = u0 + warp;   // next unit to fetch
    int fstage = 0, pending = 0;  // tiles in flight
    if (ahead < u1) fetch_seek(ahead);
    for (; pending < kAtStages && ahead < u1; ++pending, ahead += kAtWarps) fetch(ahead, pending);
    int stage = 0;
    uint32_t phase = 0;
    int64_t u = u0 + warp;       // next unit to consume

    int b = -1;
    SeqWork sw{};
    bool alive = true;
    for (int64_t seg = u0; seg < u1;) {
        // ---- one job (sequence, key head, row tile), units [seg, seg_end) of it are ours ----
        if (b < 0 || seg >= base[b + 1]) {
            b = find(seg);
            sw = seq_work(p, b, kRows);
        }
        const int64_t job = (seg - base[b]) / sw.tiles;
        const int64_t job_u0 = base[b] + job * sw.tiles, job_u1 = job_u0 + sw.tiles;
        const int64_t seg_end = min(u1, job_u1);
        const int rt = (int)(job % sw.row_tiles), head = (int)(job / sw.row_tiles);
        const int row0 = rt * kRows, nrows = min(kRows, sw.n * heads - row0);

        // queries: rows are (token, head of the group); fp16 under a common power of two
        if (threadIdx.x == 0) misc[0] = 0;
        __syncthreads();
        float qv[(kRows + kAtWarps - 1) / kAtWarps][D / 32];
        float big = 0.0f;
#pragma unroll
        for (int i = 0; i < (kRows + kAtWarps - 1) / kAtWarps; ++i) {
            const int r = warp + i * kAtWarps;
            const int row = row0 + r;
            const bool in = r < nrows;
            const T *src = static_cast<const T *>(p.a.q) + (int64_t)(sw.q0 + (in ? row / heads : 0)) * p.a.q_token +
                           (int64_t)(head * heads + (in ? row % heads : 0)) * p.a.q_head;
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
                qv[i][d] = in ? to_f32(src[d * 32 + lane]) : 0.0f;
                const float m = fabsf(qv[i][d]);
                if (m < 3.4e38f) big = fmaxf(big, m);  // infinities and NaN keep to their rows
            }
            if (lane == 0 && r < kRows) {
                const int pos = sw.len - sw.n + row / heads;
                const int hi = p.a.causal ? max(0, min(sw.len, pos + 1)) : sw.len;
                const int lo = p.a.window ? max(0, pos - (int)p.a.window + 1) : 0;
                lim[r] = in ? make_int2(lo, hi) : make_int2(0, 0);
            }
        }
#pragma unroll
        for (int m = 16; m; m >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, m));
        if (lane == 0) atomicMax(const_cast<int *>(&misc[0]), __float_as_int(big));
        __syncthreads();
        // 2^qe brings the largest |q| into [2^13, 2^14)
        const float qmax = __int_as_float(misc[0]);
        const int qe = qmax > 0.0f ? max(-114, min(126, 13 - ilogbf(qmax))) : 0;
        const float qpow = ldexpf(1.0f, qe);
        const float qf = p.a.scale * kLog2e;
#pragma unroll
        for (int i = 0; i < (kRows + kAtWarps - 1) / kAtWarps; ++i) {
            const int r = warp + i * kAtWarps;
            if (r < kRows) {
                __half *dst = reinterpret_cast<__half *>(qfrag);
#pragma unroll
                for (int d = 0; d < D / 32; ++d) {
                    // dimension -> (word of 8, nibble) -> (group, lane t, word of the lane)
                    const int dim = d * 32 + lane, word = dim / 8, nib = dim % 8;
                    const int gr = dim / kG, wi = word - gr * (kG / 8), tt = wi / kWords, j = wi % kWords;
                    // registers: {0,4} {1,5} {2,6} {3,7}; odd nibbles carry 2^-4
                    const int reg = nib & 3, half = nib >> 2;
                    const int frag = ((r / 8) * (D / 32) + gr * kWords + j) * 32 + (r % 8) * 4 + tt;
                    dst[frag * 8 + reg * 2 + half] = __float2half_rn(qv[i][d] * qpow * (nib & 1 ? 0.0625f : 1.0f));
                }
#pragma unroll
                for (int gr = 0; gr < kNG; ++gr) {
                    float s = 0.0f;
#pragma unroll
                    for (int d = gr * (kG / 32); d < (gr + 1) * (kG / 32); ++d) s += qv[i][d];
#pragma unroll
                    for (int m = 16; m; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
                    if (lane == 0) qsum[r * kNG + gr] = s * qf;
                }
            }
        }
        __syncthreads();
        const float raw = ldexpf(qf, 24 - qe);  // of q . c as the tensor core sums it
        float qs[kNT][2][kNG];
        int2 lm[kNT][2];
        int lo_max = 0, hi_min = sw.len;
        for (int r = 0; r < nrows; ++r) {
            lo_max = max(lo_max, lim[r].x);
            hi_min = min(hi_min, lim[r].y);
        }
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                lm[n][c] = lim[n * 8 + 2 * t + c];
#pragma unroll
                for (int gr = 0; gr < kNG; ++gr) qs[n][c][gr] = qsum[(n * 8 + 2 * t + c) * kNG + gr];
            }

        float acc[kVB][4][kNT][4];
        float mx[kNT][2], ls[kNT][2], om[kNT][2][kNG];
        float ws[kNG][kNT][4];  // sum w (rows of the accumulator are alike)
#pragma unroll
        for (int v = 0; v < kVB; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < kNT; ++n)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[v][i][n][c] = 0.0f;
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                mx[n][c] = -INFINITY;
                ls[n][c] = 0.0f;
#pragma unroll
                for (int gr = 0; gr < kNG; ++gr) om[n][c][gr] = ws[gr][n][c] = ws[gr][n][c + 2] = 0.0f;
            }
        int vexp = 126;  // 2^-vexp bounds the value scales met: operands are p scale' 2^(15 + vexp)
        float vbound = 0.0f, vmul = 0.0f;

        for (; u < seg_end; u += kAtWarps) {
            const int tok0 = sw.first + (int)(u - job_u0) * kAtTile;
            if (pending) {  // (0 only after a wait ran out: nothing more is fetched then)
                alive = __all_sync(0xffffffffu, mbar_wait_bounded(bars + stage, phase, p.c.status)) && alive;
                --pending;
            }
            const unsigned char *st = ring + stage * S::kStage;
            const bool edge = tok0 + kAtTile > hi_min || tok0 < lo_max;
            // ---- scores: two tiles of 16 tokens x 8 kNT rows ----
            float s[2][kNT][4];
            const int tg = g ^ ((g >> 1) & 1);  // the token of operand row g (and + 8): see below
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
                for (int gr = 0; gr < kNG; ++gr) {
                    uint32_t wa[kWords], wb[kWords];
                    const unsigned char *ka = st + (mt * 16 + tg) * (D / 2) + gr * (kG / 2) + t * (kWords * 4);
                    if constexpr (kWords == 4) {
                        *reinterpret_cast<uint4 *>(wa) = *reinterpret_cast<const uint4 *>(ka);
                        *reinterpret_cast<uint4 *>(wb) = *reinterpret_cast<const uint4 *>(ka + 8 * (D / 2));
                    } else {
                        *reinterpret_cast<uint2 *>(wa) = *reinterpret_cast<const uint2 *>(ka);
                        *reinterpret_cast<uint2 *>(wb) = *reinterpret_cast<const uint2 *>(ka + 8 * (D / 2));
                    }
                    float d[kNT][4];
#pragma unroll
                    for (int n = 0; n < kNT; ++n)
#pragma unroll
                        for (int c = 0; c < 4; ++c) d[n][c] = 0.0f;
#pragma unroll
                    for (int j = 0; j < kWords; ++j) {
                        const uint32_t a8 = wa[j] >> 8, b8 = wb[j] >> 8;
#pragma unroll
                        for (int n = 0; n < kNT; ++n) {
                            const uint4 q = qfrag[(n * (D / 32) + gr * kWords + j) * 32 + lane];
                            mma16816<__half>(d[n], wa[j] & 0x000f000fu, wb[j] & 0x000f000fu, wa[j] & 0x00f000f0u,
                                             wb[j] & 0x00f000f0u, q.x, q.y);
                            mma16816<__half>(d[n], a8 & 0x000f000fu, b8 & 0x000f000fu, a8 & 0x00f000f0u,
                                             b8 & 0x00f000f0u, q.z, q.w);
                        }
                    }
                    const __half2 *km = reinterpret_cast<const __half2 *>(st + 2 * S::kCodes);
                    const float2 f0 = __half22float2(km[(mt * 16 + tg) * kNG + gr]);
                    const float2 f1 = __half22float2(km[(mt * 16 + 8 + tg) * kNG + gr]);
                    const float r0 = f0.x * raw, r1 = f1.x * raw;
#pragma unroll
                    for (int n = 0; n < kNT; ++n)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float low = (c < 2 ? f0.y : f1.y) * qs[n][c & 1][gr];
                            const float v = fmaf(c < 2 ? r0 : r1, d[n][c], low);
                            s[mt][n][c] = gr ? s[mt][n][c] + v : v;
                        }
                }
            }
            uint32_t hidden = 0;  // bit (mt * kNT + n) * 4 + c
            if (edge) {
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int n = 0; n < kNT; ++n)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const int tok = tok0 + mt * 16 + tg + (c >> 1) * 8;
                            const int2 l = lm[n][c & 1];
                            if (tok < l.x || tok >= l.y) {
                                s[mt][n][c] = -INFINITY;
                                hidden |= 1u << ((mt * kNT + n) * 4 + c);
                            }
                        }
            }
            // ---- running maximum ----
            float al[kNT][2];
            bool moved = false;
#pragma unroll
            for (int n = 0; n < kNT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float m = fmaxf(fmaxf(s[0][n][c], s[0][n][c + 2]), fmaxf(s[1][n][c], s[1][n][c + 2]));
                    m = fmaxf(mx[n][c], max_over_g(m));
                    const float ref = m == -INFINITY ? 0.0f : m;
                    al[n][c] = ex2(mx[n][c] - ref);
                    moved |= m != mx[n][c];
                    mx[n][c] = m;
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        s[mt][n][c] = ex2(s[mt][n][c] - ref);
                        s[mt][n][c + 2] = ex2(s[mt][n][c + 2] - ref);
                    }
                }
            // ---- value factors; the bound on their scales ----
            const __half2 *vm = reinterpret_cast<const __half2 *>(st + 2 * S::kCodes + S::kMeta);
            float2 vf[2][2][kNG];
            float smax = 0.0f;
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int gr = 0; gr < kNG; ++gr) {
                        const int tok = mt * 16 + tg + r * 8;
                        float2 f = __half22float2(vm[tok * kNG + gr]);
                        if (edge && tok0 + tok >= sw.len) f = make_float2(0.0f, 0.0f);
                        smax = fmaxf(smax, f.x < 65536.0f ? f.x : 0.0f);
                        f.y = fmaf(7.5f, f.x, f.y);
                        vf[mt][r][gr] = f;
                    }
            float shrink = 1.0f;
            if (__any_sync(0xffffffffu, smax > vbound)) {
                smax = max_over_g(smax);
                const int e = -(ilogbf(smax) + 1);  // smax < 2^-e
                shrink = vbound > 0.0f ? ldexpf(1.0f, e - vexp) : 1.0f;
                vexp = e;
                vbound = ldexpf(1.0f, -e);
                vmul = ldexpf(1.0f, 15 + e);
                moved = true;
            }
            if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                for (int n = 0; n < kNT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        ls[n][c] *= al[n][c];
#pragma unroll
                        for (int gr = 0; gr < kNG; ++gr) om[n][c][gr] *= al[n][c];
                        const float f = al[n][c] * shrink;
#pragma unroll
                        for (int gr = 0; gr < kNG; ++gr) ws[gr][n][c] *= f;
#pragma unroll
                        for (int v = 0; v < kVB; ++v)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                acc[v][i][n][c] *= f;
                                acc[v][i][n][c + 2] *= f;
                            }
                    }
            }
            // ---- values: per 16 tokens, p scale' transposed into the 16-deep operand ----
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                uint32_t pb[kNG][kNT][2];
#pragma unroll
                for (int n = 0; n < kNT; ++n) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) ls[n][c & 1] += s[mt][n][c];
#pragma unroll
                    for (int gr = 0; gr < kNG; ++gr) {
                        float x[4];
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float2 f = vf[mt][c >> 1][gr];
                            x[c] = s[mt][n][c] * (f.x * vmul);
                            float y = s[mt][n][c] * f.y;
                            if (edge && (hidden >> ((mt * kNT + n) * 4 + c) & 1)) x[c] = y = 0.0f;
                            om[n][c & 1][gr] += y;
                        }
                        pb[gr][n][0] = transpose8x8(pack_half2(x[0], x[1]));
                        pb[gr][n][1] = transpose8x8(pack_half2(x[2], x[3]));
                        constexpr uint32_t one = 0x3c003c00u;
                        mma16816<__half>(ws[gr][n], one, one, one, one, pb[gr][n][0], pb[gr][n][1]);
                    }
                }
                // Operand row r of a 16-token tile is token r ^ (r >> 1 & 1): the four lanes t of
                // a value load then read rows of both parities, two bank halves instead of one.
                const int r0 = 2 * t, k0 = r0 ^ (t & 1), k1 = (r0 + 1) ^ (t & 1);
                const unsigned char *vc = st + S::kCodes + mt * 16 * (D / 2) + g * 4;
#pragma unroll
                for (int v = 0; v < kVB; ++v) {
                    const uint32_t w0 = *reinterpret_cast<const uint32_t *>(vc + k0 * (D / 2) + v * 32);
                    const uint32_t w1 = *reinterpret_cast<const uint32_t *>(vc + k1 * (D / 2) + v * 32);
                    const uint32_t w2 = *reinterpret_cast<const uint32_t *>(vc + (k0 + 8) * (D / 2) + v * 32);
                    const uint32_t w3 = *reinterpret_cast<const uint32_t *>(vc + (k1 + 8) * (D / 2) + v * 32);
                    uint32_t x[4], y[4];  // by nibble pair: tokens (2t, 2t + 1) and (+ 8)
                    x[0] = __byte_perm(w0, w1, 0x5410), x[2] = __byte_perm(w0, w1, 0x7632);
                    y[0] = __byte_perm(w2, w3, 0x5410), y[2] = __byte_perm(w2, w3, 0x7632);
                    x[1] = x[0] >> 8, x[3] = x[2] >> 8, y[1] = y[0] >> 8, y[3] = y[2] >> 8;
                    const int gr = v * 64 / kG;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int n = 0; n < kNT; ++n)
                            mma16816<__half>(acc[v][i][n], x[i] & 0x000f000fu, x[i] & 0x00f000f0u,
                                             y[i] & 0x000f000fu, y[i] & 0x00f000f0u, pb[gr][n][0], pb[gr][n][1]);
                }
            }
            // ---- the stage is read: refill it ----
            __syncwarp();
            if (ahead < u1 && alive) {
                fetch(ahead, fstage);
                ahead += kAtWarps;
                ++pending;
            }
            if (++fstage == kAtStages) fstage = 0;
            if (++stage == kAtStages) {
                stage = 0;
                phase ^= 1;
            }
        }

        // ---- join the warps ----
        const float opow = ldexpf(1.0f, 9 - vexp);  // 2^24 of the codes, 2^-(15 + vexp) of the operand
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float l = sum_over_g(ls[n][c]);
                const int r = n * 8 + 2 * t + c;
                if (g == 0) stat[warp * kRows + r] = make_float2(mx[n][c], l);
#pragma unroll
                for (int gr = 0; gr < kNG; ++gr) {
                    const float o = fmaf(ws[gr][n][c], -7.5f * 5.9604644775390625e-8f * opow, sum_over_g(om[n][c][gr]));
                    if (g == 0) omw[(warp * kRows + r) * kNG + gr] = o;
                }
            }
        __syncthreads();
        if (threadIdx.x < kRows) {
            float m = -INFINITY, l = 0.0f;
            for (int w = 0; w < kAtWarps; ++w) m = fmaxf(m, stat[w * kRows + threadIdx.x].x);
            for (int w = 0; w < kAtWarps; ++w) {
                const float2 f = stat[w * kRows + threadIdx.x];
                l += f.y * ex2(f.x == -INFINITY ? -INFINITY : f.x - m);
            }
            fin[threadIdx.x] = make_float2(m, l);
        }
        const bool whole = seg == job_u0 && seg_end == job_u1;
        // A block's first job may have begun in an earlier block (slot 0); its last may go on (1).
        const int slot = 2 * blockIdx.x + (seg == job_u0 ? 1 : 0);
        float *po = p.part + (size_t)slot * kRows * D;
        float *ps = p.part + (size_t)2 * gridDim.x * kRows * D + (size_t)slot * kRows * 2;
        __syncthreads();
        float wf[kNT][2];
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float m = fin[n * 8 + 2 * t + c].x;
                wf[n][c] = mx[n][c] == -INFINITY ? 0.0f : ex2(mx[n][c] - m);
            }
        T *out = static_cast<T *>(p.a.out);
        for (int v = 0; v < kVB; ++v) {
#pragma unroll
            for (int n = 0; n < kNT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int r = n * 8 + 2 * t + c;
                    const float o = omw[(warp * kRows + r) * kNG + v * 64 / kG];
                    float x[8];
#pragma unroll
                    for (int vv = 0; vv < kVB; ++vv)
                        if (vv == v) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                x[2 * i] = wf[n][c] * fmaf(acc[vv][i][n][c], opow, o);
                                x[2 * i + 1] = wf[n][c] * fmaf(acc[vv][i][n][c + 2], opow * 0.0625f, o);
                            }
                        }
                    if (wf[n][c] == 0.0f) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = 0.0f;
                    }
                    float4 *dst = reinterpret_cast<float4 *>(red + (warp * kRows + r) * 64 + g * 8);
                    dst[0] = make_float4(x[0], x[1], x[2], x[3]);
                    dst[1] = make_float4(x[4], x[5], x[6], x[7]);
                }
            __syncthreads();
            for (int e = threadIdx.x; e < kRows * 64; e += kAtThreads) {
                const int r = e / 64, d = v * 64 + e % 64;
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kAtWarps; ++w) sum += red[w * kRows * 64 + e];
                if (!whole) {
                    __stcg(po + r * D + d, sum);
                } else if (r < nrows) {
                    const float l = fin[r].y;
                    const int row = row0 + r;
                    out[((int64_t)(sw.q0 + row / heads) * p.a.q_heads + head * heads + row % heads) * D + d] =
                        from_f32<T>(l == 0.0f ? 0.0f : sum / l);
                }
            }
            __syncthreads();
        }
        if (threadIdx.x < nrows) {
            const float2 f = fin[threadIdx.x];
            if (!whole) {
                __stcg(reinterpret_cast<float2 *>(ps) + threadIdx.x, f);
            } else if (p.a.lse) {
                const int row = row0 + threadIdx.x;
                p.a.lse[(int64_t)(sw.q0 + row / heads) * p.a.q_heads + head * heads + row % heads] =
                    f.y == 0.0f ? -INFINITY : (f.x + log2f(f.y)) / kLog2e;
            }
        }
        if (!whole) {
            // the blocks that hold parts of this job: the first is named by the job's first unit
            // (the run that holds unit x is the last i with i U / B < x + 1)
            auto owner = [&](int64_t x) { return (int)(((x + 1) * blocks - 1) / units); };
            const int first = owner(job_u0), last = owner(job_u1 - 1);
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) misc[1] = (int)atomicAdd(p.arrived + first, 1u) == last - first;
            __syncthreads();
            if (misc[1]) {
                __threadfence();
                if (threadIdx.x == 0) p.arrived[first] = 0;
                const float *ap = p.part, *as = p.part + (size_t)2 * gridDim.x * kRows * D;
                // the first block's part is in its slot 1, the others' in their slot 0
                if (threadIdx.x < nrows) {
                    float m = -INFINITY, l = 0.0f;
                    for (int i = first; i <= last; ++i)
                        m = fmaxf(m, __ldcg(as + ((size_t)(2 * i + (i == first)) * kRows + threadIdx.x) * 2));
                    for (int i = first; i <= last; ++i) {
                        const float2 f = __ldcg(reinterpret_cast<const float2 *>(as) + (size_t)(2 * i + (i == first)) * kRows + threadIdx.x);
                        l += f.y * ex2(f.x == -INFINITY ? -INFINITY : f.x - m);
                    }
                    fin[threadIdx.x] = make_float2(m, l);
                    if (p.a.lse) {
                        const int row = row0 + threadIdx.x;
                        p.a.lse[(int64_t)(sw.q0 + row / heads) * p.a.q_heads + head * heads + row % heads] =
                            l == 0.0f ? -INFINITY : (m + log2f(l)) / kLog2e;
                    }
                }
                __syncthreads();
                for (int e = threadIdx.x; e < nrows * (D / 4); e += kAtThreads) {
                    const int r = e / (D / 4), d = e % (D / 4) * 4;
                    const float2 f = fin[r];
                    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
                    for (int i = first; i <= last; ++i) {
                        const size_t sl = (size_t)(2 * i + (i == first)) * kRows + r;
                        const float m = __ldcg(as + sl * 2);
                        const float4 x = __ldcg(reinterpret_cast<const float4 *>(ap + sl * D + d));
                        const float k = m == -INFINITY ? 0.0f : ex2(m - f.x);
                        sum.x = fmaf(k, x.x, sum.x), sum.y = fmaf(k, x.y, sum.y);
                        sum.z = fmaf(k, x.z, sum.z), sum.w = fmaf(k, x.w, sum.w);
                    }
                    const float inv = f.y == 0.0f ? 0.0f : 1.0f / f.y;
                    const int row = row0 + r;
                    T *dst = out + ((int64_t)(sw.q0 + row / heads) * p.a.q_heads + head * heads + row % heads) * D + d;
                    dst[0] = from_f32<T>(sum.x * inv), dst[1] = from_f32<T>(sum.y * inv);
                    dst[2] = from_f32<T>(sum.z * inv), dst[3] = from_f32<T>(sum.w * inv);
                }
            }
        }
        __syncthreads();
        seg = seg_end;
    }
}

}  // namespace cora
