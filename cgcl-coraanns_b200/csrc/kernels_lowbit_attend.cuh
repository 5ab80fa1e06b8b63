// Attention of a few query rows per key head over the paged 4-bit cache (cora_kv4_attend).
//
//   score_t = (scale_t (q . c_t) + low_t sum(q)) * softmax scale
//   out     = sum_t p_t (scale'_t c'_t + low'_t),   p = softmax(score)
//
// so codes enter the matrix instructions as integers and a token's factors are applied once per
// (token, query), to fp32 sums. What has to be done is to read the cache once; what bounds it is
// instruction latency (two warps per scheduler, 1080 warp instructions per 64 tokens and key head in one
// group, issue slots 42% used), then memory. Hence:
//  - tokens (then value dimensions) are the 16-row side of m16n8k16, query rows the 8-column
//    side: the query heads that share a key head fill one instruction;
//  - a code becomes an fp16 operand by one AND: nibble 0 of a 16-bit half is the subnormal
//    c 2^-24, nibble 1 is c 2^-20, both exact in the tensor core. The powers of two go into q
//    (a power of two per row, so fp16 holds every bit of a bf16 or fp16 q that is within 2^-24 of
//    its row's largest) and into the final scaling of the output;
//  - w = fp16(p scale') is the operand of the second product (11 bits; scaled by a power of two
//    per row that follows the largest scale' met, or the largest p scale' where that is far less, so
//    it uses the normal range). What the rounding of w
//    loses would be multiplied by codes of 0..15 although values spread around the middle of
//    their group's range; so the sum is taken as sum w (c' - 7.5) + sum p (low' + 7.5 scale'),
//    sum w by one more product with ones: the loss is then 2^-12 of |value - middle|.
//    Statistics, sums and accumulators are fp32;
//  - scores are taken relative to the maximum met before, and only where one exceeds it by more
//    than 2^8 (or value scales outgrow their bound) are maxima exchanged and sums rescaled: p
//    stays below 2^8, w below 2^15;
//  - a value factor that is not finite is left out of the products and makes the rows that see
//    the token NaN (0 times it would reach the rows that do not);
//  - each warp streams tiles of kAtTile tokens through a private ring of bulk copies and keeps its
//    own running maximum and sum: warps wait for one another only where they share a job;
//  - the work, (sequence, key head, row tile) jobs of token tiles plus one unit for a job's own
//    cost, is cut into equal runs, one per warp, so that long, short and ragged batches balance.
//    A job inside one run is written by its warp; one cut over the warps of a block is joined in
//    shared memory; one cut over blocks by the last block to arrive, from partial results in
//    the workspace. Where all jobs are short, each block takes one instead (no join over blocks).
// Measured, 8 key heads of 128: 131072 tokens 47 us (3.0 TB/s over the call; from 65536 to 262144
// tokens 34 -> 77 us, 4.9 TB/s, so some 18 us are start and joins), 64 ragged sequences of 200 to
// 16384 tokens in two groups 77 us (2.8 TB/s).
#pragma once
#include <cuda_fp16.h>

#include "../../include/cora_b200.h"
#include "common.cuh"
#include "kernels_lowbit_append.cuh"
#include "kernels_lowbit_matvec.cuh"

namespace cora {

// One block of 8 warps per SM: with 255 registers a thread nothing is spilled (spills would go
// past the little L1 that the ring leaves) and a tile of 64 tokens gives each warp enough
// independent work. Measured on 131072 tokens x 8 key heads / a ragged batch of 64: 16 warps x 32
// tokens 57 / 100 us, 12 x 32 53 / 93 us, 9 x 64 58 / 97 us, 8 x 64 47 / 76 us.
constexpr int kAtWarps = 8;
// Tiles of a warp's ring, and tokens of a tile (two tiles per warp have to fit shared memory).
constexpr int kAtStages = 2;
constexpr int at_tile(int D) { return D == 256 ? 32 : 64; }
constexpr int kAtRows = 8;         // query rows of a job
constexpr int kAtMinRun = 2;       // units of a warp, at least
// Tokens of a job that one block takes whole, at most, where the grid has a block for each job. Cut
// over blocks, whole, in us, heads of 128: 8 jobs of 512 / 1280 / 2048 / 3072 tokens 17.0, 22.5, 19.5,
// 19.5 against 14.2, 16.6, 20.7, 24.7; 64 jobs 22.7, 22.6, 23.0, 24.9 against 14.6, 18.4, 22.3, 25.6.
constexpr int kAtShort = 1280;
constexpr int kAtMaxSeqs = 512;    // sequences of one launch (their work is kept in smem)
constexpr float kLog2e = 1.4426950408889634f;

struct AttendParams {
    cora_kv4_cache c;
    cora_kv4_attend_args a;
    uint32_t seq0, seqs;      // this launch's sequences
    int64_t q_tokens;         // rows of q
    float *part;              // partial results
    uint32_t *arrived;        // per block, zero between launches
};

// A partial result of 8 rows: unnormalised outputs, then (maximum, sum) per row.
template <int D>
constexpr int kAtPart = kAtRows * (D + 2);

// The shared memory of a block, in order (each part a multiple of 16 bytes).
template <int D, int kNG>
struct AttendSmem {
    static constexpr int kAtTile = at_tile(D);
    static constexpr uint32_t kCodes = kAtTile * D / 2, kMeta = kAtTile * kNG * 4;
    static constexpr uint32_t kStage = 2 * kCodes + 2 * kMeta;
    static constexpr uint32_t kRing = kAtStages * kStage;   // of a warp; at the end its partial result
    static_assert(kRing >= kAtPart<D> * 4, "");
    static constexpr uint32_t ring = 0;
    static constexpr uint32_t qfrag = ring + kAtWarps * kRing;       // [warp][D / 32][32] x 16 bytes
    static constexpr uint32_t keys = qfrag + kAtWarps * (D / 32) * 512;  // [2 warps] job of each partial result
    static constexpr uint32_t info = keys + kAtWarps * 2 * 8;            // [2 warps] int4: q0, head, row0 << 4 | rows, units
    static constexpr uint32_t misc = info + kAtWarps * 2 * 16;
    static constexpr uint32_t bars = misc + 32;
    static constexpr uint32_t work = bars + kAtWarps * kAtStages * 8;    // int4[seqs], int64[seqs + 1]
    static constexpr size_t bytes(uint32_t seqs) { return work + 24 * (size_t)seqs + 8; }
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
// 2^e, and the e of the largest 2^e up to x (-127 for 0 and what is below the normal range).
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ int exponent_of(float x) { return (__float_as_int(x) >> 23) - 127; }
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
__device__ __forceinline__ SeqWork seq_work(const AttendParams &p, int b, int rows, int tile) {
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
    s.first = w ? max(0, len - s.n - w + 1) / tile * tile : 0;
    if (s.first > len) s.first = len / tile * tile;
    s.tiles = max(1, (len - s.first + tile - 1) / tile);  // an empty one still writes zeros
    s.row_tiles = (s.n * (int)(p.a.q_heads / p.c.kv_heads) + rows - 1) / rows;
    return s;
}

// Rows [from, to) that no sequence asks for: zeros, log-sums -inf. By all threads of the grid.
__device__ __forceinline__ void clear_rows(const AttendParams &p, int64_t from, int64_t to, uint32_t thread, uint32_t threads) {
    const int64_t heads = p.a.q_heads, chunks = p.c.head_dim / 8;
    uint4 *const out = static_cast<uint4 *>(p.a.out);
    for (int64_t i = from * heads * chunks + thread; i < to * heads * chunks; i += threads) out[i] = make_uint4(0, 0, 0, 0);
    if (p.a.lse)
        for (int64_t i = from * heads + thread; i < to * heads; i += threads) p.a.lse[i] = -INFINITY;
}
// Those of a launch: before the first range (first launch), after the last (last launch).
__device__ __forceinline__ void clear_gaps(const AttendParams &p, int64_t q0, int64_t q1, uint32_t thread, uint32_t threads) {
    if (p.seq0 == 0 && q0 > 0) clear_rows(p, 0, q0, thread, threads);
    if (p.seq0 + p.seqs == p.a.seqs && q1 < p.q_tokens) clear_rows(p, q1, p.q_tokens, thread, threads);
}
// A call without sequences.
__global__ void kv4_clear_kernel(const AttendParams p) {
    clear_rows(p, 0, p.q_tokens, blockIdx.x * blockDim.x + threadIdx.x, gridDim.x * blockDim.x);
}

template <typename T, int D, int kNG>
__global__ void __launch_bounds__(kAtWarps * 32, 1) kv4_attend_kernel(const AttendParams p) {
    using S = AttendSmem<D, kNG>;
    constexpr int kAtThreads = kAtWarps * 32, kAtTile = at_tile(D);
    constexpr int kMt = kAtTile / 16;
    constexpr int kG = D / kNG, kWords = kG / 32;  // words of one lane and group
    constexpr int kVB = D / 64;                    // 64-dimension blocks of the values
    extern __shared__ __align__(128) unsigned char at_smem[];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    unsigned char *ring = at_smem + S::ring + warp * S::kRing;
    uint4 *qfrag = reinterpret_cast<uint4 *>(at_smem + S::qfrag) + warp * (D / 32) * 32;
    int64_t *keys = reinterpret_cast<int64_t *>(at_smem + S::keys);
    int4 *info = reinterpret_cast<int4 *>(at_smem + S::info);
    volatile int *misc = reinterpret_cast<volatile int *>(at_smem + S::misc);
    uint64_t *bars = reinterpret_cast<uint64_t *>(at_smem + S::bars) + warp * kAtStages;
    int4 *work = reinterpret_cast<int4 *>(at_smem + S::work);
    int64_t *base = reinterpret_cast<int64_t *>(work + p.seqs);

    const int H = p.c.kv_heads, heads = p.a.q_heads / H, P = p.c.page_size;
    const Kv4Block blk(P, D, kG);

    if (lane == 0) {
        for (int s = 0; s < kAtStages; ++s) mbar_init(bars + s, 1);
        keys[2 * warp] = keys[2 * warp + 1] = -1;
        fence_barrier_init();
    }
    for (int b = threadIdx.x; b < (int)p.seqs; b += kAtThreads) {
        const SeqWork s = seq_work(p, b, kAtRows, kAtTile);
        work[b] = make_int4(s.q0, s.n, s.len, s.first);
    }
    __syncthreads();
    auto seq = [&](int b) {
        const int4 w = work[b];
        SeqWork s;
        s.q0 = w.x, s.n = w.y, s.len = w.z, s.first = w.w;
        s.tiles = max(1, (s.len - s.first + kAtTile - 1) / kAtTile);
        s.row_tiles = (s.n * heads + kAtRows - 1) / kAtRows;
        return s;
    };
    if (warp == 0) {  // first units of the sequences, 32 at a time; jobs and the longest
        int64_t run = 0, jobs = 0;
        int longest = 0;
        if (lane == 0) base[0] = 0;
        for (int b0 = 0; b0 < (int)p.seqs; b0 += 32) {
            int64_t v = 0, j = 0;
            if (b0 + lane < (int)p.seqs) {
                const SeqWork s = seq(b0 + lane);
                j = (int64_t)s.row_tiles * H;
                v = (s.tiles + 1) * j;
                if (j) longest = max(longest, s.tiles);
            }
            int64_t all = v;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int64_t o = __shfl_up_sync(0xffffffffu, all, off);
                if (lane >= off) all += o;
                j += __shfl_xor_sync(0xffffffffu, j, off);
            }
            if (b0 + lane < (int)p.seqs) base[b0 + lane + 1] = run + all;
            run += __shfl_sync(0xffffffffu, all, 31);
            jobs += j;
        }
        longest = __reduce_max_sync(0xffffffffu, longest);
        if (lane == 0) misc[2] = (int64_t)longest * kAtTile <= kAtShort && jobs <= gridDim.x ? (int)jobs : 0;
    } else if (warp == 1) {  // (meanwhile)
        clear_gaps(p, work[0].x, (int64_t)work[p.seqs - 1].x + work[p.seqs - 1].y, blockIdx.x * 32 + lane, gridDim.x * 32);
    }
    __syncthreads();
    const int64_t units = base[p.seqs];
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
    // Equal runs: with W warps, warp i holds units [cut(i), cut(i + 1)), cut(i) = floor(i U / W).
    const bool aligned = misc[2] != 0;
    const int blocks = aligned ? misc[2] : (int)max((int64_t)1, min((int64_t)gridDim.x, units / (kAtMinRun * kAtWarps)));
    if (blockIdx.x >= blocks || !units) return;
    const uint32_t workers = blocks * kAtWarps;
    const int64_t each = units >> 32 ? units / workers : (uint32_t)units / workers;
    const uint32_t more = (uint32_t)(units - each * workers);
    auto even = [&](uint32_t i) { return each * i + more * i / workers; };  // more i < 2^32
    int64_t b0 = 0, b1 = 0;  // this block's units
    if (aligned) {  // one job per block: the block's number counts jobs
        int64_t job = blockIdx.x;
        for (int b = 0;; ++b) {
            const SeqWork s = seq(b);
            const int64_t n = (int64_t)s.row_tiles * H;
            if (job < n) {
                b0 = base[b] + job * (s.tiles + 1), b1 = b0 + s.tiles + 1;
                break;
            }
            job -= n;
        }
    } else {
        b0 = even(blockIdx.x * kAtWarps), b1 = even((blockIdx.x + 1) * kAtWarps);
    }
    auto cut = [&](uint32_t w) {
        return aligned ? b0 + w * (uint32_t)(b1 - b0) / kAtWarps : even(blockIdx.x * kAtWarps + w);
    };
    const int64_t u0 = cut(warp), u1 = cut(warp + 1);

    // ---- the warp's stream of tiles ----
    // Copies of one tile: lane 4 i + k copies section k of the tile's i-th page piece.
    const int per = min(P, kAtTile), shift = 31 - __clz(P);  // tokens of a piece
    const int piece = lane >> 2, kind = lane & 3;
    const uint32_t rowb = kind < 2 ? D / 2 : kNG * 4;
    const uint32_t src_at = (kind & 1 ? (kind < 2 ? blk.codes : blk.metas) : 0) + (kind < 2 ? 0 : 2 * blk.codes);
    const uint32_t dst_at = (kind & 1 ? (kind < 2 ? S::kCodes : S::kMeta) : 0) + (kind < 2 ? 0 : 2 * S::kCodes) +
                            piece * per * rowb;
    int64_t ahead = u0;                                // the unit that the next tile to fetch is
    int fb = -1, ftile = 0, frt = 0, fhead = 0;
    SeqWork fs{};
    const int *ftable = nullptr;
    int pages = 0, pbase = 0;  // lane i holds the number of the sequence's page pbase + i
    auto load_pages = [&](int first) {
        pbase = first;
        pages = (first + lane) << shift < fs.len ? __ldg(ftable + first + lane) : -1;
    };
    auto fetch_q = [&]() {  // the job's queries, into L2 ahead of the copies that crowd the memory
        constexpr int kLines = D / 64;  // 128-byte lines of a row
        const int row = frt * kAtRows + lane / kLines, tk = row / heads;
        if (lane < kAtRows * kLines && row < fs.n * heads)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const T *>(p.a.q) + (int64_t)(fs.q0 + tk) * p.a.q_token +
                                                          (int64_t)(fhead * heads + row - tk * heads) * p.a.q_head +
                                                          lane % kLines * 64));
    };
    // Copies the tile that is next (if there is one yet) and moves on to the one after.
    auto fetch = [&](int stage) {
        if (fb >= 0) {
            const int tok = fs.first + ftile * kAtTile + piece * per;
            if (((fs.first + ftile * kAtTile + kAtTile - 1) >> shift) - pbase >= 32) load_pages((fs.first + ftile * kAtTile) >> shift);
            const int page = __shfl_sync(0xffffffffu, pages, (tok >> shift) - pbase);
            const bool got = piece * per < kAtTile && tok < fs.len, ok = got && page >= 0 && (uint32_t)page < p.c.num_pages;
            const uint32_t lanes = __ballot_sync(0xffffffffu, ok);
            if (got && !ok) atomicOr(p.c.status, kDevBadInput);
            // sections of a piece are copied by four neighbouring lanes, all or none
            if (lane == 0) mbar_arrive_expect_tx(bars + stage, __popc(lanes) / 4 * per * (D + 8 * kNG));
            __syncwarp();
            if (ok)
                bulk_g2s(ring + stage * S::kStage + dst_at,
                         p.c.pool + ((uint64_t)page * H + fhead) * blk.bytes + src_at + (uint32_t)(tok & (P - 1)) * rowb,
                         per * rowb, bars + stage);
            ++ahead, ++ftile;
        }
        if (ahead >= u1) return;
        if (fb < 0 || ftile == fs.tiles) {  // another job
            if (fb < 0 || ahead >= base[fb + 1]) {  // of another sequence
                fb = find(ahead);
                fs = seq(fb);
                ftable = p.a.page_table + (int64_t)(p.seq0 + fb) * p.a.table_stride;
                const uint32_t r = (uint32_t)(ahead - base[fb]), n = fs.tiles + 1, job = r / n;
                ftile = (int)(r - job * n) - 1;
                fhead = (int)(job / fs.row_tiles);
                frt = (int)(job - fhead * fs.row_tiles);
            } else {
                ftile = -1;
                if (++frt == fs.row_tiles) frt = 0, ++fhead;
            }
            if (ftile < 0) ++ahead, ftile = 0;  // past the job's own unit
            if (ahead >= u1) return;
            load_pages((fs.first + ftile * kAtTile) >> shift);
            fetch_q();
        }
    };
    int fstage = 0, stage = 0, pending = 0;  // next stage to fill, to read; tiles in flight
    uint32_t phase = 0;
    bool alive = true;

    // partial results: two per block, then one per warp (a first job that goes on before it ends)
    float *const part_warp = p.part + (size_t)2 * gridDim.x * kAtPart<D> + (size_t)(blockIdx.x * kAtWarps + warp) * kAtPart<D>;

    T *const out = static_cast<T *>(p.a.out);
    const bool q_vec = reinterpret_cast<uintptr_t>(p.a.q) % 8 == 0 && p.a.q_token % 4 == 0 && p.a.q_head % 4 == 0;
    float acc[kVB][4][4], om[2][kNG], ws[kNG][4];  // sum w c'; sum p (low' + 7.5 scale'); sum w (rows alike)
    float mx[2], ref[2], over[2], ls[2];           // per row: maximum, what scores are relative to, how far
                                                   // they may exceed it, sum of p
    float qs[2][kNG], raw[2] = {};                 // sums of q; the unit of these and of q . c
    int2 lm[2];                                    // tokens that rows 2 t and 2 t + 1 see
    int lo_max = 0, hi_min = 0;
    float vmul[2] = {};                            // w = p scale' vmul, a power of two: 2^7 / vmul bounds the value
    float vbound = 0.0f;                           // scales met (0: none yet); the less of both rows' bounds
    int b = -1, head = 0, row0 = 0, nrows = 0, tile = 0, tile_end = 0;
    int64_t u = u0, seg_end = 0, job_u0 = 0, job_u1 = 0;
    SeqWork sw{};
    const int tg = g ^ ((g >> 1) & 1);  // the token of operand row g (and + 8): see the values below

    constexpr int kLoads = kAtRows * D / 4 / 32;
    T qv[kLoads][4];
    for (bool fresh = true;;) {
        if (fresh) {
        // ---- the next job: tiles [tile, tile_end) of it are this warp's ----
        for (tile = 0, tile_end = 0; u < u1 && tile_end <= tile; u = tile_end <= tile ? seg_end : u) {
            if (b < 0 || u >= base[b + 1]) {
                b = find(u);
                sw = seq(b);
            }
            const uint32_t jr = (uint32_t)(u - base[b]), jn = sw.tiles + 1, job = jr / jn;
            job_u0 = base[b] + (int64_t)job * jn, job_u1 = job_u0 + jn;
            seg_end = min(u1, job_u1);
            head = (int)(job / sw.row_tiles);
            row0 = (int)(job - head * sw.row_tiles) * kAtRows;
            nrows = min(kAtRows, sw.n * heads - row0);
            tile = max(0, (int)(u - job_u0) - 1);
            tile_end = (int)(seg_end - job_u0) - 1;  // (none: only the job's own unit)
        }
        if (u >= u1) break;
        // its queries, 4 dimensions of a row a lane and load, ahead of the copies
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = (i * 32 + lane) / (D / 4), d = (i * 32 + lane) % (D / 4) * 4;
            const int row = row0 + min(r, nrows - 1), tk = row / heads;
            const T *src = static_cast<const T *>(p.a.q) + (int64_t)(sw.q0 + tk) * p.a.q_token +
                           (int64_t)(head * heads + row - tk * heads) * p.a.q_head + d;
            if (q_vec) {
                *reinterpret_cast<uint2 *>(qv[i]) = *reinterpret_cast<const uint2 *>(src);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) qv[i][e] = src[e];
            }
        }
        }
        while (pending < kAtStages && ahead < u1 && alive) {
            const bool copies = fb >= 0;
            fetch(fstage);
            if (copies) {
                ++pending;
                fstage = fstage + 1 == kAtStages ? 0 : fstage + 1;
            }
        }
        if (fresh) {
        fresh = false;
        // queries: rows are (token, head of the group); fp16 under a power of two per row: 2^qe brings
        // the row's largest |q| into [2^13, 2^14). qe[i] is that of the lane's row of load i
        int qe[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            float big = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float m = fabsf(to_f32(qv[i][e]));
                big = m < 3.4e38f ? fmaxf(big, m) : big;  // infinities and NaN have no say
            }
            uint32_t top = __float_as_uint(big);
            if constexpr (D == 64) {  // a row is half a load
#pragma unroll
                for (int o = 8; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            } else {
                top = __reduce_max_sync(0xffffffffu, top);
            }
            qe[i] = (int)(top >> 23);
        }
        if constexpr (D == 256) {  // a row is two loads
#pragma unroll
            for (int i = 0; i < kLoads; i += 2) qe[i] = qe[i + 1] = max(qe[i], qe[i + 1]);
        }
        const float qf = p.a.scale * kLog2e;
        float qpow[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            qe[i] = max(-100, min(126, 13 + 127 - qe[i]));
            qpow[i] = power_of_two(qe[i]);
        }
        int qe2[2];  // of rows 2 t and 2 t + 1
        if constexpr (D == 64) {
            const int mine = t == 0 ? qe[0] : t == 1 ? qe[1] : t == 2 ? qe[2] : qe[3], other = __shfl_xor_sync(0xffffffffu, mine, 16);
            qe2[0] = lane < 16 ? mine : other, qe2[1] = lane < 16 ? other : mine;
        } else {
            constexpr int kPer = D / 128;  // loads of a row
#pragma unroll
            for (int c = 0; c < 2; ++c)
                qe2[c] = t == 0 ? qe[c * kPer] : t == 1 ? qe[(2 + c) * kPer] : t == 2 ? qe[(4 + c) * kPer] : qe[(6 + c) * kPer];
        }
        raw[0] = ldexpf(qf, 24 - qe2[0]), raw[1] = ldexpf(qf, 24 - qe2[1]);  // of q . c as the tensor core sums it
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = (i * 32 + lane) / (D / 4), d = (i * 32 + lane) % (D / 4) * 4;
            // Dimensions d .. d + 3 are nibbles 0..3 (even lanes) or 4..7 (odd ones) of their
            // word of 8; the operand pairs nibbles {0,4} {1,5} {2,6} {3,7}, the odd ones under
            // 2^-4: neighbouring lanes swap halves, and each stores two pairs.
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = r < nrows ? to_f32(qv[i][e]) * qpow[i] * (e & 1 ? 0.0625f : 1.0f) : 0.0f;
            const uint32_t lo = pack_half2(x[0], x[1]), hi = pack_half2(x[2], x[3]);
            const uint32_t other = __shfl_xor_sync(0xffffffffu, lane & 1 ? lo : hi, 1);
            uint2 w;
            w.x = lane & 1 ? __byte_perm(other, hi, 0x5410) : __byte_perm(lo, other, 0x5410);
            w.y = lane & 1 ? __byte_perm(other, hi, 0x7632) : __byte_perm(lo, other, 0x7632);
            // word -> (group, lane t, word of the lane)
            const int word = d / 8, gr = d / kG, wi = word - gr * (kG / 8), tt = wi / kWords, j = wi % kWords;
            reinterpret_cast<uint2 *>(qfrag + (gr * kWords + j) * 32 + r * 4 + tt)[lane & 1] = w;
        }
        __syncwarp();
        // sums of q per group, by the same operands against ones (and 16s)
#pragma unroll
        for (int gr = 0; gr < kNG; ++gr) {
            float d[4] = {};
            constexpr uint32_t one = 0x3c003c00u, sixteen = 0x4c004c00u;
#pragma unroll
            for (int j = 0; j < kWords; ++j) {
                const uint4 q = qfrag[(gr * kWords + j) * 32 + lane];
                mma16816<__half>(d, one, one, sixteen, sixteen, q.x, q.y);
                mma16816<__half>(d, one, one, sixteen, sixteen, q.z, q.w);
            }
            qs[0][gr] = d[0] * 5.9604644775390625e-8f, qs[1][gr] = d[1] * 5.9604644775390625e-8f;  // 2^-24
        }
        lo_max = 0, hi_min = 0x7fffffff;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int r = 2 * t + c, pos = sw.len - sw.n + (row0 + r) / heads;
            lm[c].y = p.a.causal ? max(0, min(sw.len, pos + 1)) : sw.len;
            lm[c].x = p.a.window ? max(0, pos - (int)p.a.window + 1) : 0;
            if (r < nrows) lo_max = max(lo_max, lm[c].x), hi_min = min(hi_min, lm[c].y);
            mx[c] = over[c] = -INFINITY;
            ref[c] = ls[c] = 0.0f;
#pragma unroll
            for (int gr = 0; gr < kNG; ++gr) om[c][gr] = ws[gr][c] = ws[gr][c + 2] = 0.0f;
        }
        lo_max = __reduce_max_sync(0xffffffffu, lo_max);
        hi_min = __reduce_min_sync(0xffffffffu, hi_min);
#pragma unroll
        for (int v = 0; v < kVB; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[v][i][c] = 0.0f;
        vbound = vmul[0] = vmul[1] = 0.0f;
        }

        {
            // ---- a tile: scores of 16 tokens x 8 rows at a time ----
            const int tok0 = sw.first + tile * kAtTile;
            if (pending) {  // (0 only after a wait ran out: nothing more is fetched then)
                alive = __all_sync(0xffffffffu, mbar_wait_short(bars + stage, phase, p.c.status)) && alive;
                --pending;
            }
            const unsigned char *st = ring + stage * S::kStage;
            float s[kMt][4];
#pragma unroll
            for (int mt = 0; mt < kMt; ++mt) {
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
                    float d[4] = {};
#pragma unroll
                    for (int j = 0; j < kWords; ++j) {
                        const uint32_t a8 = wa[j] >> 8, b8 = wb[j] >> 8;
                        const uint4 q = qfrag[(gr * kWords + j) * 32 + lane];
                        mma16816<__half>(d, wa[j] & 0x000f000fu, wb[j] & 0x000f000fu, wa[j] & 0x00f000f0u,
                                         wb[j] & 0x00f000f0u, q.x, q.y);
                        mma16816<__half>(d, a8 & 0x000f000fu, b8 & 0x000f000fu, a8 & 0x00f000f0u, b8 & 0x00f000f0u,
                                         q.z, q.w);
                    }
                    const __half2 *km = reinterpret_cast<const __half2 *>(st + 2 * S::kCodes);
                    const float2 f0 = __half22float2(km[(mt * 16 + tg) * kNG + gr]);
                    const float2 f1 = __half22float2(km[(mt * 16 + 8 + tg) * kNG + gr]);
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        s[mt][c] = fmaf(c < 2 ? f0.x : f1.x, d[c], fmaf(c < 2 ? f0.y : f1.y, qs[c & 1][gr], gr ? s[mt][c] : 0.0f));
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) s[mt][c] = fmaf(s[mt][c], raw[c & 1], -ref[c & 1]);
            }
            const uint32_t *vm = reinterpret_cast<const uint32_t *>(st + 2 * S::kCodes + S::kMeta);
            uint32_t vf[kMt][2][kNG];  // the tokens' value factors
#pragma unroll
            for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int gr = 0; gr < kNG; ++gr) vf[mt][r][gr] = vm[(mt * 16 + tg + r * 8) * kNG + gr];
            if (tok0 + kAtTile > hi_min || tok0 < lo_max) {  // some row does not see some token
                // tokens that the job's rows see between them
                const int past = sw.len - sw.n, first = past + row0 / heads, last = past + (row0 + nrows - 1) / heads;
                const int job_hi = p.a.causal ? min(sw.len, last + 1) : sw.len;
                const int job_lo = p.a.window ? first - (int)p.a.window + 1 : 0;
#pragma unroll
                for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int tok = tok0 + mt * 16 + tg + r * 8;
#pragma unroll
                        for (int c = 0; c < 2; ++c)
                            if (tok < lm[c].x || tok >= lm[c].y) s[mt][2 * r + c] = -INFINITY;
                        if (tok < job_lo || tok >= job_hi) {  // nobody does: the bytes may be anything, and have no
                                                              // part in the bound of the value scales
#pragma unroll
                            for (int gr = 0; gr < kNG; ++gr) vf[mt][r][gr] = 0;
                        }
                    }
            }
            // ---- maxima, bound of the value scales: the rare way out of the tile's course ----
            __half2 most = __half2half2(__ushort_as_half(0));
#pragma unroll
            for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
                for (int r = 0; r < 2; ++r)
#pragma unroll
                    for (int gr = 0; gr < kNG; ++gr) most = __hmax2_nan(most, __habs2(*reinterpret_cast<__half2 *>(&vf[mt][r][gr])));
            const float2 mf = __half22float2(most);
            bool out_of_course = !(mf.x <= vbound) || !(mf.y <= 65504.0f);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float m = fmaxf(s[0][c], s[0][c + 2]);
#pragma unroll
                for (int mt = 1; mt < kMt; ++mt) m = fmaxf(m, fmaxf(s[mt][c], s[mt][c + 2]));
                out_of_course |= m > over[c];
            }
            if (__any_sync(0xffffffffu, out_of_course)) {
                float k[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float m = fmaxf(s[0][c], s[0][c + 2]);
#pragma unroll
                    for (int mt = 1; mt < kMt; ++mt) m = fmaxf(m, fmaxf(s[mt][c], s[mt][c + 2]));
                    m = max_over_g(m) + ref[c];
                    const bool grew = m > mx[c] + (mx[c] == -INFINITY ? 0.0f : 8.0f);
                    k[c] = grew ? ex2(mx[c] - m) : 1.0f;
                    if (grew) {
                        const float shift = ref[c] - m;
                        mx[c] = ref[c] = m, over[c] = 8.0f;
#pragma unroll
                        for (int mt = 0; mt < kMt; ++mt) s[mt][c] += shift, s[mt][c + 2] += shift;
                    }
                }
                // A row's bound: the largest value scale, or 2^6 times its largest p scale (p up to 1)
                // where that is less: a token that it all but ignores does not cost it its bits.
                float smax = 0.0f, pmax[2] = {};
#pragma unroll
                for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float p0 = ex2(fminf(0.0f, s[mt][2 * r])), p1 = ex2(fminf(0.0f, s[mt][2 * r + 1]));
#pragma unroll
                        for (int gr = 0; gr < kNG; ++gr) {
                            const float2 f = __half22float2(*reinterpret_cast<__half2 *>(&vf[mt][r][gr]));
                            if (fabsf(f.x) <= 65504.0f && fabsf(f.y) <= 65504.0f) {
                                smax = fmaxf(smax, fabsf(f.x));
                                pmax[0] = fmaxf(pmax[0], fabsf(f.x) * p0), pmax[1] = fmaxf(pmax[1], fabsf(f.x) * p1);
                                continue;
                            }
                            vf[mt][r][gr] = 0;
#pragma unroll
                            for (int c = 0; c < 2; ++c)
                                if (s[mt][2 * r + c] != -INFINITY) ls[c] = __int_as_float(0x7fc00000);
                        }
                    }
                smax = max_over_g(smax);
                vbound = 65504.0f;  // (of rows that saw a token; another comes this way with its first)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float most = fminf(smax, 64.0f * max_over_g(pmax[c]));
                    float f = k[c];
                    if (most * vmul[c] > 128.0f || (vmul[c] == 0.0f && most > 0.0f)) {
                        const float to = power_of_two(min(100, 6 - exponent_of(most)));  // most < 2^7 / to
                        if (vmul[c] > 0.0f) f *= to * power_of_two(-exponent_of(vmul[c]));
                        vmul[c] = to;
                    }
                    if (mx[c] != -INFINITY) vbound = fminf(vbound, vmul[c] > 0.0f ? power_of_two(7 - exponent_of(vmul[c])) : 0.0f);
                    ls[c] *= k[c];
#pragma unroll
                    for (int gr = 0; gr < kNG; ++gr) om[c][gr] *= k[c], ws[gr][c] *= f;
#pragma unroll
                    for (int v = 0; v < kVB; ++v)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[v][i][c] *= f, acc[v][i][c + 2] *= f;
                }
            }
            // ---- values: per 16 tokens, p scale' transposed into the 16-deep operand ----
#pragma unroll
            for (int mt = 0; mt < kMt; ++mt) {
                uint32_t pb[kNG][2];
                float sv[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    s[mt][c] = ex2(s[mt][c]);
                    ls[c & 1] += s[mt][c];
                    sv[c] = s[mt][c] * vmul[c & 1];
                }
#pragma unroll
                for (int gr = 0; gr < kNG; ++gr) {
                    float x[4];
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float2 f = __half22float2(*reinterpret_cast<__half2 *>(&vf[mt][r][gr]));
                        const float fm = fmaf(7.5f, f.x, f.y);
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            x[2 * r + c] = sv[2 * r + c] * f.x;
                            om[c][gr] = fmaf(s[mt][2 * r + c], fm, om[c][gr]);
                        }
                    }
                    pb[gr][0] = transpose8x8(pack_half2(x[0], x[1]));
                    pb[gr][1] = transpose8x8(pack_half2(x[2], x[3]));
                    constexpr uint32_t one = 0x3c003c00u;
                    mma16816<__half>(ws[gr], one, one, one, one, pb[gr][0], pb[gr][1]);
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
                        mma16816<__half>(acc[v][i], x[i] & 0x000f000fu, x[i] & 0x00f000f0u, y[i] & 0x000f000fu,
                                         y[i] & 0x00f000f0u, pb[gr][0], pb[gr][1]);
                }
            }
            __syncwarp();  // the stage is read
            if (++stage == kAtStages) {
                stage = 0;
                phase ^= 1;
            }
        }
        if (++tile < tile_end) continue;
        u = seg_end;
        fresh = true;

        // ---- the warp's result of this job: acc becomes sum p v, ls the sum over its tokens ----
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const float opow = vmul[c] > 0.0f ? power_of_two(24 - exponent_of(vmul[c])) : 0.0f;  // 2^24 of the codes, the operand's factor
            ls[c] = sum_over_g(ls[c]);
#pragma unroll
            for (int gr = 0; gr < kNG; ++gr) {
                const float o = fmaf(ws[gr][c], -7.5f * 5.9604644775390625e-8f * opow, sum_over_g(om[c][gr]));
#pragma unroll
                for (int v = gr * (kG / 64); v < (gr + 1) * (kG / 64); ++v)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        acc[v][i][c] = fmaf(acc[v][i][c], opow, o);
                        acc[v][i][c + 2] = fmaf(acc[v][i][c + 2], opow * 0.0625f, o);
                    }
            }
        }
        const bool whole = u0 <= job_u0 + 1 && seg_end == job_u1;  // all its tiles are ours
        if (whole) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int r = 2 * t + c, row = row0 + r;
                if (r < nrows) {
                    const int tk = row / heads;
                    const int64_t at = (int64_t)(sw.q0 + tk) * p.a.q_heads + head * heads + row - tk * heads;
                    const float inv = ls[c] == 0.0f ? 0.0f : 1.0f / ls[c];
#pragma unroll
                    for (int v = 0; v < kVB; ++v) {
                        float x[8];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            x[2 * i] = ls[c] == 0.0f ? 0.0f : acc[v][i][c] * inv;
                            x[2 * i + 1] = ls[c] == 0.0f ? 0.0f : acc[v][i][c + 2] * inv;
                        }
                        store8(out + at * D + v * 64 + g * 8, x);
                    }
                    if (p.a.lse && g == 0) p.a.lse[at] = ls[c] == 0.0f ? -INFINITY : (mx[c] + log2f(ls[c])) / kLog2e;
                }
            }
            continue;
        }
        // Not whole: it waits for the other warps. The last job's part goes to shared memory (the
        // ring has run dry), an earlier one's (the run's first job) to the workspace.
        const bool last = u >= u1;
        if (lane == 0) {
            keys[2 * warp + (last ? 1 : 0)] = job_u0;
            info[2 * warp + (last ? 1 : 0)] = make_int4(sw.q0, head, row0 << 4 | nrows, (int)(job_u1 - job_u0));
        }
        float *dst = last ? reinterpret_cast<float *>(ring) : part_warp;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int r = 2 * t + c;
#pragma unroll
            for (int v = 0; v < kVB; ++v) {
                float4 *at = reinterpret_cast<float4 *>(dst + r * D + v * 64 + g * 8);
                at[0] = make_float4(acc[v][0][c], acc[v][0][c + 2], acc[v][1][c], acc[v][1][c + 2]);
                at[1] = make_float4(acc[v][2][c], acc[v][2][c + 2], acc[v][3][c], acc[v][3][c + 2]);
            }
            if (g == 0) *reinterpret_cast<float2 *>(dst + kAtRows * D + 2 * r) = make_float2(mx[c], ls[c]);
        }
    }

    // ---- jobs cut over this block's warps: entries 2 w, 2 w + 1 are warp w's parts. Warp r joins
    // row r of each: a lane weighs an entry, then each takes 4 dimensions ----
    __syncthreads();
    const int64_t key = lane < 2 * kAtWarps ? keys[lane] : -1;
    const float *entry = lane & 1 ? reinterpret_cast<const float *>(at_smem + S::ring + (lane >> 1) % kAtWarps * S::kRing)
                                  : p.part + (size_t)2 * gridDim.x * kAtPart<D> +
                                        (size_t)(blockIdx.x * kAtWarps + (lane >> 1) % kAtWarps) * kAtPart<D>;
    // A part that saw nothing has maximum -inf and sum 0; a sum that is not 0 there is NaN and
    // must show.
    auto weigh = [&](float2 f, float m) { return f.x == -INFINITY ? 0.0f : ex2(f.x - m); };
    auto share = [&](float2 f, float k) { return f.y * (f.x == -INFINITY && f.y != 0.0f ? 1.0f : k); };
    int4 in{};  // of the job at hand
    auto row_at = [&](int r) {  // of out and lse
        const int row = (in.z >> 4) + r, tk = row / heads;
        return (int64_t)(in.x + tk) * p.a.q_heads + in.y * heads + row - tk * heads;
    };
    auto lse_of = [&](float m, float l) { return l == 0.0f ? -INFINITY : (m + log2f(l)) / kLog2e; };
    uint32_t cut_jobs = 0;  // entries that begin jobs cut over blocks: at most two
    for (uint32_t left = __ballot_sync(0xffffffffu, key >= 0); left;) {
        const int e0 = __ffs(left) - 1;
        job_u0 = __shfl_sync(0xffffffffu, key, e0);
        const uint32_t mine = __ballot_sync(0xffffffffu, key == job_u0);
        left &= ~mine;
        in = info[e0];
        const bool starts = b0 <= job_u0 + 1, whole = starts && b1 >= job_u0 + in.w;
        if (!whole) cut_jobs |= 1u << e0;
        if (warp >= (in.z & 15)) continue;
        const float2 f = mine >> lane & 1 ? *reinterpret_cast<const float2 *>(entry + kAtRows * D + 2 * warp)
                                          : make_float2(-INFINITY, 0.0f);
        float m = f.x;
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float k = weigh(f, m);
        float l = share(f, k);
#pragma unroll
        for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        float *slot = p.part + (size_t)(2 * blockIdx.x + (starts ? 1 : 0)) * kAtPart<D>;
        const int64_t at = row_at(warp);
#pragma unroll 1
        for (int d = lane * 4; d < D + 127 - (D + 127) % 128; d += 128) {
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
            for (uint32_t rest = mine; rest; rest &= rest - 1) {
                const int e = __ffs(rest) - 1;
                const float *en = reinterpret_cast<const float *>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(entry), e));
                const float w = __shfl_sync(0xffffffffu, k, e);
                if (w != 0.0f && d < D) {
                    const float4 x = *reinterpret_cast<const float4 *>(en + warp * D + d);
                    sum.x = fmaf(w, x.x, sum.x), sum.y = fmaf(w, x.y, sum.y);
                    sum.z = fmaf(w, x.z, sum.z), sum.w = fmaf(w, x.w, sum.w);
                }
            }
            if (d >= D) continue;
            if (whole) store4(out + at * D + d, sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
            else __stcg(reinterpret_cast<float4 *>(slot + warp * D + d), sum);
        }
        if (lane == 0) {
            if (!whole) __stcg(reinterpret_cast<float2 *>(slot + kAtRows * D + 2 * warp), make_float2(m, l));
            else if (p.a.lse) p.a.lse[at] = lse_of(m, l);
        }
    }
    if (!cut_jobs) return;
    __threadfence();
    __syncthreads();
    float2 *const fin = reinterpret_cast<float2 *>(at_smem + S::qfrag);  // [row] (maximum, 1 / sum)
    for (; cut_jobs; cut_jobs &= cut_jobs - 1) {
        const int e0 = __ffs(cut_jobs) - 1;
        job_u0 = keys[e0], in = info[e0];
        const int nrows = in.z & 15;
        // ---- cut over blocks: the last to arrive joins. Unit x is the run of worker i, the last
        // with cut(i) <= x, that is i U < (x + 1) W ----
        auto owner = [&](int64_t x) { return (int)(((x + 1) * workers - 1) / units) / kAtWarps; };
        const int first = owner(job_u0 + 1), last = owner(job_u0 + in.w - 1), parts = last - first + 1;
        if (threadIdx.x == 0) misc[1] = (int)atomicAdd(p.arrived + first, 1u) == last - first;
        __syncthreads();
        const bool joins = misc[1];
        __syncthreads();  // (misc is free again)
        if (!joins) continue;
        __threadfence();
        if (threadIdx.x == 0) p.arrived[first] = 0;
        // the first block's part is in its slot 1, the others' in their slot 0
        auto slot_of = [&](int i) { return p.part + (size_t)(2 * (first + i) + (i == 0 ? 1 : 0)) * kAtPart<D>; };
        if (warp < kAtRows) {
            constexpr int kOf = (148 + 31) / 32;  // parts of a lane, read at once
            float2 f[kOf];
            float m = -INFINITY, l = 0.0f;
#pragma unroll
            for (int i = 0; i < kOf; ++i)
                f[i] = i * 32 + lane < parts ? __ldcg(reinterpret_cast<const float2 *>(slot_of(i * 32 + lane) + kAtRows * D) + warp)
                                             : make_float2(-INFINITY, 0.0f);
            for (int i = kOf * 32 + lane; i < parts; i += 32)  // (a larger device)
                m = fmaxf(m, __ldcg(slot_of(i) + kAtRows * D + 2 * warp));
#pragma unroll
            for (int i = 0; i < kOf; ++i) m = fmaxf(m, f[i].x);
#pragma unroll
            for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
            for (int i = 0; i < kOf; ++i) l += share(f[i], weigh(f[i], m));
            for (int i = kOf * 32 + lane; i < parts; i += 32) {
                const float2 x = __ldcg(reinterpret_cast<const float2 *>(slot_of(i) + kAtRows * D) + warp);
                l += share(x, weigh(x, m));
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            if (lane == 0) {
                fin[warp] = make_float2(m, l == 0.0f ? 0.0f : 1.0f / l);
                if (warp < nrows && p.a.lse) p.a.lse[row_at(warp)] = lse_of(m, l);
            }
        }
        __syncthreads();
        // threads: (a share of the parts, if there are threads to spare) x (row, 4 dimensions)
        const int items = nrows * (D / 4), groups = max(1, kAtThreads / items);
        float4 *red = reinterpret_cast<float4 *>(at_smem + S::qfrag + 1024);
        for (int i0 = 0; i0 < items; i0 += kAtThreads) {
            const int gi = threadIdx.x / items, i = groups > 1 ? threadIdx.x % items : i0 + threadIdx.x;
            const bool on = i < items && gi < groups;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const int r = i / (D / 4), d = i % (D / 4) * 4;
            if (on) {
                const float m = fin[r].x;
#pragma unroll 4
                for (int k = groups > 1 ? gi : 0; k < parts; k += groups) {
                    const float4 x = __ldcg(reinterpret_cast<const float4 *>(slot_of(k) + r * D + d));
                    const float pm = __ldcg(slot_of(k) + kAtRows * D + 2 * r);
                    const float w = pm == -INFINITY ? 0.0f : ex2(pm - m);
                    sum.x += w != 0.0f ? w * x.x : 0.0f, sum.y += w != 0.0f ? w * x.y : 0.0f;
                    sum.z += w != 0.0f ? w * x.z : 0.0f, sum.w += w != 0.0f ? w * x.w : 0.0f;
                }
            }
            if (groups > 1) {
                if (on) red[gi * items + i] = sum;
                __syncthreads();
                if (on && gi == 0)
                    for (int k = 1; k < groups; ++k) {
                        const float4 x = red[k * items + i];
                        sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
                    }
            }
            if (on && gi == 0) {
                const float inv = fin[r].y;
                store4(out + row_at(r) * D + d, sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
            }
        }
        __syncthreads();
    }
}

}  // namespace cora
