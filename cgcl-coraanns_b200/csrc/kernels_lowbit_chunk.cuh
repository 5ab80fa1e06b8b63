// Attention of many query rows per key head over the paged 4-bit cache: cora_kv4_attend for
// chunks of a prompt and wide head groups (more than 32 rows per key head). Measured: 2048 queries
// x 32 heads of 128 on 16384 tokens (8 key heads) 756 us, 682 TFLOP/s (in turn with variants on
// unchanged inputs 745; 730 when the other figures below were taken).
//
// Tensor cores and exponentials are each a third busy, issue slots 46%: what bounds it is the chain of
// one row tile (softmax, hand-over, second product, next scores), of which the other row tile's
// work covers a part. Rows (query token, head of the group) fill tiles of 128; one block takes kNQ = 2 tiles
// (1 for few rows or head size 256) against the same keys, so each unpacked key tile serves 256
// rows. Warp roles:
//   0-3, 4-7  softmax of row tile 0 / 1, 32 rows per warp: sums of q . c from TMEM, the token's
//             factors from shared memory, running maximum and sum in fp32, probabilities back to
//             TMEM as the fp16 operand of the second product. A thread holds 8 columns of 4 rows
//             at a time (accumulator fragments), so that a factor it reads serves 4 rows: with a
//             thread per row the factors alone took 2048 of 7200 cycles of shared memory a tile.
//             One pass: probabilities refer to the maximum met before; only where it grows by more than
//             2^8 are the sums (and the tile's earlier probabilities) rescaled. All are times 2^7, so
//             that they stay below 2^15, which fp16 holds, and that of a token is off by at most
//             2^-32 of the largest: a long tail of tiny ones keeps its share.
//   8-15      unpack, into 128-byte swizzled tiles: key codes as the fp16 subnormals c 2^-24 and
//             c 2^-20, exact (the scores keep fp32 accuracy); value codes to fp16 scale c + low,
//             one rounding each (2^-12 of the value, as of the probability). The format goes up to
//             16 x 65504: from a tile that holds a value past 65504 on, a stretch's values are
//             unpacked under 2^-5 (values below 2^-9 then keep an absolute 2^-20) and the sums follow.
//   16        copies code tiles from the cache's pages (bulk copies into a ring).
//   17        issues the tcgen05 products: S_g = Q_g C_g^T per factor group (keys K-major) and
//             O += P V (P in TMEM, values as stored, token-major: the N-major operand). The whole
//             warp runs the loop; from a branch to one lane the issue itself was the bound
//             (802 against 730 us).
//   18        looks for values past 65504 in a copied tile's factors before it is unpacked (by the
//             unpacking warps themselves it cost 80 cycles a tile).
//   19        clears rows of the output that no sequence asks for.
// Units (sequence, key head, row tile, token tile) are cut into equal runs, one per block; a job
// cut over blocks is joined by the last to arrive. Every wait is bounded.
//
// Within 8 dimensions, operands and accumulator hold the order 0 4 1 5 2 6 3 7: two nibbles of a
// word that one AND isolates are neighbours.
#pragma once
#include "kernels_lowbit_attend.cuh"
#include "umma.cuh"

namespace cora {

// Registers per thread: 640 x 96 at launch; then softmax 144, unpack 72, the last group 48
// (256 x 144 + 256 x 72 + 128 x 48 = 61440). Spilled variables would go to L2: shared
// memory leaves almost no L1.
constexpr int kCkThreads = 640, kCkMinRun = 2;
constexpr int kCkRegsSoftmax = 144, kCkRegsUnpack = 72, kCkRegsRest = 48;
static_assert(256 * kCkRegsSoftmax + 256 * kCkRegsUnpack + 128 * kCkRegsRest <= kCkThreads * 96, "");
constexpr float kCkShift = 7.0f;  // probabilities are 2^(score - m), m = maximum - kCkShift
template <int kRegs>
__device__ __forceinline__ void more_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void fewer_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

template <int D, int kNG, int kNQ>
struct ChunkSmem {
    static constexpr int kTN = 128 / kNG;             // tokens of a tile: 128 columns of scores
    // Score buffers per row tile. One row tile alone needs two (the next scores are formed while
    // softmax runs); two row tiles take turns with one each (64-token tiles with two buffers
    // each measured 788 against 730 us at 2048 queries, 16384 tokens: more issue per token).
    static constexpr int kBufs = kNQ == 1 ? 2 : 1;
    static constexpr uint32_t kQ = 128 * D * 2, kSlot = kTN * D * 2;
    static constexpr int kFit = (160 * 1024 - kNQ * kQ) / kSlot;
    static constexpr int kSlots = kFit < 3 ? 3 : kFit < 6 ? kFit : 6;  // unpacked tiles, keys and values in turn
    static constexpr int kRaw = 3;
    // Tables of key factors (and marks of bad values) in use at once: keys of tile t + m are
    // unpacked once the slot's last tile is free: with 6 slots keys of t + m - 3, multiplied after
    // the softmax of t + m - 5; with 4, t + m - 2 and t + m - 4; with 3, values of t + m - 2.
    static constexpr int kTables = kSlots > 4 ? 8 : 4;
    static constexpr uint32_t kCodes = kTN * D / 2, kMeta = kTN * kNG * 4;
    static constexpr uint32_t kRawBytes = 2 * kCodes + 2 * kMeta;
    static constexpr uint32_t q = 0;
    static constexpr uint32_t slot = q + kNQ * kQ;
    static constexpr uint32_t raw = slot + kSlots * kSlot;
    static constexpr uint32_t fac = raw + kRaw * kRawBytes;         // [kTables][kNG][kTN / 2] (two scales, two lows)
    static constexpr uint32_t poison = fac + kTables * 2 * kNG * kTN * 4;  // [kTables][4] bits: value is not finite
    static constexpr uint32_t misc = poison + kTables * 16;                   // tmem slot, last-to-arrive flags
    static constexpr uint32_t bars = misc + 32;
    static constexpr uint32_t kBarBytes = 320;
    static constexpr uint32_t walk = bars + kBarBytes;              // [warp] Walker
    // Marks of tiles whose values are under 2^-5. That of tile t is written once tile t - kRaw is
    // unpacked, its values' slot thus free of tile t - kRaw - 2 (t - kRaw - 3 with 6 slots or, by the
    // scores ahead, with 3), which softmax has then left: it reads marks from t - 5 on.
    static constexpr int kLarge = 8;
    static constexpr uint32_t large = walk + 19 * 160;              // [kLarge]
    static constexpr uint32_t base = large + kLarge * 4;            // int64[seqs + 1]
    static constexpr size_t bytes(uint32_t seqs) { return 1024 + base + 8 * (size_t)(seqs + 1); }
};

// One block's stretch of one job.
struct Segment {
    SeqWork s;
    int seq, head, row0, rows;       // rows: of this job's tiles (<= 128 kNQ)
    int tok0, tiles;                 // first token and tiles of the stretch
    int64_t u0, job_u0, job_u1;      // unit of its first tile; units of the whole job
    bool first, last;                // holds the job's first / last tile
};

// Walks the stretches of units [u, end); every role of a block sees the same ones. One per warp,
// in shared memory, moved by lane 0: its state would crowd out the registers of the tile loops.
template <int kTN, int kRows>
struct Walker {
    int64_t u, end;
    SeqWork s;
    int b;
    int more;   // whether g holds a stretch
    Segment g;
    // tokens that row tile rt's queries see: [lo, hi)
    __device__ static int2 sees(const AttendParams &p, const SeqWork &s, int rt) {
        const int heads = p.a.q_heads / p.c.kv_heads;
        const int i0 = rt * kRows / heads, i1 = min(s.n * heads, (rt + 1) * kRows) - 1;
        const int first = s.len - s.n + i0, last = s.len - s.n + i1 / heads;
        const int hi = p.a.causal ? max(0, min(s.len, last + 1)) : s.len;
        const int lo = p.a.window ? min(hi, max(0, first - (int)p.a.window + 1)) : 0;
        return make_int2(lo, hi);
    }
    __device__ static int tiles(int2 r) { return max(1, (r.y + kTN - 1) / kTN - r.x / kTN); }
    __device__ static int64_t units_of_head(const AttendParams &p, const SeqWork &s) {
        int64_t n = 0;
        for (int rt = 0; rt < s.row_tiles; ++rt) n += tiles(sees(p, s, rt));
        return n;
    }
    __device__ bool next(const AttendParams &p, const int64_t *base) {
        if (u >= end) return false;
        if (b < 0 || u >= base[b + 1]) {
            int lo = 0, hi = (int)p.seqs - 1;
            while (lo < hi) {
                const int mid = (lo + hi) / 2;
                if (base[mid + 1] > u) hi = mid;
                else lo = mid + 1;
            }
            b = lo;
            s = seq_work(p, b, kRows, kTN);
        }
        const int64_t per_head = (base[b + 1] - base[b]) / p.c.kv_heads, r = u - base[b];
        g.s = s;
        g.seq = p.seq0 + b;
        g.head = (int)(r / per_head);
        int64_t at = base[b] + g.head * per_head;
        int rt = 0;
        int2 see = sees(p, s, 0);
        while (at + tiles(see) <= u) {
            at += tiles(see);
            see = sees(p, s, ++rt);
        }
        g.row0 = rt * kRows;
        g.rows = min(kRows, s.n * (int)(p.a.q_heads / p.c.kv_heads) - g.row0);
        g.job_u0 = at;
        g.job_u1 = at + tiles(see);
        g.u0 = u;
        const int64_t stop = min(end, g.job_u1);
        g.tok0 = (see.x / kTN + (int)(u - at)) * kTN;
        g.tiles = (int)(stop - u);
        g.first = u == at;
        g.last = stop == g.job_u1;
        u = stop;
        return true;
    }
};

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)), "l"(reinterpret_cast<uint64_t &>(c)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<uint64_t &>(d))
        : "l"(reinterpret_cast<uint64_t &>(a)), "l"(reinterpret_cast<uint64_t &>(b)));
    return d;
}

template <typename T, int D, int kNG, int kNQ>
__global__ void __launch_bounds__(kCkThreads, 1) kv4_chunk_kernel(const AttendParams p) {
    using S = ChunkSmem<D, kNG, kNQ>;
    constexpr int kTN = S::kTN, kRows = 128 * kNQ, kG = D / kNG;
    constexpr uint32_t kQBlock = 128 * 128, kTBlock = kTN * 128;  // bytes of 64 dimensions of a tile
    constexpr uint32_t kOCol = 0, kSCol = kNQ * D;                // TMEM columns: O tiles, then S buffers
    constexpr uint32_t kSCols = kNG * kTN;                        // of one buffer: a block per group
    constexpr int kBufs = S::kBufs;
    static_assert(kNQ * (D + kBufs * kSCols) <= 512, "");
    extern __shared__ unsigned char ck_raw[];
    unsigned char *sm = reinterpret_cast<unsigned char *>((reinterpret_cast<uintptr_t>(ck_raw) + 1023) & ~uintptr_t(1023));
    float *fac = reinterpret_cast<float *>(sm + S::fac);
    volatile uint32_t *poison = reinterpret_cast<volatile uint32_t *>(sm + S::poison);
    volatile uint32_t *large = reinterpret_cast<volatile uint32_t *>(sm + S::large);
    volatile uint32_t *misc = reinterpret_cast<volatile uint32_t *>(sm + S::misc);
    uint64_t *bars = reinterpret_cast<uint64_t *>(sm + S::bars);
    uint64_t *raw_full = bars, *raw_empty = raw_full + S::kRaw;
    uint64_t *deq_full = raw_empty + S::kRaw, *deq_empty = deq_full + S::kSlots;
    uint64_t *q_full = deq_empty + S::kSlots, *o_free = q_full + 2;
    // (pv_done has a barrier per tile parity: a wait on one knows a phase by its parity alone, and
    // the softmax may be two second products ahead)
    uint64_t *s_full = o_free + 2, *p_full = s_full + 4, *pv_done = p_full + 4, *mma_done = pv_done + 4;
    uint64_t *looked = mma_done + 1, *joined = looked + S::kRaw;
    static_assert((3 * S::kRaw + 2 * S::kSlots + 19) * 8 <= S::kBarBytes, "");
    int64_t *base = reinterpret_cast<int64_t *>(sm + S::base);
    int *err = p.c.status;

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int H = p.c.kv_heads, heads = p.a.q_heads / H, P = p.c.page_size;
    using Walk = Walker<kTN, kRows>;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kRaw; ++i) mbar_init(raw_full + i, 1), mbar_init(raw_empty + i, 8), mbar_init(looked + i, 1);
        for (int i = 0; i < S::kSlots; ++i) mbar_init(deq_full + i, 8), mbar_init(deq_empty + i, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(q_full + i, 4), mbar_init(o_free + i, 4), mbar_init(joined + i, 4);  // (an arrival per warp)
        }
        for (int i = 0; i < 4; ++i) mbar_init(s_full + i, 1), mbar_init(p_full + i, 4), mbar_init(pv_done + i, 1);
        mbar_init(mma_done, 1);
        fence_barrier_init();
    }
    if (warp == 17) tmem_alloc(const_cast<uint32_t *>(misc), 512);
    if (warp == 0) {  // unit offsets of the sequences
        int64_t run = 0;
        if (lane == 0) base[0] = 0;
        for (int b0 = 0; b0 < (int)p.seqs; b0 += 32) {
            int64_t v = 0;
            if (b0 + lane < (int)p.seqs) v = Walk::units_of_head(p, seq_work(p, b0 + lane, kRows, kTN)) * H;
#pragma unroll
            for (int off = 1; off < 32; off <<= 1) {
                const int64_t o = __shfl_up_sync(0xffffffffu, v, off);
                if (lane >= off) v += o;
            }
            if (b0 + lane < (int)p.seqs) base[b0 + lane + 1] = run + v;
            run += __shfl_sync(0xffffffffu, v, 31);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = misc[0];
    const int64_t units = base[p.seqs], blocks = max((int64_t)1, min((int64_t)gridDim.x, units / kCkMinRun));
    static_assert(sizeof(Walk) <= 160, "");
    Walk &walk = *reinterpret_cast<Walk *>(sm + S::walk + (warp < 19 ? warp : 0) * 160);
    const Segment &g = walk.g;
    if (lane == 0 && warp < 19) {
        walk.u = blockIdx.x < blocks ? blockIdx.x * units / blocks : 0;
        walk.end = blockIdx.x < blocks ? (blockIdx.x + 1) * units / blocks : 0;
        walk.b = -1;
    }
    auto next = [&]() {  // by a whole warp
        __syncwarp();
        if (lane == 0) walk.more = walk.next(p, base);
        __syncwarp();
        return walk.more != 0;
    };

    if (warp < 4 * kNQ) {
        // ---------------- softmax: thread = row of tile q ----------------
        more_registers<kCkRegsSoftmax>();
        const int q = warp / 4, row = (warp % 4) * 32 + lane;
        const uint32_t lanes = tmem + (uint32_t((warp % 4) * 32) << 16);
        const uint32_t t_o = lanes + kOCol + q * D;
        unsigned char *sq = sm + S::q + q * S::kQ;
        const bool vec = reinterpret_cast<uintptr_t>(p.a.q) % 16 == 0 && p.a.q_token % 8 == 0 && p.a.q_head % 8 == 0;
        const float f0 = fabsf(p.a.scale) * kLog2e;
        const float sign = p.a.scale < 0.0f ? -1.0f : 1.0f;
        T *out = static_cast<T *>(p.a.out);
        uint32_t tile_no = 0;  // tiles this thread has done (phases of the barriers)
        bool ok = true;
        // The four warps of this row tile meet, twice for each part of a cut job (so that the phases
        // are known); false once one of them has given up (it does not come: the wait is bounded).
        auto meet = [&](uint32_t parity) {
            __syncwarp();
            if (lane == 0) mbar_arrive(joined + q);
            return __all_sync(0xffffffffu, mbar_wait_short(joined + q, parity, err)) != 0;
        };
        while (ok && next()) {
            const int r = q * 128 + row, grow = g.row0 + r;
            const bool in = r < g.rows;
            const int i = in ? grow / heads : 0, hh = g.head * heads + (in ? grow % heads : 0);
            const T *src = static_cast<const T *>(p.a.q) + (int64_t)(g.s.q0 + i) * p.a.q_token + (int64_t)hh * p.a.q_head;
            // the row under its own power of two, largest |q| in [2^13, 2^14); kBatch loads at once
            constexpr int kBatch = 8;
            auto load = [&](int d, uint4 (&w)[kBatch]) {
#pragma unroll
                for (int e = 0; e < kBatch; ++e) {
                    if (vec) {
                        w[e] = __ldg(reinterpret_cast<const uint4 *>(src + d + e * 8));
                    } else {
                        const uint16_t *h = reinterpret_cast<const uint16_t *>(src + d + e * 8);
                        w[e] = make_uint4(h[0] | uint32_t(h[1]) << 16, h[2] | uint32_t(h[3]) << 16, h[4] | uint32_t(h[5]) << 16,
                                          h[6] | uint32_t(h[7]) << 16);
                    }
                }
            };
            float big = 0.0f;
#pragma unroll 1
            for (int d = 0; d < (in ? D : 0); d += kBatch * 8) {
                uint4 w[kBatch];
                load(d, w);
#pragma unroll
                for (int e = 0; e < kBatch * 8; ++e) {
                    const float x = fabsf(to_f32(reinterpret_cast<const T *>(w)[e]));
                    big = x < 3.4e38f ? fmaxf(big, x) : big;
                }
            }
            const int qe = big > 0.0f ? max(-100, min(126, 13 - ilogbf(big))) : 0;
            const float qpow = in && f0 != 0.0f ? ldexpf(sign, qe) : 0.0f;
            float qs[kNG];  // sums of q per group, in the units of the products
#pragma unroll
            for (int gr = 0; gr < kNG; ++gr) {
                float sum = 0.0f;
#pragma unroll 1
                for (int d = gr * kG; d < (gr + 1) * kG; d += kBatch * 8) {
                    uint4 w[kBatch];
#pragma unroll
                    for (int e = 0; e < kBatch; ++e) w[e] = make_uint4(0, 0, 0, 0);
                    if (in) load(d, w);
#pragma unroll
                    for (int e = 0; e < kBatch; ++e) {
                        float x[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            x[k] = to_f32(reinterpret_cast<const T *>(&w[e])[k]) * qpow;
                            sum += x[k];
                        }
                        const float odd = 0.0625f;  // against the odd nibbles' 2^-20
                        uint4 o;
                        o.x = pack_half2(x[0], x[4]), o.y = pack_half2(x[1] * odd, x[5] * odd);
                        o.z = pack_half2(x[2], x[6]), o.w = pack_half2(x[3] * odd, x[7] * odd);
                        *reinterpret_cast<uint4 *>(sq + (d / 64) * kQBlock + row * 128 + ((e ^ (row & 7)) << 4)) = o;
                    }
                }
                qs[gr] = sum * 5.9604644775390625e-8f;  // 2^-24
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full + q);
            // From here a thread holds rows 8 k + lane / 4 of its warp, k = 0..3.
            float fr[4], qr[4][kNG], m[4], over[4];  // unit of the scores; sums of q; maximum - kCkShift, room above it
            int lo[4], hi[4];                        // tokens that the row sees
            float2 l2[4];                            // sum of p, over even and odd columns
            float unit = 1.0f;                       // of the sums of p v: 1, or 2^5 from a large tile on
            int hi_min = 0x7fffffff, lo_max = 0;
            {
                // scale 0: scores 0, whatever the products are
                const float f = f0 == 0.0f ? 1.0f : ldexpf(f0, 24 - qe);
                const int pos = g.s.len - g.s.n + i;
                const int h1 = !in ? 0x7fffffff : p.a.causal ? max(0, min(g.s.len, pos + 1)) : g.s.len;
                const int l1 = in && p.a.window ? max(0, pos - (int)p.a.window + 1) : 0;
                hi_min = __reduce_min_sync(0xffffffffu, h1), lo_max = __reduce_max_sync(0xffffffffu, l1);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int from = 8 * k + lane / 4;
                    fr[k] = __shfl_sync(0xffffffffu, f, from);
                    lo[k] = __shfl_sync(0xffffffffu, l1, from);
                    hi[k] = __shfl_sync(0xffffffffu, h1, from);
#pragma unroll
                    for (int gr = 0; gr < kNG; ++gr) qr[k][gr] = __shfl_sync(0xffffffffu, qs[gr], from);
                    m[k] = over[k] = -INFINITY;
                    l2[k] = make_float2(0.0f, 0.0f);
                }
            }
            // The sums of p v so far, times a factor for each of the thread's rows.
            auto rescale_o = [&](float k0, float k1, float k2, float k3) {
                if (!__all_sync(0xffffffffu, mbar_wait_short(pv_done + 2 * q + ((tile_no - 1) & 1), (tile_no - 1) >> 1 & 1, err)))
                    return false;
                tc_fence_after();
#pragma unroll 1
                for (int d = 0; d < D; d += 32) {
                    uint32_t x[16], y[16];
                    tmem_ld_frag(t_o + d, x);
                    tmem_ld_frag(t_o + d + (16u << 16), y);
                    tmem_wait_frag(x, y);
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        x[e] = __float_as_uint(__uint_as_float(x[e]) * (e & 2 ? k1 : k0));
                        y[e] = __float_as_uint(__uint_as_float(y[e]) * (e & 2 ? k3 : k2));
                    }
                    tmem_st_frag(t_o + d, x);
                    tmem_st_frag(t_o + d + (16u << 16), y);
                }
                return true;
            };
            for (int j = 0; j < g.tiles && ok; ++j, ++tile_no) {
                const int buf = q * kBufs + (int)(tile_no % kBufs);
                const uint32_t sph = tile_no / kBufs & 1;
                const uint32_t t_s = lanes + kSCol + buf * kSCols;
                const int tok0 = g.tok0 + j * kTN;
                const bool edge = tok0 + kTN > hi_min || tok0 < lo_max;
                ok = __all_sync(0xffffffffu, mbar_wait_short(s_full + buf, sph, err));
                if (!ok) break;
                tc_fence_after();
                const float4 *tf = reinterpret_cast<const float4 *>(fac + (tile_no % S::kTables) * 2 * kNG * kTN) + lane % 4;
#pragma unroll 1
                for (int c = 0; c < kTN / 32; ++c) {
                    // scores of 32 tokens x 32 rows: u[k][j] columns 8 j + 2 t, + 1 of row 8 k + g
                    float2 u[4][4];
#pragma unroll
                    for (int gr = 0; gr < kNG; ++gr) {
                        uint32_t x[16], y[16];
                        tmem_ld_frag(t_s + gr * kTN + c * 32, x);
                        tmem_ld_frag(t_s + gr * kTN + c * 32 + (16u << 16), y);
                        float4 ft[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) ft[j] = tf[gr * (kTN / 2) + c * 16 + j * 4];
                        tmem_wait_frag(x, y);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const uint32_t *v = k < 2 ? x : y;
                                const float2 d = make_float2(__uint_as_float(v[4 * j + (k & 1) * 2]), __uint_as_float(v[4 * j + (k & 1) * 2 + 1]));
                                const float2 q2 = make_float2(qr[k][gr], qr[k][gr]), low = make_float2(ft[j].z, ft[j].w);
                                u[k][j] = fma2(d, make_float2(ft[j].x, ft[j].y), gr ? fma2(low, q2, u[k][j]) : mul2(low, q2));
                            }
                    }
                    if (edge) {
                        const int t0 = tok0 + c * 32 + 2 * (lane % 4);
#pragma unroll
                        for (int k = 0; k < 4; ++k)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const int tk = t0 + 8 * j;
                                if (tk < lo[k] || tk >= hi[k]) u[k][j].x = -INFINITY;
                                if (tk + 1 < lo[k] || tk + 1 >= hi[k]) u[k][j].y = -INFINITY;
                            }
                    }
                    float tm[4];
                    bool grew = false;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        tm[k] = fmaxf(fmaxf(fmaxf(u[k][0].x, u[k][0].y), fmaxf(u[k][1].x, u[k][1].y)),
                                      fmaxf(fmaxf(u[k][2].x, u[k][2].y), fmaxf(u[k][3].x, u[k][3].y)));
                        grew |= tm[k] > over[k];
                    }
                    if (__any_sync(0xffffffffu, grew)) {
                        // rescale the rows' sums, this tile's earlier probabilities among them
                        float kf[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            tm[k] = fmaxf(tm[k], __shfl_xor_sync(0xffffffffu, tm[k], 1));
                            tm[k] = fmaxf(tm[k], __shfl_xor_sync(0xffffffffu, tm[k], 2));
                            kf[k] = 1.0f;
                            if (tm[k] > over[k]) {
                                const float to = tm[k] * fr[k];
                                kf[k] = ex2(m[k] + kCkShift - to);
                                m[k] = to - kCkShift;
                                over[k] = tm[k] + 8.0f / fr[k];
                                l2[k].x *= kf[k], l2[k].y *= kf[k];
                            }
                        }
                        tmem_wait_st();
#pragma unroll 1
                        for (int cc = 0; cc < c; ++cc) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                uint32_t w[8];
                                const uint32_t at = t_s + cc * 16 + (uint32_t(16 * h) << 16);
                                tmem_ld_frag16(at, w);
#pragma unroll
                                for (int e = 0; e < 8; ++e) {
                                    const float2 v = __half22float2(*reinterpret_cast<__half2 *>(&w[e]));
                                    w[e] = pack_half2(v.x * kf[2 * h + (e & 1)], v.y * kf[2 * h + (e & 1)]);
                                }
                                tmem_st_frag16(at, w);
                            }
                        }
                        if (j > 0) {
                            ok = rescale_o(kf[0], kf[1], kf[2], kf[3]);
                            if (!ok) break;
                        }
                        tmem_wait_st();
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t w[8];
#pragma unroll
                        for (int kk = 0; kk < 2; ++kk) {
                            const int k = 2 * h + kk;
                            const float mr = m[k] == -INFINITY ? 0.0f : -m[k];
#pragma unroll
                            for (int jj = 0; jj < 4; ++jj) {
                                float2 pr = fma2(u[k][jj], make_float2(fr[k], fr[k]), make_float2(mr, mr));
                                pr.x = ex2(pr.x), pr.y = ex2(pr.y);
                                l2[k] = add2(l2[k], pr);
                                w[2 * jj + kk] = pack_half2(pr.x, pr.y);
                            }
                        }
                        tmem_st_frag16(t_s + c * 16 + (uint32_t(16 * h) << 16), w);
                    }
                }
                if (!ok) break;
                // values that are not finite are kept out of the product: rows that see one say so here;
                // from the first large tile on the sums are under 2^-5
                {
                    const volatile uint32_t *bits = poison + 4 * (tile_no % S::kTables);
                    uint32_t any = large[tile_no % S::kLarge];
#pragma unroll
                    for (int c = 0; c < kTN / 32; ++c) any |= bits[c];
                    if (any) {
                        if (large[tile_no % S::kLarge] && unit == 1.0f) {
                            unit = 32.0f;
                            if (j > 0) ok = rescale_o(0.03125f, 0.03125f, 0.03125f, 0.03125f);
                            if (!ok) break;
                        }
                        for (int e = 0; e < kTN; ++e)
                            if (bits[e / 32] >> (e % 32) & 1) {
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    if (tok0 + e >= lo[k] && tok0 + e < hi[k]) l2[k].x = __int_as_float(0x7fc00000);
                            }
                    }
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + buf);
            }
            if (!ok) break;
            // ---- the stretch is done: result, or this block's part of it ----
            ok = __all_sync(0xffffffffu, mbar_wait_short(pv_done + 2 * q + ((tile_no - 1) & 1), (tile_no - 1) >> 1 & 1, err));
            if (!ok) break;
            tc_fence_after();
            float mrow = 0.0f, l = 0.0f;  // a thread per row again
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float sum = l2[k].x + l2[k].y;
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                const float a = __shfl_sync(0xffffffffu, m[k], (lane & 7) * 4), b = __shfl_sync(0xffffffffu, sum, (lane & 7) * 4);
                if (lane / 8 == k) mrow = a, l = b;
            }
            const bool whole = g.first && g.last;
            T *dst = out + ((int64_t)(g.s.q0 + i) * p.a.q_heads + hh) * D;
            const size_t slots = (size_t)2 * gridDim.x * kNQ;
            const size_t sl = (size_t)(2 * blockIdx.x + (g.first ? 1 : 0)) * kNQ + q;
            float *po = p.part + sl * D * 128 + row;
            float2 *ps = reinterpret_cast<float2 *>(p.part + slots * D * 128) + sl * 128 + row;
            const float inv = l == 0.0f ? 0.0f : unit / l;
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t x[32];
                tmem_ld32_async(t_o + c, x);
                tmem_wait_ld(x);
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) __stcg(po + (c + e) * 128, __uint_as_float(x[e]) * unit);
                } else if (in) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        float v[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[(k >> 1) + (k & 1) * 4] = l == 0.0f ? 0.0f : __uint_as_float(x[e + k]) * inv;
                        store8(dst + c + e, v);
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(o_free + q);
            if (whole) {
                if (in && p.a.lse)
                    p.a.lse[(int64_t)(g.s.q0 + i) * p.a.q_heads + hh] = l == 0.0f ? -INFINITY : (mrow + log2f(l)) / kLog2e;
                continue;
            }
            __stcg(ps, make_float2(mrow, l));
            __threadfence();
            if (!meet(0)) break;
            const int first = (int)(((g.job_u0 + 1) * blocks - 1) / units), last = (int)((g.job_u1 * blocks - 1) / units);
            uint32_t *count = p.arrived + first * kNQ + q;
            if (row == 0) misc[1 + q] = atomicAdd(count, 1u) == (uint32_t)(last - first);
            if (!meet(1)) break;
            if (misc[1 + q]) {
                __threadfence();
                if (row == 0) *count = 0;
                const float2 *as = reinterpret_cast<const float2 *>(p.part + slots * D * 128) + row;
                auto at = [&](int bk) { return (size_t)(2 * bk + (bk == first ? 1 : 0)) * kNQ + q; };
                float jm = -INFINITY, jl = 0.0f;
                for (int bk = first; bk <= last; ++bk) jm = fmaxf(jm, __ldcg(as + at(bk) * 128).x);
                for (int bk = first; bk <= last; ++bk) {
                    const float2 st = __ldcg(as + at(bk) * 128);
                    jl += st.y * (st.x == -INFINITY ? (st.y == 0.0f ? 0.0f : 1.0f) : ex2(st.x - jm));
                }
                const float jinv = jl == 0.0f ? 0.0f : 1.0f / jl;
#pragma unroll 1
                for (int c = 0; c < D; c += 8) {
                    float v[8] = {};
                    for (int bk = first; bk <= last; ++bk) {
                        const float sm_ = __ldcg(as + at(bk) * 128).x;
                        const float k = sm_ == -INFINITY ? 0.0f : ex2(sm_ - jm);
                        const float *src2 = p.part + at(bk) * D * 128 + (size_t)c * 128 + row;
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[(e >> 1) + (e & 1) * 4] = fmaf(k, __ldcg(src2 + e * 128), v[(e >> 1) + (e & 1) * 4]);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = jl == 0.0f ? 0.0f : v[e] * jinv;
                    if (in) store8(dst + c, v);
                }
                if (in && p.a.lse)
                    p.a.lse[(int64_t)(g.s.q0 + i) * p.a.q_heads + hh] = jl == 0.0f ? -INFINITY : (jm + log2f(jl)) / kLog2e;
            }
            // (misc is written again after the next part's first meeting, when all have read it)
        }
    } else if (warp >= 8 && warp < 16) {
        // ---------------- unpack ----------------
        fewer_registers<kCkRegsUnpack>();
        const int tid = threadIdx.x - 256, t3 = lane & 7, quarter0 = lane >> 3;
        const int rot = D == 128 ? t3 >> 1 : D == 256 ? t3 : 0;  // 16-byte reads and writes of 8 lanes hit all banks
        constexpr int kQuads = D / 32;                            // 16-byte pieces of a token's codes
        uint32_t raw_no = 0, item = 0;
        bool ok = true;
        while (ok && next()) {
            int see_lo = 0x7fffffff, see_hi = 0;  // tokens that any row of this job sees
            {
                const int2 see = Walk::sees(p, g.s, g.row0 / kRows);
                see_lo = see.x, see_hi = see.y;
            }
            for (int j = 0; j < g.tiles && ok; ++j, ++raw_no) {
                const int rs = raw_no % S::kRaw, tok0 = g.tok0 + j * kTN;
                const unsigned char *rw = sm + S::raw + rs * S::kRawBytes;
                ok = mbar_wait_short(looked + rs, (raw_no / S::kRaw) & 1, err);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                // Value codes become k c (and lows k low), k = 1 or 2^-5: fma(1024 + c, k, -1024 k) and,
                // from the odd nibbles, fma(1024 + 16 c, k / 16, -64 k), exact.
                const bool big = large[raw_no % S::kLarge] != 0;
                const __half2 k1 = __half2half2(__ushort_as_half(big ? 0x2800 : 0x3c00));
                const __half2 k1024 = __half2half2(__ushort_as_half(big ? 0xd000 : 0xe400));
                const __half2 k16 = __half2half2(__ushort_as_half(big ? 0x1800 : 0x2c00));
                const __half2 k64 = __half2half2(__ushort_as_half(big ? 0xc000 : 0xd400));
#pragma unroll
                for (int kv = 0; kv < 2; ++kv, ++item) {
                    const int sl = item % S::kSlots;
                    ok = mbar_wait_short(deq_empty + sl, ((item / S::kSlots) & 1) ^ 1, err);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    unsigned char *dst = sm + S::slot + sl * S::kSlot;
                    const unsigned char *codes = rw + kv * S::kCodes;
                    const __half2 *meta = reinterpret_cast<const __half2 *>(rw + 2 * S::kCodes + kv * S::kMeta);
                    if (kv == 0 && tid < kTN) {  // the keys' factors; which values are not finite
                        const __half2 *vm = reinterpret_cast<const __half2 *>(rw + 2 * S::kCodes + S::kMeta);
                        float *tf = fac + (raw_no % S::kTables) * 2 * kNG * kTN;
                        const int tok = tok0 + tid;
                        const bool seen = tok >= see_lo && tok < see_hi;
                        bool bad = false;
#pragma unroll
                        for (int gr = 0; gr < kNG; ++gr) {
                            const float2 kf = __half22float2(meta[tid * kNG + gr]);
                            float *at = tf + (gr * (kTN / 2) + tid / 2) * 4 + (tid & 1);
                            at[0] = seen ? kf.x : 0.0f;
                            at[2] = seen ? kf.y : 0.0f;
                            const uint32_t u = *reinterpret_cast<const uint32_t *>(vm + tid * kNG + gr);
                            bad |= (u & 0x7c00u) == 0x7c00u || (u & 0x7c000000u) == 0x7c000000u;
                        }
                        const uint32_t bits = __ballot_sync(0xffffffffu, bad && seen);
                        if (lane == 0) poison[4 * (raw_no % S::kTables) + tid / 32] = bits;
                    }
#pragma unroll
                    for (int it = 0; it < (kTN * kQuads + 255) / 256; ++it) {
                        // 8 tokens x 4 pieces per warp and step
                        const int step = it * 8 + (warp - 8);
                        if (kTN * kQuads % 256 && step >= kTN * kQuads / 32) break;
                        constexpr int kParts = kQuads > 4 ? kQuads / 4 : 1;
                        const int tg8 = step / kParts, part = step % kParts;
                        int tk, quad;
                        if (kQuads == 2) {  // 16 tokens x 2 pieces
                            tk = step * 16 + (quarter0 >> 1) * 8 + t3;
                            quad = quarter0 & 1;
                        } else {
                            tk = tg8 * 8 + t3;
                            quad = (part * 4 + quarter0 + rot) & (kQuads - 1);
                        }
                        const uint4 w4 = *reinterpret_cast<const uint4 *>(codes + tk * (D / 2) + quad * 16);
                        const uint32_t ws[4] = {w4.x, w4.y, w4.z, w4.w};
                        __half2 sc, lw;
                        if (kv) {
                            const int tok = tok0 + tk;
                            __half2 f = meta[tk * kNG + quad * 32 / kG];
                            const uint32_t fu = *reinterpret_cast<const uint32_t *>(&f);
                            const bool bad = (fu & 0x7c00u) == 0x7c00u || (fu & 0x7c000000u) == 0x7c000000u;
                            // unseen tokens count as 0, and so do values that are marked above
                            if (tok < see_lo || tok >= see_hi || bad) f = __halves2half2(__ushort_as_half(0), __ushort_as_half(0));
                            sc = __low2half2(f), lw = __hmul2(__high2half2(f), k1);
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t w = ws[k], w8 = w >> 8;
                            uint32_t o[4] = {w & 0x000f000fu, w & 0x00f000f0u, w8 & 0x000f000fu, w8 & 0x00f000f0u};
                            if (kv) {
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    o[e] |= 0x64006400u;  // 1024 + c or 1024 + 16 c
                                    __half2 v = *reinterpret_cast<__half2 *>(&o[e]);
                                    v = e & 1 ? __hfma2(v, k16, k64) : __hfma2(v, k1, k1024);
                                    v = __hfma2(v, sc, lw);
                                    o[e] = *reinterpret_cast<uint32_t *>(&v);
                                }
                            }
                            const int chunk = quad * 4 + k, c = chunk & 7;
                            *reinterpret_cast<uint4 *>(dst + (chunk >> 3) * kTBlock + tk * 128 + ((c ^ (tk & 7)) << 4)) =
                                make_uint4(o[0], o[1], o[2], o[3]);
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(deq_full + sl);
                        if (kv) mbar_arrive(raw_empty + rs);
                    }
                }
            }
        }
    } else if (warp < 16) {
        fewer_registers<kCkRegsRest>();  // (no second row tile)
    } else {
        fewer_registers<kCkRegsRest>();
        if (warp == 16) {
        // ---------------- copies from the pages ----------------
        const Kv4Block blk(P, D, kG);
        const int per = min(P, kTN), piece = lane >> 2, kind = lane & 3;
        const uint32_t rowb = kind < 2 ? blk.code_row : blk.meta_row;
        const uint32_t src_at = (kind & 1 ? (kind < 2 ? blk.codes : blk.metas) : 0) + (kind < 2 ? 0 : 2 * blk.codes);
        const uint32_t dst_at = (kind & 1 ? (kind < 2 ? S::kCodes : S::kMeta) : 0) + (kind < 2 ? 0 : 2 * S::kCodes);
        uint32_t raw_no = 0;
        bool ok = true;
        while (ok && next()) {
            for (int j = 0; j < g.tiles; ++j, ++raw_no) {
                const int rs = raw_no % S::kRaw, tok0 = g.tok0 + j * kTN;
                ok = __all_sync(0xffffffffu, mbar_wait_short(raw_empty + rs, ((raw_no / S::kRaw) & 1) ^ 1, err));
                if (!ok) break;
                const int pieces = max(0, min(kTN / per, (g.s.len - tok0 + per - 1) / per));
                uint32_t bytes = 0;
                const unsigned char *src = nullptr;
                if (piece < pieces) {
                    const int tok = tok0 + piece * per;
                    const int page = __ldg(p.a.page_table + (int64_t)g.seq * p.a.table_stride + tok / P);
                    if (page >= 0 && (uint64_t)page < p.c.num_pages) {
                        src = p.c.pool + ((uint64_t)page * H + g.head) * blk.bytes + src_at + (uint32_t)(tok % P) * rowb;
                        bytes = per * rowb;
                    } else {
                        atomicOr(err, kDevBadInput);
                    }
                }
                const uint32_t total = __reduce_add_sync(0xffffffffu, bytes);
                if (lane == 0) mbar_arrive_expect_tx(raw_full + rs, total);
                __syncwarp();
                if (bytes) bulk_g2s(sm + S::raw + rs * S::kRawBytes + dst_at + piece * per * rowb, src, bytes, raw_full + rs);
            }
        }
        // the last copy into each stage has landed before the block exits
        for (uint32_t k = raw_no > S::kRaw ? raw_no - S::kRaw : 0; k < raw_no; ++k)
            mbar_wait_short(raw_full + k % S::kRaw, (k / S::kRaw) & 1, err);
        } else if (warp == 18) {
        // ---------------- values past 65504 ----------------
        uint32_t raw_no = 0;
        bool ok = true;
        while (ok && next()) {
            const int2 see = Walk::sees(p, g.s, g.row0 / kRows);
            bool big = false;  // from the first such tile of a stretch on
            for (int j = 0; j < g.tiles; ++j, ++raw_no) {
                const int rs = raw_no % S::kRaw, tok0 = g.tok0 + j * kTN;
                ok = __all_sync(0xffffffffu, mbar_wait_short(raw_full + rs, (raw_no / S::kRaw) & 1, err));
                if (!ok) break;
                const uint4 f4 = reinterpret_cast<const uint4 *>(sm + S::raw + rs * S::kRawBytes + 2 * S::kCodes + S::kMeta)[lane];
                const uint32_t f[4] = {f4.x, f4.y, f4.z, f4.w};
                bool past = false;  // some row sees it, its factors are finite, its largest value rounds to infinity
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&f[e]));
                    const int tok = tok0 + (lane * 4 + e) / kNG;
                    past |= tok >= see.x && tok < see.y && fabsf(v.x) <= 65504.0f && fabsf(v.y) <= 65504.0f &&
                            fabsf(fmaf(15.0f, v.x, v.y)) >= 65520.0f;
                }
                big |= __any_sync(0xffffffffu, past) != 0;
                if (lane == 0) {
                    large[raw_no % S::kLarge] = big;
                    mbar_arrive(looked + rs);
                }
            }
        }
        } else if (warp == 19) {
        // ---------------- rows that no sequence asks for ----------------
        const SeqWork head = seq_work(p, 0, kRows, kTN), tail = seq_work(p, (int)p.seqs - 1, kRows, kTN);
        clear_gaps(p, head.q0, (int64_t)tail.q0 + tail.n, blockIdx.x * 32 + lane, gridDim.x * 32);
        } else if (warp == 17) {
        // ---------------- products ----------------
        constexpr uint32_t id_qk = idesc_f16(128, kTN, false), id_pv = idesc_f16(128, D, true);
        uint32_t seg_no = 0, done = 0;  // stretches and tiles before this one
        bool ok = true;
        const uint32_t leader = elect_one();
        const uint32_t sm0 = __shfl_sync(0xffffffffu, smem_u32(sm), 0), tm0 = __shfl_sync(0xffffffffu, tmem, 0);
        auto slot_wait = [&](uint32_t item) {
            const bool w = mbar_wait_short(deq_full + item % S::kSlots, (item / S::kSlots) & 1, err);
            tc_fence_after();
            return w;
        };
        auto buffer = [&](int q, uint32_t tile) { return q * kBufs + (int)(tile % kBufs); };
        auto qk = [&](int q, uint32_t tile) {  // scores of row tile q against key tile `tile`
            const uint32_t kt = sm0 + S::slot + (2 * tile) % S::kSlots * S::kSlot;
            const uint32_t a0 = desc_low(sm0 + S::q + q * S::kQ), b0 = desc_low(kt);
            const uint32_t d = tm0 + kSCol + buffer(q, tile) * kSCols;
#pragma unroll
            for (int k = 0; k < D / 16; ++k) {
                const int gr = k / (kG / 16);
                mma_f16(leader, d + gr * kTN, a0 + (k / 4) * (kQBlock >> 4) + (k % 4) * 2, b0 + (k / 4) * (kTBlock >> 4) + (k % 4) * 2,
                        id_qk, k % (kG / 16) != 0);
            }
            mma_commit_by(leader, s_full + buffer(q, tile));
            if (q == kNQ - 1) mma_commit_by(leader, deq_empty + (2 * tile) % S::kSlots);
        };
        auto pv = [&](int q, uint32_t tile, bool add) {
            const uint32_t vt = sm0 + S::slot + (2 * tile + 1) % S::kSlots * S::kSlot;
            const uint32_t b0 = desc_low(vt, kTBlock);
            const uint32_t a = tm0 + kSCol + buffer(q, tile) * kSCols;
#pragma unroll
            for (int k = 0; k < kTN / 16; ++k) mma_f16_ta(leader, tm0 + kOCol + q * D, a + k * 8, b0 + k * (2048 >> 4), id_pv, add || k != 0);
            mma_commit_by(leader, pv_done + 2 * q + (tile & 1));
            if (q == kNQ - 1) mma_commit_by(leader, deq_empty + (2 * tile + 1) % S::kSlots);
        };
        while (ok && next()) {
            const int tiles = __shfl_sync(0xffffffffu, g.tiles, 0);
            for (int q = 0; q < kNQ && ok; ++q) ok = mbar_wait_short(q_full + q, seg_no & 1, err);
            tc_fence_after();
            constexpr int kAhead = kBufs;  // score tiles issued ahead of the second product
            for (int a = 0; a < min(kAhead, tiles) && ok; ++a) {
                ok = slot_wait(2 * (done + a));
                for (int q = 0; q < kNQ && ok; ++q) qk(q, done + a);
            }
            for (int j = 0; j < tiles && ok; ++j) {
                const uint32_t tile = done + j;
                for (int q = 0; q < kNQ && ok; ++q) {
                    if (q == 0) ok = slot_wait(2 * tile + 1);
                    if (j == 0 && ok) ok = mbar_wait_short(o_free + q, (seg_no & 1) ^ 1, err);
                    if (ok) ok = mbar_wait_short(p_full + buffer(q, tile), tile / kBufs & 1, err);
                    if (!ok) break;
                    tc_fence_after();
                    pv(q, tile, j > 0);
                    if (j + kAhead < tiles) {
                        if (q == 0) ok = slot_wait(2 * (tile + kAhead));
                        if (ok) qk(q, tile + kAhead);
                    }
                }
            }
            done += tiles;
            ++seg_no;
        }
        mma_commit_by(leader, mma_done);  // every product has finished before TMEM is freed
        mbar_wait_short(mma_done, 0, err);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 17) tmem_dealloc(tmem, 512);
}

}  // namespace cora
