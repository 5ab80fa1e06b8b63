// Host side of the 4-bit reader operators: argument checks, choice of kernel variant, launches.
#include <climits>
#include <cstdint>

#include "kernels_lowbit_append.cuh"
#include "kernels_lowbit_attend.cuh"
#include "kernels_lowbit_chunk.cuh"
#include "kernels_lowbit_matvec.cuh"
#include "status.hpp"

namespace cora {
namespace {

constexpr uint64_t kMaxGrid = 65535;

bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
void need(bool ok, const char *what) {
    if (!ok) fail(CORA_EINVAL, what);
}

// Multiprocessors of the current device.
int sm_count() {
    static thread_local int dev_seen = -1, sms = 0;
    int dev = 0;
    CUDA_TRY(cudaGetDevice(&dev));
    if (dev != dev_seen) {
        CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
        dev_seen = dev;
    }
    return sms;
}

void check_cache(const cora_kv4_cache *c) {
    need(c, "null cache");
    need(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, "head_dim must be 64, 128 or 256");
    need((c->group == 64 || c->group == 128) && c->group <= c->head_dim && c->group * 4 >= c->head_dim,
         "group must be 64 or 128 and at most head_dim");
    need(c->page_size >= 16 && c->page_size <= 1024 && (c->page_size & (c->page_size - 1)) == 0,
         "page_size must be a power of two from 16 to 1024");
    need(c->kv_heads >= 1 && c->kv_heads <= 65535, "kv_heads must be in [1, 65535]");
    need(c->pool && aligned16(c->pool), "the pool must be 16-byte aligned device memory");
    need(c->num_pages <= INT_MAX, "num_pages must fit an int");
    need(c->status, "null status word");
}

template <typename F>
void by_dtype(uint32_t dtype, F &&f) {
    if (dtype == CORA_BF16) return f(__nv_bfloat16{});
    if (dtype == CORA_FP16) return f(__half{});
    fail(CORA_EINVAL, "dtype must be CORA_BF16 or CORA_FP16");
}
template <int N>
using Int = std::integral_constant<int, N>;

// Takes back the bits that were reported, and only those: calls on other streams may set more.
__global__ void clear_bits_kernel(int32_t *status, int32_t bits) { atomicAnd(status, ~bits); }

// Raises a kernel's dynamic shared memory limit, once per device and kernel.
template <typename K>
void allow_smem(K kernel, size_t bytes, int (&seen)[64]) {
    int dev = 0;
    CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 64 && seen[dev] >= (int)bytes) return;
    CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    if (dev < 64) seen[dev] = (int)bytes;
}

// ---- append ------------------------------------------------------------------------------

template <typename T, int D, bool kOne, bool kVec>
void launch_append(const cora_kv4_cache &c, const cora_kv4_append_args &a, cudaStream_t st) {
    const uint64_t per = kAppendThreads / (D / 16), bx = (a.tokens + per - 1) / per;
    const uint64_t heads = 2ull * c.kv_heads + (a.q ? a.q_heads : 0);
    // Few tokens: one head per thread, for latency. Many: runs of heads share one read of the
    // rotation's factors, as long as 16 blocks per SM remain to hide the loads.
    const uint64_t want = 16ull * sm_count();
    uint64_t run = bx * heads <= want ? 1 : std::min(heads, bx * heads / want);
    while ((heads + run - 1) / run > kMaxGrid) ++run;
    need(bx <= INT_MAX, "too many tokens");
    const int turn = !a.rotary ? kTurnNone : a.interleaved ? kTurnInterleaved : a.rotary == D ? kTurnFull : kTurnPart;
    kv4_append_kernel<T, D, kOne, kVec><<<dim3((unsigned)bx, (unsigned)((heads + run - 1) / run)), kAppendThreads, 0, st>>>(
        c, a, (int)run, turn);
    CUDA_TRY(cudaGetLastError());
}

void append(const cora_kv4_cache *c, const cora_kv4_append_args *a, cudaStream_t st) {
    check_cache(c);
    need(a, "null arguments");
    if (a->tokens == 0) return;
    need(a->k && a->v && a->slots, "k, v and slots are needed");
    need(!a->q || (a->q_out && a->q_heads >= 1 && a->q_heads <= 65535), "q needs q_out and q_heads in [1, 65535]");
    need(a->rotary % 16 == 0 && a->rotary <= c->head_dim, "rotary must be a multiple of 16, at most head_dim");
    need(!a->rotary || (a->rope_cos && a->rope_sin && a->positions && a->rope_rows), "rotation needs cos, sin and positions");
    need(aligned16(a->rope_cos) && aligned16(a->rope_sin), "cos and sin must be 16-byte aligned");
    need(aligned16(a->k_out) && aligned16(a->v_out) && aligned16(a->q_out), "outputs must be 16-byte aligned");
    const bool vec = aligned16(a->k) && aligned16(a->v) && aligned16(a->q) && a->k_token % 8 == 0 && a->k_head % 8 == 0 &&
                     a->v_token % 8 == 0 && a->v_head % 8 == 0 && (!a->q || (a->q_token % 8 == 0 && a->q_head % 8 == 0));
    by_dtype(a->dtype, [&](auto z) {
        using T = decltype(z);
        auto go = [&](auto d) {
            constexpr int D = decltype(d)::value;
            const bool one = c->group == c->head_dim;
            if (vec) one ? launch_append<T, D, true, true>(*c, *a, st) : launch_append<T, D, false, true>(*c, *a, st);
            else one ? launch_append<T, D, true, false>(*c, *a, st) : launch_append<T, D, false, false>(*c, *a, st);
        };
        if (c->head_dim == 64) go(Int<64>{});
        else if (c->head_dim == 128) go(Int<128>{});
        else go(Int<256>{});
    });
}

// ---- attend ------------------------------------------------------------------------------

// Rows of one key head and sequence. Up to 32 the streaming kernel takes tiles of 8, reading the
// cache again for each (from L2); more go to the tile kernel. Both measured, 16 sequences of 4096
// tokens, 8 key heads, in us at 8 / 16 / 32 / 40 / 48 / 64 rows: head size 64, streaming 29 / 41 / 65 /
// 76 / 87 / 111, tiles 92 throughout; head size 128, 35 / 50 / 80 / 95 / 109 / 139 against 107 to 109;
// head size 256, 55 / 84 / 144 / 175 / 205 / 264 against 172 to 177.
uint64_t attend_rows(const cora_kv4_cache &c, uint64_t q_heads, uint64_t max_queries) {
    return std::max<uint64_t>(1, max_queries) * (q_heads / c.kv_heads);
}
constexpr uint64_t kFewRows = 32;
uint64_t attend_counters() { return ((uint64_t)sm_count() * 2 * 4 + 255) / 256 * 256; }
// Workspace: the arrival counters first (they are the part that has to start at zero), then two
// partial results per block.
uint64_t attend_workspace(const cora_kv4_cache &c, uint64_t rows) {
    const uint64_t blocks = sm_count();
    // few rows: two parts of 8 rows per block and one per warp
    const uint64_t parts = rows <= kFewRows ? blocks * (2 + kAtWarps) * kAtRows
                                            : 2 * blocks * (rows <= 128 || c.head_dim == 256 ? 128 : 256);
    return attend_counters() + parts * (c.head_dim + 2) * 4;
}

template <typename T, int D, int kNG>
void launch_attend(AttendParams p, cudaStream_t st) {
    auto *kern = kv4_attend_kernel<T, D, kNG>;
    using S = AttendSmem<D, kNG>;
    static_assert(S::bytes(kAtMaxSeqs) <= 232448, "");
    static int seen[64] = {};
    allow_smem(kern, S::bytes(kAtMaxSeqs), seen);
    const uint32_t seqs = p.a.seqs;
    for (uint32_t s0 = 0; s0 < seqs; s0 += kAtMaxSeqs) {
        p.seq0 = s0;
        p.seqs = std::min<uint32_t>(kAtMaxSeqs, seqs - s0);
        kern<<<sm_count(), kAtWarps * 32, S::bytes(p.seqs), st>>>(p);
        CUDA_TRY(cudaGetLastError());
    }
}

template <typename T, int D, int kNG, int kNQ>
void launch_chunk(AttendParams p, cudaStream_t st) {
    auto *kern = kv4_chunk_kernel<T, D, kNG, kNQ>;
    using S = ChunkSmem<D, kNG, kNQ>;
    static_assert(S::bytes(kAtMaxSeqs) <= 232448, "");
    static int seen[64] = {};
    static const int regs = [&] {
        cudaFuncAttributes at{};
        CUDA_TRY(cudaFuncGetAttributes(&at, kern));
        return at.numRegs;
    }();
    // The roles' shares are drawn from what the block is launched with; with less they would wait.
    if (regs < 96) fail(CORA_ERUNTIME, "kv4_chunk_kernel was compiled to fewer registers than its roles share");
    allow_smem(kern, S::bytes(kAtMaxSeqs), seen);
    const uint32_t seqs = p.a.seqs;
    for (uint32_t s0 = 0; s0 < seqs; s0 += kAtMaxSeqs) {
        p.seq0 = s0;
        p.seqs = std::min<uint32_t>(kAtMaxSeqs, seqs - s0);
        kern<<<sm_count(), kCkThreads, S::bytes(p.seqs), st>>>(p);
        CUDA_TRY(cudaGetLastError());
    }
}

void attend(const cora_kv4_cache *c, const cora_kv4_attend_args *a, cudaStream_t st) {
    check_cache(c);
    need(a, "null arguments");
    if (a->q_tokens == 0) return;
    need(a->q && a->out && (!a->seqs || (a->page_table && a->lens)), "q, out, page_table and lens are needed");
    need(aligned16(a->out), "out must be 16-byte aligned");
    need(a->q_heads >= 1 && a->q_heads % c->kv_heads == 0, "q_heads must be a multiple of kv_heads");
    need(a->q_tokens <= INT_MAX && a->seqs <= INT_MAX, "too many rows");
    need(a->q_start || a->q_tokens >= a->seqs, "q needs a row per sequence where q_start is null");
    // Positions, from -q_tokens to the table's last token, and up to 32 pages read ahead are ints in the
    // kernels.
    const uint64_t room = (uint64_t)a->table_width * c->page_size;
    need(room + 32ull * c->page_size + a->q_tokens <= INT_MAX, "table_width * page_size must fit an int, with q_tokens and 32 pages");
    need(!a->window || a->causal, "a window needs causal attention");
    need(a->window <= INT_MAX, "window must fit an int");
    AttendParams p{};
    p.c = *c;
    p.a = *a;
    p.q_tokens = (int64_t)a->q_tokens;
    if (!a->seqs) {
        by_dtype(a->dtype, [](auto) {});
        kv4_clear_kernel<<<sm_count(), 256, 0, st>>>(p);
        CUDA_TRY(cudaGetLastError());
        return;
    }
    const uint64_t rows = attend_rows(*c, a->q_heads, a->max_queries);
    need(a->workspace && aligned16(a->workspace) && a->workspace_bytes >= attend_workspace(*c, rows),
         "the workspace is smaller than cora_kv4_attend_workspace()");
    // units (token tiles x row tiles x key heads) of a sequence are counted in 32 bits
    const double tiles = (double)a->table_width * c->page_size / 32 + 2;
    const double row_tiles = (double)a->q_tokens * (a->q_heads / c->kv_heads) / kAtRows + 1;
    need(tiles * row_tiles * c->kv_heads < 4.0e9, "too much work for one call: split the queries");
    // A captured call readies its counters itself: whoever ran before a replay of the graph, and
    // whether the memory was ever zeroed outside it, is not known here.
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    CUDA_TRY(cudaStreamIsCapturing(st, &capture));
    if (capture != cudaStreamCaptureStatusNone) CUDA_TRY(cudaMemsetAsync(a->workspace, 0, attend_counters(), st));
    // No sequence is longer than its table: a wider window hides nothing, and position - window would
    // wrap for the queries of a sequence that has more of them than cached tokens.
    if (a->window >= room) p.a.window = 0;
    p.arrived = static_cast<uint32_t *>(a->workspace);
    p.part = reinterpret_cast<float *>(static_cast<char *>(a->workspace) + attend_counters());
    by_dtype(a->dtype, [&](auto z) {
        using T = decltype(z);
        auto go = [&](auto d, auto ng) {
            constexpr int D = decltype(d)::value, NG = decltype(ng)::value;
            if (rows <= kFewRows) launch_attend<T, D, NG>(p, st);
            else if (rows <= 128 || D == 256) launch_chunk<T, D, NG, 1>(p, st);
            else launch_chunk<T, D, NG, D == 256 ? 1 : 2>(p, st);
        };
        if (c->head_dim == 64) go(Int<64>{}, Int<1>{});
        else if (c->head_dim == 128 && c->group == 128) go(Int<128>{}, Int<1>{});
        else if (c->head_dim == 128) go(Int<128>{}, Int<2>{});
        else if (c->group == 128) go(Int<256>{}, Int<2>{});
        else go(Int<256>{}, Int<4>{});
    });
}

// ---- matvec ------------------------------------------------------------------------------

// 32 weight rows per warp halve what is done once per activation (its loads, its sums); 16 give
// twice the blocks, which matrices with fewer rows than fill the SMs twice need more. One bf16 row,
// weights from HBM, us with 16 / 32 rows per warp: 4736 x 4096 6.1 / 6.8, 7000 x 4096 8.5 / 8.4,
// 9472 x 4096 10.0 / 8.8, 18944 x 4096 17.1 / 15.2, 32768 x 8192 46.5 / 42.2; eight rows alike. From
// 9 rows of x on the products' registers spill with 32 (10007 x 5000, 13 rows: 27 us against 20).
uint64_t wide_rows() { return 32ull * 2 * sm_count(); }

template <typename T, int kGroup, int kMT, int kNT, bool kVec>
void launch_matvec(const cora_w4_weight &w, const cora_w4_matvec_args &a, cudaStream_t st) {
    const uint64_t bx = (w.rows + 16 * kMT - 1) / (16 * kMT), by = (a.rows + 8 * kNT - 1) / (8 * kNT);
    need(by <= kMaxGrid, "too many activation rows");
    const size_t sm = (size_t)kMvWarps * 8 * kNT * 16 * kMT * 4;
    auto *kern = w4_matvec_kernel<T, kGroup, kMT, kNT, kVec>;
    static_assert((size_t)kMvWarps * 8 * kNT * 16 * kMT * 4 <= 48 * 1024, "");
    kern<<<dim3((unsigned)bx, (unsigned)by), kMvWarps * 32, sm, st>>>(w, a);
    CUDA_TRY(cudaGetLastError());
}

void matvec(const cora_w4_weight *w, const cora_w4_matvec_args *a, cudaStream_t st) {
    need(w && a, "null arguments");
    need(w->group == 32 || w->group == 64 || w->group == 128, "group must be 32, 64 or 128");
    need(w->cols >= 1 && w->cols <= INT_MAX / 2 && w->rows <= INT_MAX / 2, "weight sizes must be positive and fit an int");
    if (a->rows == 0 || w->rows == 0) return;
    need(w->codes && w->meta && aligned16(w->codes) && aligned16(w->meta), "codes and meta must be 16-byte aligned device memory");
    need(a->x && a->y, "x and y are needed");
    const bool vec = aligned16(a->x) && a->x_stride % 8 == 0 && w->cols % 8 == 0;
    by_dtype(a->dtype, [&](auto z) {
        using T = decltype(z);
        auto go = [&](auto gr) {
            constexpr int G = decltype(gr)::value;
            auto wide = [&](auto nt, auto mt) {
                constexpr int NT = decltype(nt)::value, MT = decltype(mt)::value;
                vec ? launch_matvec<T, G, MT, NT, true>(*w, *a, st) : launch_matvec<T, G, MT, NT, false>(*w, *a, st);
            };
            const bool two = w->rows >= wide_rows();
            if (a->rows <= 8) two ? wide(Int<1>{}, Int<2>{}) : wide(Int<1>{}, Int<1>{});
            else if (a->rows <= 16) wide(Int<2>{}, Int<1>{});
            else wide(Int<4>{}, Int<1>{});
        };
        if (w->group == 32) go(Int<32>{});
        else if (w->group == 64) go(Int<64>{});
        else go(Int<128>{});
    });
}

}  // namespace
}  // namespace cora

extern "C" {

uint64_t cora_kv4_block_bytes(uint32_t page_size, uint32_t head_dim, uint32_t group) {
    if (!group || head_dim % group) return 0;
    return (uint64_t)page_size * head_dim + 8ull * page_size * (head_dim / group);
}

int cora_kv4_status(const cora_kv4_cache *cache, void *stream) {
    return cora::guarded([&] {
        if (!cache || !cache->status) cora::fail(CORA_EINVAL, "null cache");
        int32_t word = 0;
        auto st = static_cast<cudaStream_t>(stream);
        CUDA_TRY(cudaMemcpyAsync(&word, cache->status, sizeof word, cudaMemcpyDeviceToHost, st));
        CUDA_TRY(cudaStreamSynchronize(st));
        if (word) {
            cora::clear_bits_kernel<<<1, 1, 0, st>>>(cache->status, word);
            CUDA_TRY(cudaGetLastError());
            CUDA_TRY(cudaStreamSynchronize(st));
        }
        if (word & cora::kDevWaitTimeout) cora::fail(CORA_ERUNTIME, "a device-side wait timed out");
        if (word & cora::kDevBadInput)
            cora::fail(CORA_ERUNTIME, "a slot, position, page or row range lies outside its tensor");
    });
}

int cora_kv4_append(const cora_kv4_cache *cache, const cora_kv4_append_args *args, void *stream) {
    return cora::guarded([&] { cora::append(cache, args, static_cast<cudaStream_t>(stream)); });
}

uint64_t cora_kv4_attend_workspace(const cora_kv4_cache *cache, uint32_t q_heads, uint32_t max_queries) {
    uint64_t bytes = 0;
    const int rc = cora::guarded([&] {
        cora::check_cache(cache);
        bytes = cora::attend_workspace(*cache, cora::attend_rows(*cache, q_heads, max_queries));
    });
    return rc == CORA_OK ? bytes : 0;
}

int cora_kv4_attend(const cora_kv4_cache *cache, const cora_kv4_attend_args *args, void *stream) {
    return cora::guarded([&] { cora::attend(cache, args, static_cast<cudaStream_t>(stream)); });
}

int cora_w4_matvec(const cora_w4_weight *weight, const cora_w4_matvec_args *args, void *stream) {
    return cora::guarded([&] { cora::matvec(weight, args, static_cast<cudaStream_t>(stream)); });
}

}  // extern "C"
