// Appending keys and values to the paged 4-bit cache (cora_kv4_append): rotate keys (and
// queries) by position, quantise keys and values group by group, store codes and factors.
//
//   rotation of a pair (a, b) by the angle of its position:  a cos - b sin,  b cos + a sin
//   group of G values:  low = fp16(min),  scale = fp16((max - min) * (1 / 15)),
//                       code = clamp(rne((x - low) * (1 / scale)), 0, 15)   (0 where scale is 0)
//
// Every step is one IEEE fp32 operation in the order written (no contraction), so codes do not
// depend on the launch shape and equal those of any fp32 implementation of the same formulas.
// A NaN in a group makes its factors NaN (min.NaN below), so that it is read back as NaN;
// factors past the fp16 range saturate.
//
// What bounds it: memory, for prompts. A thread owns dimensions 8c .. 8c + 7 and D / 2 + 8c .. of
// one token (two 16-byte loads per head), the two sides of a full rotation's pairs, and walks
// over heads, so that cos and sin are read once per token and not once per head; a group's
// threads are neighbouring lanes.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/cora_b200.h"
#include "common.cuh"

namespace cora {

// Byte offsets inside one (page, key head) block: key codes, value codes, key factors, value
// factors, each token-major.
struct Kv4Block {
    uint32_t code_row, codes, meta_row, metas;  // bytes per token and per section
    uint32_t bytes;
    __host__ __device__ Kv4Block(uint32_t page, uint32_t dim, uint32_t group)
        : code_row(dim / 2), codes(page * dim / 2), meta_row(dim / group * 4),
          metas(page * (dim / group) * 4), bytes(2 * codes + 2 * metas) {}
};

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }

// min and max that keep NaN.
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// 8 consecutive values; kVec: one 16-byte load (the host has checked alignment and strides).
template <typename T, bool kVec>
__device__ __forceinline__ void load8(const T *p, float (&x)[8]) {
    T t[8];
    if constexpr (kVec) {
        *reinterpret_cast<uint4 *>(t) = __ldg(reinterpret_cast<const uint4 *>(p));
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) t[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(t[i]);
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
    alignas(16) T t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = from_f32<T>(x[i]);
    *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(t);
}

template <typename T>
__device__ __forceinline__ void store4(T *p, float a, float b, float c, float d) {
    alignas(8) T t[4] = {from_f32<T>(a), from_f32<T>(b), from_f32<T>(c), from_f32<T>(d)};
    *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(t);
}

constexpr int kAppendThreads = 256;
enum AppendTurn { kTurnNone, kTurnFull, kTurnInterleaved, kTurnPart };

// Quantises 8 values of a group whose extremes are known: the word of codes, the values they
// stand for in x, the factors.
__device__ __forceinline__ uint32_t quantize8(float (&x)[8], float lo, float hi, __half2 &factors) {
    const float s = __fmul_rn(__fsub_rn(hi, lo), 1.0f / 15.0f);
    const __half hs = __float2half_rn(s > 65504.0f ? 65504.0f : s);
    const __half hl = __float2half_rn(lo > 65504.0f ? 65504.0f : lo < -65504.0f ? -65504.0f : lo);
    factors = __halves2half2(hs, hl);
    const float scale = __half2float(hs), low = __half2float(hl);
    const float inv = scale > 0.0f ? __frcp_rn(scale) : 0.0f;
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float r = fminf(fmaxf(__fmul_rn(__fsub_rn(x[i], low), inv), 0.0f), 15.0f);
        // 2^23 + r: rounds to the nearest integer, halves to even, in the low mantissa bits
        const float n = __fadd_rn(r, 8388608.0f);
        word |= (__float_as_uint(n) & 15u) << (4 * i);
        x[i] = fmaf(scale, __fsub_rn(n, 8388608.0f), low);
    }
    return word;
}

// grid: x over tokens (kAppendThreads / (D / 16) of them per block), y over runs of `run` heads
// of the list [key heads | value heads | query heads]. kOne: one group per head (group = D).
// Four blocks per SM: 93 us for 16384 tokens (32 + 8 + 8 heads of 128, 430 MB, 4.6 TB/s); without
// the bound, 80 registers and three blocks, 100 us; five (spills) 97 us.
template <typename T, int D, bool kOne, bool kVec>
__global__ void __launch_bounds__(kAppendThreads, 4) kv4_append_kernel(const cora_kv4_cache c,
                                                                    const cora_kv4_append_args a,
                                                                    int run, int turn) {
    constexpr int kLanes = D / 16;
    const int chunk = threadIdx.x % kLanes, d0 = chunk * 8, d1 = D / 2 + d0;
    const uint64_t token = (uint64_t)blockIdx.x * (kAppendThreads / kLanes) + threadIdx.x / kLanes;
    const bool live = token < a.tokens;
    const uint64_t tok = live ? token : a.tokens - 1;  // spare threads follow the last token's loads
    const uint32_t group = kOne ? D : c.group;
    const Kv4Block blk(c.page_size, D, group);
    const int H = c.kv_heads, heads = 2 * H + (a.q ? (int)a.q_heads : 0);
    const int h0 = blockIdx.y * run, h1 = min(heads, h0 + run);

    uint8_t *base = nullptr;  // this token in head 0 of its page; null: not stored
    uint32_t off = 0;
    if (h0 < 2 * H) {
        const int64_t slot = __ldg(a.slots + tok);
        if (live && slot >= 0) {
            const uint32_t shift = 31 - __clz(c.page_size);
            const uint64_t page = (uint64_t)slot >> shift;
            off = (uint32_t)slot & (c.page_size - 1);
            if (page < c.num_pages) base = c.pool + page * H * (uint64_t)blk.bytes;
            else if (chunk == 0) atomicOr(c.status, kDevBadInput);
        }
    }
    const int R = a.rotary, half = R / 2;
    float cs[8], sn[8];  // full: of the pairs (d0 + i, d1 + i); interleaved: 4 of d0's, 4 of d1's
    const float *pc = nullptr, *ps = nullptr;
    if (turn != kTurnNone) {
        int32_t pos = __ldg(a.positions + tok);
        if (pos < 0 || (uint64_t)pos >= a.rope_rows) {
            if (live && chunk == 0) atomicOr(c.status, kDevBadInput);
            pos = 0;
        }
        pc = a.rope_cos + (uint64_t)pos * half, ps = a.rope_sin + (uint64_t)pos * half;
        if (turn != kTurnPart) {
            const int i0 = turn == kTurnFull ? d0 : d0 / 2, i1 = turn == kTurnFull ? d0 + 4 : d1 / 2;
            const bool t0 = turn == kTurnFull || d0 < R, t1 = turn == kTurnFull || d1 < R;
            const float4 one = make_float4(1.0f, 1.0f, 1.0f, 1.0f), zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            *reinterpret_cast<float4 *>(cs) = t0 ? __ldg(reinterpret_cast<const float4 *>(pc + i0)) : one;
            *reinterpret_cast<float4 *>(sn) = t0 ? __ldg(reinterpret_cast<const float4 *>(ps + i0)) : zero;
            *reinterpret_cast<float4 *>(cs + 4) = t1 ? __ldg(reinterpret_cast<const float4 *>(pc + i1)) : one;
            *reinterpret_cast<float4 *>(sn + 4) = t1 ? __ldg(reinterpret_cast<const float4 *>(ps + i1)) : zero;
        }
    }

    // A partial rotation's pairs (i, i + R / 2) lie in other threads' chunks: those are read again.
    auto turn_part = [&](const T *src, float (&x)[8], int d) {
        if (d >= R) return;
        float y[8];
        load8<T, kVec>(src + (d < half ? d + half : d - half), y);
        const int i0 = d < half ? d : d - half;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float m = __fmul_rn(x[i], __ldg(pc + i0 + i)), n = __fmul_rn(y[i], __ldg(ps + i0 + i));
            x[i] = d < half ? __fsub_rn(m, n) : __fadd_rn(m, n);
        }
    };
    auto load = [&](const T *src, float (&x)[8], float (&y)[8], bool turned) {
        load8<T, kVec>(src + d0, x);
        load8<T, kVec>(src + d1, y);
        if (!turned) return;
        if (turn == kTurnFull) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float u = x[i], v = y[i];
                x[i] = __fsub_rn(__fmul_rn(u, cs[i]), __fmul_rn(v, sn[i]));
                y[i] = __fadd_rn(__fmul_rn(v, cs[i]), __fmul_rn(u, sn[i]));
            }
        } else if (turn == kTurnInterleaved) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float u = x[2 * i], v = x[2 * i + 1];
                if (d0 < R) {
                    x[2 * i] = __fsub_rn(__fmul_rn(u, cs[i]), __fmul_rn(v, sn[i]));
                    x[2 * i + 1] = __fadd_rn(__fmul_rn(v, cs[i]), __fmul_rn(u, sn[i]));
                }
                u = y[2 * i], v = y[2 * i + 1];
                if (d1 < R) {
                    y[2 * i] = __fsub_rn(__fmul_rn(u, cs[4 + i]), __fmul_rn(v, sn[4 + i]));
                    y[2 * i + 1] = __fadd_rn(__fmul_rn(v, cs[4 + i]), __fmul_rn(u, sn[4 + i]));
                }
            }
        } else if (turn == kTurnPart) {
            turn_part(src, x, d0);
            turn_part(src, y, d1);
        }
    };

    // queries: heads [2 H, heads)
    if (h1 > 2 * H) {
        const int q0 = max(h0, 2 * H) - 2 * H, q1 = h1 - 2 * H;
        const T *src = static_cast<const T *>(a.q) + (int64_t)tok * a.q_token + (int64_t)q0 * a.q_head;
        T *dst = static_cast<T *>(a.q_out) + (tok * a.q_heads + q0) * D;
#pragma unroll 2
        for (int h = q0; h < q1; ++h, src += a.q_head, dst += D) {
            float x[8], y[8];
            load(src, x, y, turn != kTurnNone);
            if (live) {
                store8(dst + d0, x);
                store8(dst + d1, y);
            }
        }
    }
    // keys: heads [0, H), values: [H, 2 H)
    for (int h = h0; h < min(h1, 2 * H); ++h) {
        const bool val = h >= H;
        const int hh = val ? h - H : h;
        const T *src = val ? static_cast<const T *>(a.v) + (int64_t)tok * a.v_token + (int64_t)hh * a.v_head
                           : static_cast<const T *>(a.k) + (int64_t)tok * a.k_token + (int64_t)hh * a.k_head;
        float x[8], y[8];
        load(src, x, y, !val && turn != kTurnNone);
        float lo = x[0], hi = x[0], lo2 = y[0], hi2 = y[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            lo = min_nan(lo, x[i]), hi = max_nan(hi, x[i]);
            lo2 = min_nan(lo2, y[i]), hi2 = max_nan(hi2, y[i]);
        }
        if (kOne) {
            lo = min_nan(lo, lo2), hi = max_nan(hi, hi2);
#pragma unroll
            for (int m = 1; m < kLanes; m <<= 1) {
                lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, m));
                hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, m));
            }
            lo2 = lo, hi2 = hi;
        } else {
            for (int m = 1; m < (int)group / 8; m <<= 1) {
                lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, m));
                hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, m));
                lo2 = min_nan(lo2, __shfl_xor_sync(0xffffffffu, lo2, m));
                hi2 = max_nan(hi2, __shfl_xor_sync(0xffffffffu, hi2, m));
            }
        }
        __half2 f, f2;
        const uint32_t w = quantize8(x, lo, hi, f), w2 = quantize8(y, lo2, hi2, f2);
        if (base) {
            uint8_t *codes = base + (uint64_t)hh * blk.bytes + (val ? blk.codes : 0) + off * blk.code_row;
            *reinterpret_cast<uint32_t *>(codes + d0 / 2) = w;
            *reinterpret_cast<uint32_t *>(codes + d1 / 2) = w2;
            uint8_t *meta = base + (uint64_t)hh * blk.bytes + 2 * blk.codes + (val ? blk.metas : 0) + off * blk.meta_row;
            if (d0 % group == 0) *reinterpret_cast<__half2 *>(meta + d0 / group * 4) = f;
            if (!kOne && d1 % group == 0) *reinterpret_cast<__half2 *>(meta + d1 / group * 4) = f2;
        }
        T *out = static_cast<T *>(val ? a.v_out : a.k_out);
        if (out && live) {
            out += (tok * H + hh) * D;
            store8(out + d0, x);
            store8(out + d1, y);
        }
    }
}

}  // namespace cora
