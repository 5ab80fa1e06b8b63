// Appending keys and values to the paged 4-bit cache (cora_kv4_append): rotate keys (and
// queries) by position, quantise keys and values group by group, store codes and factors.
//
//   rotation of a pair (a, b) by the angle of its position:  a cos - b sin,  b cos + a sin
//   group of G values:  low = fp16(min),  scale = fp16((max - min) / 15),
//                       code = clamp(rne((x - low) * (1 / scale)), 0, 15)   (0 where scale is 0)
//
// Every step is one IEEE fp32 operation in the order written (no contraction), so codes do not
// depend on the launch shape and equal those of any fp32 implementation of the same formulas.
// A NaN in a group makes its factors NaN (min.NaN below), so that it is read back as NaN;
// factors past the fp16 range saturate.
//
// What bounds it: memory, for prompts. A thread owns 8 consecutive dimensions of one token (one
// 16-byte load per head) and walks over heads, so that the rotation's cos and sin are read once
// per token and chunk instead of once per head; a group's 8 or 16 threads are neighbouring lanes.
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

constexpr int kAppendThreads = 256;

// grid: x over tokens (kAppendThreads / (D / 8) of them per block), y over runs of `run` heads
// of the list [key heads | value heads | query heads].
template <typename T, int D, bool kVec>
__global__ void __launch_bounds__(kAppendThreads) kv4_append_kernel(const cora_kv4_cache c,
                                                                    const cora_kv4_append_args a,
                                                                    int run) {
    constexpr int kChunks = D / 8;
    const int chunk = threadIdx.x % kChunks, d0 = chunk * 8;
    const uint64_t token = (uint64_t)blockIdx.x * (kAppendThreads / kChunks) + threadIdx.x / kChunks;
    const bool live = token < a.tokens;
    const uint64_t tok = live ? token : a.tokens - 1;  // spare threads follow the last token's loads
    const Kv4Block blk(c.page_size, D, c.group);

    int64_t slot = __ldg(a.slots + tok);
    bool store = live && slot >= 0;
    if (store && (uint64_t)slot >= c.num_pages * c.page_size) {
        if (chunk == 0) atomicOr(c.status, kDevBadInput);
        store = false;
    }
    uint64_t page = 0;
    uint32_t off = 0;
    if (store) {
        page = (uint64_t)slot / c.page_size;
        off = (uint32_t)((uint64_t)slot - page * c.page_size);
    }

    const int R = a.rotary, half = R / 2;
    const bool turns = d0 < R;
    float cs[8], sn[8];
    if (turns) {
        int32_t pos = __ldg(a.positions + tok);
        if (pos < 0 || (uint64_t)pos >= a.rope_rows) {
            if (live && chunk == 0) atomicOr(c.status, kDevBadInput);
            pos = 0;
        }
        const int i0 = a.interleaved ? d0 / 2 : d0 < half ? d0 : d0 - half;
        const float4 *pc = reinterpret_cast<const float4 *>(a.rope_cos + (uint64_t)pos * half + i0);
        const float4 *ps = reinterpret_cast<const float4 *>(a.rope_sin + (uint64_t)pos * half + i0);
        *reinterpret_cast<float4 *>(cs) = __ldg(pc);
        *reinterpret_cast<float4 *>(sn) = __ldg(ps);
        if (!a.interleaved) {
            *reinterpret_cast<float4 *>(cs + 4) = __ldg(pc + 1);
            *reinterpret_cast<float4 *>(sn + 4) = __ldg(ps + 1);
        }
    }

    const int H = c.kv_heads, heads = 2 * H + (a.q ? (int)a.q_heads : 0);
    const int h1 = min(heads, (int)(blockIdx.y + 1) * run);
    for (int h = blockIdx.y * run; h < h1; ++h) {
        const int kind = h < H ? 0 : h < 2 * H ? 1 : 2;
        const int hh = kind == 0 ? h : kind == 1 ? h - H : h - 2 * H;
        const T *src = kind == 0   ? static_cast<const T *>(a.k) + tok * a.k_token + hh * a.k_head
                       : kind == 1 ? static_cast<const T *>(a.v) + tok * a.v_token + hh * a.v_head
                                   : static_cast<const T *>(a.q) + tok * a.q_token + hh * a.q_head;
        float x[8];
        load8<T, kVec>(src + d0, x);
        if (kind != 1 && turns) {
            if (a.interleaved) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float u = x[2 * i], v = x[2 * i + 1];
                    x[2 * i] = __fsub_rn(__fmul_rn(u, cs[i]), __fmul_rn(v, sn[i]));
                    x[2 * i + 1] = __fadd_rn(__fmul_rn(v, cs[i]), __fmul_rn(u, sn[i]));
                }
            } else {
                float y[8];  // the other halves of the pairs: a neighbour's load, in L1
                load8<T, kVec>(src + (d0 < half ? d0 + half : d0 - half), y);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float m = __fmul_rn(x[i], cs[i]), n = __fmul_rn(y[i], sn[i]);
                    x[i] = d0 < half ? __fsub_rn(m, n) : __fadd_rn(m, n);
                }
            }
        }
        if (kind == 2) {
            if (live) store8(static_cast<T *>(a.q_out) + (tok * a.q_heads + hh) * D + d0, x);
            continue;
        }
        float lo = x[0], hi = x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            lo = min_nan(lo, x[i]);
            hi = max_nan(hi, x[i]);
        }
        for (int m = 1; m < (int)c.group / 8; m <<= 1) {
            lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, m));
            hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, m));
        }
        const float s = __fdiv_rn(__fsub_rn(hi, lo), 15.0f);
        const __half hs = __float2half_rn(s > 65504.0f ? 65504.0f : s);
        const __half hl = __float2half_rn(lo > 65504.0f ? 65504.0f : lo < -65504.0f ? -65504.0f : lo);
        const float scale = __half2float(hs), low = __half2float(hl);
        const float inv = scale > 0.0f ? __frcp_rn(scale) : 0.0f;
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float r = __fmul_rn(__fsub_rn(x[i], low), inv);
            r = fminf(fmaxf(r, 0.0f), 15.0f);
            // 2^23 + r: rounds to the nearest integer, halves to even, in the low mantissa bits
            const uint32_t code = __float_as_uint(__fadd_rn(r, 8388608.0f)) & 15u;
            word |= code << (4 * i);
            x[i] = fmaf(scale, (float)code, low);
        }
        if (store) {
            uint8_t *base = c.pool + (page * H + hh) * (uint64_t)blk.bytes;
            *reinterpret_cast<uint32_t *>(base + (kind ? blk.codes : 0) + off * blk.code_row + d0 / 2) = word;
            if (d0 % c.group == 0)
                *reinterpret_cast<__half2 *>(base + 2 * blk.codes + (kind ? blk.metas : 0) +
                                             off * blk.meta_row + d0 / c.group * 4) = __halves2half2(hs, hl);
        }
        T *out = static_cast<T *>(kind ? a.v_out : a.k_out);
        if (out && live) store8(out + (tok * H + hh) * D + d0, x);
    }
}

}  // namespace cora
