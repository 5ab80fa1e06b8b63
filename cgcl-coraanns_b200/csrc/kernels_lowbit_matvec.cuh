// Products of a few activation rows with a 4-bit weight matrix (cora_w4_matvec):
//
//   y[m][n] = sum over groups ( scale[n] * sum_k x[m][k] c[n][k]  +  low[n] * sum_k x[m][k] )
//
// so that codes enter the matrix instructions as small integers and each group's two factors are
// applied once to fp32 sums. Weights are the 16-row side of m16n8k16, activations the 8-column
// side: up to 8 rows of x cost what one costs.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/cora_b200.h"
#include "common.cuh"
#include "kernels_lowbit_append.cuh"

namespace cora {

// D (16 x 8, fp32) += A (16 x 16) B (16 x 8).
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
            "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
            "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kMvWarps = 8;

// 16 bytes that are read once: they do not displace the activations from L1.
__device__ __forceinline__ uint4 ld_stream(const void *p) {
    uint4 v;
    asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
        : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
        : "l"(p));
    return v;
}
template <int kWords>
__device__ __forceinline__ void ld_factors(const uint32_t *p, uint32_t (&f)[kWords]) {
    if constexpr (kWords == 1) {
        asm("ld.global.nc.u32 %0, [%1];" : "=r"(f[0]) : "l"(p));
    } else if constexpr (kWords == 2) {
        asm("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(f[0]), "=r"(f[1]) : "l"(p));
    } else {
        asm("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(f[0]), "=r"(f[1]), "=r"(f[2]), "=r"(f[3]) : "l"(p));
    }
}

// One warp: kMT tiles of 16 weight rows, segments of 128 columns warp, warp + 8, ...; the
// block's warps split the columns and add up in shared memory. grid: x over 16 kMT weight rows,
// y over 8 kNT activation rows. kVec: x rows may be read 16 bytes at a time.
//
// A lane holds row g = lane / 4 (and g + 8), 16 bytes at t = lane % 4: by the packed order, its
// word j is columns 32 j + 8 t .. + 7 of the segment, so one k-step of the tensor instruction
// stays inside 32 columns (any group of 32, 64 or 128) and x is read in its own order. Nibbles
// 0, 4 | 2, 6 | 1, 5 | 3, 7 of a word are columns (0, 1) (2, 3) (4, 5) (6, 7).
//   fp16 x: a masked nibble is the fp16 subnormal c 2^-24 (low nibble of a byte) or c 2^-20
//           (high nibble), exact in the tensor core; the two go to separate sums.
//   bf16 x: 0x4300 | c is 128 + c; the 128 sum(x) is taken off with the low term. The sums hold
//           24 bits, of which the offset costs about five, and the result keeps eight.
// sum(x) of a group comes from one more product with a matrix of ones.
//
// What has to be done is to read the weights: codes and factors of the next kMvDepth segments are in
// flight in registers (a warp and segment: 1 or 2 KB). What bounds it is the wait for the activations,
// which are loaded where they are used (long scoreboard first, issue slots 42% used). Measured:
// 32768 x 8192, one fp16 row, 39 us (3.6 TB/s); 10007 x 5000, 13 bf16 rows, 20 us.
template <typename T, int kGroup, int kMT, int kNT, bool kVec>
__global__ void __launch_bounds__(kMvWarps * 32, kNT >= 4 ? 1 : 2) w4_matvec_kernel(const cora_w4_weight w,
                                                                                    const cora_w4_matvec_args p) {
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr int kGroups = 128 / kGroup, kSteps = kGroup / 32;
    constexpr int kMvDepth = kNT == 1 && kMT == 1 ? 3 : 2;
    extern __shared__ float mv_red[];  // [warp][row of x][weight row]
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int n0 = blockIdx.x * 16 * kMT, m0 = blockIdx.y * 8 * kNT;
    const int segs = (int)((w.cols + 127) / 128);
    const uint64_t row_bytes = (uint64_t)segs * 64, row_groups = (uint64_t)segs * kGroups;
    const int rows = (int)w.rows;
    const uint8_t *cp[2 * kMT];
    const uint32_t *mp[2 * kMT];
#pragma unroll
    for (int i = 0; i < 2 * kMT; ++i) {
        const int r = min(n0 + i * 8 + g, rows - 1);
        cp[i] = w.codes + r * row_bytes + t * 16;
        mp[i] = static_cast<const uint32_t *>(w.meta) + r * row_groups;
    }
    const T *xp[kNT];
    bool xin[kNT];
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
        xin[n] = m0 + n * 8 + g < (int)p.rows;
        xp[n] = static_cast<const T *>(p.x) + (uint64_t)(xin[n] ? m0 + n * 8 + g : 0) * p.x_stride + t * 8;
    }
    float y[kMT][kNT][4];
#pragma unroll
    for (int i = 0; i < kMT; ++i)
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) y[i][n][c] = 0.0f;

    uint4 code[kMvDepth][2 * kMT];
    uint32_t fac[kMvDepth][2 * kMT][kGroups];
    auto fetch = [&](int s, uint4 (&c)[2 * kMT], uint32_t (&f)[2 * kMT][kGroups]) {
        if (s >= segs) return;
#pragma unroll
        for (int i = 0; i < 2 * kMT; ++i) {
            c[i] = ld_stream(cp[i] + (uint32_t)s * 64);
            ld_factors<kGroups>(mp[i] + (uint32_t)s * kGroups, f[i]);
        }
    };
#pragma unroll
    for (int d = 0; d < kMvDepth; ++d) fetch(warp + d * kMvWarps, code[d], fac[d]);

    for (int s0 = warp; s0 < segs; s0 += kMvWarps * kMvDepth) {
#pragma unroll
        for (int d = 0; d < kMvDepth; ++d) {
            const int s = s0 + d * kMvWarps;
            if (s >= segs) break;
            uint4 bx[kNT][4];  // the segment's activations, word j of the lane
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t k = (uint32_t)s * 128 + j * 32;  // (xp starts at the lane's own 8)
#pragma unroll
                for (int n = 0; n < kNT; ++n) {
                    bx[n][j] = make_uint4(0, 0, 0, 0);
                    if (kVec) {
                        if (xin[n] && k + t * 8 < w.cols) bx[n][j] = __ldg(reinterpret_cast<const uint4 *>(xp[n] + k));
                    } else if (xin[n]) {
                        uint32_t e[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            e[i] = k + t * 8 + i < w.cols ? reinterpret_cast<const uint16_t *>(xp[n])[k + i] : 0;
                        bx[n][j] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
                    }
                }
            }
#pragma unroll
            for (int gr = 0; gr < kGroups; ++gr) {
                float a1[kMT][kNT][4], a2[kMT][kNT][4], xs[kNT][4];
#pragma unroll
                for (int n = 0; n < kNT; ++n)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        xs[n][c] = 0.0f;
#pragma unroll
                        for (int i = 0; i < kMT; ++i) a1[i][n][c] = a2[i][n][c] = 0.0f;
                    }
#pragma unroll
                for (int j = gr * kSteps; j < (gr + 1) * kSteps; ++j) {
                    constexpr uint32_t one = kHalf ? 0x3c003c00u : 0x3f803f80u;
#pragma unroll
                    for (int n = 0; n < kNT; ++n) {
                        mma16816<T>(xs[n], one, one, one, one, bx[n][j].x, bx[n][j].y);
                        mma16816<T>(xs[n], one, one, one, one, bx[n][j].z, bx[n][j].w);
                    }
#pragma unroll
                    for (int i = 0; i < kMT; ++i) {
                        const uint4 &cu = code[d][2 * i], &cv = code[d][2 * i + 1];
                        const uint32_t u = j == 0 ? cu.x : j == 1 ? cu.y : j == 2 ? cu.z : cu.w;
                        const uint32_t v = j == 0 ? cv.x : j == 1 ? cv.y : j == 2 ? cv.z : cv.w;
                        const uint32_t u8 = u >> 8, v8 = v >> 8;
                        uint32_t f[8];
                        if constexpr (kHalf) {
                            f[0] = u & 0x000f000fu, f[1] = v & 0x000f000fu, f[2] = u8 & 0x000f000fu, f[3] = v8 & 0x000f000fu;
                            f[4] = u & 0x00f000f0u, f[5] = v & 0x00f000f0u, f[6] = u8 & 0x00f000f0u, f[7] = v8 & 0x00f000f0u;
                        } else {
                            f[0] = (u & 0x000f000fu) | 0x43004300u, f[1] = (v & 0x000f000fu) | 0x43004300u;
                            f[2] = (u8 & 0x000f000fu) | 0x43004300u, f[3] = (v8 & 0x000f000fu) | 0x43004300u;
                            f[4] = ((u >> 4) & 0x000f000fu) | 0x43004300u, f[5] = ((v >> 4) & 0x000f000fu) | 0x43004300u;
                            f[6] = ((u >> 12) & 0x000f000fu) | 0x43004300u, f[7] = ((v >> 12) & 0x000f000fu) | 0x43004300u;
                        }
#pragma unroll
                        for (int n = 0; n < kNT; ++n) {
                            mma16816<T>(a1[i][n], f[0], f[1], f[2], f[3], bx[n][j].x, bx[n][j].y);
                            mma16816<T>(kHalf ? a2[i][n] : a1[i][n], f[4], f[5], f[6], f[7], bx[n][j].z, bx[n][j].w);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < kMT; ++i) {
                    float2 f0 = __half22float2(*reinterpret_cast<const __half2 *>(&fac[d][2 * i][gr]));
                    float2 f1 = __half22float2(*reinterpret_cast<const __half2 *>(&fac[d][2 * i + 1][gr]));
                    if constexpr (kHalf) {  // 2^24 of the subnormal codes
                        f0.x *= 16777216.0f, f1.x *= 16777216.0f;
                    } else {  // the 128 of 128 + c
                        f0.y = fmaf(-128.0f, f0.x, f0.y), f1.y = fmaf(-128.0f, f1.x, f1.y);
                    }
#pragma unroll
                    for (int n = 0; n < kNT; ++n)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float2 f = c < 2 ? f0 : f1;
                            const float sum = kHalf ? fmaf(a2[i][n][c], 0.0625f, a1[i][n][c]) : a1[i][n][c];
                            y[i][n][c] = fmaf(f.x, sum, fmaf(f.y, xs[n][c], y[i][n][c]));
                        }
                }
            }
            fetch(s + kMvWarps * kMvDepth, code[d], fac[d]);
        }
    }

    // the warps' column shares, added in warp order
    constexpr int kR = 16 * kMT;
#pragma unroll
    for (int i = 0; i < kMT; ++i)
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                mv_red[(warp * 8 * kNT + n * 8 + 2 * t + (c & 1)) * kR + i * 16 + g + (c >> 1) * 8] = y[i][n][c];
    __syncthreads();
    for (int e = threadIdx.x; e < 8 * kNT * kR; e += kMvWarps * 32) {
        const int m = m0 + e / kR, n = n0 + e % kR;
        if (m >= (int)p.rows || n >= rows) continue;
        float sum = 0.0f;
#pragma unroll
        for (int q = 0; q < kMvWarps; ++q) sum += mv_red[q * 8 * kNT * kR + e];
        if (p.bias) sum += to_f32(static_cast<const T *>(p.bias)[n]);
        static_cast<T *>(p.y)[(uint64_t)m * p.y_stride + n] = from_f32<T>(sum);
    }
}

}  // namespace cora
