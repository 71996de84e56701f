// Product of e4m3 operands with a scale for each block of 128:
//   out[m, n] = sum_b a_scales[m, b] w_scales[n / 128, b] (sum over k in block b of a[m, k] w[n, k]) + bias[n]
// b = k / 128.  The inner sums come from the matrix cores, from zero for each block; the outer ones are fp32 multiply-adds with the product
// of the two scales.  The product is formed transposed (MFMA rows = n), so that a lane holds one row of `out`, whose scale it multiplies
// with, and four consecutive columns.
//
// The matrix instructions for 8-bit operands add up to 16 neighbouring products at a time in about 14 bits below the largest of them (measured: a
// product of 2^-14 beside one of 1 is lost, beyond those 16 one of 2^-23 is kept).  2-norm relative 1.5e-5 for normally distributed operands: a
// hundredth of the rounding of a bf16 result, but not fp32.  Results in fp32 take their operands as bf16, which hold every e4m3 value
// exactly, at half the rate: 4e-9 so.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "launch_internal.h"
#include "mfma_tiles.h"
#include "profiler.h"
#include "row_chunks.h"

namespace {
using namespace kutacc_dev;

typedef __attribute__((ext_vector_type(8))) int i32x8;

struct LinearParams {
    const uint8_t *a, *w;
    const float *a_scales, *w_scales, *bias;
    void *out;
    int64_t a_ld, w_ld, a_scales_ld, w_scales_ld, out_ld;
    int M, N, K, MT, NT;
};

// 16 rows of w by 16 rows of a, 128 k: lane l holds 32 bytes of row l & 15 of either, and columns 4 (l >> 4) .. + 3 of the sums of row l & 15 of a
__device__ __forceinline__ f32x4 mfma_fp8(i32x8 w, i32x8 a, f32x4 c)
{
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, a, c, 0, 0, 0, 0, 0, 0);
}

__device__ __forceinline__ i32x8 fp8_operand(uint4 lo, uint4 hi)
{
    union {
        uint4 u[2];
        i32x8 v;
    } c;
    c.u[0] = lo, c.u[1] = hi;
    return c.v;
}

// eight e4m3 values as bf16
__device__ __forceinline__ bf16x8 widened(uint32_t lo, uint32_t hi)
{
    union {
        bf16x2 p[4];
        bf16x8 v;
    } c;
    c.p[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), c.p[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    c.p[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), c.p[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return c.v;
}

// the same product with sums in full fp32
struct WideOperand {
    bf16x8 piece[4];
};
__device__ __forceinline__ WideOperand widened(i32x8 v)
{
    WideOperand o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        o.piece[i] = widened((uint32_t)v[2 * i], (uint32_t)v[2 * i + 1]);
    }
    return o;
}
__device__ __forceinline__ f32x4 mfma_wide(const WideOperand &w, const WideOperand &a, f32x4 c)
{
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.piece[i], a.piece[i], c, 0, 0, 0);
    }
    return c;
}

// 16 bytes of a row of `length`, from byte `at` on, zeros past its end
__device__ __forceinline__ uint4 load16_checked(const uint8_t *row, int at, int length)
{
    union {
        uint4 u;
        uint8_t b[16];
    } c;
    if (at + 16 <= length) {
        __builtin_memcpy(&c.u, row + at, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            c.b[i] = at + i < length ? row[at + i] : 0;
        }
    }
    return c.u;
}

// 128 x 128 of `out` a workgroup, 64 x 64 a wave; a block of 128 k a step.  In the LDS a row's 128 bytes are eight slots of 16, the slots of
// row i XOR-ed with i & 7.
constexpr int TILE = 128;

template <typename T>
__global__ __launch_bounds__(256, 2) void fp8_tiles_kernel(const LinearParams p)
{
    __shared__ uint4 lds[2 * TILE * 8];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 15, q = lane >> 4, wm = wave >> 1, wn = wave & 1;
    const int m0 = (int)(blockIdx.x / (unsigned)p.NT) * TILE, n0 = (int)(blockIdx.x % (unsigned)p.NT) * TILE;
    const int blocks = (p.K + FP8_BLOCK - 1) / FP8_BLOCK;

    // a thread brings 16 bytes (slot tid & 7) of rows tid / 8 + 32 i of either operand
    const uint8_t *a_row[4], *w_row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a_row[i] = p.a + (int64_t)min(m0 + (tid >> 3) + 32 * i, p.M - 1) * p.a_ld;
        w_row[i] = p.w + (int64_t)min(n0 + (tid >> 3) + 32 * i, p.N - 1) * p.w_ld;
    }
    uint4 next_a[4], next_w[4];
    float next_scale[4];
    const float *scale_row[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        scale_row[j] = p.a_scales + (int64_t)min(m0 + 64 * wm + 16 * j + r, p.M - 1) * p.a_scales_ld;
    }
    const float *w_scales = p.w_scales + (int64_t)(n0 / FP8_BLOCK) * p.w_scales_ld;
    auto fetch = [&](int b) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            next_a[i] = load16_checked(a_row[i], b * FP8_BLOCK + (tid & 7) * 16, p.K);
            next_w[i] = load16_checked(w_row[i], b * FP8_BLOCK + (tid & 7) * 16, p.K);
        }
        const float ws = w_scales[b];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            next_scale[j] = scale_row[j][b] * ws;
        }
    };
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    fetch(0);
    for (int b = 0; b < blocks; ++b) {
        __syncthreads(); // the last step's operands have been read
        float scale[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = (tid >> 3) + 32 * i, slot = row * 8 + ((tid & 7) ^ (row & 7));
            lds[slot] = next_a[i];
            lds[TILE * 8 + slot] = next_w[i];
            scale[i] = next_scale[i];
        }
        __syncthreads();
        if (b + 1 < blocks) {
            fetch(b + 1);
        }
        auto operand = [&](const uint4 *rows, int block) {
            const uint4 *row = rows + (16 * block + r) * 8;
            return fp8_operand(row[q ^ (r & 7)], row[(4 + q) ^ (r & 7)]);
        };
        constexpr bool WIDE = std::is_same<T, float>::value;
        typename std::conditional<WIDE, WideOperand, i32x8>::type w[4], a;
        auto take = [&](auto &to, const uint4 *rows, int block) {
            if constexpr (WIDE) {
                to = widened(operand(rows, block));
            } else {
                to = operand(rows, block);
            }
        };
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            take(w[i], lds + TILE * 8, 4 * wn + i);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            take(a, lds, 4 * wm + j);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
                f32x4 part;
                if constexpr (WIDE) {
                    part = mfma_wide(w[i], a, zero);
                } else {
                    part = mfma_fp8(w[i], a, zero);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    acc[i][j][e] = fmaf(part[e], scale[j], acc[i][j][e]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = n0 + 64 * wn + 16 * i + 4 * q;
        float bias[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            bias[e] = p.bias != nullptr && n + e < p.N ? p.bias[n + e] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int m = m0 + 64 * wm + 16 * j + r;
            T *to = (T *)p.out + (int64_t)m * p.out_ld + n;
            if (m < p.M) {
                T o[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    o[e] = from_f32<T>(acc[i][j][e] + bias[e]);
                }
                if (n + 4 <= p.N) {
                    __builtin_memcpy(to, o, sizeof(o));
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (n + e < p.N) {
                            to[e] = o[e];
                        }
                    }
                }
            }
        }
    }
}
} // namespace

namespace kutacc_launch {

int linear_fp8(const kutacc_hip_linear_fp8_args_t &a, hipStream_t stream)
{
    LinearParams p = {(const uint8_t *)a.a, (const uint8_t *)a.w, a.a_scales, a.w_scales, a.bias, a.out, a.a_ld, a.w_ld, a.a_scales_ld,
                      a.w_scales_ld, a.out_ld, (int)a.m, (int)a.n, (int)a.k, 0, 0};
    p.MT = (p.M + TILE - 1) / TILE, p.NT = (p.N + TILE - 1) / TILE;
    const int64_t tiles = (int64_t)p.MT * p.NT;
    if (tiles > INT32_MAX) {
        return KUTACC_HIP_EUNSUPPORTED;
    }
    kutacc_prof::KernelTimer t("fp8_tiles_kernel", 2.0 * (double)a.m * (double)a.n * (double)a.k, stream);
    if (a.dtype == KUTACC_DTYPE_BF16) {
        fp8_tiles_kernel<bf16_t><<<dim3((unsigned)tiles), 256, 0, stream>>>(p);
    } else {
        fp8_tiles_kernel<float><<<dim3((unsigned)tiles), 256, 0, stream>>>(p);
    }
    return kutacc_hip_status(hipGetLastError());
}

} // namespace kutacc_launch
