// Rows held eight values a lane, in 32 bits, for the kernels that normalise or quantise rows of any length and address: chunk c of a
// row is its elements 8 c .. 8 c + 7, and what lies past the row's end is zero.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "device_util.h"

namespace kutacc_dev {

// Elements past `size` are neither read nor written; rows start on any address of their type (the hardware's unaligned 16-byte accesses).
template <typename T>
__device__ __forceinline__ void load_chunk(float (&v)[8], const T *row, int at, int size)
{
    if (at + 8 <= size) {
        T raw[8];
        __builtin_memcpy(raw, row + at, sizeof(raw));
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = to_f32(raw[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = at + e < size ? to_f32(row[at + e]) : 0.f;
        }
    }
}

template <typename T>
__device__ __forceinline__ void store_chunk(const float (&v)[8], T *row, int at, int size)
{
    if (at + 8 <= size) {
        T raw[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            raw[e] = from_f32<T>(v[e]);
        }
        __builtin_memcpy(row + at, raw, sizeof(raw));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (at + e < size) {
                row[at + e] = from_f32<T>(v[e]);
            }
        }
    }
}

// A chunk on its way, as it lies in memory: asked for without a branch, so that nothing waits for it before unpack() does.  Rows of at least eight elements; a
// chunk past the row's end is read in front of it, and unpack() shifts it into place.
template <typename T>
struct RawChunk {
    uint4 v[sizeof(T) / 2];
};
__device__ __forceinline__ int past_end(int at, int size) { return max(0, at + 8 - size); }
template <typename T>
__device__ __forceinline__ void ask_chunk(RawChunk<T> &raw, const T *row, int at, int size)
{
    __builtin_memcpy(&raw, row + at - past_end(at, size), sizeof(raw));
}
template <typename T>
__device__ __forceinline__ void unpack(float (&v)[8], const RawChunk<T> &raw, int at, int size)
{
    T values[8];
    __builtin_memcpy(values, &raw, sizeof(values));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        v[e] = to_f32(values[e]);
    }
    const int past = past_end(at, size);
    if (size % 8 != 0) {
#pragma unroll
        for (int shift = 1; shift < 8; shift *= 2) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = (past & shift) == 0 ? v[e] : e + shift < 8 ? v[e + shift] : 0.f;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        v[e] = past < 8 ? v[e] : 0.f;
    }
}

// ---- e4m3 (OCP: largest value 448, no infinities) with a scale ----

constexpr int FP8_BLOCK = 128; // values along a row that share a scale
constexpr float FP8_LARGEST = 448.0f;
constexpr float FP8_SMALLEST_SCALE = 0x1p-126f; // what a block of zeros gets: its quotients are zeros, not 0 / 0

__device__ __forceinline__ float abs_max(const float (&v)[8])
{
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        m = __builtin_elementwise_maximum(m, fabsf(v[e])); // keeps a NaN, so that its block's scale is one
    }
    return m;
}

// the largest over 16 lanes (LANES = 16) or 8, in every one of them
template <int LANES>
__device__ __forceinline__ float lanes_max(float v)
{
    auto step = [&](auto ctrl) {
        const int moved = __builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, false);
        v = __builtin_elementwise_maximum(v, __int_as_float(moved));
    };
    step(std::integral_constant<int, 0xB1>{});  // lane ^ 1
    step(std::integral_constant<int, 0x4E>{});  // lane ^ 2
    step(std::integral_constant<int, 0x141>{}); // pairs the two quads of 8 lanes
    if constexpr (LANES == 16) {
        step(std::integral_constant<int, 0x140>{}); // pairs the two halves of 16 lanes
    }
    return v;
}

__device__ __forceinline__ float fp8_scale(float largest) { return __builtin_elementwise_maximum(largest / FP8_LARGEST, FP8_SMALLEST_SCALE); }

// Eight values over their scale, rounded to 32 bits as a division rounds and then to nearest even in e4m3.  The quotient is one Newton step
// on the product with the rounded reciprocal (P. W. Markstein, Computation of elementary functions on the IBM RISC System/6000 processor,
// 1990): 3 instructions where a division takes some 10.  A scale far from 1, where that step's remainder is no normal number, or one
// that is no finite number, takes divisions.  No quotient passes 464, from where on e4m3 would round up.
__device__ __forceinline__ uint2 fp8_quotients(const float (&v)[8], float scale)
{
    float q[8];
    if (scale > 0x1p-60f && scale < 0x1p100f) {
        const float r = 1.0f / scale;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float q0 = v[e] * r;
            q[e] = fmaf(fmaf(-q0, scale, v[e]), r, q0);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            q[e] = v[e] / scale;
        }
    }
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}

__device__ __forceinline__ void store_fp8_chunk(uint2 q, uint8_t *row, int at, int size)
{
    if (at + 8 <= size) {
        __builtin_memcpy(row + at, &q, 8);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (at + e < size) {
                row[at + e] = (uint8_t)((e < 4 ? q.x : q.y) >> (8 * (e & 3)));
            }
        }
    }
}

} // namespace kutacc_dev
