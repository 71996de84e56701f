// Product of e4m3 operands with a scale for each block of 128:
//   out[m, n] = sum_b a_scales[m, b] w_scales[n / 128, b] (sum over k in block b of a[m, k] w[n, k]) + bias[n]
// b = k / 128.  The inner sums come from the matrix cores, from zero for each block; the outer ones are fp32 multiply-adds with the product
// of the two scales.  The product is formed transposed (MFMA rows = n), so that a lane holds one row of `out`, whose scale it multiplies
// with, and four consecutive columns.
//
// The matrix instructions for 8-bit operands add up to 16 neighbouring products at a time in about 14 bits below the largest of them (measured: a
// product of 2^-14 beside one of 1 is lost, beyond those 16 one of 2^-23 is kept).  2-norm relative 1.5e-5 for normally distributed operands: a
// hundredth of the rounding of a bf16 result, but not fp32.  Results in fp32 take their operands as bf16, which hold every e4m3 value
// exactly, at half the rate (8192 x 4096 x 8192 522 us, 1050 TFLOP/s): 4e-9 so.
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

// four consecutive columns of a row of `out`, with the bias
template <typename T>
__device__ __forceinline__ void store_four(const LinearParams &p, int m, int n, f32x4 v)
{
    if (m >= p.M || n >= p.N) {
        return;
    }
    T o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        o[e] = from_f32<T>(p.bias != nullptr && n + e < p.N ? v[e] + p.bias[n + e] : v[e]);
    }
    T *to = (T *)p.out + (int64_t)m * p.out_ld + n;
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

// Tile `index` of the MT x NT tiles of `out`.  Workgroup ids are dealt round robin over the 8 XCDs: each gets a contiguous run of the walk, which
// goes through bands of 8 tiles of rows, column by column, so that the workgroups that run at one time share both operands in their L2.
struct TileOrder {
    int m, n;
};
__device__ __forceinline__ TileOrder tile_order(const LinearParams &p, unsigned index)
{
    const unsigned total = (unsigned)p.MT * (unsigned)p.NT, per = total / 8;
    if (index < per * 8) {
        index = index % 8 * per + index / 8;
    }
    const unsigned band = index / (8u * (unsigned)p.NT), height = min(8u, (unsigned)p.MT - 8 * band), in = index - band * 8u * (unsigned)p.NT;
    return TileOrder{(int)(8 * band + in % height), (int)(in / height)};
}

// ---- rows of fewer than 16 bytes, or very far apart: the waves of a workgroup share the blocks of k ----
//
// 16 MB rows of `out` by 16 NB columns a workgroup, all of them in every wave: wave w takes blocks w, w + W, ... of k, straight from memory
// into registers, and the waves' sums meet in the LDS at the end, in one order.
struct Piece { // 32 bytes of a row of 128: 16 from 16 q on, and 16 from 64 + 16 q on
    uint4 lo, hi;
};

// the last 16 - n bytes of v, then zeros
__device__ __forceinline__ uint4 without_first_bytes(uint4 v, int n)
{
    union {
        uint4 u;
        unsigned __int128 v;
    } c;
    c.u = v;
    c.v = n < 16 ? c.v >> (8 * n) : 0;
    return c.u;
}

// `row`: the row's bytes of this block, `before` of which lie in front of it.  A cut block ends after `left` < 128 bytes; what follows is zero and not read.
__device__ __forceinline__ uint4 load16_cut(const uint8_t *row, int64_t before, int at, int left)
{
    union {
        uint4 u;
        unsigned __int128 v;
    } c;
    c.u = zero_u4();
    if (at >= left) {
        return c.u;
    }
    const int past = at + 16 - left; // of the 16 bytes
    if (past <= 0) {
        __builtin_memcpy(&c.u, row + at, 16);
    } else if (before + at >= past) {
        __builtin_memcpy(&c.u, row + at - past, 16);
        return without_first_bytes(c.u, past);
    } else { // a row of fewer than 16 bytes
#pragma unroll
        for (int i = 0; i < 15; ++i) {
            if (at + i < left) {
                c.v |= (unsigned __int128)row[at + i] << (8 * i);
            }
        }
    }
    return c.u;
}
template <bool CUT>
__device__ __forceinline__ Piece load_piece(const uint8_t *row, int64_t before, int q, int left)
{
    Piece p;
    if constexpr (CUT) {
        p.lo = load16_cut(row, before, 16 * q, left), p.hi = load16_cut(row, before, 64 + 16 * q, left);
    } else {
        __builtin_memcpy(&p.lo, row + 16 * q, 16);
        __builtin_memcpy(&p.hi, row + 64 + 16 * q, 16);
    }
    return p;
}

template <typename T, int MB, int NB, int W>
__global__ __launch_bounds__(64 * W) void fp8_any_kernel(const LinearParams p)
{
    constexpr bool WIDE = std::is_same<T, float>::value || MB == 1; // full fp32 sums, also where memory bounds the time anyway
    extern __shared__ f32x4 sums[]; // [W][NB][MB][64]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int n0 = (int)(blockIdx.x % (unsigned)p.NT) * 16 * NB, m0 = (int)(blockIdx.x / (unsigned)p.NT) * 16 * MB;
    const int whole = p.K / FP8_BLOCK;
    const uint8_t *w_row[NB], *a_row[MB];
    const float *a_scale[MB], *w_scale[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        w_row[i] = p.w + (int64_t)min(n0 + 16 * i + r, p.N - 1) * p.w_ld;
        w_scale[i] = p.w_scales + (int64_t)(min(n0 + 16 * i, p.N - 1) / FP8_BLOCK) * p.w_scales_ld;
    }
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        const int64_t m = min(m0 + 16 * j + r, p.M - 1);
        a_row[j] = p.a + m * p.a_ld, a_scale[j] = p.a_scales + m * p.a_scales_ld;
    }
    f32x4 acc[NB][MB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    struct Block {
        Piece w[NB], a[MB];
        float ws[NB], as[MB];
    };
    auto load = [&](Block &t, int b, auto cut) {
        const int64_t at = (int64_t)b * FP8_BLOCK;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            t.w[i] = load_piece<decltype(cut)::value>(w_row[i] + at, at, q, p.K - (int)at);
            t.ws[i] = w_scale[i][b];
        }
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            t.a[j] = load_piece<decltype(cut)::value>(a_row[j] + at, at, q, p.K - (int)at);
            t.as[j] = a_scale[j][b];
        }
    };
    auto multiply = [&](const Block &t) {
        typename std::conditional<WIDE, WideOperand, i32x8>::type w[NB], a;
        auto take = [&](auto &to, const Piece &piece) {
            if constexpr (WIDE) {
                to = widened(fp8_operand(piece.lo, piece.hi));
            } else {
                to = fp8_operand(piece.lo, piece.hi);
            }
        };
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            take(w[i], t.w[i]);
        }
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            take(a, t.a[j]);
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
                f32x4 part;
                if constexpr (WIDE) {
                    part = mfma_wide(w[i], a, zero);
                } else {
                    part = mfma_fp8(w[i], a, zero);
                }
                const float scale = t.as[j] * t.ws[i];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    acc[i][j][e] = fmaf(part[e], scale, acc[i][j][e]);
                }
            }
        }
    };
    int b = wave;
    for (; b < whole; b += W) {
        Block t;
        load(t, b, std::false_type{});
        multiply(t);
    }
    if (b == whole && p.K % FP8_BLOCK != 0) { // this wave's turn
        Block t;
        load(t, b, std::true_type{});
        multiply(t);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            sums[((wave * NB + i) * MB + j) * 64 + lane] = acc[i][j];
        }
    }
    __syncthreads();
    for (int t = wave; t < NB * MB; t += W) {
        const int i = t / MB, j = t % MB;
        f32x4 sum = sums[t * 64 + lane];
#pragma unroll
        for (int v = 1; v < W; ++v) {
            sum += sums[(v * NB * MB + t) * 64 + lane];
        }
        store_four<T>(p, m0 + 16 * j + r, n0 + 16 * i + 4 * q, sum);
    }
}

int64_t tiles_of(const LinearParams &p, int rows, int columns) { return ((int64_t)p.M + rows - 1) / rows * (((int64_t)p.N + columns - 1) / columns); }

template <typename T, int MB, int NB, int W>
int launch_any(LinearParams p, hipStream_t stream)
{
    const int64_t groups = tiles_of(p, 16 * MB, 16 * NB);
    if (!kutacc_grid_fits(groups, 64 * W)) {
        return KUTACC_HIP_EUNSUPPORTED;
    }
    p.NT = (p.N + 16 * NB - 1) / (16 * NB);
    fp8_any_kernel<T, MB, NB, W><<<dim3((unsigned)groups), 64 * W, (size_t)W * NB * MB * 1024, stream>>>(p);
    return kutacc_hip_status(hipGetLastError());
}

// a dword for each lane, as load_to_lds
__device__ __forceinline__ void load_dword_to_lds(uint32_t to, const void *from, uint32_t lane_bytes)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(to), "v"(lane_bytes), "s"(from) : "memory");
}

// ---- few rows, or few tiles: the same, but a wave brings its blocks into a part of the LDS of its own ----
//
// Eight rows of 128 bytes a load, straight there, the next block while this one is multiplied, and without barriers.  (In the order of the operands, 16 bytes of
// another row in every lane, a load takes the address path some 42 cycles instead of 16.)  Scales come the same way, a lane for each row.  With ANY, where rows are not whole
// 16-byte pieces, a block passes through registers: it is asked for when the operands of the one before are in theirs, and goes into the LDS behind its
// products; past a row's end it is as in the tiles below.  (us, so and with the operands' order: 1000 x 200 x 8001 18 and 86, 16 x 3001 x 8001 10 and 22,
// 1 x 4097 x 4097 7.8 and 10.9, 40 x 3001 x 2001 7.0 and 21.)
template <typename T, int MB, int NB, int W, bool ANY>
__global__ __launch_bounds__(64 * W) void fp8_split_kernel(const LinearParams p)
{
    constexpr bool WIDE = std::is_same<T, float>::value || MB == 1; // full fp32 sums, also where memory bounds the time anyway
    constexpr int SLOTS = (MB + NB) * 128 + 16; // of a block: operands and 64 scales
    extern __shared__ uint4 lds[];              // [W][SLOTS], and at the end sums [W][NB][MB][64]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int n0 = (int)(blockIdx.x % (unsigned)p.NT) * 16 * NB, m0 = (int)(blockIdx.x / (unsigned)p.NT) * 16 * MB;
    const int blocks = (p.K + FP8_BLOCK - 1) / FP8_BLOCK;
    const int chunk = (lane & 7) ^ (lane >> 3);
    const uint8_t *a_tile = p.a + (int64_t)m0 * p.a_ld, *w_tile = p.w + (int64_t)n0 * p.w_ld;
    uint32_t a_from[2 * MB], w_from[2 * NB];
#pragma unroll
    for (int u = 0; u < 2 * MB; ++u) {
        a_from[u] = (uint32_t)min(8 * u + (lane >> 3), p.M - m0 - 1) * (uint32_t)p.a_ld + 16u * (uint32_t)chunk;
    }
#pragma unroll
    for (int u = 0; u < 2 * NB; ++u) {
        w_from[u] = (uint32_t)min(8 * u + (lane >> 3), p.N - n0 - 1) * (uint32_t)p.w_ld + 16u * (uint32_t)chunk;
    }
    const uint32_t scale_from = 4u * (uint32_t)min(lane, min(16 * MB, p.M - m0) - 1) * (uint32_t)p.a_scales_ld;
    const float *a_scales = p.a_scales + (int64_t)m0 * p.a_scales_ld, *w_scales = p.w_scales + (int64_t)(n0 / FP8_BLOCK) * p.w_scales_ld;
    uint4 *mine = lds + wave * SLOTS;
    const uint32_t to = (uint32_t)(uintptr_t)(const lds_char *)mine;
    uint4 held[ANY ? 2 * (MB + NB) : 1];
    float held_scale;
    auto past_end = [&](int b) { return max(0, 16 * chunk + 16 - (p.K - b * FP8_BLOCK)); };
    auto park = [&](int b) {
        if constexpr (ANY) {
            reinterpret_cast<float *>(mine + (MB + NB) * 128)[lane] = held_scale;
            if (p.K - b * FP8_BLOCK >= FP8_BLOCK) {
#pragma unroll
                for (int u = 0; u < 2 * (MB + NB); ++u) {
                    mine[u * 64 + lane] = held[u];
                }
            } else {
#pragma unroll
                for (int u = 0; u < 2 * (MB + NB); ++u) {
                    mine[u * 64 + lane] = without_first_bytes(held[u], past_end(b));
                }
            }
        }
    };
    auto ask = [&](int b) {
        if constexpr (ANY) {
            const int64_t at = (int64_t)b * FP8_BLOCK - past_end(b);
            held_scale = *reinterpret_cast<const float *>(reinterpret_cast<const char *>(a_scales + b) + scale_from);
#pragma unroll
            for (int u = 0; u < 2 * MB; ++u) {
                __builtin_memcpy(&held[u], a_tile + at + a_from[u], 16);
            }
#pragma unroll
            for (int u = 0; u < 2 * NB; ++u) {
                __builtin_memcpy(&held[2 * MB + u], w_tile + at + w_from[u], 16);
            }
            return;
        }
        const uint32_t stage = (uint32_t)__builtin_amdgcn_readfirstlane((int)to); // (known to be the same in all lanes, the compiler keeps its sums in vector registers)
        load_dword_to_lds(stage + (MB + NB) * 2048u, a_scales + b, scale_from);
        if (16 * chunk < p.K - b * FP8_BLOCK) {
#pragma unroll
            for (int u = 0; u < 2 * MB; ++u) {
                load_to_lds(stage + u * 1024u, a_tile + (int64_t)b * FP8_BLOCK, a_from[u]);
            }
#pragma unroll
            for (int u = 0; u < 2 * NB; ++u) {
                load_to_lds(stage + (2 * MB + u) * 1024u, w_tile + (int64_t)b * FP8_BLOCK, w_from[u]);
            }
        } else { // of a cut block, past the end
#pragma unroll
            for (int u = 0; u < 2 * (MB + NB); ++u) {
                mine[u * 64 + lane] = zero_u4();
            }
        }
    };
    f32x4 acc[NB][MB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    if (wave < blocks) {
        ask(wave);
        park(wave);
    }
    float w_scale = wave < blocks ? w_scales[wave] : 0.f;
    for (int b = wave; b < blocks; b += W) {
        if constexpr (!ANY) {
            wait_for_loads<0>();
        }
        const float ws = w_scale;
        if (b + W < blocks) {
            w_scale = w_scales[b + W];
        }
        const float *scales = reinterpret_cast<const float *>(mine + (MB + NB) * 128);
        auto operand_of = [&](int block16) {
            const uint4 *row = mine + (16 * block16 + r) * 8;
            return fp8_operand(row[q ^ (r & 7)], row[(4 + q) ^ (r & 7)]);
        };
        i32x8 w8[NB], a8[MB];
        float scale[MB];
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            w8[i] = operand_of(MB + i);
        }
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            a8[j] = operand_of(j);
            scale[j] = scales[16 * j + r] * ws;
        }
        if (b + W < blocks) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the operands are out of the LDS
            ask(b + W);
        }
        typename std::conditional<WIDE, WideOperand, i32x8>::type w[NB], a;
        auto take = [&](auto &to, i32x8 v) {
            if constexpr (WIDE) {
                to = widened(v);
            } else {
                to = v;
            }
        };
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            take(w[i], w8[i]);
        }
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            take(a, a8[j]);
#pragma unroll
            for (int i = 0; i < NB; ++i) {
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
        if (b + W < blocks) {
            park(b + W);
        }
    }
    __syncthreads(); // the sums take the operands' place
    f32x4 *sums = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
    for (int i = 0; i < NB; ++i) {
#pragma unroll
        for (int j = 0; j < MB; ++j) {
            sums[((wave * NB + i) * MB + j) * 64 + lane] = acc[i][j];
        }
    }
    __syncthreads();
    for (int t = wave; t < NB * MB; t += W) {
        const int i = t / MB, j = t % MB;
        f32x4 sum = sums[t * 64 + lane];
#pragma unroll
        for (int v = 1; v < W; ++v) {
            sum += sums[(v * NB * MB + t) * 64 + lane];
        }
        store_four<T>(p, m0 + 16 * j + r, n0 + 16 * i + 4 * q, sum);
    }
}

template <typename T, int MB, int NB, int W, bool ANY>
int launch_split(LinearParams p, hipStream_t stream)
{
    static_assert(64 * MB * NB <= (MB + NB) * 128 + 16, "the sums lie where the operands were");
    constexpr size_t bytes = (size_t)W * ((MB + NB) * 128 + 16) * 16;
    static size_t configured[KUTACC_DEVICE_SLOTS] = {};
    const auto kernel = &fp8_split_kernel<T, MB, NB, W, ANY>;
    const int64_t groups = tiles_of(p, 16 * MB, 16 * NB);
    if (!kutacc_grid_fits(groups, 64 * W)) {
        return KUTACC_HIP_EUNSUPPORTED;
    }
    p.NT = (p.N + 16 * NB - 1) / (16 * NB);
    if (const hipError_t e = kutacc_opt_in_lds(reinterpret_cast<const void *>(kernel), bytes, configured)) {
        return kutacc_hip_status(e);
    }
    kernel<<<dim3((unsigned)groups), 64 * W, bytes, stream>>>(p);
    return kutacc_hip_status(hipGetLastError());
}

// ---- many rows: WM x WN waves a workgroup, 16 MI rows x 64 columns of `out` a wave: 256 x 256 by 2 x 4 waves or 128 x 128 by 2 x 2 ----
//
// Operands come straight into the LDS (a wave's 64 lanes bring eight rows of 128 bytes a load), a block of 128 k a stage, two stages: a block
// is asked for when the one before the last has been read by all.  The sums of a block are added to a wave's 128 by vector
// instructions, which cannot reach the accumulation registers: more than 128 a wave would not fit beside its operands.
// Two waves a SIMD: one multiplies while the other scales.  8192 x 4096 x 8192: 262 us, 2100 TFLOP/s (a large library product: 2690): the matrix pipe works in
// 47 % of the clocks, the vector issue port in 35 %, four multiply-adds a product.
constexpr int SPAN = 8; // blocks whose scales are brought at a time
constexpr size_t tiles_lds(int side) { return 2 * 2 * side * 128 + 2 * SPAN * side * 4 + 2 * 64 * 4; }

template <typename T, int MI, int WM, int WN, bool ANY>
__global__ __launch_bounds__(64 * WM * WN, 2) void fp8_tiles_kernel(const LinearParams p)
{
    constexpr bool WIDE = std::is_same<T, float>::value;
    constexpr int SIDE = 16 * MI * WM, STAGE = 2 * SIDE * 8; // rows and columns of the tile; 16-byte slots of a stage
    constexpr int HALF = WM * WN / 2;                        // waves that bring a, and as many that bring w
    static_assert(SIDE == 64 * WN && SIDE == 64 * HALF && SPAN % (HALF == 4 ? 2 : 1) == 0, "a wave brings 64 rows");
    extern __shared__ uint4 lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, q = lane >> 4, wm = wave / WN, wn = wave % WN;
    const TileOrder at = tile_order(p, blockIdx.x);
    const int m0 = at.m * SIDE, n0 = at.n * SIDE;
    const int blocks = (p.K + FP8_BLOCK - 1) / FP8_BLOCK;

    // The first half of the waves brings a, the second w: 64 rows each, eight a load; a row's slots are XOR-ed with its number & 7
    const bool brings_a = wave < HALF;
    const int first = 64 * (wave % HALF), rows = (brings_a ? p.M - m0 : p.N - n0) - 1; // rows past the last one bring that one
    const int64_t ld = brings_a ? p.a_ld : p.w_ld;
    const uint8_t *operand = brings_a ? p.a + (int64_t)m0 * ld : p.w + (int64_t)n0 * ld;
    const int chunk = (lane & 7) ^ (lane >> 3);
    uint32_t from[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        from[u] = (uint32_t)min(first + 8 * u + (lane >> 3), rows) * (uint32_t)ld + 16u * (uint32_t)chunk;
    }
    const uint32_t to = (uint32_t)(uintptr_t)(const lds_char *)lds + (brings_a ? 0u : SIDE * 128u) + (uint32_t)first * 128u;
    // With ANY, where rows are not whole 16-byte pieces, a block passes through registers: asked for a block ahead as well, and put into the LDS before the
    // barrier that it has to be there at.  Of a cut block a piece past the row's end is the row's last 16 bytes, shifted by as many as are past it.
    uint4 held[ANY ? 8 : 1];
    auto past_end = [&](int b) { return max(0, 16 * chunk + 16 - (p.K - b * FP8_BLOCK)); };
    auto park = [&](int b, int half) {
        if constexpr (ANY) {
            uint4 *slot = lds + half * STAGE + (brings_a ? 0 : SIDE * 8) + first * 8 + lane;
            if (p.K - b * FP8_BLOCK >= FP8_BLOCK) {
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    slot[u * 64] = held[u];
                }
            } else {
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    slot[u * 64] = without_first_bytes(held[u], past_end(b));
                }
            }
        }
    };
    auto ask = [&](int b, int half) {
        const uint32_t stage = to + (uint32_t)half * (STAGE * 16u);
        const uint8_t *block = operand + (int64_t)b * FP8_BLOCK;
        if constexpr (ANY) {
            block -= past_end(b);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                __builtin_memcpy(&held[u], block + from[u], 16);
            }
            return;
        }
        if (16 * chunk < p.K - b * FP8_BLOCK) {
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                load_to_lds(stage + u * 1024u, block, from[u]);
            }
        } else { // of a cut block, past the end
            uint4 *slot = lds + half * STAGE + (brings_a ? 0 : SIDE * 8) + first * 8 + lane;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                slot[u * 64] = zero_u4();
            }
        }
    };
    // Scales come the same way, for SPAN blocks at a time: [2][SPAN][SIDE rows of a], then [2][2 x SPAN] of w and what else its load brings.  Read
    // where they are needed, a line for each row and block, they were a third of all that the L2 was asked for.
    const float *scales = reinterpret_cast<const float *>(lds + 2 * STAGE);
    const uint32_t scales_to = (uint32_t)(uintptr_t)(const lds_char *)(lds + 2 * STAGE);
    const uint32_t scale_from = 4u * (uint32_t)min(64 * (wave % HALF) + lane, p.M - m0 - 1) * (uint32_t)p.a_scales_ld;
    const int w_blocks_left = (p.N - 1) / FP8_BLOCK - n0 / FP8_BLOCK;
    auto load_scales = [&](int span, int place) {
        const float *a_scales = p.a_scales + (int64_t)m0 * p.a_scales_ld, *w_scales = p.w_scales + (int64_t)(n0 / FP8_BLOCK) * p.w_scales_ld;
#pragma unroll
        for (int u = 0; u < SPAN / 2; ++u) {
            const int k = SPAN / 2 * (wave / HALF) + u;
            load_dword_to_lds(scales_to + 4u * (uint32_t)((place * SPAN + k) * SIDE + 64 * (wave % HALF)), a_scales + min(SPAN * span + k, blocks - 1), scale_from);
        }
        if (wave == 0) {
            const uint32_t from = 4u * ((uint32_t)min((lane / SPAN) & 1, w_blocks_left) * (uint32_t)p.w_scales_ld + (uint32_t)min(SPAN * span + lane % SPAN, blocks - 1));
            load_dword_to_lds(scales_to + 4u * (uint32_t)(2 * SPAN * SIDE + 64 * place), w_scales, from);
        }
    };

    f32x4 acc[4][MI];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < MI; ++j) {
            acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    // Tiles of neighbouring columns start at different blocks: with rows a power of two apart, all rows' bytes of one block lie in one or two
    // channels of the L2.
    int block = (int)((unsigned)at.n * 2u % (unsigned)blocks);
    auto after = [&](int b) { return b + 1 < blocks ? b + 1 : 0; };
    const int odd = r & 7;
    auto operand_of = [&](const uint4 *rows16) {
        const uint4 *row = rows16 + r * 8;
        const i32x8 v = fp8_operand(row[q ^ odd], row[(4 + q) ^ odd]);
        if constexpr (WIDE) {
            return widened(v);
        } else {
            return v;
        }
    };
    auto product = [](const auto &w, const auto &a) {
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        if constexpr (WIDE) {
            return mfma_wide(w, a, zero);
        } else {
            return mfma_fp8(w, a, zero);
        }
    };
    typename std::conditional<WIDE, WideOperand, i32x8>::type w[4], a[2];
    float now[MI], scale_w; // a's scales of the current block, and w's
    auto take_scales = [&](int b, int place) {
        scale_w = scales[2 * SPAN * SIDE + 64 * place + SPAN * (wn / 2) + b % SPAN];
#pragma unroll
        for (int j = 0; j < MI; ++j) {
            now[j] = scales[(place * SPAN + b % SPAN) * SIDE + 16 * MI * wm + 16 * j + r];
        }
    };
    int place = 0, next = after(block); // where the next block's scales lie; the block after this one
    load_scales(block / SPAN, 0);
    ask(block, 0);
    park(block, 0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (blocks > 1) {
        if (next / SPAN != block / SPAN) {
            place = 1;
            load_scales(next / SPAN, 1);
        }
        ask(next, 1);
    }
    take_scales(block, 0);
    a[0] = operand_of(lds + 16 * MI * wm * 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = operand_of(lds + (SIDE + 64 * wn + 16 * i) * 8);
    }
    for (int b = 0; b < blocks; ++b) {
        const uint4 *stage = lds + (b & 1) * STAGE, *other = lds + ((b + 1) & 1) * STAGE;
        float scale[MI];
#pragma unroll
        for (int j = 0; j < MI; ++j) {
            scale[j] = now[j] * scale_w;
        }
        // In a fixed order: product n, the operand that product n + 4 or later takes, and the addition of product n - LAG, whose sums are there by
        // then.  The last four products run behind the barrier at which the stage is given back, and hide the first reads of the next.
        constexpr int LAG = 2;
        f32x4 part[LAG + 1];
        auto add = [&](int n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[n % 4][n / 4][e] = fmaf(part[n % (LAG + 1)][e], scale[n / 4], acc[n % 4][n / 4][e]);
            }
            asm volatile("" : "+v"(acc[n % 4][n / 4])); // stays here: sunk behind the barrier, 112 registers of sums would wait for it
        };
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < 4 * (MI - 1); ++n) {
            const int i = n % 4, j = n / 4;
            part[n % (LAG + 1)] = product(w[i], a[j % 2]);
            if (i == 0) {
                a[(j + 1) % 2] = operand_of(stage + (16 * MI * wm + 16 * (j + 1)) * 8);
            }
            if (n >= LAG) {
                add(n - LAG);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (b + 1 < blocks) {
            park(next, (b + 1) & 1);
        }
        // The next block is there, and all have read this one.  (Behind the last block what is read is never used.)
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        take_scales(next, place);
        if (b + 2 < blocks) {
            const int then = after(next);
            if (then / SPAN != next / SPAN) {
                place ^= 1; // the readers of what lay there have met this barrier
                load_scales(then / SPAN, place);
            }
            ask(then, b & 1);
            next = then;
        }
        a[0] = operand_of(other + 16 * MI * wm * 8);
#pragma unroll
        for (int n = 4 * (MI - 1); n < 4 * MI; ++n) {
            __builtin_amdgcn_sched_barrier(0);
            part[n % (LAG + 1)] = product(w[n % 4], a[1]);
            __builtin_amdgcn_sched_barrier(0);
            w[n % 4] = operand_of(other + (SIDE + 64 * wn + 16 * (n % 4)) * 8);
            add(n - LAG);
        }
#pragma unroll
        for (int n = 4 * MI - LAG; n < 4 * MI; ++n) {
            add(n);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < MI; ++j) {
            store_four<T>(p, m0 + 16 * MI * wm + 16 * j + r, n0 + 64 * wn + 16 * i + 4 * q, acc[i][j]);
        }
    }
}

template <typename T, int MI, int WM, int WN, bool ANY>
int launch_tiles(LinearParams p, hipStream_t stream)
{
    constexpr int SIDE = 16 * MI * WM;
    static size_t configured[KUTACC_DEVICE_SLOTS] = {};
    const auto kernel = &fp8_tiles_kernel<T, MI, WM, WN, ANY>;
    p.MT = (p.M + SIDE - 1) / SIDE, p.NT = (p.N + SIDE - 1) / SIDE;
    const int64_t tiles = tiles_of(p, SIDE, SIDE);
    if (!kutacc_grid_fits(tiles, 64 * WM * WN)) {
        return KUTACC_HIP_EUNSUPPORTED;
    }
    if (const hipError_t e = kutacc_opt_in_lds(reinterpret_cast<const void *>(kernel), tiles_lds(SIDE), configured)) {
        return kutacc_hip_status(e);
    }
    kernel<<<dim3((unsigned)tiles), 64 * WM * WN, tiles_lds(SIDE), stream>>>(p);
    return kutacc_hip_status(hipGetLastError());
}

// Up to 16 rows: columns in blocks of 16, or of 64 where these make half a workgroup a CU and more (us, 16 or 64 wide: 1 x 2048 x 8192 5.6, 8.5;
// 1 x 4096 x 4096 6.1, 6.2; 1 x 8192 x 4096 8.8, 9.0; 1 x 8192 x 8192 13.3, 11.7; 1 x 16384 x 4096 14.1, 11.8).  More rows: the
// largest tile of which there are enough for five in eight of the CUs, or three in four where a tile is a CU's whole work (us: 64 x 4096 x 4096
// on 32 x 32 7.4, on 32 x 64 8.0, on 64 x 64 10.9; 128 rows 12.8, 8.6, 11.0; 256 rows on 32 x 64 14.9, on 64 x 64 11.5, on 128 x 128 26.5;
// 512 rows on 64 x 64 20.7, on 128 x 128 26.4; 700 rows 28.9, 27.0; 1024 rows 41, 28.8, on 256 x 256 58; 3000 rows on 128 x 128 65.3, on
// 256 x 256 64.5; 4096 rows 83, 77).
bool enough(const LinearParams &p, int rows, int columns) { return 8 * tiles_of(p, rows, columns) >= 5 * kutacc_cu_count(); }
bool takes_large_tiles(const LinearParams &p, bool bf16) { return bf16 && 4 * tiles_of(p, 256, 256) >= 3 * kutacc_cu_count(); }
bool takes_tiles(const LinearParams &p, bool bf16) { return p.M > 16 && (takes_large_tiles(p, bf16) || enough(p, 128, 128)); }

template <typename T>
int launch_pieces(const LinearParams &p, hipStream_t stream)
{
    if (p.M <= 16) {
        return 2 * tiles_of(p, 16, 64) >= kutacc_cu_count() ? launch_split<T, 1, 4, 8, false>(p, stream) : launch_split<T, 1, 1, 16, false>(p, stream);
    }
    if constexpr (std::is_same<T, bf16_t>::value) { // in fp32 a wave of these has no registers for its widened operands
        if (takes_large_tiles(p, true)) {
            return launch_tiles<T, 8, 2, 4, false>(p, stream);
        }
    }
    if (takes_tiles(p, false)) {
        return launch_tiles<T, 4, 2, 2, false>(p, stream);
    }
    return enough(p, 64, 64) ? launch_split<T, 4, 4, 8, false>(p, stream) : enough(p, 32, 64) ? launch_split<T, 2, 4, 8, false>(p, stream) : launch_split<T, 2, 2, 16, false>(p, stream);
}

// Rows on any address, of 16 bytes and more: what passes through registers leaves less of them, so 64 x 64 is not among these, nor with fp32 results 32 x 32;
// tiles from three for eight CUs on (us, 32 x 32, 32 x 64 and 128 x 128, bf16 results: 40 x 3001 x 2001 7.0, 8.5, 21; 1000 x 200 x 8001 18, 24, 77;
// 3814 x 112 x 6088 22, 16, 49; 300 x 3001 x 2001 23, 18, 24; 675 x 1751 x 4081 46, 37, 42; 12417 x 128 x 861 27, 20, 13; 4001 x 3001 x 2001 248, 174, 57).
bool takes_any_tiles(const LinearParams &p) { return p.M > 16 && 8 * tiles_of(p, 128, 128) >= 3 * kutacc_cu_count(); }

template <typename T>
int launch_bytes(const LinearParams &p, hipStream_t stream)
{
    if (p.M <= 16) {
        return 2 * tiles_of(p, 16, 64) >= kutacc_cu_count() ? launch_split<T, 1, 4, 8, true>(p, stream) : launch_split<T, 1, 1, 16, true>(p, stream);
    }
    if (takes_any_tiles(p)) {
        return launch_tiles<T, 4, 2, 2, true>(p, stream);
    }
    if constexpr (std::is_same<T, bf16_t>::value) {
        if (!enough(p, 32, 64)) {
            return launch_split<T, 2, 2, 16, true>(p, stream);
        }
    }
    return launch_split<T, 2, 4, 8, true>(p, stream);
}
} // namespace

namespace kutacc_launch {

int linear_fp8(const kutacc_hip_linear_fp8_args_t &a, hipStream_t stream)
{
    const LinearParams p = {(const uint8_t *)a.a, (const uint8_t *)a.w, a.a_scales, a.w_scales, a.bias, a.out, a.a_ld, a.w_ld, a.a_scales_ld,
                            a.w_scales_ld, a.out_ld, (int)a.m, (int)a.n, (int)a.k, 0, 0};
    // rows of a tile within 32 bits of its first; whole 16-byte pieces; at least one piece
    const bool near = a.a_ld < (1 << 23) && a.w_ld < (1 << 23) && a.a_scales_ld < (1 << 21) && a.w_scales_ld < (1 << 21);
    const bool pieces = near && kutacc_hip_aligned16(a.a) && kutacc_hip_aligned16(a.w) && a.a_ld % 16 == 0 && a.w_ld % 16 == 0 && a.k % 16 == 0;
    const bool bytes = near && a.k >= 16;
    const bool tiles = pieces ? takes_tiles(p, a.dtype == KUTACC_DTYPE_BF16) : bytes && takes_any_tiles(p);
    const auto run = [&](auto type) {
        using T = decltype(type);
        return pieces ? launch_pieces<T>(p, stream) : bytes ? launch_bytes<T>(p, stream) : launch_any<T, 4, 4, 4>(p, stream);
    };
    kutacc_prof::KernelTimer t(tiles ? "fp8_tiles_kernel" : pieces || bytes ? "fp8_split_kernel" : "fp8_any_kernel", 2.0 * (double)a.m * (double)a.n * (double)a.k, stream);
    return a.dtype == KUTACC_DTYPE_BF16 ? run(bf16_t{}) : run(float{});
}

} // namespace kutacc_launch
