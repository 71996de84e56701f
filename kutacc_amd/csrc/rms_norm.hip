// RMS norm with the residual's addition, into the storage type and / or 8 bits with a scale for 128 channels, its backward pass, and the
// quantiser by itself.
//
//   s = x + residual,  r = 1 / sqrt(mean(s^2) + eps),  y = s r gamma
//   scale = max(max |y| / 448, 2^-126) over a row's channels 128 g .. 128 g + 127,  q = e4m3(y / scale)
// backward, with h = gamma dy:
//   ds = d_sum + r (h - s r^2 mean(h s)),  dgamma = sum over the rows of dy s r
//
// All sums are fp32, and y is formed from s before its rounding to storage.  Memory bounds them: a row is read once, held in
// registers (8 values a lane and chunk) over its reduction, and written once.  TPR threads share a row, each with NV chunks, chunk
// TPR i + thread: whole lines a load, and the 16 lanes whose chunks make up a block of 128 are neighbours, so that a scale costs four DPP
// steps.  8191 x 4096 with a residual and an 8-bit result: 46.5 us, 5.1 TB/s; backward 147456 x 128: 34.6 us, 4.4 TB/s.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "launch_internal.h"
#include "profiler.h"
#include "row_chunks.h"

namespace {
using namespace kutacc_dev;

constexpr int MAX_SIZE = 16384; // of a row: what 1024 threads hold with two chunks each (with four the backward pass has no registers)

// the sum over the TPR threads of a row, in all of them; `waves` where these are a whole workgroup: one float for each of its waves
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float *waves)
{
    if constexpr (TPR <= 64) {
        return group_sum<TPR>(v);
    } else {
        v = group_sum<64>(v);
        if ((threadIdx.x & 63) == 0) {
            waves[threadIdx.x >> 6] = v;
        }
        __syncthreads();
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < TPR / 64; ++w) {
            sum += waves[w];
        }
        return sum;
    }
}

// two sums at once
template <int TPR>
__device__ __forceinline__ void row_sums(float &a, float &b, float *waves)
{
    if constexpr (TPR <= 64) {
        a = group_sum<TPR>(a), b = group_sum<TPR>(b);
    } else {
        a = group_sum<64>(a), b = group_sum<64>(b);
        __syncthreads(); // the last row's sums have been read
        if ((threadIdx.x & 63) == 0) {
            waves[2 * (threadIdx.x >> 6)] = a, waves[2 * (threadIdx.x >> 6) + 1] = b;
        }
        __syncthreads();
        a = b = 0.f;
#pragma unroll
        for (int w = 0; w < TPR / 64; ++w) {
            a += waves[2 * w], b += waves[2 * w + 1];
        }
    }
}

struct NormParams {
    const void *x, *residual;
    void *sum, *out;
    uint8_t *out8;
    const float *gamma;
    float *scales;
    int64_t x_ld, residual_ld, sum_ld, out_ld, out8_ld, scales_ld, rows;
    int size;
    float eps;
};

template <int TPR>
constexpr int threads_of() { return TPR > 256 ? TPR : 256; }

template <typename T, int TPR, int NV>
__global__ __launch_bounds__(threads_of<TPR>()) void rms_norm_kernel(const NormParams p)
{
    constexpr int ROWS = threads_of<TPR>() / TPR;
    __shared__ float waves[threads_of<TPR>() / 64];
    const int t = (int)threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * ROWS + (int)threadIdx.x / TPR;
    const bool there = row < p.rows;
    const int64_t at = there ? row : 0;
    const int size = there ? p.size : 0; // a row past the end reads and writes nothing
    const T *x = (const T *)p.x + at * p.x_ld;
    float v[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        load_chunk(v[i], x, 8 * (TPR * i + t), size);
    }
    if (p.residual != nullptr) {
        const T *residual = (const T *)p.residual + at * p.residual_ld;
        float add[NV][8];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            load_chunk(add[i], residual, 8 * (TPR * i + t), size);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[i][e] += add[i][e];
            }
        }
    }
    float squares = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            squares = fmaf(v[i][e], v[i][e], squares);
        }
    }
    if (p.sum != nullptr) {
        T *sum = (T *)p.sum + at * p.sum_ld;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            store_chunk(v[i], sum, 8 * (TPR * i + t), size);
        }
    }
    const float r = 1.0f / sqrtf(row_sum<TPR>(squares, waves) / (float)p.size + p.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = 8 * (TPR * i + t);
        if (p.gamma != nullptr) {
            float gamma[8];
            load_chunk(gamma, p.gamma, c, p.size);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[i][e] = v[i][e] * r * gamma[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[i][e] *= r;
            }
        }
        if (p.out != nullptr) {
            store_chunk(v[i], (T *)p.out + at * p.out_ld, c, size);
        }
        if (p.out8 != nullptr) {
            const float scale = fp8_scale(lanes_max<(TPR < 16 ? 8 : 16)>(abs_max(v[i])));
            store_fp8_chunk(fp8_quotients(v[i], scale), p.out8 + at * p.out8_ld, c, size);
            if (c < size && c % FP8_BLOCK == 0) {
                p.scales[at * p.scales_ld + c / FP8_BLOCK] = scale;
            }
        }
    }
}

struct BackwardParams {
    const void *x, *grad_out, *grad_sum;
    const float *gamma;
    void *grad_x;
    float *partial; // [workgroups][size]: each one's share of dgamma
    int64_t x_ld, grad_out_ld, grad_sum_ld, grad_x_ld, rows;
    int size;
    float eps;
};

// A workgroup walks rows, ROWS at a time, and keeps its share of dgamma in registers.  The shares meet in the LDS and then, in another kernel,
// over the workgroups, always in one order.  With AHEAD the next rows are on their way while these are reduced and written, as they lie in memory: values
// that a load's own branch converts are waited for there.  us, so and with converted values: bf16 with grad_sum, 5696 x 4096 43.9 and 66.8 (floor 38.3),
// 4238 x 2334 33 and 62, 147456 x 128 35.8 and 37.7 (31.0); fp32 50000 x 256 41.9 (42.0).  TINY: rows of fewer than eight elements.
template <typename T, int TPR, int NV, bool TINY>
__global__ __launch_bounds__(threads_of<TPR>()) void rms_norm_backward_kernel(const BackwardParams p)
{
    constexpr int THREADS = threads_of<TPR>(), ROWS = THREADS / TPR;
    __shared__ float waves[THREADS / 32];
    __shared__ float shares[ROWS > 1 ? THREADS * 8 : 1];
    const int t = (int)threadIdx.x % TPR, group = (int)threadIdx.x / TPR;
    constexpr bool AHEAD = TPR * NV < 2048; // beyond, a thread has no registers for two rows, nor for gamma
    float gamma[NV][8], share[NV][8];
    auto load_gamma = [&](float (&to)[8], int i) {
        if (p.gamma != nullptr) {
            load_chunk(to, p.gamma, 8 * (TPR * i + t), p.size);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            to[e] = p.gamma != nullptr ? to[e] : 1.f;
        }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if constexpr (AHEAD) {
            load_gamma(gamma[i], i);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            share[i][e] = 0.f;
        }
    }
    const bool adds = p.grad_sum != nullptr;
    struct Row {
        RawChunk<T> x[AHEAD ? NV : 1], dy[AHEAD ? NV : 1], ds[AHEAD ? NV : 1];
        float x32[AHEAD ? 1 : NV][8], dy32[AHEAD ? 1 : NV][8];
        bool there;
        int64_t at;
    } now, next;
    auto load = [&](Row &row, int64_t first) {
        row.there = first + group < p.rows;
        row.at = row.there ? first + group : 0; // a row past the last brings the first one, and leaves nothing
        const T *x = (const T *)p.x + row.at * p.x_ld, *dy = (const T *)p.grad_out + row.at * p.grad_out_ld;
        if constexpr (AHEAD && !TINY) {
            const T *ds = adds ? (const T *)p.grad_sum + row.at * p.grad_sum_ld : dy; // without grad_sum, grad_out once more: a branch would wait for what it brings
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = 8 * (TPR * i + t);
                ask_chunk(row.x[i], x, c, p.size), ask_chunk(row.dy[i], dy, c, p.size), ask_chunk(row.ds[i], ds, c, p.size);
            }
        } else if constexpr (!AHEAD) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                load_chunk(row.x32[i], x, 8 * (TPR * i + t), p.size);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                load_chunk(row.dy32[i], dy, 8 * (TPR * i + t), p.size);
            }
        }
    };
    const int64_t step = (int64_t)gridDim.x * ROWS;
    int64_t first = (int64_t)blockIdx.x * ROWS;
    if constexpr (AHEAD) {
        load(now, first);
    }
    for (; first < p.rows; first += step) {
        const bool more = first + step < p.rows;
        if constexpr (!AHEAD) {
            load(now, first);
        } else if (more) {
            load(next, first + step);
        }
        auto take = [&](float (&x)[8], float (&dy)[8], int i) {
            const int c = 8 * (TPR * i + t);
            if constexpr (TINY) {
                load_chunk(x, (const T *)p.x + now.at * p.x_ld, c, p.size), load_chunk(dy, (const T *)p.grad_out + now.at * p.grad_out_ld, c, p.size);
            } else if constexpr (AHEAD) {
                unpack(x, now.x[i], c, p.size), unpack(dy, now.dy[i], c, p.size);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = now.x32[i][e], dy[e] = now.dy32[i][e];
                }
            }
        };
        float squares = 0.f, products = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (!AHEAD) {
                load_gamma(gamma[0], i);
            }
            constexpr int KEPT = AHEAD ? 1 : 0;
            float x[8], dy[8];
            take(x, dy, i);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                squares = fmaf(x[e], x[e], squares);
                products = fmaf(dy[e] * gamma[KEPT * i][e], x[e], products);
            }
        }
        const float n = (float)p.size;
        row_sums<TPR>(squares, products, waves);
        const float r = 1.0f / sqrtf(squares / n + p.eps);
        const float pull = r * (r * (products / n)); // (r^2 may be past 2^128 where x r^2 is not)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = 8 * (TPR * i + t);
            if constexpr (!AHEAD) {
                load_gamma(gamma[0], i);
            }
            constexpr int KEPT = AHEAD ? 1 : 0;
            float x[8], dy[8], dx[8];
            take(x, dy, i);
            if (adds && AHEAD && !TINY) {
                unpack(dx, now.ds[AHEAD ? i : 0], c, p.size);
            } else if (adds) {
                load_chunk(dx, (const T *)p.grad_sum + now.at * p.grad_sum_ld, c, p.size);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float own = r * (dy[e] * gamma[KEPT * i][e] - x[e] * pull);
                dx[e] = adds ? dx[e] + own : own;
                share[i][e] = now.there ? fmaf(dy[e] * x[e], r, share[i][e]) : share[i][e];
            }
            if (p.grad_x != nullptr) {
                store_chunk(dx, (T *)p.grad_x + now.at * p.grad_x_ld, c, now.there ? p.size : 0);
            }
        }
        if (AHEAD && more) {
            now = next;
        }
    }
    if (p.partial == nullptr) {
        return;
    }
    float *partial = p.partial + (int64_t)blockIdx.x * p.size;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if constexpr (ROWS > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                shares[(group * TPR + t) * 8 + e] = share[i][e];
            }
            __syncthreads();
            for (int j = threadIdx.x; j < TPR * 8; j += THREADS) {
                float sum = 0.f;
                for (int g = 0; g < ROWS; ++g) {
                    sum += shares[g * TPR * 8 + j];
                }
                if (8 * TPR * i + j < p.size) {
                    partial[8 * TPR * i + j] = sum;
                }
            }
        } else {
            store_chunk(share[i], partial, 8 * (TPR * i + t), p.size);
        }
    }
}

// dgamma from its shares: 16 columns a workgroup, 64 threads a column
__global__ __launch_bounds__(1024) void column_sums_kernel(const float *partial, float *out, int count, int size)
{
    __shared__ float part[64][17];
    const int c = (int)threadIdx.x & 15, slice = (int)threadIdx.x >> 4, column = (int)blockIdx.x * 16 + c;
    float sum = 0.f;
    if (column < size) {
#pragma unroll 8
        for (int i = slice; i < count; i += 64) {
            sum += partial[(int64_t)i * size + column];
        }
    }
    part[slice][c] = sum;
    __syncthreads();
    if (threadIdx.x < 256) { // 16 threads a column now, each with four of the shares
        const int col = (int)threadIdx.x >> 4, lane = (int)threadIdx.x & 15;
        const float four = (part[lane][col] + part[lane + 16][col]) + (part[lane + 32][col] + part[lane + 48][col]);
        const float all = group_sum<16>(four);
        if (lane == 0 && (int)blockIdx.x * 16 + col < size) {
            out[(int)blockIdx.x * 16 + col] = all;
        }
    }
}

// Blocks of BLOCK_ROWS x 128 values with a scale each: 16 lanes a row of a block, and 256 threads a block of 128 rows (8 rows each)
// or 16 blocks of one row.  Memory bounds blocks of 128 rows, 8192 x 8192 of bf16 42.8 us, 4.7 TB/s, of fp32 59.5 us, 5.6 TB/s; with one row a thread has a
// single load on its way, and two divisions of 64 bits in front of it: 65.7 us, 3.1 TB/s, and 67.1 us, 5.0 TB/s.
struct QuantizeParams {
    const void *x;
    uint8_t *out;
    float *scales;
    int64_t x_ld, out_ld, scales_ld, rows;
    int size, blocks_across;
};

template <typename T, int BLOCK_ROWS>
__global__ __launch_bounds__(256) void quantize_fp8_kernel(const QuantizeParams p)
{
    constexpr int NV = BLOCK_ROWS == 1 ? 1 : BLOCK_ROWS / 16;
    __shared__ float waves[4];
    const int lane16 = (int)threadIdx.x & 15, sub = (int)threadIdx.x >> 4;
    int64_t row0;
    int block;
    bool there = true;
    if constexpr (BLOCK_ROWS == 1) {
        const int64_t unit = (int64_t)blockIdx.x * 16 + sub;
        there = unit < p.rows * p.blocks_across;
        row0 = there ? unit / p.blocks_across : 0;
        block = there ? (int)(unit % p.blocks_across) : 0;
    } else {
        row0 = (int64_t)(blockIdx.x / (unsigned)p.blocks_across) * BLOCK_ROWS + sub;
        block = (int)(blockIdx.x % (unsigned)p.blocks_across);
    }
    const int c = block * FP8_BLOCK + lane16 * 8;
    float v[NV][8], largest = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int64_t row = row0 + 16 * i;
        load_chunk(v[i], (const T *)p.x + (row < p.rows ? row : 0) * p.x_ld, c, there && row < p.rows ? p.size : 0);
        largest = __builtin_elementwise_maximum(largest, abs_max(v[i]));
    }
    largest = lanes_max<16>(largest);
    if constexpr (BLOCK_ROWS != 1) {
        largest = __builtin_elementwise_maximum(largest, __shfl_xor(largest, 16, 64));
        largest = __builtin_elementwise_maximum(largest, __shfl_xor(largest, 32, 64));
        if ((threadIdx.x & 63) == 0) {
            waves[threadIdx.x >> 6] = largest;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            largest = __builtin_elementwise_maximum(largest, waves[w]);
        }
    }
    const float scale = fp8_scale(largest);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int64_t row = row0 + 16 * i;
        if (there && row < p.rows) {
            store_fp8_chunk(fp8_quotients(v[i], scale), p.out + row * p.out_ld, c, p.size);
        }
    }
    if (there && lane16 == 0 && (BLOCK_ROWS == 1 || sub == 0)) {
        p.scales[row0 / BLOCK_ROWS * p.scales_ld + block] = scale;
    }
}

// Threads a row and chunks a thread for a row of `size`, as f(TPR, NV): the fewest that hold it, up to a wave with two chunks ...
template <typename F>
int by_size(int64_t size, F f)
{
    using std::integral_constant;
#define KUTACC_ROW(limit, tpr, nv)                                                   \
    if (size <= (limit)) {                                                            \
        return f(integral_constant<int, tpr>{}, integral_constant<int, nv>{});        \
    }
    KUTACC_ROW(64, 8, 1)
    KUTACC_ROW(128, 16, 1)
    KUTACC_ROW(256, 32, 1)
    KUTACC_ROW(512, 64, 1)
    KUTACC_ROW(1024, 64, 2)
    KUTACC_ROW(2048, 256, 1) // ... then workgroups
    KUTACC_ROW(4096, 256, 2)
    KUTACC_ROW(8192, 512, 2)
    KUTACC_ROW(MAX_SIZE, 1024, 2)
#undef KUTACC_ROW
    return KUTACC_HIP_EUNSUPPORTED;
}

template <typename F>
int by_type(int32_t dtype, F f)
{
    return dtype == KUTACC_DTYPE_BF16 ? f(bf16_t{}) : f(float{});
}

// Workgroups of the backward pass, each with its share of dgamma: as many as are on the chip at a time.  One alone writes dgamma itself, which saves the second
// kernel where it has few rounds of rows to go through (us, so and with shares: 2 x 1256 4.7 and 8.1, 8 x 1024 5.3 and 7.3, 16 x 512 (four rounds) 5.4 and 7.3,
// 3 x 8192 (three) 8.1 and 7.4, 4 x 8192 10.2 and 7.8).  Four for a CU with short rows of bf16, else two (two, four and eight: 147456 x 128 bf16 33.7, 28.9, 31.0,
// fp32 45, 50, 50; 20000 x 512 20.5, 19.4, 21.6, fp32 28, 32, 33; 10000 x 1024 18.4, 21.4, 24.7), and one where a row's
// threads fill the CU (one and two: 2000 x 8192 34.4 and 40.2, 700 x 12000 24.3 and 30.7).
int64_t backward_groups(int64_t rows, int64_t size, bool bf16)
{
    int per_group = 1;
    (void)by_size(size, [&](auto tpr, auto) {
        per_group = threads_of<decltype(tpr)::value>() / decltype(tpr)::value;
        return 0;
    });
    const int64_t needed = (rows + per_group - 1) / per_group;
    if (needed <= (size <= 2048 ? 4 : 2)) {
        return 1;
    }
    return std::min<int64_t>(needed, (size <= 512 && bf16 ? 4 : size <= 4096 ? 2 : 1) * (int64_t)kutacc_cu_count());
}
} // namespace

namespace kutacc_launch {

int rms_norm(const kutacc_hip_rms_norm_args_t &a, hipStream_t stream)
{
    return by_type(a.dtype, [&](auto type) {
        return by_size(a.size, [&](auto tpr, auto nv) {
            using T = decltype(type);
            constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value, THREADS = threads_of<TPR>(), PER_GROUP = THREADS / TPR;
            constexpr int64_t MOST = (int64_t)(UINT32_MAX / THREADS) * PER_GROUP; // rows of a launch
            kutacc_prof::KernelTimer t("rms_norm_kernel", 8.0 * (double)a.rows * (double)a.size, stream);
            for (int64_t first = 0; first < a.rows; first += MOST) {
                const auto from = [&](auto *rows, int64_t ld) { return rows != nullptr ? rows + first * ld : nullptr; };
                const int64_t rows = std::min(a.rows - first, MOST);
                const NormParams p = {from((const T *)a.x, a.x_ld), from((const T *)a.residual, a.residual_ld), from((T *)a.sum, a.sum_ld), from((T *)a.out, a.out_ld),
                                      from((uint8_t *)a.out8, a.out8_ld), a.gamma, from(a.scales, a.scales_ld),
                                      a.x_ld, a.residual_ld, a.sum_ld, a.out_ld, a.out8_ld, a.scales_ld, rows, (int)a.size, a.eps};
                rms_norm_kernel<T, TPR, NV><<<dim3((unsigned)((rows + PER_GROUP - 1) / PER_GROUP)), THREADS, 0, stream>>>(p);
                if (const hipError_t e = hipGetLastError()) {
                    return kutacc_hip_status(e);
                }
            }
            return 0;
        });
    });
}

int64_t rms_norm_backward_workspace(int64_t rows, int64_t size) { return backward_groups(rows, size, true) * size * (int64_t)sizeof(float); }

int rms_norm_backward(const kutacc_hip_rms_norm_backward_args_t &a, hipStream_t stream)
{
    const int64_t groups = backward_groups(a.rows, a.size, a.dtype == KUTACC_DTYPE_BF16);
    const BackwardParams p = {a.x, a.grad_out, a.grad_sum, a.gamma, a.grad_x, groups == 1 || a.grad_gamma == nullptr ? a.grad_gamma : (float *)a.workspace,
                              a.x_ld, a.grad_out_ld, a.grad_sum_ld, a.grad_x_ld, a.rows, (int)a.size, a.eps};
    const int rc = by_type(a.dtype, [&](auto type) {
        return by_size(a.size, [&](auto tpr, auto nv) {
            constexpr int TPR = decltype(tpr)::value, NV = decltype(nv)::value;
            kutacc_prof::KernelTimer t("rms_norm_backward_kernel", 12.0 * (double)p.rows * (double)p.size, stream);
            if (TPR == 8 && p.size < 8) {
                rms_norm_backward_kernel<decltype(type), 8, 1, true><<<dim3((unsigned)groups), threads_of<TPR>(), 0, stream>>>(p);
            } else {
                rms_norm_backward_kernel<decltype(type), TPR, NV, false><<<dim3((unsigned)groups), threads_of<TPR>(), 0, stream>>>(p);
            }
            return kutacc_hip_status(hipGetLastError());
        });
    });
    if (rc != 0 || a.grad_gamma == nullptr || groups == 1) {
        return rc;
    }
    kutacc_prof::KernelTimer t("column_sums_kernel", (double)groups * (double)a.size, stream);
    column_sums_kernel<<<dim3((unsigned)((a.size + 15) / 16)), 1024, 0, stream>>>(p.partial, a.grad_gamma, (int)groups, (int)a.size);
    return kutacc_hip_status(hipGetLastError());
}

int quantize_fp8(const void *x, int64_t x_ld, void *out, int64_t out_ld, float *scales, int64_t scales_ld, int64_t rows, int64_t size,
                 int32_t block_rows, int32_t dtype, hipStream_t stream)
{
    const int across = (int)((size + FP8_BLOCK - 1) / FP8_BLOCK);
    const int64_t groups = UINT32_MAX / 256, most = block_rows == 1 ? groups * 16 / across : groups / across * FP8_BLOCK; // rows of a launch
    return by_type(dtype, [&](auto type) {
        using T = decltype(type);
        kutacc_prof::KernelTimer t("quantize_fp8_kernel", (double)rows * (double)size, stream);
        for (int64_t first = 0; first < rows; first += most) {
            const int64_t count = std::min(rows - first, most);
            const QuantizeParams p = {(const T *)x + first * x_ld, (uint8_t *)out + first * out_ld, scales + first / block_rows * scales_ld, x_ld, out_ld, scales_ld, count, (int)size, across};
            if (block_rows == 1) {
                quantize_fp8_kernel<T, 1><<<dim3((unsigned)((count * across + 15) / 16)), 256, 0, stream>>>(p);
            } else {
                quantize_fp8_kernel<T, FP8_BLOCK><<<dim3((unsigned)((count + FP8_BLOCK - 1) / FP8_BLOCK * across)), 256, 0, stream>>>(p);
            }
            if (const hipError_t e = hipGetLastError()) {
                return kutacc_hip_status(e);
            }
        }
        return 0;
    });
}

bool rms_norm_supports(int64_t size) { return size <= MAX_SIZE; }

} // namespace kutacc_launch
