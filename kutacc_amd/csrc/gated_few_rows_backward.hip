// The backward pass of the gated transition of up to 64 rows, where its time is that of a few round trips to memory: one kernel and the addition of shares.
//
// A workgroup of eight waves owns 32 hidden units.  First g, u and dh of all rows: the waves share the channels, operands straight into registers but the
// columns of Wd, which leave the LDS by its transposing reads; their sums meet in the LDS, in one order.  What the activation and its derivative make of them is
// rounded to bf16 once and stays in the LDS: h, dg and du of 32 units, and what that rounding left, for results that have few values or are sums of few rows,
// and so little to average over: 16 bits of them, for little here (us, with rests and without: 25 x 128 x 512 10.3 and 9.8, 16 x 512 x 2048 20.6 and 19.7).  Then the waves go through
// the channels in blocks of 32, each with its own: the units' rows of the three weights' gradients are whole, as the rows are few enough to be contracted at once,
// and the gradient of x is a share of 32 units, in fp32.
// What bounds it are those trips and the code itself, which is run once: some 6 us at 25 x 128 -> 512, of which the operands of the first products take 1.5, the sums and
// the activation 1.5 (2.7 as straight-line code), the blocks of channels 2.5.  us for the whole pass, this and the kernels for any number of rows: 25 x 128 x 512
// 10.3 and 26, 3 x 256 x 1024 11.6 and 28, 50 x 256 x 896 16.9 and 30, 16 x 512 x 2048 20.6 and 35, 64 x 512 x 2048 28 and 35, 64 x 1024 x 4096 (34 MB of shares) 53 and 51.
//
// All blocks in the LDS are rows of 64 bytes, their four 16-byte slots XOR-ed with bits 2 and 3 of the row's number: 16 rows are 1 KB, which one load of 64 lanes
// brings.  Of such 16 rows a transposing read gives the fragment with k along the rows, column (lane & 31).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "gated_activation.h"
#include "launch_internal.h"
#include "mfma_tiles.h"
#include "profiler.h"

namespace {
using namespace kutacc_dev;

constexpr int UNITS = 32, WAVES = 8, MAX_CHANNELS = 2048; // (of channels, what leaves the LDS room for the columns of Wd)

struct FewRowsParams {
    const bf16_t *x, *grad_out, *gate_w, *up_w, *down_w;
    bf16_t *grad_x, *grad_gate_w, *grad_up_w, *grad_down_w; // or null
    float *shares;                                          // [c_i / 32][rows][c_o]
    int64_t x_ld, grad_out_ld, grad_x_ld;
    int rows, c_o, c_i, activation;
};

// MB blocks of 32 rows
template <int MB, int ACTIVATION>
__global__ __launch_bounds__(64 * WAVES, 2) void gated_few_rows_backward_kernel(const FewRowsParams p)
{
    constexpr int PARTS = WAVES / MB;                         // ways that the channels are split in the first products
    constexpr int ROWS_KB = 2 * MB;                           // of 64-byte rows: two loads for 32
    constexpr int OWN = (2 * ROWS_KB + 4) * 1024;             // a wave's blocks of x and the gradient, Wg and Wu
    extern __shared__ uint4 lds[];                            // [h, dg, du, the rests of dg, du and h: ROWS_KB each], then the columns of Wd, then the sums, then the waves' blocks
    lds_char *const bytes = (lds_char *)lds;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, g = lane >> 5;
    const int unit0 = (int)blockIdx.x * UNITS;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(const lds_char *)lds;
    constexpr bool ALL_RESTS = MB == 1;                              // of two blocks of rows the weights' gradients do without: no registers
    constexpr int REST = (ALL_RESTS ? 6 : 5) * ROWS_KB * 1024;       // where what follows h, dg, du and what their rounding left begins
    // this lane's 16 bytes of 16 rows of 64 bytes, `ld` elements apart
    auto lane_bytes = [&](int64_t ld, int row0, int last) { return 2u * ((uint32_t)min(row0 + (lane >> 2), last) * (uint32_t)ld + 8u * (uint32_t)((lane & 3) ^ ((lane >> 4) & 3))); };
    const int a4 = (lane & 15) >> 2, half16 = (lane >> 4) & 1, quad = lane & 3;
    const int transposed_lane[2] = {(8 * g + a4) * 64 + ((2 * half16 + (quad >> 1)) ^ (2 * g)) * 16 + (quad & 1) * 8,
                                    (8 * g + a4 + 4) * 64 + ((2 * half16 + (quad >> 1)) ^ (2 * g + 1)) * 16 + (quad & 1) * 8};
    auto transposed = [&](int base) { return lds_transposed_fragment(bytes + base + transposed_lane[0], bytes + base + transposed_lane[1]); };

    // ---- g, u and dh: D[unit][row], channels k in steps of 16 ----
    const int rb = MB == 1 ? 0 : wave % MB, part = wave / MB, steps = p.c_o / 16;
    const int first = steps * part / PARTS, end = steps * (part + 1) / PARTS;
    const int row = min(32 * rb + r, p.rows - 1);
    const bf16_t *const x_row = p.x + (int64_t)row * p.x_ld + 8 * g, *const dy_row = p.grad_out + (int64_t)row * p.grad_out_ld + 8 * g;
    const bf16_t *const gate_row = p.gate_w + (int64_t)(unit0 + r) * p.c_o + 8 * g, *const up_row = p.up_w + (int64_t)(unit0 + r) * p.c_o + 8 * g;
    for (int k = first + (MB == 1 ? 0 : rb); k < end; k += MB) { // (the waves of a part share them)
        load_to_lds(lds0 + REST + k * 1024u, same_in_all_lanes(p.down_w + (int64_t)16 * k * p.c_i + unit0), lane_bytes(p.c_i, 0, 15));
    }
    f32x16 sum[3] = {zero16(), zero16(), zero16()};
    bool waits = true; // for the columns of Wd, which all of a part bring
    auto batch = [&](int k, auto count) __attribute__((always_inline)) {
        constexpr int COUNT = decltype(count)::value;
        uint4 xs[COUNT], dys[COUNT], gates[COUNT], ups[COUNT];
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            gates[i] = *reinterpret_cast<const uint4 *>(gate_row + 16 * (k + i)), ups[i] = *reinterpret_cast<const uint4 *>(up_row + 16 * (k + i));
            xs[i] = *reinterpret_cast<const uint4 *>(x_row + 16 * (k + i)), dys[i] = *reinterpret_cast<const uint4 *>(dy_row + 16 * (k + i));
        }
        if (waits) {
            asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
            waits = false;
        }
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
            sum[0] = mfma(as_bf16x8(gates[i]), as_bf16x8(xs[i]), sum[0]);
            sum[1] = mfma(as_bf16x8(ups[i]), as_bf16x8(xs[i]), sum[1]);
            sum[2] = mfma(transposed(REST + (k + i) * 1024), as_bf16x8(dys[i]), sum[2]);
        }
    };
    int k = first;
    for (; k + 4 <= end; k += 4) {
        batch(k, std::integral_constant<int, 4>());
    }
    for (; k < end; ++k) {
        batch(k, std::integral_constant<int, 1>());
    }
    if (waits) { // a part without channels
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    }
    __syncthreads(); // the sums take the place of Wd's columns
    f32x4 *const sums = reinterpret_cast<f32x4 *>(lds + REST / 16);
#pragma unroll
    for (int n = 0; n < 3; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            sums[((wave * 3 + n) * 4 + e) * 64 + lane] = f32x4{sum[n][4 * e], sum[n][4 * e + 1], sum[n][4 * e + 2], sum[n][4 * e + 3]};
        }
    }
    __syncthreads();
    // two units of a row for each thread (and block of rows); loops rather than long code, which is run once and comes from memory as the rest does
    typedef __attribute__((ext_vector_type(2))) float f32x2;
    typedef __attribute__((ext_vector_type(2))) __bf16 two_bf16;
#pragma unroll 1
    for (int of = 0; of < MB; ++of) {
        const int half = wave & 1, e = wave >> 1, at_row = 32 * of + r;
        const f32x2 *from = reinterpret_cast<const f32x2 *>(sums) + (((of * 3) * 4 + e) * 64 + lane) * 2 + half;
        f32x2 v[3] = {from[0], from[512], from[1024]};
#pragma unroll 1
        for (int q = 1; q < PARTS; ++q) {
            from += MB * 3 * 4 * 64 * 2;
            v[0] += from[0], v[1] += from[512], v[2] += from[1024];
        }
        const bool valid = at_row < p.rows; // rows past the last are zeros, and so is all they give
        two_bf16 h, dg, du, h_rest, dg_rest, du_rest;
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            float slope;
            const float a = activate<true>(v[0][f], ACTIVATION, slope);
            const float h32 = valid ? a * v[1][f] : 0.f, dg32 = valid ? v[2][f] * v[1][f] * slope : 0.f, du32 = valid ? v[2][f] * a : 0.f;
            h[f] = (bf16_t)h32, dg[f] = (bf16_t)dg32, du[f] = (bf16_t)du32;
            h_rest[f] = rounding_rest(h32, h[f]), dg_rest[f] = rounding_rest(dg32, dg[f]), du_rest[f] = rounding_rest(du32, du[f]);
        }
        const int to = at_row * 64 + ((e ^ ((at_row >> 2) & 3)) * 16) + g * 8 + half * 4; // units 8 e + 4 g + 2 half ..
        *(__attribute__((address_space(3))) two_bf16 *)(bytes + to) = h;
        *(__attribute__((address_space(3))) two_bf16 *)(bytes + ROWS_KB * 1024 + to) = dg;
        *(__attribute__((address_space(3))) two_bf16 *)(bytes + 2 * ROWS_KB * 1024 + to) = du;
        *(__attribute__((address_space(3))) two_bf16 *)(bytes + 3 * ROWS_KB * 1024 + to) = dg_rest;
        *(__attribute__((address_space(3))) two_bf16 *)(bytes + 4 * ROWS_KB * 1024 + to) = du_rest;
        if constexpr (ALL_RESTS) {
            *(__attribute__((address_space(3))) two_bf16 *)(bytes + 5 * ROWS_KB * 1024 + to) = h_rest;
        }
    }
    __syncthreads();

    // ---- the gradients, 32 channels at a time ----
    bf16x8 h_t[ROWS_KB], dg_t[ROWS_KB], du_t[ROWS_KB]; // k along the rows
    bf16x8 h_rest_t[ALL_RESTS ? ROWS_KB : 1], dg_rest_t[ALL_RESTS ? ROWS_KB : 1], du_rest_t[ALL_RESTS ? ROWS_KB : 1];
    bf16x8 dg[MB][2], du[MB][2], dg_rest[MB][2], du_rest[MB][2]; // k along the units
#pragma unroll
    for (int k = 0; k < ROWS_KB; ++k) {
        h_t[k] = transposed(k * 1024), dg_t[k] = transposed((ROWS_KB + k) * 1024), du_t[k] = transposed((2 * ROWS_KB + k) * 1024);
        if constexpr (ALL_RESTS) {
            dg_rest_t[k] = transposed((3 * ROWS_KB + k) * 1024), du_rest_t[k] = transposed((4 * ROWS_KB + k) * 1024), h_rest_t[k] = transposed((5 * ROWS_KB + k) * 1024);
        }
    }
#pragma unroll
    for (int m = 0; m < MB; ++m) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int slot = (32 * m + r) * 4 + ((2 * s + g) ^ ((r >> 2) & 3));
            dg[m][s] = as_bf16x8(lds[ROWS_KB * 64 + slot]), du[m][s] = as_bf16x8(lds[2 * ROWS_KB * 64 + slot]);
            dg_rest[m][s] = as_bf16x8(lds[3 * ROWS_KB * 64 + slot]), du_rest[m][s] = as_bf16x8(lds[4 * ROWS_KB * 64 + slot]);
        }
    }
    const int own = REST + wave * OWN;
    for (int c0 = 32 * wave; c0 < p.c_o; c0 += 32 * WAVES) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the block before is out of the LDS
#pragma unroll
        for (int k = 0; k < ROWS_KB; ++k) {
            load_to_lds(lds0 + own + k * 1024u, same_in_all_lanes(p.x + c0), lane_bytes(p.x_ld, 16 * k, p.rows - 1));
            load_to_lds(lds0 + own + (ROWS_KB + k) * 1024u, same_in_all_lanes(p.grad_out + c0), lane_bytes(p.grad_out_ld, 16 * k, p.rows - 1));
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            load_to_lds(lds0 + own + (2 * ROWS_KB + k) * 1024u, same_in_all_lanes(p.gate_w + (int64_t)(unit0 + 16 * k) * p.c_o + c0), lane_bytes(p.c_o, 0, 15));
            load_to_lds(lds0 + own + (2 * ROWS_KB + 2 + k) * 1024u, same_in_all_lanes(p.up_w + (int64_t)(unit0 + 16 * k) * p.c_o + c0), lane_bytes(p.c_o, 0, 15));
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        for (int i = 4 * p.rows + lane; i < 4 * 32 * MB; i += 64) { // what was brought in place of rows past the last: 0 times an infinity is no zero
            lds[own / 16 + i] = zero_u4(), lds[own / 16 + 64 * ROWS_KB + i] = zero_u4();
        }
        f32x16 gate_g = zero16(), up_g = zero16(), down_g = zero16(), x_g[MB];
        bf16x8 x_t[ALL_RESTS ? ROWS_KB : 1], dy_t[ALL_RESTS ? ROWS_KB : 1], gate_t[2], up_t[2];
#pragma unroll
        for (int k = 0; k < ROWS_KB; ++k) {
            constexpr int KEPT = ALL_RESTS ? 1 : 0;
            x_t[KEPT * k] = transposed(own + k * 1024), dy_t[KEPT * k] = transposed(own + (ROWS_KB + k) * 1024);
            gate_g = mfma(x_t[KEPT * k], dg_t[k], gate_g);
            up_g = mfma(x_t[KEPT * k], du_t[k], up_g);
            down_g = mfma(h_t[k], dy_t[KEPT * k], down_g);
        }
        // channels c0 + 8 e + 4 g .. of unit or row r; units 8 e + 4 g .. of channel c0 + r
        auto store = [&](bf16_t *to, const f32x16 &v) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                *reinterpret_cast<bf16x4 *>(to + 8 * e) = bf16x4{(bf16_t)v[4 * e], (bf16_t)v[4 * e + 1], (bf16_t)v[4 * e + 2], (bf16_t)v[4 * e + 3]};
            }
        };
        auto store_weights = [&]() {
            const int64_t of_unit = (int64_t)(unit0 + r) * p.c_o + c0 + 4 * g;
            if (p.grad_gate_w != nullptr) {
                store(p.grad_gate_w + of_unit, gate_g);
            }
            if (p.grad_up_w != nullptr) {
                store(p.grad_up_w + of_unit, up_g);
            }
            if (p.grad_down_w != nullptr) {
                store(p.grad_down_w + (int64_t)(c0 + r) * p.c_i + unit0 + 4 * g, down_g);
            }
        };
        if constexpr (!ALL_RESTS) { // now: beside what follows they would not all have registers
            store_weights();
        }
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            x_g[m] = zero16();
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            gate_t[s] = transposed(own + (2 * ROWS_KB + s) * 1024), up_t[s] = transposed(own + (2 * ROWS_KB + 2 + s) * 1024);
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                x_g[m] = mfma(gate_t[s], dg[m][s], x_g[m]);
                x_g[m] = mfma(up_t[s], du[m][s], x_g[m]);
            }
        }
        // What the rounding left, on top.  An infinity among the other operands makes a sum what it is: a rest of the other sign, or of zero, would make it no
        // number.  So where a block has a sum that is not finite, its rests' sums are formed apart, and added to those that are.
        float finite = 0.f; // else no number
        auto look = [&](const f32x16 &v) {
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                finite = fmaf(v[e], 0.f, finite);
            }
        };
        auto rests_of_x = [&](int m, f32x16 &to) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                to = mfma(gate_t[s], dg_rest[m][s], to);
                to = mfma(up_t[s], du_rest[m][s], to);
            }
        };
        [[maybe_unused]] auto rests_of_weights = [&](int which, f32x16 &to) {
            if constexpr (ALL_RESTS) {
#pragma unroll
                for (int k = 0; k < ROWS_KB; ++k) {
                    to = which == 0 ? mfma(x_t[k], dg_rest_t[k], to) : which == 1 ? mfma(x_t[k], du_rest_t[k], to) : mfma(h_rest_t[k], dy_t[k], to);
                }
            }
        };
#pragma unroll
        for (int m = 0; m < MB; ++m) {
            look(x_g[m]);
        }
        if constexpr (ALL_RESTS) {
            look(gate_g), look(up_g), look(down_g);
        }
        if (__builtin_expect(__any(finite != 0.f) == 0, 1)) {
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                rests_of_x(m, x_g[m]);
            }
            rests_of_weights(0, gate_g), rests_of_weights(1, up_g), rests_of_weights(2, down_g);
        } else {
            auto add = [&](f32x16 &sum, const f32x16 &rests) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    sum[e] = __builtin_isfinite(sum[e]) ? sum[e] + rests[e] : sum[e];
                }
            };
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                f32x16 rests = zero16();
                rests_of_x(m, rests);
                add(x_g[m], rests);
            }
            if constexpr (ALL_RESTS) {
                f32x16 rests[3] = {zero16(), zero16(), zero16()};
                rests_of_weights(0, rests[0]), rests_of_weights(1, rests[1]), rests_of_weights(2, rests[2]);
                add(gate_g, rests[0]), add(up_g, rests[1]), add(down_g, rests[2]);
            }
        }
        if constexpr (ALL_RESTS) {
            store_weights();
        }
        if (p.grad_x != nullptr) {
#pragma unroll
            for (int m = 0; m < MB; ++m) {
                if (32 * m + r < p.rows) {
                    float *const to = p.shares + ((int64_t)blockIdx.x * p.rows + 32 * m + r) * p.c_o + c0 + 4 * g;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        *reinterpret_cast<f32x4 *>(to + 8 * e) = f32x4{x_g[m][4 * e], x_g[m][4 * e + 1], x_g[m][4 * e + 2], x_g[m][4 * e + 3]};
                    }
                }
            }
        }
    }
}

// The gradient of x from its shares: four channels of a row a lane; wave w of a workgroup adds shares w, w + 4, ..., and the four sums meet, always in that order.
__global__ __launch_bounds__(256) void gated_few_rows_shares_kernel(const FewRowsParams p)
{
    __shared__ f32x4 sums[3][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row_four = p.c_o / 4, all = p.rows * row_four;
    const int at = (int)blockIdx.x * 64 + lane, shares = p.c_i / UNITS;
    const f32x4 *share = reinterpret_cast<const f32x4 *>(p.shares) + min(at, all - 1);
    f32x4 sum = {0, 0, 0, 0};
#pragma unroll 8
    for (int s = wave; s < shares; s += 4) {
        sum += share[(int64_t)s * all];
    }
    if (wave > 0) {
        sums[wave - 1][lane] = sum;
    }
    __syncthreads();
    if (wave == 0 && at < all) {
        sum = sum + sums[0][lane] + sums[1][lane] + sums[2][lane];
        const bf16x4 o = {(bf16_t)sum[0], (bf16_t)sum[1], (bf16_t)sum[2], (bf16_t)sum[3]};
        *reinterpret_cast<bf16x4 *>(p.grad_x + (int64_t)(at / row_four) * p.grad_x_ld + 4 * (at % row_four)) = o;
    }
}

template <int MB, int ACTIVATION>
hipError_t launch(const FewRowsParams &p, hipStream_t stream)
{
    static size_t configured[KUTACC_DEVICE_SLOTS] = {};
    const auto kernel = &gated_few_rows_backward_kernel<MB, ACTIVATION>;
    constexpr size_t OPERANDS = (MB == 1 ? 6 : 5) * 2 * MB * 1024, SUMS = WAVES * 12 * 1024, BLOCKS = WAVES * (4 * MB + 4) * 1024;
    const size_t bytes = OPERANDS + std::max({SUMS, BLOCKS, (size_t)p.c_o * 64});
    // opted in for the widest rows at once, not for these: a later call with wider ones must not have to, in a capture or beside another thread's first call
    if (const hipError_t e = kutacc_opt_in_lds(reinterpret_cast<const void *>(kernel), OPERANDS + std::max({SUMS, BLOCKS, (size_t)MAX_CHANNELS * 64}), configured)) {
        return e;
    }
    kernel<<<dim3((unsigned)(p.c_i / UNITS)), 64 * WAVES, bytes, stream>>>(p);
    return hipGetLastError();
}
} // namespace

namespace kutacc_launch {

// widths in blocks of 32, and shares of no more than 16 MB
bool gated_few_rows_backward_fits(int64_t rows, int64_t c_o, int64_t c_i)
{
    return rows > 0 && rows <= 64 && c_o > 0 && c_i > 0 && c_o % 32 == 0 && c_i % 32 == 0 && c_o <= MAX_CHANNELS && c_i < (1 << 23) && gated_few_rows_backward_workspace(rows, c_o, c_i) <= (16 << 20);
}

int64_t gated_few_rows_backward_workspace(int64_t rows, int64_t c_o, int64_t c_i) { return c_i / UNITS * rows * c_o * 4; }

bool gated_few_rows_backward_takes(const kutacc_hip_gated_transition_backward_args_t &a)
{
    const int64_t limit = 1 << 23;
    return gated_few_rows_backward_fits(a.rows, a.c_o, a.c_i) && a.x_ld % 8 == 0 && a.grad_out_ld % 8 == 0 && a.grad_x_ld % 4 == 0 && a.x_ld < limit && a.grad_out_ld < limit &&
           kutacc_hip_aligned16(a.x) && kutacc_hip_aligned16(a.grad_out) && kutacc_hip_aligned16(a.grad_x) && kutacc_hip_aligned16(a.gate_w) && kutacc_hip_aligned16(a.up_w) &&
           kutacc_hip_aligned16(a.down_w) && kutacc_hip_aligned16(a.grad_gate_w) && kutacc_hip_aligned16(a.grad_up_w) && kutacc_hip_aligned16(a.grad_down_w);
}

int gated_few_rows_backward(const kutacc_hip_gated_transition_backward_args_t &a, hipStream_t stream)
{
    FewRowsParams p = {(const bf16_t *)a.x, (const bf16_t *)a.grad_out, (const bf16_t *)a.gate_w, (const bf16_t *)a.up_w, (const bf16_t *)a.down_w};
    p.grad_x = (bf16_t *)a.grad_x, p.grad_gate_w = (bf16_t *)a.grad_gate_w, p.grad_up_w = (bf16_t *)a.grad_up_w, p.grad_down_w = (bf16_t *)a.grad_down_w;
    p.shares = (float *)a.workspace;
    p.x_ld = a.x_ld, p.grad_out_ld = a.grad_out_ld, p.grad_x_ld = a.grad_x_ld;
    p.rows = (int)a.rows, p.c_o = (int)a.c_o, p.c_i = (int)a.c_i, p.activation = a.activation;
    kutacc_prof::KernelTimer t("gated_few_rows_backward_kernel", 16.0 * (double)a.rows * (double)a.c_o * (double)a.c_i, stream);
    const bool gelu = a.activation == KUTACC_HIP_GELU;
    const hipError_t e = a.rows <= 32 ? (gelu ? launch<1, KUTACC_HIP_GELU>(p, stream) : launch<1, KUTACC_HIP_SILU>(p, stream))
                                      : (gelu ? launch<2, KUTACC_HIP_GELU>(p, stream) : launch<2, KUTACC_HIP_SILU>(p, stream));
    if (e != hipSuccess || a.grad_x == nullptr) {
        return kutacc_hip_status(e);
    }
    gated_few_rows_shares_kernel<<<dim3((unsigned)((a.rows * a.c_o / 4 + 63) / 64)), 256, 0, stream>>>(p);
    return kutacc_hip_status(hipGetLastError());
}

} // namespace kutacc_launch
