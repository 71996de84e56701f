// The backward pass of the gated transition of 64 and 128 channels: the hidden layer stays on chip, formed once for the gradient of x and once more for those
// of the weights.  With so few channels that costs less than its way through memory: at 65536 rows, 128 -> 512, 94 GFLOP in place of 69, but h, dg and du are
// 200 MB to write and to read again (us for the whole pass: 112; a kernel that stored them beside the gradient of x, and products of tiles: 88 + 60; products of
// tiles alone: 174).
//
// The gradient of x: a wave owns 32 rows of x and of the gradient of out as operand fragments in registers, and walks the hidden layer in slices of 32 units
// that come straight into the LDS: g and u from x, dh from the gradient, in 32 bits; what the activation and its derivative make of them is rounded to bf16
// once, as operands (row i of a first product is hidden unit sigma(i), bits 2 and 3 of i swapped, so that a lane's eight values per k-step are consecutive
// units).  The gradient of x is two more products with the same slices: these contract over the slice's rows, and dh over the rows of Wd, so their operands
// leave the LDS by its transposing reads.  65536 rows, 128 -> 512: 46 us, 920 TFLOP/s of the 1380 that a large product reaches; the activation takes a third
// of the vector instructions' time, and the other wave of a SIMD hides only part of it.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "gated_activation.h"
#include "launch_internal.h"
#include "mfma_tiles.h"
#include "profiler.h"

namespace {
using namespace kutacc_dev;

struct BackwardParams {
    const bf16_t *x, *grad_out, *gate_w, *up_w, *down_w;
    bf16_t *grad_x;
    bf16_t *grad_gate_w, *grad_up_w, *grad_down_w; // or null
    float *shares;                                 // [splits][units of 32][3][CO / 32][4][64] times four values
    int64_t x_ld, grad_out_ld, grad_x_ld, rows;
    int splits, split_blocks;                      // blocks of 32 rows in a split
    int c_i, activation;
    int full_groups, tail_waves; // workgroups whose waves all have rows, and how many waves of the others have
};

template <int CO, int WAVES, int GROUPS, int ACTIVATION>
__global__ __launch_bounds__(64 * WAVES, GROUPS * WAVES / 4) void gated_input_gradient_kernel(const BackwardParams p)
{
    constexpr int KS = CO / 16, CP = CO / 64, CB = CO / 32;
    constexpr int MATRIX = 4 * CO, STAGE = 3 * MATRIX; // 16-byte slots: 32 hidden units of a matrix, and of all three
    constexpr int MATRIX_UNITS = CO / 16, UPW = 3 * MATRIX_UNITS / WAVES;
    static_assert(UPW * WAVES == 3 * MATRIX_UNITS, "all waves bring as much");
    extern __shared__ uint4 lds[]; // [2][gate, up, down], and what the waves' panels take beyond the second
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, g = lane >> 5, slices = p.c_i / 32;

    const int past = (int)blockIdx.x - p.full_groups;
    const bool has_rows = past < 0 || wave < p.tail_waves; // the other waves only bring weights
    int64_t row0 = (past < 0 ? (int64_t)blockIdx.x * WAVES + wave : (int64_t)p.full_groups * WAVES + (int64_t)past * p.tail_waves + wave) * 32;
    const bool active = has_rows && row0 < p.rows;
    if (!active) {
        row0 = p.rows - 1; // keeps every address valid; nothing is stored
    }
    const int last_local = (int)(p.rows - row0 < 32 ? p.rows - row0 : 32) - 1;
    PanelRegs x_panels[CP], dy_panels[CP];
#pragma unroll
    for (int cp = 0; cp < CP; ++cp) {
        x_panels[cp] = panel_load(p.x + row0 * p.x_ld, p.x_ld, 0, last_local, cp * 64, lane);
        dy_panels[cp] = panel_load(p.grad_out + row0 * p.grad_out_ld, p.grad_out_ld, 0, last_local, cp * 64, lane);
    }

    const uint32_t lds0 = (uint32_t)(uintptr_t)(const lds_char *)lds + (uint32_t)(wave * UPW) * 1024u;
    uint32_t lane_bytes[UPW];
    const char *source[UPW];
    int64_t pitch[UPW]; // bytes from a slice to the next
#pragma unroll
    for (int i = 0; i < UPW; ++i) {
        const int unit = wave * UPW + i, matrix = unit / MATRIX_UNITS, u = unit % MATRIX_UNITS, rl = lane >> 3;
        if (matrix < 2) { // row i of the panel is hidden unit sigma(i); rows 16 - 31 swizzle with bit 0 flipped
            source[i] = reinterpret_cast<const char *>((matrix == 0 ? p.gate_w : p.up_w) + (4 * (u & 1) + 16 * ((u >> 1) & 1)) * CO + (u >> 2) * 64);
            lane_bytes[i] = 2u * (uint32_t)(((rl & 3) | ((rl & 4) << 1)) * CO + 8 * ((lane & 7) ^ rl ^ ((u >> 1) & 1)));
            pitch[i] = 64 * CO;
        } else {
            source[i] = reinterpret_cast<const char *>(p.down_w + (int64_t)u * 16 * p.c_i);
            lane_bytes[i] = 2u * (uint32_t)((lane >> 2) * p.c_i + 8 * ((lane & 3) ^ ((lane >> 4) & 3)));
            pitch[i] = 64;
        }
    }
    auto ask = [&](int half) { // the next slice
#pragma unroll
        for (int i = 0; i < UPW; ++i) {
            load_to_lds(lds0 + (uint32_t)half * (STAGE * 16u) + i * 1024u, same_in_all_lanes(source[i]), lane_bytes[i]);
            source[i] += pitch[i];
        }
    };
    ask(0);

    bf16x8 x[KS], dy[KS];
    uint4 *const panel = lds + STAGE + wave * 256; // the second stage is still free
#pragma unroll
    for (int cp = 0; cp < CP; ++cp) {
        panel_store(panel, lane, x_panels[cp]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            x[cp * 4 + k] = as_bf16x8(panel[panel_slot(r, 2 * k + g)]);
        }
    }
#pragma unroll
    for (int cp = 0; cp < CP; ++cp) {
        panel_store(panel, lane, dy_panels[cp]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            dy[cp * 4 + k] = as_bf16x8(panel[panel_slot(r, 2 * k + g)]);
        }
    }
    f32x16 sum[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        sum[cb] = zero16();
    }
    const int w1_lane = panel_slot(r, g);
    auto gate_slot = [&](int k) { return (k / 4) * 256 + (w1_lane ^ (2 * (k % 4))); };
    // Transposed fragments.  Within 16 lanes a lane points at row a = (lane & 15) >> 2 of four, and at four columns.  Of the gate's and the other
    // projection's panels: rows are hidden units 16 s + 8 g + 4 t + a, at i = sigma of that, columns the channels 32 cb + 16 ((lane >> 4) & 1) + 4 (lane & 3).
    const int a4 = (lane & 15) >> 2, half16 = (lane >> 4) & 1, quad = lane & 3;
    const lds_char *const bytes = (const lds_char *)lds;
    auto panel_transposed = [&](int base, int cb, int s) { // `base` in bytes
        const int slot = ((cb & 1) * 4 + 2 * half16 + (quad >> 1)) ^ (a4 + 4 * g) ^ s;
        const int at = base + (cb >> 1) * 4096 + (a4 + 4 * g + 16 * s) * 128 + slot * 16 + (quad & 1) * 8;
        return lds_transposed_fragment(bytes + at, bytes + at + 8 * 128);
    };
    // Of Wd's slice: rows are channels 16 k + 8 g + 4 t + a, columns the hidden units of row sigma(lane & 31) of the product, so of two quads of columns the
    // inner ones change places.
    const int hidden_quad = 4 * half16 + ((quad & 1) << 1 | quad >> 1);
    auto down_transposed = [&](int base, int k) {
        const int row = 16 * k + 8 * g + a4;
        const int lo = base + row * 64 + (((hidden_quad >> 1) ^ (2 * g)) * 16) + (hidden_quad & 1) * 8;
        const int hi = base + (row + 4) * 64 + (((hidden_quad >> 1) ^ (2 * g + 1)) * 16) + (hidden_quad & 1) * 8;
        return lds_transposed_fragment(bytes + lo, bytes + hi);
    };
    __syncthreads(); // the panels
    for (int j = 0; j < slices; ++j) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); // this slice is there, and all are done with the one before
        if (j + 1 < slices) {
            ask((j + 1) & 1);
        }
        if (!active) {
            continue;
        }
        const uint4 *stage = lds + (j & 1) * STAGE;
        const int at = (j & 1) * STAGE * 16;
        f32x16 gate = zero16(), up = zero16(), dh = zero16();
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            gate = mfma(as_bf16x8(stage[gate_slot(k)]), x[k], gate);
            up = mfma(as_bf16x8(stage[MATRIX + gate_slot(k)]), x[k], up);
            dh = mfma(down_transposed(at + 2 * MATRIX * 16, k), dy[k], dh);
        }
        bf16x8 dg[2], du[2];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            float slope;
            const float a = activate<true>(gate[e], ACTIVATION, slope);
            dg[e / 8][e % 8] = (bf16_t)(dh[e] * up[e] * slope);
            du[e / 8][e % 8] = (bf16_t)(dh[e] * a);
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                sum[cb] = mfma(panel_transposed(at, cb, s), dg[s], sum[cb]);
                sum[cb] = mfma(panel_transposed(at + MATRIX * 16, cb, s), du[s], sum[cb]);
            }
        }
    }
    __syncthreads(); // the results take the stages' place
    if (!active) {
        return;
    }
    uint4 *const strip = lds + wave * 256;
#pragma unroll
    for (int cp = 0; cp < CP; ++cp) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                bf16x4 o;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    o[c] = (bf16_t)sum[2 * cp + n][4 * a + c];
                }
                *(reinterpret_cast<bf16x4 *>(strip + panel_slot(r, n * 4 + a)) + g) = o;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int row = 8 * i + (lane >> 3);
            if (row <= last_local) {
                *reinterpret_cast<uint4 *>(p.grad_x + (row0 + row) * p.grad_x_ld + cp * 64 + (lane & 7) * 8) = strip[panel_slot(row, lane & 7)];
            }
        }
    }
}

// ---- the gradients of the weights ----
//
// A wave owns 32 hidden units: their rows of Wg and Wu and their column of Wd as operands in registers, and the three sums.  It walks blocks of 32 rows that
// come straight into the LDS for all waves of the workgroup, x and the gradient of out, in the order sigma, and forms what the other kernel forms, the other
// way round (MFMA columns = hidden units): rounded to bf16, h, dg and du are operands of products that contract over the rows, whose other operands leave the
// LDS by the transposing reads.  Nothing of the hidden layer goes to memory.  The sums of 32 units, three times 32 x 128, are 192 registers and the weights 96:
// one wave a SIMD, whose products run beside its own activation.  The rows are split over as many workgroups as there are CUs, each with a share of the sums:
// 65536 rows, 128 -> 512: 59 us and 8 for adding the shares (50 MB).  Without activation and LDS reads it would take 48: the products
// themselves, at the rate that they reach here, bound it.
template <int CO, int ACTIVATION>
__global__ __launch_bounds__(256, 1) void gated_weight_gradients_kernel(const BackwardParams p)
{
    constexpr int KS = CO / 16, CB = CO / 32, WAVES = 4, STAGES = 6, AHEAD = 6;
    constexpr int PANEL = 4 * CO, STAGE = 2 * PANEL;      // 16-byte slots of 32 rows of x, and of both
    constexpr int UNITS = CO / 16, UPW = 2 * UNITS / WAVES; // loads of 1 KB: of 32 rows of x, and of a wave
    extern __shared__ uint4 lds[];                          // [STAGES][x, gradient of out]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 31, g = lane >> 5;
    const int groups = (p.c_i + 127) / 128, group = (int)blockIdx.x % groups, split = (int)blockIdx.x / groups;
    const int unit0 = 128 * group + 32 * wave;
    const bool active = unit0 < p.c_i;
    const int64_t row_blocks = (p.rows + 31) / 32, block0 = (int64_t)split * p.split_blocks;
    const int blocks = (int)(row_blocks - block0 < p.split_blocks ? row_blocks - block0 : p.split_blocks);
    const int64_t last_row0 = (block0 + blocks - 1) * 32; // the walk is from the last block to the first, so that one with fewer rows comes first
    const int valid = (int)(p.rows - last_row0 < 32 ? p.rows - last_row0 : 32);

    const uint32_t lds0 = (uint32_t)(uintptr_t)(const lds_char *)lds + (uint32_t)(wave * UPW) * 1024u;
    uint32_t lane_bytes[UPW], first_bytes[UPW];
    const char *source[UPW];
    int64_t pitch[UPW];
#pragma unroll
    for (int i = 0; i < UPW; ++i) { // row i of a panel is row sigma(i) of the block; rows 16 - 31 swizzle with bit 0 flipped
        const int unit = wave * UPW + i, of = unit / UNITS, u = unit % UNITS, rl = lane >> 3;
        const int64_t ld = of == 0 ? p.x_ld : p.grad_out_ld;
        const int row = ((rl & 3) | ((rl & 4) << 1)) + 4 * (u & 1) + 16 * ((u >> 1) & 1), chunk = 16 * ((lane & 7) ^ rl ^ ((u >> 1) & 1));
        source[i] = reinterpret_cast<const char *>((of == 0 ? p.x : p.grad_out) + last_row0 * ld + (u >> 2) * 64);
        first_bytes[i] = 2u * (uint32_t)(row < valid ? row : valid - 1) * (uint32_t)ld + (uint32_t)chunk;
        lane_bytes[i] = blocks == 1 ? first_bytes[i] : 2u * (uint32_t)row * (uint32_t)ld + (uint32_t)chunk;
        pitch[i] = 64 * ld;
    }
    auto ask_unit = [&](int i, int b, uint32_t bytes) {
        load_to_lds(lds0 + (uint32_t)(b % STAGES) * (STAGE * 16u) + i * 1024u, same_in_all_lanes(source[i] - (b < blocks ? b : blocks - 1) * pitch[i]), bytes);
    };
#pragma unroll
    for (int i = 0; i < UPW; ++i) {
        ask_unit(i, 0, first_bytes[i]);
    }

#pragma unroll
    for (int b = 1; b < STAGES - 2; ++b) {
#pragma unroll
        for (int i = 0; i < UPW; ++i) {
            ask_unit(i, b, lane_bytes[i]); // behind the last block, that block again
        }
    }
    // the columns of Wd, rows of 64 bytes, into the last two stages
    const bf16_t *down = p.down_w + (active ? unit0 : 0);
    const uint32_t down_to = (uint32_t)(uintptr_t)(const lds_char *)lds + (uint32_t)((STAGES - 2) * STAGE * 16 + wave * 64 * CO);
    static_assert(WAVES * 64 * CO <= 2 * STAGE * 16, "as much as two stages hold");
#pragma unroll
    for (int u = 0; u < CO / 16; ++u) {
        load_to_lds(down_to + u * 1024u, same_in_all_lanes(down + (int64_t)u * 16 * p.c_i), 2u * (uint32_t)((lane >> 2) * p.c_i + 8 * ((lane & 3) ^ ((lane >> 4) & 3))));
    }
    const int64_t unit = active ? unit0 + r : 0;
    bf16x8 wg[KS], wu[KS], wd[KS]; // of unit r
#pragma unroll
    for (int k = 0; k < KS; ++k) {
        wg[k] = as_bf16x8(*reinterpret_cast<const uint4 *>(p.gate_w + unit * CO + 16 * k + 8 * g));
        wu[k] = as_bf16x8(*reinterpret_cast<const uint4 *>(p.up_w + unit * CO + 16 * k + 8 * g));
    }
    const int a4 = (lane & 15) >> 2, half16 = (lane >> 4) & 1, quad = lane & 3; // transposed, within 16 lanes a lane points at one row of four, and at four columns
    const lds_char *const bytes = (const lds_char *)lds;
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
    for (int k = 0; k < KS; ++k) { // rows are channels 16 k + 8 g + 4 t + (0 .. 3)
        const lds_char *const from = bytes + (STAGES - 2) * STAGE * 16 + wave * 64 * CO + (16 * k + 8 * g + a4) * 64 + (quad & 1) * 8;
        const int chunk = 2 * half16 + (quad >> 1);
        wd[k] = lds_transposed_fragment(from + (chunk ^ (2 * g)) * 16, from + 256 + (chunk ^ (2 * g + 1)) * 16);
    }
    if (valid < 32) { // rows past the last are zeros, and so is all they give
        for (int i = tid; i < 2 * 32 * (CO / 8); i += 256) {
            const int at = i / 8 % 32, row = (at & 19) | ((at & 4) << 1) | ((at & 8) >> 1);
            if (row >= valid) {
                lds[i] = make_uint4(0, 0, 0, 0);
            }
        }
    }
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); // Wd's columns are in registers
#pragma unroll
    for (int i = 0; i < UPW; ++i) {
        ask_unit(i, STAGES - 2, lane_bytes[i]);
    }

    // until block b is there for all: what is younger may be on its way
    auto meet = [&]() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"((STAGES - 3) * UPW) : "memory"); };
    if (!active) { // brings rows only
        for (int b = 0; b < blocks; ++b) {
            meet();
#pragma unroll
            for (int i = 0; i < UPW; ++i) {
                ask_unit(i, b + STAGES - 1, lane_bytes[i]);
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        return;
    }
    f32x16 sum[3][CB];
#pragma unroll
    for (int n = 0; n < 3 * CB; ++n) {
        sum[n / CB][n % CB] = zero16();
    }
    const int row_lane = panel_slot(r, g);
    auto rows_fragment = [&](int stage, int of, int k) { return as_bf16x8(lds[stage * STAGE + of * PANEL + (k / 4) * 256 + (row_lane ^ (2 * (k % 4)))]); };
    auto transposed = [&](int stage, int of, int cb, int s) {
        const int slot = ((cb & 1) * 4 + 2 * half16 + (quad >> 1)) ^ (a4 + 4 * g) ^ s;
        const int at = (stage * STAGE + of * PANEL) * 16 + (cb >> 1) * 4096 + (a4 + 4 * g + 16 * s) * 128 + slot * 16 + (quad & 1) * 8;
        return lds_transposed_fragment(bytes + at, bytes + at + 8 * 128);
    };
    // Fragments and products of a step, in the order that they are formed: of block j the first products (fragment 2 k of x: g and u; 2 k + 1 of the gradient:
    // dh), of block j - 1 the last ones (fragment 2 n of x: dWg and dWu; 2 n + 1 of the gradient: dWd).
    constexpr int FIRST = 2 * KS, EARLY = FIRST * 3 / 4, LAST = 2 * CB, TOTAL = FIRST + 2 * LAST;
    f32x16 gate, up, dh;
    bf16x8 h[2], dg[2], du[2], ready[AHEAD];
    auto index_of = [](int m) { // first ones 0 .. FIRST - 1, last ones from FIRST on
        return m < EARLY ? m : m < EARLY + LAST ? FIRST + m - EARLY : m < FIRST + LAST ? m - LAST : m;
    };
    float t[16], a[16];
    auto part = [&](int n) { // of the activation: the exponential of value n, the sigmoid of value n - 1, the operands of value n - 2
        if (n < 16) {
            t[n] = 1.0f + __builtin_amdgcn_exp2f(activation_exponent(gate[n], ACTIVATION));
        }
        if (n >= 1 && n < 17) {
            t[n - 1] = __builtin_amdgcn_rcpf(t[n - 1]);
        }
        if (n >= 2) {
            const int e = n - 2;
            float slope;
            const float act = activation_of_sigmoid(gate[e], t[e], ACTIVATION, slope);
            h[e / 8][e % 8] = (bf16_t)(act * up[e]);
            dg[e / 8][e % 8] = (bf16_t)(dh[e] * up[e] * slope);
            du[e / 8][e % 8] = (bf16_t)(dh[e] * act);
        }
    };
    auto last_product = [&](int i, const bf16x8 &w) { // of fragment i of the last ones
        const int of = i % 2, cb = i / 2 % CB, s = i / 2 / CB;
        if (of == 0) {
            sum[0][cb] = mfma(w, dg[s], sum[0][cb]);
            sum[1][cb] = mfma(w, du[s], sum[1][cb]);
        } else {
            sum[2][cb] = mfma(w, h[s], sum[2][cb]);
        }
    };
    auto step = [&](int j, int stage, int before, auto has_last) __attribute__((always_inline)) {
        constexpr bool BOTH = decltype(has_last)::value;
        constexpr int COUNT = BOTH ? TOTAL : FIRST;
        const int next = stage + 1 == STAGES ? 0 : stage + 1;
        auto fragment = [&](int m) {
            const int i = BOTH ? index_of(m) : m;
            return i < FIRST ? rows_fragment(stage, i % 2, i / 2) : transposed(before, (i - FIRST) % 2, (i - FIRST) / 2 % CB, (i - FIRST) / 2 / CB);
        };
        f32x16 next_gate = zero16(), next_up = zero16(), next_dh = zero16();
        bf16x8 w[COUNT];
#pragma unroll
        for (int m = 0; m < AHEAD; ++m) {
            w[m] = ready[m];
        }
#pragma unroll
        for (int m = 0; m < COUNT; ++m) {
            if (m == COUNT - AHEAD) {
                meet();
            }
            const int i = BOTH ? index_of(m) : m;
            if (i >= FIRST) {
                last_product(i - FIRST, w[m]);
            } else if (i % 2 == 0) {
                next_gate = mfma(w[m], wg[i / 2], next_gate);
                next_up = mfma(w[m], wu[i / 2], next_up);
            } else {
                next_dh = mfma(w[m], wd[i / 2], next_dh);
            }
            if (m + AHEAD < COUNT) {
                w[m + AHEAD] = fragment(m + AHEAD);
            } else {
                const int n = m + AHEAD - COUNT;
                ready[n] = rows_fragment(next, n % 2, n / 2); // behind the last block, what is not used
                if (n < UPW) {
                    ask_unit(n, j + STAGES - 1, lane_bytes[n]);
                }
            }
            if constexpr (BOTH) {
                constexpr int LATER = FIRST + LAST - EARLY;
                const int from = m < EARLY ? 10 * m / EARLY : m < FIRST + LAST ? 10 + 8 * (m - EARLY) / LATER : 18;
                const int to = m < EARLY ? 10 * (m + 1) / EARLY : m < FIRST + LAST ? 10 + 8 * (m + 1 - EARLY) / LATER : 18;
#pragma unroll
                for (int n = from; n < to; ++n) {
                    part(n);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        gate = next_gate, up = next_up, dh = next_dh;
    };
    static_assert(UPW <= AHEAD && EARLY >= AHEAD && FIRST > AHEAD);
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) {
        ready[n] = rows_fragment(0, n % 2, n / 2);
    }
    __builtin_amdgcn_sched_barrier(0);
    step(0, 0, 0, std::false_type{});
    if (valid < 32) { // the first block's rows past the last: of zeros, but an infinity among the weights makes no numbers of these
#pragma unroll
        for (int e = 0; e < 16; ++e) { // (row i of a product is row sigma(i) of the block)
            const int i = 8 * (e / 4) + 4 * g + e % 4, row = (i & 19) | ((i & 4) << 1) | ((i & 8) >> 1);
            gate[e] = row < valid ? gate[e] : 0.f, up[e] = row < valid ? up[e] : 0.f, dh[e] = row < valid ? dh[e] : 0.f;
        }
    }
    int stage = 0;
    for (int j = 1; j < blocks; ++j) {
        const int before = stage;
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        step(j, stage, before, std::true_type{});
    }
#pragma unroll
    for (int n = 0; n < 18; ++n) {
        part(n);
    }
#pragma unroll
    for (int i = 0; i < 2 * LAST; ++i) {
        last_product(i, transposed(stage, i % 2, i / 2 % CB, i / 2 / CB));
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // requests past the last block: let them land before the LDS is given back
    f32x4 *share = reinterpret_cast<f32x4 *>(p.shares) + ((int64_t)split * (p.c_i / 32) + unit0 / 32) * (3 * CB * 256) + lane;
#pragma unroll
    for (int n = 0; n < 3 * CB; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const f32x16 &v = sum[n / CB][n % CB];
            share[(n * 4 + e) * 64] = f32x4{v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]};
        }
    }
}

// The weights' gradients from their shares: wave w of a workgroup adds those of splits w, w + 4, ..., and the four sums meet, always in that order.
template <int CO>
__global__ __launch_bounds__(256) void gated_weight_shares_kernel(const BackwardParams p)
{
    constexpr int CB = CO / 32;
    __shared__ f32x4 sums[3][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, at = (int)blockIdx.x;
    const int64_t pitch = (int64_t)(p.c_i / 32) * (3 * CB * 256);
    const f32x4 *share = reinterpret_cast<const f32x4 *>(p.shares) + (int64_t)at * 64 + lane;
    f32x4 sum = {0, 0, 0, 0};
#pragma unroll 8
    for (int s = wave; s < p.splits; s += 4) {
        sum += share[s * pitch];
    }
    if (wave > 0) {
        sums[wave - 1][lane] = sum;
    }
    __syncthreads();
    if (wave > 0) {
        return;
    }
    sum = sum + sums[0][lane] + sums[1][lane] + sums[2][lane];
    const int e = at & 3, cb = at / 4 % CB, matrix = at / (4 * CB) % 3, unit = at / (12 * CB) * 32 + (lane & 31), channel = 32 * cb + 8 * e + 4 * (lane >> 5);
    const bf16x4 o = {(bf16_t)sum[0], (bf16_t)sum[1], (bf16_t)sum[2], (bf16_t)sum[3]};
    if (matrix == 2) {
        if (p.grad_down_w != nullptr) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                p.grad_down_w[(int64_t)(channel + c) * p.c_i + unit] = o[c];
            }
        }
    } else if (bf16_t *const to = matrix == 0 ? p.grad_gate_w : p.grad_up_w) {
        *reinterpret_cast<bf16x4 *>(to + (int64_t)unit * CO + channel) = o;
    }
}

template <int CO>
hipError_t launch_weights(const BackwardParams &p, hipStream_t stream)
{
    static size_t configured[2][KUTACC_DEVICE_SLOTS] = {};
    constexpr size_t LDS = (size_t)6 * 8 * CO * 16;
    const bool gelu = p.activation == KUTACC_HIP_GELU;
    const auto kernel = gelu ? &gated_weight_gradients_kernel<CO, KUTACC_HIP_GELU> : &gated_weight_gradients_kernel<CO, KUTACC_HIP_SILU>;
    if (const hipError_t e = kutacc_opt_in_lds(reinterpret_cast<const void *>(kernel), LDS, configured[gelu])) {
        return e;
    }
    kernel<<<dim3((unsigned)((p.c_i + 127) / 128 * p.splits)), 256, LDS, stream>>>(p);
    gated_weight_shares_kernel<CO><<<dim3((unsigned)(p.c_i / 32 * 3 * (CO / 32) * 4)), 256, 0, stream>>>(p);
    return hipGetLastError();
}

// Blocks of 32 rows that a workgroup walks, so that there are as many workgroups as CUs, but at least two
int64_t weight_split_blocks(int64_t rows, int64_t c_i)
{
    const int64_t row_blocks = (rows + 31) / 32, splits = std::max<int64_t>(1, kutacc_cu_count() / ((c_i + 127) / 128));
    return std::max<int64_t>(2, (row_blocks + splits - 1) / splits);
}

template <int CO, int WAVES, int GROUPS>
hipError_t launch(BackwardParams p, hipStream_t stream)
{
    static size_t configured[2][KUTACC_DEVICE_SLOTS] = {};
    constexpr size_t LDS = (size_t)std::max(2 * 12 * CO, 12 * CO + WAVES * 256) * 16;
    const bool gelu = p.activation == KUTACC_HIP_GELU;
    const auto kernel = gelu ? &gated_input_gradient_kernel<CO, WAVES, GROUPS, KUTACC_HIP_GELU> : &gated_input_gradient_kernel<CO, WAVES, GROUPS, KUTACC_HIP_SILU>;
    if (const hipError_t e = kutacc_opt_in_lds(reinterpret_cast<const void *>(kernel), LDS, configured[gelu])) {
        return e;
    }
    // Full rounds of workgroups, then the rest dealt evenly over the CUs, as few waves with rows per workgroup as that takes
    const int64_t row_blocks = (p.rows + 31) / 32, cus = kutacc_cu_count();
    p.full_groups = (int)(row_blocks / (cus * GROUPS * WAVES) * cus * GROUPS);
    const int64_t rest = row_blocks - (int64_t)p.full_groups * WAVES, per_cu = std::max<int64_t>(1, (rest + cus - 1) / cus);
    const int64_t groups = (per_cu + WAVES - 1) / WAVES;
    p.tail_waves = (int)((per_cu + groups - 1) / groups);
    const int64_t blocks = p.full_groups + (rest + p.tail_waves - 1) / p.tail_waves;
    kernel<<<dim3((unsigned)blocks), 64 * WAVES, LDS, stream>>>(p);
    return hipGetLastError();
}
} // namespace

namespace kutacc_launch {

// The walk over the slices takes 1.3 us a slice however few the rows, the tiles of the other kernels about 40 us whatever the width (us, these kernels and
// those; rows x channels -> hidden units): 1000 x 128 -> 128 22 and 30, 8192 x 128 -> 128 33 and 32, 1000 x 64 -> 256 20 and 30, 6000 x 128 -> 512 51 and 43,
// 20000 x 128 -> 512 60 and 76, 8192 x 128 -> 2048 116 and 109, 16000 x 128 -> 2048 136 and 163, 4000 x 64 -> 1024 53 and 50, 8192 x 64 -> 1024 54 and 62.
bool gated_rows_backward_takes(const kutacc_hip_gated_transition_backward_args_t &a)
{
    const int64_t row_blocks = (a.rows + 31) / 32, cus = kutacc_cu_count(), limit = 1 << 23;
    const bool pays = a.c_i <= 256 || (a.c_o == 64 ? row_blocks >= cus : 2 * row_blocks >= 3 * cus);
    return (a.c_o == 64 || a.c_o == 128) && pays && a.rows > 0 && a.c_i > 0 && a.c_i % 32 == 0 && a.c_i < limit && row_blocks < limit && a.x_ld % 8 == 0 && a.grad_out_ld % 8 == 0 &&
           a.x_ld < limit && a.grad_out_ld < limit && a.grad_x_ld % 8 == 0 && kutacc_hip_aligned16(a.x) && kutacc_hip_aligned16(a.grad_out) && kutacc_hip_aligned16(a.grad_x) &&
           kutacc_hip_aligned16(a.gate_w) && kutacc_hip_aligned16(a.up_w) && kutacc_hip_aligned16(a.down_w) && kutacc_hip_aligned16(a.grad_gate_w) &&
           kutacc_hip_aligned16(a.grad_up_w) && kutacc_hip_aligned16(a.grad_down_w);
}

int64_t gated_rows_backward_workspace(int64_t rows, int64_t c_o, int64_t c_i)
{
    const int64_t row_blocks = (rows + 31) / 32, per_split = weight_split_blocks(rows, c_i);
    return (row_blocks + per_split - 1) / per_split * c_i * c_o * 12;
}

int gated_rows_backward(const kutacc_hip_gated_transition_backward_args_t &a, hipStream_t stream)
{
    const int64_t row_blocks = (a.rows + 31) / 32, per_split = weight_split_blocks(a.rows, a.c_i);
    BackwardParams p = {(const bf16_t *)a.x, (const bf16_t *)a.grad_out, (const bf16_t *)a.gate_w, (const bf16_t *)a.up_w, (const bf16_t *)a.down_w};
    p.grad_x = (bf16_t *)a.grad_x, p.grad_gate_w = (bf16_t *)a.grad_gate_w, p.grad_up_w = (bf16_t *)a.grad_up_w, p.grad_down_w = (bf16_t *)a.grad_down_w;
    p.shares = (float *)a.workspace;
    p.x_ld = a.x_ld, p.grad_out_ld = a.grad_out_ld, p.grad_x_ld = a.grad_x_ld, p.rows = a.rows;
    p.splits = (int)((row_blocks + per_split - 1) / per_split), p.split_blocks = (int)per_split;
    p.c_i = (int)a.c_i, p.activation = a.activation;
    const double flops = 2.0 * (double)a.rows * (double)a.c_o * (double)a.c_i;
    if (a.grad_x != nullptr) {
        kutacc_prof::KernelTimer t("gated_rows_input_gradient", 5 * flops, stream);
        if (const hipError_t e = a.c_o == 128 ? launch<128, 4, 2>(p, stream) : launch<64, 4, 3>(p, stream)) {
            return kutacc_hip_status(e);
        }
    }
    if (a.grad_gate_w != nullptr || a.grad_up_w != nullptr || a.grad_down_w != nullptr) {
        kutacc_prof::KernelTimer t("gated_rows_weight_gradients", 6 * flops, stream);
        return kutacc_hip_status(a.c_o == 128 ? launch_weights<128>(p, stream) : launch_weights<64>(p, stream));
    }
    return 0;
}

} // namespace kutacc_launch
