// The gated transition of 64, 128 and 256 channels in one kernel: out = (act(x Wg^T) * (x Wu^T)) Wd^T, the hidden layer on chip.
//
// A wave owns 32 rows of x as operand fragments in registers and walks the hidden layer in slices of 32 units: two products of the slice's weights with
// x, the activation, and the product of the slice of Wd with what they gave.  All are formed transposed (MFMA rows = hidden units, then output channels;
// columns = rows of x): the accumulators of the first two, rounded to bf16, are the operand of the third without leaving the registers.  For that, row i
// of a slice in the LDS is hidden unit sigma(i) (bits 2 and 3 of i swapped), which makes the eight values a lane holds per k-step consecutive hidden units.
// The slices come straight into the LDS, into a ring with one barrier a slice.
//
// 147456 x 128 -> 512: 65.7 us, 880 TFLOP/s of the 1380 that a large product reaches here (142 us with the hidden layer in memory).  The matrix pipe works in 37 %
// of the clocks, the vector issue port in 42 %, both in 19 %, and neither in 40 %: a SIMD has two waves, which wait for 28 % of their time, at a slice's barrier among
// others.  The activation is as much work as the products, and the clock falls under the two together.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "gated_activation.h"
#include "launch_internal.h"
#include "mfma_tiles.h"
#include "profiler.h"

namespace {
using namespace kutacc_dev;

struct RowsParams {
    const bf16_t *x, *gate_w, *up_w, *down_w;
    bf16_t *out;
    int64_t x_ld, out_ld, rows;
    int c_i, activation;
    int full_groups, tail_waves; // workgroups whose waves all have rows, and how many waves of the others have
};

// until at most N of a wave's own loads are on their way and none of its LDS reads
template <int N>
__device__ __forceinline__ void wait_and_barrier()
{
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(N) : "memory");
}

template <int CO, int STAGES, int WAVES, int GROUPS, bool APART, int ACTIVATION>
__global__ __launch_bounds__(64 * WAVES, GROUPS * WAVES / 4) void gated_rows_kernel(const RowsParams p)
{
    constexpr int KS = CO / 16, CP = CO / 64, CB = CO / 32;       // k-steps of the first products, panels of 64 channels, blocks of 32
    constexpr int MATRIX = 4 * CO, STAGE = 3 * MATRIX;            // 16-byte slots: 32 hidden units of a matrix, and of all three
    constexpr int MATRIX_UNITS = CO / 16, UPW = 3 * MATRIX_UNITS / WAVES; // loads of 1 KB: of a matrix, and of a wave for all three
    static_assert(UPW * WAVES == 3 * MATRIX_UNITS && WAVES * 256 <= STAGES * STAGE, "all waves bring as much; their panels lie where the stages do");
    extern __shared__ uint4 lds[]; // [STAGES][gate, up, down], and what the panels take beyond the last
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
    PanelRegs panels[CP];
#pragma unroll
    for (int cp = 0; cp < CP; ++cp) {
        panels[cp] = panel_load(p.x + row0 * p.x_ld, p.x_ld, 0, last_local, cp * 64, lane);
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
    // Batch b of the loads: the gate's and the other projection's slice b, and Wd's, or with APART Wd's slice b - 1, which meets them in step b
    constexpr int LATE = APART ? 1 : 0;
    const int batches = slices + LATE;
    // (a batch past either end of its matrix in no lane: without a branch, beside the products)
    auto ask_unit = [&](int i, int batch) {
        const bool is_down = wave * UPW + i >= 2 * MATRIX_UNITS;
        const int lanes = __builtin_amdgcn_readfirstlane((is_down ? batch >= LATE && batch < batches : batch < slices) ? -1 : 0);
        asm volatile("s_mov_b32 exec_lo, %3\n\ts_mov_b32 exec_hi, %3\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b64 exec, -1" ::"s"(
                         __builtin_amdgcn_readfirstlane((int)(lds0 + (uint32_t)(batch % STAGES) * (STAGE * 16u) + i * 1024u))),
                     "v"(lane_bytes[i]), "s"(same_in_all_lanes(source[i] + (int64_t)(is_down ? batch - LATE : batch) * pitch[i])), "s"(lanes)
                     : "memory");
    };
    auto ask = [&](int batch) {
#pragma unroll
        for (int i = 0; i < UPW; ++i) {
            ask_unit(i, batch);
        }
    };
    constexpr int AT_FIRST = APART ? 1 : STAGES - 1; // the panels of x take the last stage, or all but the first
    for (int b = 0; b < AT_FIRST; ++b) {
        ask(b);
    }

    // x as operands of the first products, through a panel in the stage that is still free
    bf16x8 x[KS];
    uint4 *const panel = lds + AT_FIRST * STAGE + wave * 256;
#pragma unroll
    for (int cp = 0; cp < CP; ++cp) {
        panel_store(panel, lane, panels[cp]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            x[cp * 4 + k] = as_bf16x8(panel[panel_slot(r, 2 * k + g)]);
        }
    }
    f32x16 sum[CB];
#pragma unroll
    for (int cb = 0; cb < CB; ++cb) {
        sum[cb] = zero16();
    }
    const int w1_lane = panel_slot(r, g), w2_lane = r * 4 + (g ^ ((r >> 2) & 3));
    auto gate_slot = [&](int k) { return (k / 4) * 256 + (w1_lane ^ (2 * (k % 4))); };
    auto down_slot = [&](int cb, int s) { return 2 * MATRIX + cb * 128 + (w2_lane ^ (2 * s)); };
    if constexpr (!APART) {
        for (int j = 0; j < slices; ++j) {
            // slice j has landed (later ones may be under way), and every wave is done with the stage of the one before
            if (STAGES > 2 && j + STAGES - 2 < slices) {
                wait_and_barrier<(STAGES - 2) * UPW>();
            } else {
                wait_and_barrier<0>();
            }
            ask(j + STAGES - 1);
            if (!active) {
                continue;
            }
            const uint4 *stage = lds + j % STAGES * STAGE;
            f32x16 gate = zero16(), up = zero16();
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                gate = mfma(as_bf16x8(stage[gate_slot(k)]), x[k], gate);
                up = mfma(as_bf16x8(stage[MATRIX + gate_slot(k)]), x[k], up);
            }
            bf16x8 h[2];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float none;
                h[e / 8][e % 8] = (bf16_t)(activate<false>(gate[e], ACTIVATION, none) * up[e]);
            }
#pragma unroll
            for (int n = 0; n < 2 * CB; ++n) {
                sum[n % CB] = mfma(as_bf16x8(stage[down_slot(n % CB, n / CB)]), h[n / CB], sum[n % CB]);
            }
        }
    } else {
        // Step j: the products of slice j with x, and beside them slice j - 1: its activation, then its product.  Every fragment leaves the LDS AHEAD
        // products before its own.  The last AHEAD products, whose fragments are there, run behind the barrier of the next step: beside them the first
        // fragments of that step leave the LDS and the batch after it is asked for, into the stage that all are done with.
        static_assert(STAGES == 2, "a batch is all that is on its way");
        constexpr int AHEAD = 6;
        __syncthreads(); // the panels
        ask(1);
        auto meet = [&]() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
        if (!active) { // brings weights only
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"(0) : "memory");
            for (int j = 0; j < slices; ++j) {
                meet();
                ask(j + 2);
            }
        } else {
            f32x16 gate, up;
            bf16x8 h[2], first[AHEAD];
            constexpr int GU = 2 * KS, EARLY = GU * 3 / 4;
            auto gate_up = [&](const uint4 *stage, int i) { return as_bf16x8(stage[(i % 2) * MATRIX + gate_slot(i / 2)]); };
            auto step = [&](int j, auto has_second) __attribute__((always_inline)) {
                constexpr bool SECOND = decltype(has_second)::value;
                const uint4 *stage = lds + (j & 1) * STAGE, *next = lds + ((j + 1) & 1) * STAGE;
                constexpr int D = SECOND ? CB : 0, TOTAL = GU + 2 * D;
                static_assert(TOTAL > 2 * AHEAD && EARLY >= AHEAD, "the first fragments are of the first products");
                // the order: three quarters of the first products, half of Wd's, the rest of the first, the other half
                auto index_of = [](int m) { // first products 0 .. GU - 1, Wd's from GU on
                    return m < EARLY ? m : m < EARLY + D ? GU + m - EARLY : m < GU + D ? m - D : m;
                };
                auto fragment = [&](int m) {
                    const int i = index_of(m);
                    return i < GU ? gate_up(stage, i) : as_bf16x8(stage[down_slot((i - GU) % CB, (i - GU) / CB)]);
                };
                f32x16 next_gate = zero16(), next_up = zero16();
                // the activation of a value in three parts, a product apart, none of which waits for the one before
                float t[16];
                auto part = [&](int n) { // 0 .. 17: the exponential of value n, the sigmoid of value n - 1, the operand of value n - 2
                    if (n < 16) {
                        t[n] = 1.0f + __builtin_amdgcn_exp2f(activation_exponent(gate[n], ACTIVATION));
                    }
                    if (n >= 1 && n < 17) {
                        t[n - 1] = gate[n - 1] * __builtin_amdgcn_rcpf(t[n - 1]);
                    }
                    if (n >= 2) {
                        h[(n - 2) / 8][(n - 2) % 8] = (bf16_t)(t[n - 2] * up[n - 2]);
                    }
                };
                bf16x8 w[TOTAL];
#pragma unroll
                for (int m = 0; m < AHEAD; ++m) {
                    w[m] = first[m];
                }
#pragma unroll
                for (int m = 0; m < TOTAL; ++m) {
                    if (m == TOTAL - AHEAD) {
                        meet();
                    }
                    const int i = index_of(m);
                    if (i < GU) {
                        if (i % 2 == 0) {
                            next_gate = mfma(w[m], x[i / 2], next_gate);
                        } else {
                            next_up = mfma(w[m], x[i / 2], next_up);
                        }
                    } else {
                        sum[(i - GU) % CB] = mfma(w[m], h[(i - GU) / CB], sum[(i - GU) % CB]);
                    }
                    if (m + AHEAD < TOTAL) {
                        w[m + AHEAD] = fragment(m + AHEAD);
                    } else {
                        const int n = m + AHEAD - TOTAL;
                        first[n] = gate_up(next, n); // behind the last slice, what is not used
#pragma unroll
                        for (int u = n * UPW / AHEAD; u < (n + 1) * UPW / AHEAD; ++u) {
                            ask_unit(u, j + 2);
                        }
                    }
                    if constexpr (SECOND) { // parts 0 .. 9 beside the first three quarters, the others beside what follows up to the last half
                        constexpr int LATER = GU + D - EARLY;
                        const int from = m < EARLY ? 10 * m / EARLY : m < GU + D ? 10 + 8 * (m - EARLY) / LATER : 18;
                        const int to = m < EARLY ? 10 * (m + 1) / EARLY : m < GU + D ? 10 + 8 * (m + 1 - EARLY) / LATER : 18;
#pragma unroll
                        for (int n = from; n < to; ++n) {
                            part(n);
                        }
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                gate = next_gate, up = next_up;
            };
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"i"(0) : "memory");
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) {
                first[n] = gate_up(lds, n);
            }
            __builtin_amdgcn_sched_barrier(0);
            step(0, std::false_type{});
            for (int j = 1; j < slices; ++j) {
                step(j, std::true_type{});
            }
            // the last slice's activation and product
            const uint4 *stage = lds + (slices & 1) * STAGE;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float none;
                h[e / 8][e % 8] = (bf16_t)(activate<false>(gate[e], ACTIVATION, none) * up[e]);
            }
#pragma unroll
            for (int n = 0; n < 2 * CB; ++n) {
                sum[n % CB] = mfma(as_bf16x8(stage[down_slot(n % CB, n / CB)]), h[n / CB], sum[n % CB]);
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
                *reinterpret_cast<uint4 *>(p.out + (row0 + row) * p.out_ld + cp * 64 + (lane & 7) * 8) = strip[panel_slot(row, lane & 7)];
            }
        }
    }
}

template <int CO, int STAGES, int WAVES, int GROUPS, bool APART>
hipError_t launch_rows(RowsParams p, hipStream_t stream)
{
    static size_t configured[2][KUTACC_DEVICE_SLOTS] = {};
    constexpr size_t LDS = (size_t)std::max(STAGES * 12 * CO, (APART ? 1 : STAGES - 1) * 12 * CO + WAVES * 256) * 16;
    const auto kernel = p.activation == KUTACC_HIP_GELU ? &gated_rows_kernel<CO, STAGES, WAVES, GROUPS, APART, KUTACC_HIP_GELU> : &gated_rows_kernel<CO, STAGES, WAVES, GROUPS, APART, KUTACC_HIP_SILU>;
    if (const hipError_t e = kutacc_opt_in_lds(reinterpret_cast<const void *>(kernel), LDS, configured[p.activation == KUTACC_HIP_GELU])) {
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

// 64, 128 and 256 channels, and rows enough: a wave's chain through the hidden layer takes its time however few there are (us, here and with the hidden
// layer in memory: 128 -> 512 5000 rows 15.0 14.1, 12000 15.7 22.7, 147456 66 142; 128 -> 2048 8000 rows 46 39, 12000 47 60; 256 -> 1024 20000 rows 64 60,
// 40000 76 104, 195072 284 476; 64 -> 256 100 rows 7.1 9.0, 40000 10.7 30.4; 64 -> 512 60 rows 11.2 7.8).
bool gated_rows_takes(const kutacc_hip_gated_transition_args_t &a)
{
    const int64_t row_blocks = (a.rows + 31) / 32, cus = kutacc_cu_count();
    return ((a.c_o == 64 && a.rows > 64) || (a.c_o == 128 && row_blocks >= cus) || (a.c_o == 256 && 2 * row_blocks >= 5 * cus)) && a.c_i % 32 == 0 && row_blocks <= ((int64_t)1 << 31) &&
           a.c_i <= (1 << 24) && a.x_ld % 8 == 0 && a.out_ld % 8 == 0 && kutacc_hip_aligned16(a.x) && kutacc_hip_aligned16(a.out) && kutacc_hip_aligned16(a.gate_w) &&
           kutacc_hip_aligned16(a.up_w) && kutacc_hip_aligned16(a.down_w);
}

int gated_rows(const kutacc_hip_gated_transition_args_t &a, hipStream_t stream)
{
    const RowsParams p = {(const bf16_t *)a.x, (const bf16_t *)a.gate_w, (const bf16_t *)a.up_w, (const bf16_t *)a.down_w, (bf16_t *)a.out,
                          a.x_ld, a.out_ld, a.rows, (int)a.c_i, a.activation, 0, 0};
    kutacc_prof::KernelTimer t("gated_rows_kernel", 6.0 * (double)a.rows * (double)a.c_o * (double)a.c_i, stream);
    if (a.c_o == 256) {
        return kutacc_hip_status(launch_rows<256, 3, 8, 1, false>(p, stream));
    }
    if (a.c_o == 128) { // a workgroup a CU while its eight waves take all rows, else two, one of which computes while the other fetches or stores
        const bool one_round = (a.rows + 31) / 32 <= 8 * (int64_t)kutacc_cu_count();
        return kutacc_hip_status(one_round ? launch_rows<128, 2, 8, 1, true>(p, stream) : launch_rows<128, 2, 4, 2, true>(p, stream));
    }
    return kutacc_hip_status(launch_rows<64, 2, 4, 4, false>(p, stream));
}

} // namespace kutacc_launch
