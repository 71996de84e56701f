// The gated transition and its backward pass, bf16 with fp32 sums:
//   g = x Wg^T,  u = x Wu^T,  h = act(g) u,  out = h Wd^T,      act(v) = v sigmoid(t(v))
//   dh = dy Wd,  dg = dh u act'(g),  du = dh act(g),  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h
// act'(v) = s + v s (1 - s) t'(v) with s = sigmoid(t(v)).  silu: t = v; gelu (its tanh form): t = 2 sqrt(2 / pi) (v + 0.044715 v^3).
//
// g, u and dh are never rounded: the kernel that forms them holds all of them of one tile at once, and h, dg and du are rounded once, as
// operands of the products that follow.
//
// ff_tiles_kernel covers every shape: 128 x 128 of a result per workgroup of four waves, K in steps of 64 through registers and the LDS, for a list of
// products that share the tile.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "gated_activation.h"
#include "gemm_panels.h"
#include "launch_internal.h"
#include "mfma_tiles.h"
#include "profiler.h"

namespace {
using namespace kutacc_dev;

// ---- every shape ----

// C(m, n) += sum_k A(m, k) B(n, k)
struct Product {
    const bf16_t *a, *b;
    int64_t a_ld, b_ld;
};

enum Mode { PLAIN, GATED, HIDDEN_GRADIENTS, INPUT_GRADIENT, WEIGHT_GRADIENTS };

struct TilesParams {
    Product product[3];
    bf16_t *c[3];
    int64_t c_ld[3];
    int M[3], N[3], tiles[3]; // of the products of WEIGHT_GRADIENTS, which have tiles of their own; else the first alone
    int K, activation;
    int splits;   // of k, with WEIGHT_GRADIENTS and INPUT_GRADIENT; their sums then meet in `shares`
    float *shares;
};

constexpr int TILE = 128, OPERAND_SLOTS = 1024, CT_LD = 136;
constexpr size_t TILES_LDS = TILE * CT_LD * 2;

// Eight elements of a row that has `size` >= 8, on their way as they lie in memory, without a branch that would wait for them: a piece past the row's end is the row's
// last eight, and dropped() elements are too many in front.
__device__ __forceinline__ int dropped(int at, int size) { return max(0, at + 8 - size); }
__device__ __forceinline__ uint4 ask8(const bf16_t *row, int at, int size) { return load8_any(row - dropped(at, size), (uint32_t)at); }
// 32 rows by 64 k of a K-major operand, 64 columns by 32 k of an M-major one, as load_kmajor and load_mmajor divide them
__device__ __forceinline__ PanelRegs ask_kmajor(const bf16_t *base, int64_t ld, int row0, int last_row, int k0, int K, int lane)
{
    PanelRegs p;
    uint4 *dst[4] = {&p.r0, &p.r1, &p.r2, &p.r3};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        *dst[i] = ask8(base + (int64_t)min(row0 + 8 * i + (lane >> 3), last_row) * ld, k0 + (lane & 7) * 8, K);
    }
    return p;
}
__device__ __forceinline__ PanelRegs ask_mmajor(const bf16_t *base, int64_t ld, int m0, int rows, int k0, int K, int lane)
{
    PanelRegs p;
    uint4 *dst[4] = {&p.r0, &p.r1, &p.r2, &p.r3};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        *dst[i] = ask8(base + (int64_t)min(k0 + 8 * i + mm_row(lane >> 3), K - 1) * ld, m0 + (lane & 7) * 8, rows);
    }
    return p;
}
// ... and put in order, zeros past K
__device__ __forceinline__ void settle_kmajor(PanelRegs &p, int k0, int K, int lane)
{
    if (k0 + KSTEP > K) {
        const int drop = min(8, dropped(k0 + (lane & 7) * 8, K));
        p.r0 = drop_first(p.r0, drop), p.r1 = drop_first(p.r1, drop), p.r2 = drop_first(p.r2, drop), p.r3 = drop_first(p.r3, drop);
    }
}
__device__ __forceinline__ void settle_mmajor(PanelRegs &p, int m0, int rows, int k0, int K, int lane)
{
    uint4 *dst[4] = {&p.r0, &p.r1, &p.r2, &p.r3};
    if (m0 + 64 > rows) {
        const int drop = min(8, dropped(m0 + (lane & 7) * 8, rows));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            *dst[i] = drop_first(*dst[i], drop);
        }
    }
    if (k0 + 32 > K) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            *dst[i] = k0 + 8 * i + mm_row(lane >> 3) < K ? *dst[i] : zero_u4();
        }
    }
}

// The next step's operands are on their way while this one's are multiplied.  us, so and with branches around the pieces at a row's end: 7829 x 512 x 2046 89
// and 193, its backward pass 274 and 825 (with rows and hidden units split where tiles are few, as below), 5088 x 124 x 128 41 and 192.  TINY: a width of fewer than
// eight, element by element.
template <int MODE, bool TINY>
__global__ __launch_bounds__(256, MODE == GATED || MODE == HIDDEN_GRADIENTS ? 1 : 2) void ff_tiles_kernel(const TilesParams p)
{
    constexpr int SUMS = MODE == GATED ? 2 : MODE == HIDDEN_GRADIENTS ? 3 : 1;
    constexpr int PRODUCTS = MODE == INPUT_GRADIENT ? 2 : SUMS;
    extern __shared__ uint4 lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 31, g = lane >> 5, wm = wave >> 1, wn = wave & 1;
    constexpr bool SPLIT = MODE == WEIGHT_GRADIENTS || MODE == INPUT_GRADIENT;
    int which = 0, split = 0;
    unsigned tile = blockIdx.x;
    if constexpr (SPLIT) { // (all tiles of a range of k, then the next range's)
        const unsigned all = (unsigned)(p.tiles[0] + p.tiles[1] + p.tiles[2]);
        split = (int)(tile / all), tile %= all;
        while (which < 2 && tile >= (unsigned)p.tiles[which]) {
            tile -= (unsigned)p.tiles[which++];
        }
    }
    const int M = p.M[which], N = p.N[which];
    // the walk of ff_pieces_kernel, as the shares are added in its order
    const unsigned MT = (unsigned)(M + TILE - 1) / TILE, NT = (unsigned)(N + TILE - 1) / TILE;
    const unsigned band = tile / (8 * NT), height = min(8u, MT - 8 * band), in = tile - band * 8 * NT;
    const int m0 = (int)(8 * band + in % height) * TILE, n0 = (int)(in / height) * TILE;

    f32x16 acc[SUMS][2][2];
#pragma unroll
    for (int s = 0; s < SUMS; ++s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc[s][i >> 1][i & 1] = zero16();
        }
    }
    const int mm_a[2] = {mm_fragment_offset(2 * wm, lane), mm_fragment_offset(2 * wm + 1, lane)};
    const int mm_b[2] = {mm_fragment_offset(2 * wn, lane), mm_fragment_offset(2 * wn + 1, lane)};
    const int all_steps = (p.K + KSTEP - 1) / KSTEP;
    const int first = SPLIT ? (int)((int64_t)all_steps * split / p.splits) : 0, steps = SPLIT ? (int)((int64_t)all_steps * (split + 1) / p.splits) : all_steps;
#pragma unroll
    for (int n = 0; n < PRODUCTS; ++n) {
        constexpr bool A_MMAJOR = MODE == WEIGHT_GRADIENTS;
        const bool B_MMAJOR = MODE == INPUT_GRADIENT || MODE == WEIGHT_GRADIENTS || (MODE == HIDDEN_GRADIENTS && n == 2); // a constant in every copy
        const Product &q = p.product[MODE == WEIGHT_GRADIENTS ? which : n];
        auto fetch = [&](const bf16_t *base, int64_t ld, bool mmajor, int at, int extent, int k0) {
            if constexpr (TINY) {
                return mmajor ? load_mmajor<true>(base, ld, at + 64 * (wave & 1), extent, k0 + 32 * (wave >> 1), p.K, lane) : load_kmajor<true>(base, ld, at + 32 * wave, extent - 1, k0, p.K, lane);
            } else {
                return mmajor ? ask_mmajor(base, ld, at + 64 * (wave & 1), extent, k0 + 32 * (wave >> 1), p.K, lane) : ask_kmajor(base, ld, at + 32 * wave, extent - 1, k0, p.K, lane);
            }
        };
        auto settle = [&](PanelRegs &f, bool mmajor, int at, int extent, int k0) {
            if constexpr (!TINY) {
                if (mmajor) {
                    settle_mmajor(f, at + 64 * (wave & 1), extent, k0 + 32 * (wave >> 1), p.K, lane);
                } else {
                    settle_kmajor(f, k0, p.K, lane);
                }
            }
        };
        auto fetch_a = [&](int k0) { return fetch(q.a, q.a_ld, A_MMAJOR, m0, M, k0); };
        auto fetch_b = [&](int k0) { return fetch(q.b, q.b_ld, B_MMAJOR, n0, N, k0); };
        auto park = [&](uint4 *operand, bool mmajor, const PanelRegs &f) {
            if (mmajor) {
                store_mmajor(operand, 64 * (wave & 1), 32 * (wave >> 1), lane, f);
            } else {
                panel_store(operand + wave * 256, lane, f);
            }
        };
        f32x16(&sum)[2][2] = acc[SUMS == 1 ? 0 : n];
        PanelRegs ra = fetch_a(first * KSTEP), rb = fetch_b(first * KSTEP);
        for (int kt = first; kt < steps; ++kt) {
            settle(ra, A_MMAJOR, m0, M, kt * KSTEP);
            settle(rb, B_MMAJOR, n0, N, kt * KSTEP);
            __syncthreads(); // the stage is no longer being read
            park(lds, A_MMAJOR, ra);
            park(lds + OPERAND_SLOTS, B_MMAJOR, rb);
            __syncthreads();
            if (kt + 1 < steps) {
                ra = fetch_a((kt + 1) * KSTEP);
                rb = fetch_b((kt + 1) * KSTEP);
            }
            const uint4 *oa = lds + 2 * wm * 256, *ob = lds + OPERAND_SLOTS + 2 * wn * 256;
            const lds_char *ta = (const lds_char *)lds, *tb = (const lds_char *)(lds + OPERAND_SLOTS);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int slot = panel_slot(r, 2 * s + g);
                bf16x8 a[2], b[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    a[i] = A_MMAJOR ? mm_fragment(ta, mm_a[i], s) : as_bf16x8(oa[256 * i + slot]);
                    b[i] = B_MMAJOR ? mm_fragment(tb, mm_b[i], s) : as_bf16x8(ob[256 * i + slot]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    sum[i >> 1][i & 1] = mfma(b[i & 1], a[i >> 1], sum[i >> 1][i & 1]);
                }
            }
        }
    }

    if constexpr (SPLIT) {
        if (p.splits > 1) { // a share of the sums, as ff_pieces_kernel leaves it
            f32x4 *share = reinterpret_cast<f32x4 *>(p.shares) + ((int64_t)blockIdx.x * 4 + wave) * (2 * 2 * 4 * 64) + lane;
#pragma unroll
            for (int n = 0; n < 16; ++n) {
                const f32x16 &v = acc[0][n / 8][n / 4 % 2];
                share[n * 64] = f32x4{v[4 * (n % 4)], v[4 * (n % 4) + 1], v[4 * (n % 4) + 2], v[4 * (n % 4) + 3]};
            }
            return;
        }
    }
    // results as bf16 through the LDS, out as whole rows of 256 bytes
    bf16_t *ct = reinterpret_cast<bf16_t *>(lds);
    auto store = [&](const f32x16 (&v)[2][2], bf16_t *c, int64_t ld) {
        __syncthreads(); // what lay there has been read
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    bf16x4 o;
#pragma unroll
                    for (int f = 0; f < 4; ++f) {
                        o[f] = (bf16_t)v[i][j][4 * e + f];
                    }
                    *reinterpret_cast<bf16x4 *>(ct + (64 * wm + 32 * i + r) * CT_LD + 64 * wn + 32 * j + 8 * e + 4 * g) = o;
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int piece = tid + 256 * i, row = piece >> 4, chunk = piece & 15;
            const int m = m0 + row, n = n0 + chunk * 8;
            if (m >= M || n >= N) {
                continue;
            }
            const uint4 v8 = *reinterpret_cast<const uint4 *>(ct + row * CT_LD + chunk * 8);
            bf16_t *to = c + (int64_t)m * ld + n;
            if (n + 8 <= N) {
                __builtin_memcpy(to, &v8, 16);
            } else {
                const bf16x8 b = as_bf16x8(v8);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (n + e < N) {
                        to[e] = b[e];
                    }
                }
            }
        }
    };
    if constexpr (MODE == GATED || MODE == HIDDEN_GRADIENTS) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    float slope = 0.f;
                    const float a = activate<MODE == HIDDEN_GRADIENTS>(acc[0][i][j][e], p.activation, slope), u = acc[1][i][j][e];
                    acc[0][i][j][e] = a * u;
                    if constexpr (MODE == HIDDEN_GRADIENTS) {
                        const float dh = acc[2][i][j][e];
                        acc[1][i][j][e] = dh * u * slope;
                        acc[2][i][j][e] = dh * a;
                    }
                }
            }
        }
        store(acc[0], p.c[0], p.c_ld[0]);
        if constexpr (MODE == HIDDEN_GRADIENTS) {
            store(acc[1], p.c[1], p.c_ld[1]);
            store(acc[2], p.c[2], p.c_ld[2]);
        }
    } else {
        store(acc[0], p.c[which], p.c_ld[which]);
    }
}

// ---- whole 16-byte pieces: WM x WN waves a workgroup, 32 MI x 64 of the tile a wave: 256 x 256 by 2 x 4 waves or 128 x 128 by 2 x 2 ----
//
// Operands come straight into the LDS, 64 k a stage (A's rows, then B's; 128 bytes a row, its 16-byte slots XOR-ed with the row's number & 7),
// two stages: a stage is asked for when the one before it has been read by all.  M-major operands (their tile's rows contiguous) lie in sub-tiles of
// 64 k x 128 as mm_fragment expects them.  The last quarter of a stage's products runs behind the barrier at which the stage is given back and hides
// the first reads of the next; in every quarter the fragments of the next one come out of the LDS between the products.
//
// A tile of GATED is SIDE rows of x by SIDE / 2 hidden units: of every 64 columns 32 are of the gate and 32 of the other projection, so that a wave
// holds both of the same hidden units.  HIDDEN_GRADIENTS then multiplies dy with SIDE / 2 columns of down_w into sums of their own.
//
// 4001 x 1024 -> 2816, 81 us: GATED 52 (890 TFLOP/s), PLAIN 29 (800); 4096 x 1024 -> 4096, backward, 322: hidden gradients 146 (710), gradient of x 77 (890), of the
// weights 99 (1040); a large library product reaches 1380.  (A call's time, and its kernels' shares of that in a trace.)  The matrix pipe works in 30 to 44 % of the clocks: the two waves of a SIMD run in step, so that neither hides the
// other's barriers, nor a tile's activation and results another tile's products.
template <int MODE, int MI, int WM, int WN, int GROUPS>
__global__ __launch_bounds__(64 * WM * WN * GROUPS, 2) void ff_pieces_kernel(const TilesParams p)
{
    constexpr int ROWS = 32 * MI * WM, SIDE = 64 * WN, STAGE = (ROWS + SIDE) * 8; // of A and B; 16-byte slots of a stage
    constexpr int A_UNITS = ROWS / 8, UNITS = (ROWS + SIDE) / 8 / (WM * WN);      // of 1 KB: of A, and those that a wave brings
    static_assert((ROWS + SIDE) % (8 * WM * WN) == 0, "all waves bring as much");
    constexpr bool HIDDEN = MODE == GATED || MODE == HIDDEN_GRADIENTS, TWO = MODE == HIDDEN_GRADIENTS || MODE == INPUT_GRADIENT;
    constexpr int COLUMNS = HIDDEN ? SIDE / 2 : SIDE;
    constexpr bool A_MMAJOR = MODE == WEIGHT_GRADIENTS, B_MMAJOR = MODE == WEIGHT_GRADIENTS || MODE == INPUT_GRADIENT;
    static_assert(!A_MMAJOR || ROWS % 128 == 0, "sub-tiles of M-major operands");
    static_assert(GROUPS == 1 || MODE == PLAIN || MODE == INPUT_GRADIENT, "sums that meet in the LDS");
    constexpr bool SPLIT = (MODE == WEIGHT_GRADIENTS || MODE == INPUT_GRADIENT) && MI == 2 && GROUPS == 1;
    extern __shared__ uint4 all_lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int group = wave / (WM * WN), member = wave % (WM * WN);
    const int r = lane & 31, g = lane >> 5, wm = member / WN, wn = member % WN;
    uint4 *const lds = all_lds + group * 2 * STAGE;

    // Workgroup ids are dealt round robin over the 8 XCDs: each gets a contiguous run of the walk
    unsigned tile = blockIdx.x;
    {
        const unsigned per = gridDim.x / 8;
        tile = tile < per * 8 ? tile % 8 * per + tile / 8 : tile;
    }
    int which = 0, split = 0;
    const unsigned place = tile; // of a share of the sums
    if constexpr (MODE == WEIGHT_GRADIENTS || SPLIT) { // (all tiles of a range of k, which share it, and then the next range's)
        const unsigned all = (unsigned)(p.tiles[0] + p.tiles[1] + p.tiles[2]);
        split = __builtin_amdgcn_readfirstlane((int)(tile / all)), tile = (unsigned)__builtin_amdgcn_readfirstlane((int)(tile % all));
        while (which < 2 && tile >= (unsigned)p.tiles[which]) {
            tile -= (unsigned)p.tiles[which++];
        }
    }
    const int M = p.M[which], N = p.N[which];
    // ... a walk through bands of 8 tiles of rows, column by column, so that neighbours share both operands in their L2
    const unsigned MT = (unsigned)(M + ROWS - 1) / ROWS, NT = (unsigned)(N + COLUMNS - 1) / COLUMNS;
    const unsigned band = tile / (8 * NT), height = min(8u, MT - 8 * band), in = tile - band * 8 * NT;
    // (quotients come from vector instructions: back into scalar registers, for the addresses)
    const int m0 = __builtin_amdgcn_readfirstlane((int)(8 * band + in % height) * ROWS), n0 = __builtin_amdgcn_readfirstlane((int)(in / height) * COLUMNS);

    // stages of the first list of products (and of the second, as many)
    const int all_stages = (p.K + 63) / 64;
    int first_stage = 0, stages = all_stages;
    if constexpr (SPLIT) {
        first_stage = __builtin_amdgcn_readfirstlane((int)((int64_t)all_stages * split / p.splits));
        stages = __builtin_amdgcn_readfirstlane((int)((int64_t)all_stages * (split + 1) / p.splits)) - first_stage;
    }
    // of the stages a group takes every other one; a group that has one less multiplies zeros
    const int steps = (stages + GROUPS - 1) / GROUPS, total = TWO ? 2 * steps : steps;
    // Tiles of neighbouring columns start at different stages: with rows a power of two apart, all rows' bytes of one stage lie in one or two channels
    // of the L2.
    const int turn = MODE == WEIGHT_GRADIENTS ? 0 : __builtin_amdgcn_readfirstlane((int)((unsigned)(n0 / COLUMNS) * 2u % (unsigned)stages));

    const int first_unit = member * UNITS; // this wave's, of A's and then B's
    const uint32_t to = (uint32_t)(uintptr_t)(const lds_char *)lds + (uint32_t)first_unit * 1024u;
    uint4 *const slots = lds + first_unit * 64 + lane;
    const int chunk = (lane & 7) ^ (lane >> 3);                               // K-major: eight rows a unit
    const int mm_k = lane >> 4, mm_m = 8 * ((lane & 15) ^ (4 * (lane >> 4))); // M-major: four k by 128
    // this lane's elements of the operand, from the tile's first
    auto kmajor_from = [&](int row, int last, int64_t ld) { return 2u * ((uint32_t)min(row, last) * (uint32_t)ld + 8u * (uint32_t)chunk); };
    auto mmajor_from = [&](int u, int last, int64_t ld) { return 2u * ((uint32_t)(4 * (u & 15) + mm_k) * (uint32_t)ld + (uint32_t)max(0, min(128 * (u >> 4) + mm_m, last))); };
    uint32_t from[UNITS], from_second[MODE == HIDDEN_GRADIENTS ? UNITS : 1];
    const Product &q0 = p.product[which];
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
        const bool is_a = first_unit + i < A_UNITS;
        const int u = is_a ? first_unit + i : first_unit + i - A_UNITS;
        if (is_a) {
            from[i] = A_MMAJOR ? mmajor_from(u, M - m0 - 8, q0.a_ld) : kmajor_from(8 * u + (lane >> 3), M - m0 - 1, q0.a_ld);
        } else if constexpr (B_MMAJOR) {
            from[i] = mmajor_from(u, N - n0 - 8, q0.b_ld);
        } else if constexpr (HIDDEN) { // of eight units 0 .. 3 the gate's 32 rows, 4 .. 7 the other projection's
            from[i] = kmajor_from(32 * (u >> 3) + 8 * (u & 3) + (lane >> 3), N - n0 - 1, q0.b_ld);
        } else {
            from[i] = kmajor_from(8 * u + (lane >> 3), N - n0 - 1, q0.b_ld);
        }
        if constexpr (MODE == HIDDEN_GRADIENTS) {
            from_second[i] = is_a ? kmajor_from(8 * u + (lane >> 3), M - m0 - 1, p.product[2].a_ld) : mmajor_from(u, N - n0 - 8, p.product[2].b_ld);
        }
    }
    // what this wave asks for at step t of all: where its units start, and how much of k is left there
    struct Stage {
        uint64_t a, b, up; // addresses
        uint32_t to;
        int half, left;
        bool own; // the second products of HIDDEN_GRADIENTS
    };
    auto stage_of = [&](int t, int half) {
        const bool second = TWO && t >= steps;
        const int in_order = (second ? t - steps : t) * GROUPS + group; // of the stages, before their turn
        int s = in_order + turn;
        s = (s >= stages ? s - stages : s) + first_stage;
        const Product &q = p.product[MODE == HIDDEN_GRADIENTS ? (second ? 2 : 0) : MODE == INPUT_GRADIENT ? (second ? 1 : 0) : which];
        Stage st;
        st.own = MODE == HIDDEN_GRADIENTS && second;
        st.a = (uint64_t)(q.a + (A_MMAJOR ? (int64_t)64 * s * q.a_ld + m0 : (int64_t)m0 * q.a_ld + 64 * s));
        st.b = (uint64_t)(q.b + (B_MMAJOR || st.own ? (int64_t)64 * s * q.b_ld + n0 : (int64_t)n0 * q.b_ld + 64 * s));
        st.up = HIDDEN && !st.own ? (uint64_t)(p.product[1].b + (int64_t)n0 * p.product[1].b_ld + 64 * s) : st.b;
        st.to = to + (uint32_t)half * (STAGE * 16u);
        st.half = half;
        st.left = GROUPS > 1 && in_order >= stages ? 0 : p.K - 64 * s;
        return st;
    };
    auto base_of = [&](Stage st, bool is_a, int u) {
        const uint64_t b = HIDDEN && (u & 4) ? st.up : st.b;
        return same_in_all_lanes((const void *)(is_a ? st.a : b));
    };
    auto from_of = [&](Stage st, int i) {
        if constexpr (MODE == HIDDEN_GRADIENTS) {
            return st.own ? from_second[i] : from[i];
        } else {
            return from[i];
        }
    };
    auto ask = [&](Stage st) {
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const bool is_a = first_unit + i < A_UNITS;
            const int u = is_a ? first_unit + i : first_unit + i - A_UNITS;
            if ((is_a ? A_MMAJOR : B_MMAJOR || st.own) ? 4 * (u & 15) + mm_k < st.left : 8 * chunk < st.left) {
                load_to_lds(st.to + i * 1024u, base_of(st, is_a, u), from_of(st, i));
            } else {
                slots[st.half * STAGE + i * 64] = zero_u4();
            }
        }
    };
    // unit i of a whole stage in all lanes (`lanes` -1) or none (0): without a branch, beside the products
    auto ask_whole = [&](Stage st, int i, int lanes) {
        const bool is_a = first_unit + i < A_UNITS;
        const int u = is_a ? first_unit + i : first_unit + i - A_UNITS;
        asm volatile("s_mov_b32 exec_lo, %3\n\ts_mov_b32 exec_hi, %3\n\ts_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b64 exec, -1" ::"s"(st.to + i * 1024u),
                     "v"(from_of(st, i)), "s"(base_of(st, is_a, u)), "s"(lanes)
                     : "memory");
    };

    constexpr int SUMS = MODE == HIDDEN_GRADIENTS ? 3 : 2; // 32-wide column blocks of a wave
    f32x16 acc[SUMS][MI];
#pragma unroll
    for (int j = 0; j < SUMS; ++j) {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            acc[j][i] = zero16();
        }
    }
    // where this lane points the transposing reads for the wave's blocks of an M-major operand
    int a_mm[MI], b_mm[2], own_mm = mm_fragment_offset(wn & 3, lane);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        a_mm[i] = ((MI * wm + i) >> 2) * 16384 + mm_fragment_offset((MI * wm + i) & 3, lane);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        b_mm[j] = ((2 * wn + j) >> 2) * 16384 + mm_fragment_offset((2 * wn + j) & 3, lane);
    }
    const int odd = r & 7;
    auto kmajor_fragment = [&](const uint4 *operand, int block, int s) { return as_bf16x8(operand[(32 * block + r) * 8 + ((2 * s + g) ^ odd)]); };
    int t = 0; // the current stage, of all
    auto run = [&](auto is_second) {
        constexpr bool SECOND = decltype(is_second)::value;
        constexpr bool OWN = SECOND && MODE == HIDDEN_GRADIENTS; // sums of its own, one block of columns
        constexpr int NB = OWN ? 1 : 2;
        bf16x8 a[2][MI], b[2][NB];
        auto fetch = [&](int set, const uint4 *stage, int s, int n) { // fragment n of a quarter's MI + NB
            const uint4 *columns = stage + ROWS * 8;
            if (n < NB) {
                if constexpr (OWN) {
                    b[set][n] = mm_fragment((const lds_char *)columns, own_mm, s);
                } else if constexpr (B_MMAJOR) {
                    b[set][n] = mm_fragment((const lds_char *)columns, b_mm[n], s);
                } else {
                    b[set][n] = kmajor_fragment(columns, 2 * wn + n, s);
                }
            } else if constexpr (A_MMAJOR) {
                a[set][n - NB] = mm_fragment((const lds_char *)stage, a_mm[n - NB], s);
            } else {
                a[set][n - NB] = kmajor_fragment(stage, MI * wm + n - NB, s);
            }
        };
#pragma unroll
        for (int n = 0; n < MI + NB; ++n) {
            fetch(0, lds + (t & 1) * STAGE, 0, n);
        }
        // the products of 16 k, beside them the fragments of the next 16, and with ASK a wave's units of a stage
        auto quarter = [&](const uint4 *from_stage, int s, auto asks, Stage st, int lanes) {
            constexpr int STEPS = MI * NB, TOTAL = MI + NB;
#pragma unroll
            for (int n = 0; n < STEPS; ++n) {
                const int i = n / NB, j = n % NB;
                f32x16 &sum = acc[OWN ? 2 : j][i];
                sum = mfma(b[s & 1][j], a[s & 1][i], sum);
                asm volatile("" : "+a"(sum)); // not to be moved behind the barrier
#pragma unroll
                for (int f = n * TOTAL / STEPS; f < (n + 1) * TOTAL / STEPS; ++f) {
                    fetch((s + 1) & 1, from_stage, (s + 1) & 3, f);
                }
                if constexpr (decltype(asks)::value) {
#pragma unroll
                    for (int i = n * UNITS / STEPS; i < (n + 1) * UNITS / STEPS; ++i) {
                        ask_whole(st, i, lanes);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        for (const int end = t + steps; t < end; ++t) {
            const uint4 *stage = lds + (t & 1) * STAGE, *other = lds + ((t + 1) & 1) * STAGE;
            const Stage then = stage_of(t + 2, t & 1);
            __builtin_amdgcn_sched_barrier(0);
            quarter(stage, 0, std::false_type{}, then, 0);
            quarter(stage, 1, std::false_type{}, then, 0);
            quarter(stage, 2, std::false_type{}, then, 0);
            // the next stage is there, and all have read this one; behind the last one what is read is not used
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            const bool more = t + 2 < total;
            if (more && then.left < 64) {
                ask(then);
            }
            quarter(other, 3, std::true_type{}, then, __builtin_amdgcn_readfirstlane(more && then.left >= 64 ? -1 : 0));
        }
    };
    ask(stage_of(0, 0));
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (total > 1) {
        ask(stage_of(1, 1));
    }
    run(std::false_type{});
    if constexpr (TWO) {
        run(std::true_type{});
    }

    if constexpr (SPLIT) {
        if (p.splits > 1) { // a share of the sums, lane by lane: [split][tile of all three][wave][MI][2][4][64] of 16 bytes
            f32x4 *share = reinterpret_cast<f32x4 *>(p.shares) + ((int64_t)place * (WM * WN) + member) * (MI * 2 * 4 * 64) + lane;
#pragma unroll
            for (int i = 0; i < MI; ++i) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        share[((i * 2 + j) * 4 + e) * 64] = f32x4{acc[j][i][4 * e], acc[j][i][4 * e + 1], acc[j][i][4 * e + 2], acc[j][i][4 * e + 3]};
                    }
                }
            }
            return;
        }
    }
    if constexpr (GROUPS == 2) { // the second group's sums to the first
        constexpr int PER_WAVE = 2 * MI * 4 * 64;
        static_assert(WM * WN * PER_WAVE <= GROUPS * 2 * STAGE, "the sums lie where the operands were");
        __syncthreads(); // what the other waves have read ahead lies there
        f32x4 *sums = reinterpret_cast<f32x4 *>(all_lds) + member * PER_WAVE + lane;
        if (group == 1) {
#pragma unroll
            for (int n = 0; n < 2 * MI * 4; ++n) {
                const f32x16 &v = acc[n & 1][n / 8];
                const int e = n / 2 % 4;
                sums[n * 64] = f32x4{v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]};
            }
        }
        __syncthreads();
        if (group == 1) {
            return;
        }
#pragma unroll
        for (int n = 0; n < 2 * MI * 4; ++n) {
            const f32x4 v = sums[n * 64];
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                acc[n & 1][n / 8][4 * (n / 2 % 4) + f] += v[f];
            }
        }
    }
    // results as bf16 through a strip of the LDS of the wave's own, 32 rows by WIDTH columns, out in whole runs of WIDTH
    constexpr int WIDTH = HIDDEN ? 32 : 64, STRIP_LD = WIDTH + 8;
    static_assert(WM * WN * 32 * STRIP_LD * 2 <= 2 * STAGE * 16, "the strips lie where the operands were");
    if constexpr (GROUPS == 1) {
        __syncthreads(); // what the other waves have read ahead lies there
    }
    bf16_t *strip = reinterpret_cast<bf16_t *>(lds + GROUPS / 2 * 2 * STAGE) + member * 32 * STRIP_LD; // with two groups, behind the sums
    auto store = [&](bf16_t *c, int64_t ld, int i, auto value) {
#pragma unroll
        for (int j = 0; j < WIDTH / 32; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                bf16x4 o;
#pragma unroll
                for (int f = 0; f < 4; ++f) {
                    o[f] = (bf16_t)value(j, 4 * e + f);
                }
                *reinterpret_cast<bf16x4 *>(strip + r * STRIP_LD + 32 * j + 8 * e + 4 * g) = o;
            }
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int e = 0; e < WIDTH / 16; ++e) {
            const int piece = lane + 64 * e, row = piece / (WIDTH / 8), part = piece % (WIDTH / 8);
            const int m = m0 + 32 * (MI * wm + i) + row, n = n0 + WIDTH * wn + 8 * part;
            if (m < M && n < N) {
                *reinterpret_cast<uint4 *>(c + (int64_t)m * ld + n) = *reinterpret_cast<const uint4 *>(strip + row * STRIP_LD + 8 * part);
            }
        }
        __builtin_amdgcn_wave_barrier();
    };
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        if constexpr (HIDDEN) {
            f32x16 h, dg, du;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float slope = 0.f;
                const float act = activate<MODE == HIDDEN_GRADIENTS>(acc[0][i][e], p.activation, slope), u = acc[1][i][e];
                h[e] = act * u;
                if constexpr (MODE == HIDDEN_GRADIENTS) {
                    dg[e] = acc[2][i][e] * u * slope;
                    du[e] = acc[2][i][e] * act;
                }
            }
            store(p.c[0], p.c_ld[0], i, [&](int, int e) { return h[e]; });
            if constexpr (MODE == HIDDEN_GRADIENTS) {
                store(p.c[1], p.c_ld[1], i, [&](int, int e) { return dg[e]; });
                store(p.c[2], p.c_ld[2], i, [&](int, int e) { return du[e]; });
            }
        } else {
            store(p.c[which], p.c_ld[which], i, [&](int j, int e) { return acc[j][i][e]; });
        }
    }
}

// The result of split products from its shares: a thread adds four columns of a row over the splits, in one order.
template <int MI, int WM, int WN>
__global__ __launch_bounds__(256) void ff_shares_kernel(const TilesParams p)
{
    constexpr int SIDE = 32 * MI * WM, PER_TILE = WM * WN * MI * 2 * 4 * 64;
    const unsigned all = (unsigned)(p.tiles[0] + p.tiles[1] + p.tiles[2]);
    const int64_t index = (int64_t)blockIdx.x * 256 + threadIdx.x, pitch = (int64_t)all * PER_TILE;
    const f32x4 *share = reinterpret_cast<const f32x4 *>(p.shares) + index;
    f32x4 sum = share[0];
#pragma unroll 8
    for (int s = 1; s < p.splits; ++s) {
        sum += share[s * pitch];
    }
    unsigned tile = (unsigned)(index / PER_TILE);
    const int in = (int)(index % PER_TILE), lane = in & 63, e = (in >> 6) & 3, j = (in >> 8) & 1, i = (in >> 9) % MI, wave = in / (512 * MI);
    int which = 0;
    while (which < 2 && tile >= (unsigned)p.tiles[which]) {
        tile -= (unsigned)p.tiles[which++];
    }
    const int M = p.M[which], N = p.N[which];
    const unsigned MT = (unsigned)(M + SIDE - 1) / SIDE, NT = (unsigned)(N + SIDE - 1) / SIDE;
    const unsigned band = tile / (8 * NT), height = min(8u, MT - 8 * band), of = tile - band * 8 * NT;
    const int m = (int)(8 * band + of % height) * SIDE + 32 * (MI * (wave / WN) + i) + (lane & 31);
    const int n = (int)(of / height) * SIDE + 64 * (wave % WN) + 32 * j + 8 * e + 4 * (lane >> 5);
    if (m < M && n < N) {
        const bf16x4 o = {(bf16_t)sum[0], (bf16_t)sum[1], (bf16_t)sum[2], (bf16_t)sum[3]};
        bf16_t *const to = p.c[which] + (int64_t)m * p.c_ld[which] + n;
        if (n + 4 <= N) {
            __builtin_memcpy(to, &o, sizeof(o));
        } else {
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                if (n + f < N) {
                    to[f] = o[f];
                }
            }
        }
    }
}

// ---- few rows, or few tiles: the W waves of a workgroup share the blocks of 64 k ----
//
// 16 MB rows by 16 NB columns a workgroup, all of them in every wave (and with GATED of both projections): wave w takes blocks w, w + W, ... and brings
// them straight into its own part of the LDS, eight rows of 128 bytes a load, DEPTH blocks ahead and without barriers.  The waves' sums meet in the LDS at
// the end, in one order.  Memory bounds it: 3 x 2048 -> 8192, 24.7 us: GATED 14.9, 4.5 TB/s, PLAIN 9.8, 3.4.
//
// With WITH_REST half of the MB blocks of rows are what the rounding of the others left, product 1's: few enough results are bound by launches, and keep the
// hidden layer to 16 bits almost for nothing (3 x 128 -> 512 7.2 us and 7.1): a result's error is then that of its own rounding, 1.65e-3 in place of 2.35e-3.
template <int MODE, int MB, int NB, int W, int DEPTH, bool WITH_REST = false>
__global__ __launch_bounds__(64 * W) void ff_split_kernel(const TilesParams p)
{
    constexpr int ROW_BLOCKS = WITH_REST ? MB / 2 : MB;
    static_assert(!WITH_REST || (MODE == PLAIN && MB % 2 == 0), "the hidden layer is the product's operand");
    static_assert(MODE == PLAIN || MODE == GATED, "operands along k");
    constexpr int SUMS = MODE == GATED ? 2 : 1, LOADS = 2 * (MB + SUMS * NB), SLOTS = 64 * LOADS;
    static_assert(SUMS * MB * NB <= DEPTH * LOADS, "the sums lie where the operands were");
    extern __shared__ uint4 lds[]; // [W][DEPTH][SLOTS], and at the end sums [W][SUMS][NB][MB][64]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, q = lane >> 4;
    const int M = p.M[0], N = p.N[0], NT = (N + 16 * NB - 1) / (16 * NB);
    const int n0 = (int)(blockIdx.x % (unsigned)NT) * 16 * NB, m0 = (int)(blockIdx.x / (unsigned)NT) * 16 * ROW_BLOCKS;
    const int blocks = (p.K + 63) / 64;
    const int chunk = (lane & 7) ^ (lane >> 3);
    const bf16_t *const a_tile = p.product[0].a + (int64_t)m0 * p.product[0].a_ld;
    [[maybe_unused]] const bf16_t *const rest_tile = p.product[1].a + (int64_t)m0 * p.product[0].a_ld;
    uint32_t a_from[2 * MB], b_from[2 * NB];
#pragma unroll
    for (int u = 0; u < 2 * MB; ++u) {
        a_from[u] = 2u * ((uint32_t)min(8 * (u % (2 * ROW_BLOCKS)) + (lane >> 3), M - m0 - 1) * (uint32_t)p.product[0].a_ld + 8u * (uint32_t)chunk);
    }
#pragma unroll
    for (int u = 0; u < 2 * NB; ++u) {
        b_from[u] = 2u * ((uint32_t)min(8 * u + (lane >> 3), N - n0 - 1) * (uint32_t)p.product[0].b_ld + 8u * (uint32_t)chunk);
    }
    uint4 *const mine = lds + wave * DEPTH * SLOTS;
    const uint32_t to = (uint32_t)(uintptr_t)(const lds_char *)mine;
    auto ask = [&](int b, int slot) {
        const uint32_t stage = to + (uint32_t)slot * (SLOTS * 16u);
        if (8 * chunk < p.K - 64 * b) {
#pragma unroll
            for (int u = 0; u < 2 * MB; ++u) {
                load_to_lds(stage + u * 1024u, (u < 2 * ROW_BLOCKS ? a_tile : rest_tile) + (int64_t)64 * b, a_from[u]);
            }
#pragma unroll
            for (int u = 0; u < 2 * NB * SUMS; ++u) {
                load_to_lds(stage + (2 * MB + u) * 1024u, p.product[u / (2 * NB)].b + (int64_t)n0 * p.product[0].b_ld + (int64_t)64 * b, b_from[u % (2 * NB)]);
            }
        } else { // past the end of a cut block
#pragma unroll
            for (int u = 0; u < LOADS; ++u) {
                mine[slot * SLOTS + u * 64 + lane] = zero_u4();
            }
        }
    };
    f32x4 acc[SUMS][NB][MB];
#pragma unroll
    for (int n = 0; n < SUMS * NB * MB; ++n) {
        acc[n / (NB * MB)][n / MB % NB][n % MB] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
        if (wave + d * W < blocks) {
            ask(wave + d * W, d);
        }
    }
    int slot = 0;
    for (int b = wave; b < blocks; b += W) {
        if (b + (DEPTH - 1) * W < blocks) {
            wait_for_loads<(DEPTH - 1) * LOADS>();
        } else {
            wait_for_loads<0>();
        }
        const uint4 *stage = mine + slot * SLOTS;
        auto operand_of = [&](int block16, int half) { return as_bf16x8(stage[(16 * block16 + r) * 8 + ((4 * half + q) ^ (r & 7))]); };
        bf16x8 a[MB][2], w[SUMS * NB][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < MB; ++j) {
                a[j][h] = operand_of(j, h);
            }
#pragma unroll
            for (int i = 0; i < SUMS * NB; ++i) {
                w[i][h] = operand_of(MB + i, h);
            }
        }
        if (b + DEPTH * W < blocks) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the operands are out of the LDS
            ask(b + DEPTH * W, slot);
        }
        slot = slot + 1 < DEPTH ? slot + 1 : 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < SUMS * NB; ++i) {
#pragma unroll
                for (int j = 0; j < MB; ++j) {
                    f32x4 &sum = acc[i / NB][i % NB][j];
                    sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[i][h], a[j][h], sum, 0, 0, 0);
                }
            }
        }
    }
    __syncthreads(); // the sums take the operands' place
    f32x4 *sums = reinterpret_cast<f32x4 *>(lds);
#pragma unroll
    for (int n = 0; n < SUMS * NB * MB; ++n) {
        sums[(wave * SUMS * NB * MB + n) * 64 + lane] = acc[n / (NB * MB)][n / MB % NB][n % MB];
    }
    __syncthreads();
    for (int t = wave; t < NB * ROW_BLOCKS; t += W) {
        f32x4 sum[SUMS];
#pragma unroll
        for (int s = 0; s < SUMS; ++s) {
            const int at = s * NB * MB + t / ROW_BLOCKS * MB + t % ROW_BLOCKS;
            sum[s] = sums[at * 64 + lane];
#pragma unroll
            for (int v = 1; v < W; ++v) {
                sum[s] += sums[(v * SUMS * NB * MB + at) * 64 + lane];
            }
            if constexpr (WITH_REST) {
                f32x4 rests = sums[(at + ROW_BLOCKS) * 64 + lane];
#pragma unroll
                for (int v = 1; v < W; ++v) {
                    rests += sums[(v * SUMS * NB * MB + at + ROW_BLOCKS) * 64 + lane];
                }
                // an infinity among the weights makes the sum what it is: a rest of the other sign, or of zero, would make it no number
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sum[s][e] = __builtin_isfinite(sum[s][e]) ? sum[s][e] + rests[e] : sum[s][e];
                }
            }
        }
        const int m = m0 + 16 * (t % ROW_BLOCKS) + r, n = n0 + 16 * (t / ROW_BLOCKS) + 4 * q;
        bf16x4 o, rest;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float v = sum[0][e];
            if constexpr (MODE == GATED) {
                float none;
                v = activate<false>(v, p.activation, none) * sum[1][e];
            }
            o[e] = (bf16_t)v;
            rest[e] = rounding_rest(v, o[e]);
        }
        if (m < M && n < N) { // N is a multiple of 8
            *reinterpret_cast<bf16x4 *>(p.c[0] + (int64_t)m * p.c_ld[0] + n) = o;
            if (MODE == GATED && p.c[1] != nullptr) {
                *reinterpret_cast<bf16x4 *>(p.c[1] + (int64_t)m * p.c_ld[0] + n) = rest;
            }
        }
    }
}

// Whether a product's operands fill whole 16-byte pieces: pointers, pitches, and the extents along which rows are contiguous.  Rows of a tile have to lie within
// 32 bits of bytes from its first, up to 255 pitches on; ff_tiles_kernel has no such bound.
bool pieces(const void *ptr, int64_t ld, int64_t contiguous) { return kutacc_hip_aligned16(ptr) && ld % 8 == 0 && contiguous % 8 == 0 && ld < (1 << 23); }

int64_t tiles_of(int64_t m, int64_t n) { return (m + TILE - 1) / TILE * ((n + TILE - 1) / TILE); }

template <int MODE>
int launch_any(TilesParams p, double flops, const char *name, hipStream_t stream)
{
    static size_t configured[2][KUTACC_DEVICE_SLOTS] = {};
    int64_t blocks = 0;
    for (int i = 0; i < 3; ++i) {
        const int64_t tiles = tiles_of(p.M[i], p.N[i]);
        blocks += tiles;
        p.tiles[i] = (int)std::min<int64_t>(tiles, INT32_MAX);
    }
    if (MODE == WEIGHT_GRADIENTS && p.M[1] != 0 && !kutacc_grid_fits(blocks * p.splits, 256)) { // one by one
        for (int i = 0; i < 3 && p.M[i] != 0; ++i) {
            TilesParams one = p;
            one.product[0] = p.product[i], one.c[0] = p.c[i], one.c_ld[0] = p.c_ld[i], one.M[0] = p.M[i], one.N[0] = p.N[i];
            one.M[1] = one.M[2] = 0;
            if (const int rc = launch_any<MODE>(one, flops / 3, name, stream)) {
                return rc;
            }
        }
        return 0;
    }
    const bool tiny = std::min(p.N[0], MODE == WEIGHT_GRADIENTS ? p.M[0] : p.K) < 8; // contiguous extents
    const auto kernel = tiny ? &ff_tiles_kernel<MODE, true> : &ff_tiles_kernel<MODE, false>;
    if (const hipError_t e = kutacc_opt_in_lds(reinterpret_cast<const void *>(kernel), TILES_LDS, configured[tiny])) {
        return kutacc_hip_status(e);
    }
    if (!kutacc_grid_fits(blocks * p.splits, 256)) {
        return KUTACC_HIP_EUNSUPPORTED;
    }
    kutacc_prof::KernelTimer t(name, flops, stream);
    kernel<<<dim3((unsigned)(blocks * p.splits)), 256, TILES_LDS, stream>>>(p);
    if ((MODE == WEIGHT_GRADIENTS || MODE == INPUT_GRADIENT) && p.splits > 1) {
        ff_shares_kernel<2, 2, 2><<<dim3((unsigned)(blocks * 16)), 256, 0, stream>>>(p);
    }
    return kutacc_hip_status(hipGetLastError());
}

// tiles of SIDE rows by `columns`, of all products; p.tiles filled in
int64_t count_tiles(TilesParams &p, int side, int columns)
{
    int64_t all = 0;
    for (int i = 0; i < 3; ++i) {
        const int64_t tiles = ((int64_t)p.M[i] + side - 1) / side * (((int64_t)p.N[i] + columns - 1) / columns);
        p.tiles[i] = (int)std::min<int64_t>(tiles, INT32_MAX);
        all += tiles;
    }
    return all;
}

template <int MODE, int MI, int WM, int WN, int GROUPS>
int launch_pieces(TilesParams p, hipStream_t stream)
{
    constexpr int ROWS = 32 * MI * WM, SIDE = 64 * WN;
    constexpr size_t LDS = (size_t)GROUPS * 2 * (ROWS + SIDE) * 128;
    static size_t configured[KUTACC_DEVICE_SLOTS] = {};
    const auto kernel = &ff_pieces_kernel<MODE, MI, WM, WN, GROUPS>;
    const int64_t tiles = count_tiles(p, ROWS, MODE == GATED || MODE == HIDDEN_GRADIENTS ? SIDE / 2 : SIDE), groups = tiles * p.splits;
    if (!kutacc_grid_fits(groups, 64 * WM * WN * GROUPS)) {
        return KUTACC_HIP_EUNSUPPORTED;
    }
    if (const hipError_t e = kutacc_opt_in_lds(reinterpret_cast<const void *>(kernel), LDS, configured)) {
        return kutacc_hip_status(e);
    }
    kernel<<<dim3((unsigned)groups), 64 * WM * WN * GROUPS, LDS, stream>>>(p);
    if constexpr ((MODE == WEIGHT_GRADIENTS || MODE == INPUT_GRADIENT) && MI == 2 && GROUPS == 1) {
        if (p.splits > 1) {
            ff_shares_kernel<MI, WM, WN><<<dim3((unsigned)(tiles * WM * WN * MI * 2)), 256, 0, stream>>>(p);
        }
    }
    return kutacc_hip_status(hipGetLastError());
}

template <int MODE, int MB, int NB, int W, int DEPTH, bool WITH_REST = false>
int launch_split(TilesParams p, hipStream_t stream)
{
    constexpr size_t LDS = (size_t)W * DEPTH * 2 * (MB + (MODE == GATED ? 2 : 1) * NB) * 1024;
    static size_t configured[KUTACC_DEVICE_SLOTS] = {};
    const auto kernel = &ff_split_kernel<MODE, MB, NB, W, DEPTH, WITH_REST>;
    const int64_t groups = count_tiles(p, WITH_REST ? 8 * MB : 16 * MB, 16 * NB);
    if (!kutacc_grid_fits(groups, 64 * W)) {
        return KUTACC_HIP_EUNSUPPORTED;
    }
    if (const hipError_t e = kutacc_opt_in_lds(reinterpret_cast<const void *>(kernel), LDS, configured)) {
        return kutacc_hip_status(e);
    }
    kernel<<<dim3((unsigned)groups), 64 * W, LDS, stream>>>(p);
    return kutacc_hip_status(hipGetLastError());
}

// whether the weights' gradients make enough tiles of 256 x 256 without a split of their rows
bool whole_rows(TilesParams p) { return 4 * count_tiles(p, 256, 256) >= 3 * kutacc_cu_count(); }

// A kernel's tile, its threads, how many of its workgroups a CU holds, and what a round of them takes for 64 k
struct Choice {
    int rows, columns, threads, per_cu;
    float round;
};
// of those that can be started, the one that takes the fewest rounds, weighted with what they take
template <int N>
int least(TilesParams p, const Choice (&choices)[N])
{
    int best = 0;
    double time = 0;
    for (int i = 0; i < N; ++i) {
        const int64_t tiles = count_tiles(p, choices[i].rows, choices[i].columns), slots = (int64_t)kutacc_cu_count() * choices[i].per_cu;
        const double t = (double)((tiles + slots - 1) / slots) * choices[i].round;
        if (kutacc_grid_fits(tiles, choices[i].threads) && (time == 0 || t < time)) {
            best = i, time = t;
        }
    }
    return best;
}

// The rounds' times are measured, us for 64 k: 4001 x 1024 x 2816, 8192 x 2048 x 8192, 1000 x 1024 x 4096, 128 x 2048 x 8192 (rows x columns x k) and for the
// gated form 4001 x 2816 x 1024, 8192 x 8192 x 2048, 256 x 4096 x 1024, 64 x 8192 x 2048.
template <int MODE>
int launch_whole(const TilesParams &p, hipStream_t stream)
{
    if constexpr (MODE == PLAIN) {
        if (p.product[1].a != nullptr) {
            return p.M[0] <= 16 ? launch_split<MODE, 2, 1, 8, 2, true>(p, stream) : launch_split<MODE, 4, 2, 8, 1, true>(p, stream);
        }
        if (p.M[0] <= 16) {
            return launch_split<MODE, 1, 1, 16, 2>(p, stream);
        }
        constexpr Choice choices[] = {{32, 32, 1024, 1, 0.10f}, {32, 64, 512, 1, 0.13f}, {64, 64, 512, 1, 0.23f}, {128, 128, 512, 1, 0.66f}, {128, 128, 256, 2, 1.05f}, {192, 256, 512, 1, 1.41f}, {256, 256, 512, 1, 1.70f}};
        switch (least(p, choices)) {
        case 0: return launch_split<MODE, 2, 2, 16, 1>(p, stream);
        case 1: return launch_split<MODE, 2, 4, 8, 1>(p, stream);
        case 2: return launch_split<MODE, 4, 4, 8, 1>(p, stream);
        case 3: return launch_pieces<MODE, 2, 2, 2, 2>(p, stream);
        case 4: return launch_pieces<MODE, 2, 2, 2, 1>(p, stream);
        case 5: return launch_pieces<MODE, 3, 2, 4, 1>(p, stream);
        default: return launch_pieces<MODE, 4, 2, 4, 1>(p, stream);
        }
    } else if constexpr (MODE == GATED) {
        if (p.M[0] <= 16) {
            return launch_split<MODE, 1, 1, 8, 2>(p, stream);
        }
        if (p.c[1] != nullptr) {
            return launch_split<MODE, 2, 2, 8, 1>(p, stream);
        }
        constexpr Choice choices[] = {{32, 32, 512, 1, 0.23f}, {64, 32, 512, 1, 0.33f}, {128, 64, 256, 2, 1.15f}, {192, 128, 512, 1, 1.45f}, {256, 128, 512, 1, 1.90f}};
        switch (least(p, choices)) {
        case 0: return launch_split<MODE, 2, 2, 8, 1>(p, stream);
        case 1: return launch_split<MODE, 4, 2, 8, 1>(p, stream);
        case 2: return launch_pieces<MODE, 2, 2, 2, 1>(p, stream);
        case 3: return launch_pieces<MODE, 3, 2, 4, 1>(p, stream);
        default: return launch_pieces<MODE, 4, 2, 4, 1>(p, stream);
        }
    } else if constexpr (MODE == HIDDEN_GRADIENTS) {
        constexpr Choice choices[] = {{128, 64, 256, 2, 1.0f}, {192, 128, 512, 1, 1.27f}};
        return least(p, choices) == 0 ? launch_pieces<MODE, 2, 2, 2, 1>(p, stream) : launch_pieces<MODE, 3, 2, 4, 1>(p, stream);
    } else if constexpr (MODE == INPUT_GRADIENT) {
        if (p.splits > 1) {
            return launch_pieces<MODE, 2, 2, 2, 1>(p, stream);
        }
        constexpr Choice choices[] = {{128, 128, 512, 1, 0.61f}, {128, 128, 256, 2, 0.97f}, {256, 256, 512, 1, 1.55f}};
        switch (least(p, choices)) {
        case 0: return launch_pieces<MODE, 2, 2, 2, 2>(p, stream);
        case 1: return launch_pieces<MODE, 2, 2, 2, 1>(p, stream);
        default: return launch_pieces<MODE, 4, 2, 4, 1>(p, stream);
        }
    } else {
        return p.splits == 1 && whole_rows(p) ? launch_pieces<MODE, 4, 2, 4, 1>(p, stream) : launch_pieces<MODE, 2, 2, 2, 1>(p, stream);
    }
}

template <int MODE>
int launch(const TilesParams &p, bool any, double flops, const char *name, hipStream_t stream)
{
    if (any) {
        return launch_any<MODE>(p, flops, name, stream);
    }
    kutacc_prof::KernelTimer t(name, flops, stream);
    return launch_whole<MODE>(p, stream);
}

// How many ways the rows are split for the weights' gradients: 128 x 128 tiles of fewer than two workgroups a CU, into ranges of at least eight stages (us, split,
// whole, and whole in 256 x 256: 300 x 512 x 2048 10.9, 11.0, 15.5; 5000 x 256 x 1024 26, 60, 101; 20000 x 256 x 1024 48, 218, 370; 8000 x 512 x 2048 73, 92, 162;
// 2000 x 1024 x 4096 56, 63, 60; 4096 x 1024 x 4096, which has tiles of 256 x 256 enough: -, 111, 99)
int weight_splits(int64_t rows, int64_t c_o, int64_t c_i)
{
    TilesParams p = {};
    p.M[0] = p.M[1] = (int)c_i, p.N[0] = p.N[1] = (int)c_o, p.M[2] = (int)c_o, p.N[2] = (int)c_i;
    if (whole_rows(p)) {
        return 1;
    }
    const int64_t tiles = count_tiles(p, 128, 128), stages = (rows + 63) / 64;
    return (int)std::max<int64_t>(1, std::min<int64_t>(2 * kutacc_cu_count() / tiles, stages / 8));
}
// How many ways the hidden units are split for the gradient of x, where its tiles leave half of the CUs and more without work: into ranges of at least four
// stages, and only where that saves more than the shares cost, all in us: a stage of both products takes 1.15, a share of a tile 0.033 to write and read, the
// kernel that adds them 3.  (us, the whole backward pass, unsplit and split: 300 x 512 x 2048 64 and 42, 93 x 512 x 1024 42 and 35, 2 x 2048 x 8192 187 and 96,
// 1000 x 1024 x 4096 137 and 106, 4000 x 384 x 1536 87 and 85, 5618 x 256 x 1024 70 and 71.)
int input_splits(int64_t rows, int64_t c_o, int64_t c_i)
{
    TilesParams p = {};
    p.M[0] = (int)rows, p.N[0] = (int)c_o;
    const int64_t tiles = count_tiles(p, 128, 128), stages = (c_i + 63) / 64;
    if (2 * tiles > kutacc_cu_count()) {
        return 1;
    }
    const int64_t splits = std::max<int64_t>(1, std::min<int64_t>(2 * kutacc_cu_count() / std::max<int64_t>(tiles, 1), stages / 4));
    return 1.15 * (double)stages * (double)(splits - 1) > (3 + 0.033 * (double)(tiles * splits)) * (double)splits ? (int)splits : 1;
}
int64_t shares_bytes(int64_t rows, int64_t c_o, int64_t c_i)
{
    const int64_t weights = weight_splits(rows, c_o, c_i), input = input_splits(rows, c_o, c_i), across = (c_o + 127) / 128, tile = 128 * 128 * 4;
    return std::max(weights == 1 ? 0 : weights * ((c_i + 127) / 128) * across * 3 * tile, input == 1 ? 0 : input * ((rows + 127) / 128) * across * tile);
}

int64_t padded(int64_t v) { return (v + 31) / 32 * 32; }
int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }

// results few enough to keep what the rounding of the hidden layer leaves
bool keeps_rest(int64_t rows, int64_t c_o) { return rows <= 64 && rows * c_o <= 4096; }
} // namespace

namespace kutacc_launch {

int64_t gated_transition_workspace(int64_t rows, int64_t c_o, int64_t c_i) { return (keeps_rest(rows, c_o) ? 2 : 1) * align256(2 * rows * padded(c_i)); }

int gated_transition(const kutacc_hip_gated_transition_args_t &a, hipStream_t stream)
{
    if (gated_rows_takes(a)) {
        return gated_rows(a, stream);
    }
    const int64_t rows = a.rows, c_o = a.c_o, c_i = a.c_i, h_ld = padded(c_i);
    bf16_t *h = (bf16_t *)a.workspace;
    TilesParams p = {};
    p.splits = 1;
    p.product[0] = {(const bf16_t *)a.x, (const bf16_t *)a.gate_w, a.x_ld, c_o};
    p.product[1] = {(const bf16_t *)a.x, (const bf16_t *)a.up_w, a.x_ld, c_o};
    p.c[0] = h, p.c_ld[0] = h_ld;
    p.M[0] = (int)rows, p.N[0] = (int)c_i, p.K = (int)c_o, p.activation = a.activation;
    const bool widths = c_o % 8 == 0 && c_i % 8 == 0;
    const bool any_in = !widths || !pieces(h, h_ld, c_i) || !pieces(a.x, a.x_ld, c_o) || !pieces(a.gate_w, c_o, c_o) || !pieces(a.up_w, c_o, c_o);
    const bool any_out = !widths || !pieces(h, h_ld, c_i) || !pieces(a.down_w, c_i, c_i) || !pieces(a.out, a.out_ld, c_o);
    bf16_t *const rest = keeps_rest(rows, c_o) && !any_in && !any_out ? h + align256(2 * rows * h_ld) / 2 : nullptr;
    p.c[1] = rest;
    if (const int rc = launch<GATED>(p, any_in, 4.0 * (double)rows * (double)c_o * (double)c_i, "gated_transition<gated>", stream)) {
        return rc;
    }
    TilesParams d = {};
    d.splits = 1;
    d.product[0] = {h, (const bf16_t *)a.down_w, h_ld, c_i};
    d.product[1] = {rest, (const bf16_t *)a.down_w, h_ld, c_i};
    d.c[0] = (bf16_t *)a.out, d.c_ld[0] = a.out_ld;
    d.M[0] = (int)rows, d.N[0] = (int)c_o, d.K = (int)c_i;
    return launch<PLAIN>(d, any_out, 2.0 * (double)rows * (double)c_o * (double)c_i, "gated_transition<plain>", stream);
}

int64_t gated_transition_backward_workspace(int64_t rows, int64_t c_o, int64_t c_i)
{
    int64_t bytes = 3 * align256(2 * rows * padded(c_i)) + shares_bytes(rows, c_o, c_i);
    if (gated_few_rows_backward_fits(rows, c_o, c_i)) {
        bytes = std::max(bytes, gated_few_rows_backward_workspace(rows, c_o, c_i));
    }
    return c_o == 64 || c_o == 128 ? std::max(bytes, gated_rows_backward_workspace(rows, c_o, c_i)) : bytes;
}

int gated_transition_backward(const kutacc_hip_gated_transition_backward_args_t &a, hipStream_t stream)
{
    if (gated_few_rows_backward_takes(a)) {
        return gated_few_rows_backward(a, stream);
    }
    if (gated_rows_backward_takes(a)) {
        return gated_rows_backward(a, stream);
    }
    const int64_t rows = a.rows, c_o = a.c_o, c_i = a.c_i, ld = padded(c_i), each = align256(2 * rows * ld) / 2;
    bf16_t *h = (bf16_t *)a.workspace, *dg = h + each, *du = dg + each;
    float *shares = reinterpret_cast<float *>(du + each);
    const bf16_t *x = (const bf16_t *)a.x, *dy = (const bf16_t *)a.grad_out;
    const bf16_t *wg = (const bf16_t *)a.gate_w, *wu = (const bf16_t *)a.up_w, *wd = (const bf16_t *)a.down_w;
    const double flops = 2.0 * (double)rows * (double)c_o * (double)c_i;
    const bool rows_fit = pieces(x, a.x_ld, c_o) && pieces(dy, a.grad_out_ld, c_o), hidden_fit = c_o % 8 == 0 && pieces(h, ld, c_i);
    const bool weights_fit = hidden_fit && pieces(wg, c_o, c_o) && pieces(wu, c_o, c_o);
    TilesParams p = {};
    p.splits = 1;
    p.product[0] = {x, wg, a.x_ld, c_o};
    p.product[1] = {x, wu, a.x_ld, c_o};
    p.product[2] = {dy, wd, a.grad_out_ld, c_i};
    p.c[0] = h, p.c[1] = dg, p.c[2] = du, p.c_ld[0] = p.c_ld[1] = p.c_ld[2] = ld;
    p.M[0] = (int)rows, p.N[0] = (int)c_i, p.K = (int)c_o, p.activation = a.activation;
    if (const int rc = launch<HIDDEN_GRADIENTS>(p, !rows_fit || !weights_fit || !pieces(wd, c_i, c_i), 3 * flops, "gated_transition<hidden gradients>", stream)) {
        return rc;
    }
    if (a.grad_x != nullptr) {
        TilesParams d = {};
        d.splits = input_splits(rows, c_o, c_i);
        d.shares = shares;
        d.product[0] = {dg, wg, ld, c_o};
        d.product[1] = {du, wu, ld, c_o};
        d.c[0] = (bf16_t *)a.grad_x, d.c_ld[0] = a.grad_x_ld;
        d.M[0] = (int)rows, d.N[0] = (int)c_o, d.K = (int)c_i;
        if (const int rc = launch<INPUT_GRADIENT>(d, !weights_fit || !pieces(a.grad_x, a.grad_x_ld, c_o), 2 * flops, "gated_transition<input gradient>", stream)) {
            return rc;
        }
    }
    TilesParams w = {};
    w.K = (int)rows;
    int count = 0;
    auto add = [&](Product q, void *c, int64_t m, int64_t n) {
        if (c != nullptr) {
            w.product[count] = q;
            w.c[count] = (bf16_t *)c, w.c_ld[count] = n, w.M[count] = (int)m, w.N[count] = (int)n;
            ++count;
        }
    };
    add({dg, x, ld, a.x_ld}, a.grad_gate_w, c_i, c_o);
    add({du, x, ld, a.x_ld}, a.grad_up_w, c_i, c_o);
    add({dy, h, a.grad_out_ld, ld}, a.grad_down_w, c_o, c_i);
    const bool aligned = (!a.grad_gate_w || kutacc_hip_aligned16(a.grad_gate_w)) && (!a.grad_up_w || kutacc_hip_aligned16(a.grad_up_w)) && (!a.grad_down_w || kutacc_hip_aligned16(a.grad_down_w));
    w.splits = weight_splits(rows, c_o, c_i);
    w.shares = shares;
    return count == 0 ? 0 : launch<WEIGHT_GRADIENTS>(w, !rows_fit || !hidden_fit || !aligned, count * flops, "gated_transition<weight gradients>", stream);
}

} // namespace kutacc_launch
