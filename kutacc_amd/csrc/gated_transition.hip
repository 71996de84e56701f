// The gated transition and its backward pass, bf16 with fp32 sums:
//   g = x Wg^T,  u = x Wu^T,  h = act(g) u,  out = h Wd^T,      act(v) = v sigmoid(t(v))
//   dh = dy Wd,  dg = dh u act'(g),  du = dh act(g),  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dWd = dy^T h
// act'(v) = s + v s (1 - s) t'(v) with s = sigmoid(t(v)).  silu: t = v; gelu (its tanh form): t = 2 sqrt(2 / pi) (v + 0.044715 v^3).
//
// g, u and dh are never rounded: the kernel that forms them holds all of them of one tile at once, and h, dg and du are rounded once, as
// operands of the products that follow.
//
// ff_tiles_kernel covers every shape: 128 x 128 of a result per workgroup of four waves, K in steps of 64 through the LDS, for a list of
// products that share the tile.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "gemm_panels.h"
#include "launch_internal.h"
#include "mfma_tiles.h"
#include "profiler.h"

namespace {
using namespace kutacc_dev;

// ---- the activation ----

constexpr float GELU_SLOPE = 1.5957691216057308f, GELU_CUBE = 0.044715f; // 2 sqrt(2 / pi)

// act(v), and its derivative where it is asked for
template <bool DERIVATIVE>
__device__ __forceinline__ float activate(float v, int activation, float &derivative)
{
    float t = v, slope = 1.f;
    if (activation == KUTACC_HIP_GELU) {
        const float square = v * v;
        t = GELU_SLOPE * fmaf(GELU_CUBE * square, v, v);
        slope = GELU_SLOPE * fmaf(3.f * GELU_CUBE, square, 1.f);
    }
    const float s = sigmoid_fast(t), a = v * s;
    if constexpr (DERIVATIVE) {
        derivative = fmaf(a * (1.f - s), slope, s);
    }
    return a;
}

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
};

constexpr int TILE = 128, OPERAND_SLOTS = 1024, CT_LD = 136;
constexpr size_t TILES_LDS = TILE * CT_LD * 2;

template <int MODE, bool ANY>
__global__ __launch_bounds__(256, MODE == GATED || MODE == HIDDEN_GRADIENTS ? 1 : 2) void ff_tiles_kernel(const TilesParams p)
{
    constexpr int SUMS = MODE == GATED ? 2 : MODE == HIDDEN_GRADIENTS ? 3 : 1;
    constexpr int PRODUCTS = MODE == INPUT_GRADIENT ? 2 : SUMS;
    extern __shared__ uint4 lds[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = lane & 31, g = lane >> 5, wm = wave >> 1, wn = wave & 1;
    int which = 0, tile = blockIdx.x;
    if constexpr (MODE == WEIGHT_GRADIENTS) {
        while (which < 2 && tile >= p.tiles[which]) {
            tile -= p.tiles[which++];
        }
    }
    const int M = p.M[which], N = p.N[which], NT = (N + TILE - 1) / TILE;
    const int m0 = tile / NT * TILE, n0 = tile % NT * TILE;

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
    const int steps = (p.K + KSTEP - 1) / KSTEP;
#pragma unroll
    for (int n = 0; n < PRODUCTS; ++n) {
        constexpr bool A_MMAJOR = MODE == WEIGHT_GRADIENTS;
        const bool B_MMAJOR = MODE == INPUT_GRADIENT || MODE == WEIGHT_GRADIENTS || (MODE == HIDDEN_GRADIENTS && n == 2); // a constant in every copy
        const Product &q = p.product[MODE == WEIGHT_GRADIENTS ? which : n];
        auto fetch_a = [&](int k0) {
            return A_MMAJOR ? load_mmajor<ANY>(q.a, q.a_ld, m0 + 64 * (wave & 1), M, k0 + 32 * (wave >> 1), p.K, lane)
                            : load_kmajor<ANY>(q.a, q.a_ld, m0 + 32 * wave, M - 1, k0, p.K, lane);
        };
        auto fetch_b = [&](int k0) {
            return B_MMAJOR ? load_mmajor<ANY>(q.b, q.b_ld, n0 + 64 * (wave & 1), N, k0 + 32 * (wave >> 1), p.K, lane)
                            : load_kmajor<ANY>(q.b, q.b_ld, n0 + 32 * wave, N - 1, k0, p.K, lane);
        };
        auto park = [&](uint4 *operand, bool mmajor, const PanelRegs &f) {
            if (mmajor) {
                store_mmajor(operand, 64 * (wave & 1), 32 * (wave >> 1), lane, f);
            } else {
                panel_store(operand + wave * 256, lane, f);
            }
        };
        f32x16(&sum)[2][2] = acc[SUMS == 1 ? 0 : n];
        PanelRegs ra = fetch_a(0), rb = fetch_b(0);
        for (int kt = 0; kt < steps; ++kt) {
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

// Whether a product's operands fill whole 16-byte pieces: pointers, pitches, and the extents along which rows are contiguous
bool pieces(const void *ptr, int64_t ld, int64_t contiguous) { return kutacc_hip_aligned16(ptr) && ld % 8 == 0 && contiguous % 8 == 0; }

int64_t tiles_of(int64_t m, int64_t n) { return (m + TILE - 1) / TILE * ((n + TILE - 1) / TILE); }

template <int MODE>
int launch_tiles(TilesParams p, bool any, double flops, const char *name, hipStream_t stream)
{
    static size_t configured[2][KUTACC_DEVICE_SLOTS] = {};
    int64_t blocks = 0;
    for (int i = 0; i < 3; ++i) {
        const int64_t tiles = tiles_of(p.M[i], p.N[i]);
        blocks += tiles;
        if (blocks > INT32_MAX) {
            return KUTACC_HIP_EUNSUPPORTED;
        }
        p.tiles[i] = (int)tiles;
    }
    const auto kernel = any ? &ff_tiles_kernel<MODE, true> : &ff_tiles_kernel<MODE, false>;
    if (const hipError_t e = kutacc_opt_in_lds(reinterpret_cast<const void *>(kernel), TILES_LDS, configured[any])) {
        return kutacc_hip_status(e);
    }
    kutacc_prof::KernelTimer t(name, flops, stream);
    kernel<<<dim3((unsigned)blocks), 256, TILES_LDS, stream>>>(p);
    return kutacc_hip_status(hipGetLastError());
}

int64_t padded(int64_t v) { return (v + 31) / 32 * 32; }
int64_t align256(int64_t v) { return (v + 255) / 256 * 256; }
} // namespace

namespace kutacc_launch {

int64_t gated_transition_workspace(int64_t rows, int64_t c_o, int64_t c_i) { return align256(2 * rows * padded(c_i)); }

int gated_transition(const kutacc_hip_gated_transition_args_t &a, hipStream_t stream)
{
    const int64_t rows = a.rows, c_o = a.c_o, c_i = a.c_i, h_ld = padded(c_i);
    bf16_t *h = (bf16_t *)a.workspace;
    TilesParams p = {};
    p.product[0] = {(const bf16_t *)a.x, (const bf16_t *)a.gate_w, a.x_ld, c_o};
    p.product[1] = {(const bf16_t *)a.x, (const bf16_t *)a.up_w, a.x_ld, c_o};
    p.c[0] = h, p.c_ld[0] = h_ld;
    p.M[0] = (int)rows, p.N[0] = (int)c_i, p.K = (int)c_o, p.activation = a.activation;
    const bool any_in = !pieces(a.x, a.x_ld, c_o) || !kutacc_hip_aligned16(a.gate_w) || !kutacc_hip_aligned16(a.up_w);
    if (const int rc = launch_tiles<GATED>(p, any_in, 4.0 * (double)rows * (double)c_o * (double)c_i, "ff_tiles_kernel<gated>", stream)) {
        return rc;
    }
    TilesParams d = {};
    d.product[0] = {h, (const bf16_t *)a.down_w, h_ld, c_i};
    d.c[0] = (bf16_t *)a.out, d.c_ld[0] = a.out_ld;
    d.M[0] = (int)rows, d.N[0] = (int)c_o, d.K = (int)c_i;
    return launch_tiles<PLAIN>(d, !pieces(a.down_w, c_i, c_i), 2.0 * (double)rows * (double)c_o * (double)c_i, "ff_tiles_kernel<plain>", stream);
}

int64_t gated_transition_backward_workspace(int64_t rows, int64_t c_o, int64_t c_i) { return 3 * align256(2 * rows * padded(c_i)); }

int gated_transition_backward(const kutacc_hip_gated_transition_backward_args_t &a, hipStream_t stream)
{
    const int64_t rows = a.rows, c_o = a.c_o, c_i = a.c_i, ld = padded(c_i), each = align256(2 * rows * ld) / 2;
    bf16_t *h = (bf16_t *)a.workspace, *dg = h + each, *du = dg + each;
    const bf16_t *x = (const bf16_t *)a.x, *dy = (const bf16_t *)a.grad_out;
    const bf16_t *wg = (const bf16_t *)a.gate_w, *wu = (const bf16_t *)a.up_w, *wd = (const bf16_t *)a.down_w;
    const double flops = 2.0 * (double)rows * (double)c_o * (double)c_i;
    const bool rows_fit = pieces(x, a.x_ld, c_o) && pieces(dy, a.grad_out_ld, c_o), weights_fit = kutacc_hip_aligned16(wg) && kutacc_hip_aligned16(wu) && c_o % 8 == 0;
    TilesParams p = {};
    p.product[0] = {x, wg, a.x_ld, c_o};
    p.product[1] = {x, wu, a.x_ld, c_o};
    p.product[2] = {dy, wd, a.grad_out_ld, c_i};
    p.c[0] = h, p.c[1] = dg, p.c[2] = du, p.c_ld[0] = p.c_ld[1] = p.c_ld[2] = ld;
    p.M[0] = (int)rows, p.N[0] = (int)c_i, p.K = (int)c_o, p.activation = a.activation;
    if (const int rc = launch_tiles<HIDDEN_GRADIENTS>(p, !rows_fit || !weights_fit || !pieces(wd, c_i, c_i), 3 * flops, "ff_tiles_kernel<hidden gradients>", stream)) {
        return rc;
    }
    if (a.grad_x != nullptr) {
        TilesParams d = {};
        d.product[0] = {dg, wg, ld, c_o};
        d.product[1] = {du, wu, ld, c_o};
        d.c[0] = (bf16_t *)a.grad_x, d.c_ld[0] = a.grad_x_ld;
        d.M[0] = (int)rows, d.N[0] = (int)c_o, d.K = (int)c_i;
        if (const int rc = launch_tiles<INPUT_GRADIENT>(d, !weights_fit || c_i % 8 != 0, 2 * flops, "ff_tiles_kernel<input gradient>", stream)) {
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
    return count == 0 ? 0 : launch_tiles<WEIGHT_GRADIENTS>(w, !rows_fit || c_i % 8 != 0, count * flops, "ff_tiles_kernel<weight gradients>", stream);
}

} // namespace kutacc_launch
