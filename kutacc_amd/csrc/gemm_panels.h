// Operands of the bf16 matrix products on 128 x 128 tiles: steps of 64 k from global memory into the LDS and out of it as MFMA fragments, for
// operands stored K-major (rows contiguous in k) and M-major (contiguous along the tile's rows).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "mfma_tiles.h"

namespace kutacc_dev {

constexpr int KSTEP = 64;

// K-major operand: rows row0..row0+31 (clamped), 64 k from k0; chunks past K read as zero.  ANY (here and below): extents,
// pitches and pointers need not be multiples of 8 elements -- unaligned 16-byte loads, and the last piece of a row shifted
// into place.
template <bool ANY>
__device__ __forceinline__ PanelRegs load_kmajor(const bf16_t *base, int64_t ld, int row0, int last_row, int k0, int K, int lane)
{
    const int col = k0 + (lane & 7) * 8;
    const bool ok = col < K;
    const int colc = ok ? col : 0;
    PanelRegs p;
    uint4 *dst[4] = {&p.r0, &p.r1, &p.r2, &p.r3};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        int row = row0 + 8 * i + (lane >> 3);
        row = row < last_row ? row : last_row;
        if constexpr (ANY) {
            *dst[i] = k0 + KSTEP <= K ? load8_any(base + (int64_t)row * ld, col) : load8_checked(base + (int64_t)row * ld, col, K);
            continue;
        }
        uint4 v = *reinterpret_cast<const uint4 *>(base + (int64_t)row * ld + colc);
        if (!ok) {
            v = make_uint4(0u, 0u, 0u, 0u);
        }
        *dst[i] = v;
    }
    return p;
}

// M-major operand (element (m, k) at base + k*ld + m).  Its tile goes to LDS the way it lies in memory, 64 rows k of
// 128 m (256 bytes), and the MFMA fragments -- 8 consecutive k of one m per lane -- come out of the LDS transposing
// read of gfx950, ds_read_b64_tr_b16: within 16 lanes, lane i receives element (i & 3) of the 8-byte chunks that lanes
// 4j + (i >> 2), j = 0..3, point at.  With lane s of the group pointing at row k0 + (s >> 2), m = m0 + 4 (s & 3), lane
// i ends up with k0..k0+3 of m0 + i: a 4 x 16 block transposed per group and instruction, two instructions per
// fragment.  The 8-byte chunk index of a row is XOR-ed with 8 (k & 3), which spreads the four rows a group reads over
// all banks; writes are whole 16-byte pieces of a row.
//
// Loading: 64 m from m0, 32 k from k0 per wave.  Lane (kk, mc) takes 8 consecutive m of row k0 + 8i + mm_row(kk); a
// load instruction covers 8 k x 128 contiguous bytes.  mm_row orders the rows so that the 16 lanes that store together
// hold rows with different k & 3 (different bank halves after the swizzle).
__device__ __forceinline__ int mm_row(int kk) { return (kk & 4) | ((kk & 1) << 1) | ((kk >> 1) & 1); }

template <bool ANY = false>
__device__ __forceinline__ PanelRegs load_mmajor(const bf16_t *base, int64_t ld, int m0, int rows, int k0, int K, int lane)
{
    int m = m0 + (lane & 7) * 8;
    const bool whole = m + 8 <= rows;
    m = ANY || whole ? m : rows - 8; // rows past the end are never stored; any valid address will do
    PanelRegs p;
    uint4 *dst[4] = {&p.r0, &p.r1, &p.r2, &p.r3};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = k0 + 8 * i + mm_row(lane >> 3);
        const bool ok = k < K;
        if constexpr (ANY) {
            const bf16_t *row = base + (int64_t)(ok ? k : 0) * ld;
            const uint4 v = whole ? load8_any(row, m) : load8_checked(row, m, rows);
            *dst[i] = ok ? v : zero_u4();
            continue;
        }
        uint4 v = *reinterpret_cast<const uint4 *>(base + (int64_t)(ok ? k : 0) * ld + m);
        if (!ok) {
            v = make_uint4(0u, 0u, 0u, 0u);
        }
        *dst[i] = v;
    }
    return p;
}

// what load_mmajor fetched -> operand tile [64 k][128 m], m columns mcol0.., rows krow0..
__device__ __forceinline__ void store_mmajor(uint4 *operand, int mcol0, int krow0, int lane, const PanelRegs &p)
{
    const int chunk = (mcol0 >> 2) + 2 * (lane & 7); // 8-byte chunk of the row: 4 m each
    const uint4 regs[4] = {p.r0, p.r1, p.r2, p.r3};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = krow0 + 8 * i + mm_row(lane >> 3);
        operand[k * 16 + ((chunk ^ (8 * (k & 3))) >> 1)] = regs[i];
    }
}

// byte offset, inside an m-major operand tile, of the chunk a lane points ds_read_b64_tr_b16 at for the 32-row block
// mblk of the tile: row (lane >> 5) * 8 + ((lane & 15) >> 2) of a 16-k step, m = 32 mblk + 16 ((lane >> 4) & 1) + 4 (lane & 3)
__device__ __forceinline__ int mm_fragment_offset(int mblk, int lane)
{
    const int a = (lane & 15) >> 2;
    const int chunk = 8 * mblk + 4 * ((lane >> 4) & 1) + (lane & 3);
    return ((lane >> 5) * 8 + a) * 256 + ((chunk ^ (8 * a)) * 8);
}

// fragment of k-step s (16 k) from an m-major operand tile: k = 16 s + 8 (lane >> 5) + 0..7 of the lane's m
__device__ __forceinline__ bf16x8 mm_fragment(const lds_char *operand, int lane_off, int s)
{
    return lds_transposed_fragment(operand + lane_off + s * 4096, operand + lane_off + s * 4096 + 1024);
}

} // namespace kutacc_dev
