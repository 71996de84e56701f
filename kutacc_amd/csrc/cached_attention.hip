// Attention over a cache of keys and values in pages, behind a prefix that the sequences share.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q k_j - m),  m = max_j scale q k_j
//
// A row is one token's query head; the rows of a tile share a kv head: the tokens of one sequence times the heads of its group, or, over the shared prefix, all of the
// batch's.  A pass over the keys holds m, the sum and 32 x D results a wave in registers, by the transposed products of the matrix instructions: K Q^T leaves a row's
// logits in one lane (and the one 32 further on), so that maximum and sum need no more than one exchange, and P^T is in registers as the second product's operand
// wants it, V^T P^T, when V is read from the LDS transposed in the same order of keys.  K and V go straight into the LDS, double buffered, 16 bytes a lane from any
// page; rows that are not there come from a line of zeros.
//
// Waves of a workgroup are RW rows of waves, of 32 QB rows each, times KW that share the keys among themselves and join at the end.  Few rows: KW = 4, memory bounds them.
// Keys are split over workgroups where the tiles do not fill the chip, by the lengths on the device: every workgroup sums up what there is to do, takes
// the same share of it and finds its own.  The shares meet in a second kernel, in one order.
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "launch_internal.h"
#include "mfma_tiles.h"
#include "paged_cache.h"
#include "profiler.h"

namespace {
using namespace kutacc_dev;

constexpr float LN2 = 0.69314718055994530942f;

struct AttentionParams {
    const bf16_t *q;
    int64_t q_token, q_head;
    bf16_t *out;
    int64_t out_token, out_head;
    float *lse;
    const char *k, *v; // strides in bytes
    int64_t k_page, k_token, k_head, v_page, v_token, v_head;
    const float *k_scales, *v_scales;
    const int32_t *query_starts, *lengths, *page_table, *prefix_pages;
    int64_t page_table_ld;
    int sequences, tokens, heads, kv_heads, size, pages, own_limit; // own_limit: entries that the page table's columns hold
    int prefix_length;
    int joined;       // sequences' units walk the prefix too
    int causal;
    float scale_log2; // scale log2(e)
    Divisor page_size, group;
    // units: of the prefix, then of the sequences
    int prefix_units, prefix_splits, prefix_steps; // steps of keys of a split
    int targets;                                   // shares to make of the sequences' work; 0: none is split
    int least_steps;                               // of a share
    int combined;                                  // whether a second kernel joins shares
    float *prefix_partial, *partial;               // [unit][row of its tile][D]
    float2 *prefix_sums, *sums;                    // [unit][row]: m log2(e), sum
    int4 *rows;                                    // [token][head]: first unit, units (0: done), row of the tile
};

__device__ const uint4 NOTHING = {0u, 0u, 0u, 0u}; // what is read for entries that are not there

// what a workgroup does: rows row0 .. row0 + rows - 1 of its sequence (or of the batch) over entries begin .. end - 1
struct Unit {
    const int32_t *table;
    int prefix, keys; // entries on the prefix's pages, and all
    int token0, row0, rows, head;
    int limit0; // entries that token 0 sees (causal)
    int begin, end;
    int unit, share, shares, first; // its number, its place among the shares of its tile, and the first one's number
};

__device__ __forceinline__ void load_to_lds_from(uint32_t to, const char *from)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}

// infinities and what is no number replaced by zero; `wild` says whether there were any
__device__ __forceinline__ bf16x8 finite_part(bf16x8 v, uint32_t &wild)
{
    uint4 u = as_uint4(v);
    const auto part = [&](uint32_t pair) {
        const bool low = (pair & 0x7f80u) == 0x7f80u, high = (pair & 0x7f800000u) == 0x7f800000u;
        wild |= low || high ? 1u : 0u;
        return (low ? 0u : pair & 0xffffu) | (high ? 0u : pair & 0xffff0000u);
    };
    u.x = part(u.x), u.y = part(u.y), u.z = part(u.z), u.w = part(u.w);
    return as_bf16x8(u);
}

template <int D, int QB, int RW, int KW, int KT, bool FP8>
struct Shape {
    static constexpr int WAVES = RW * KW, THREADS = 64 * WAVES;
    static constexpr int ROWS = 32 * QB * RW, STEP = KW * KT;
    static constexpr int PITCH = 2 * D, CHUNKS = D / 8; // bytes and 16-byte pieces of an entry in the LDS
    static constexpr int TILE = KT * PITCH, STAGE = 2 * KW * TILE;
    static constexpr int LOADS = TILE / 1024 / RW;      // of a wave, keys and values each
    static constexpr int BYTE_LOADS = TILE / 2048 / RW; // of e4m3
    static constexpr int JOIN = KW > 1 ? KW * ROWS * ((D + 4) * 4 + 8) : 0;
    static constexpr int LDS = 2 * STAGE > JOIN ? 2 * STAGE : JOIN;
    static_assert((FP8 ? BYTE_LOADS : LOADS) >= 1 && LDS <= 156 * 1024, "");
    // 16-byte pieces stand where the banks of those that one access reads differ: a piece of 16 entries' keys, four pieces of four entries' values
    static __device__ __forceinline__ int key_swizzle(int row) { return D >= 128 ? row & 15 : (row >> 1) & 7; }
    static __device__ __forceinline__ int value_swizzle(int row) { return D >= 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }
};

// sum over the workgroup and sum over the threads in front of this one
template <int WAVES, typename T>
__device__ __forceinline__ T scan(T v, T &total, T *waves)
{
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
    T sum = v;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
        const T other = __shfl_up(sum, off, 64);
        sum += lane >= off ? other : T(0);
    }
    __syncthreads(); // the last scan has been read
    if (lane == 63) {
        waves[wave] = sum;
    }
    __syncthreads();
    T before = T(0);
    total = T(0);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        before += w < wave ? waves[w] : T(0);
        total += waves[w];
    }
    return before + sum - v;
}

struct Work {
    TokenRange tokens;
    int tiles, keys, steps, own; // own: its own entries as the array has them
};
template <typename S>
__device__ __forceinline__ Work work_of(const AttentionParams &p, int s)
{
    Work w;
    w.tokens = tokens_of(p.query_starts, s, p.tokens);
    w.own = max(p.lengths[s], 0);
    w.tiles = (int)(((int64_t)(w.tokens.end - w.tokens.first) * (int)p.group.d + S::ROWS - 1) / S::ROWS);
    w.keys = min(w.own, p.own_limit) + (p.joined ? p.prefix_length : 0);
    w.steps = max((w.keys + S::STEP - 1) / S::STEP, 1);
    return w;
}

// The unit `index` of the sequences': false where there are not as many.  Sequences in order; of one, its tiles from the last one on, which sees
// the most entries, of a tile its shares, of a share the kv heads: neighbouring workgroups, which start on neighbouring XCDs, have different heads.
template <typename S>
__device__ __forceinline__ bool find_unit(const AttentionParams &p, int index, Unit &u)
{
    __shared__ double double_waves[S::WAVES];
    __shared__ int int_waves[S::WAVES];
    __shared__ int found[3];
    const int tid = (int)threadIdx.x, of_head = index / p.kv_heads;
    Work w = {};
    int64_t steps = INT32_MAX; // of a share
    if (p.targets > 0) {
        double sum = 0.0, total;
        for (int s = tid; s < p.sequences; s += S::THREADS) {
            w = work_of<S>(p, s);
            sum += (double)w.tiles * (double)w.steps;
        }
        (void)scan<S::WAVES, double>(sum, total, double_waves);
        const double share = ceil(total * p.kv_heads / p.targets);
        steps = (int64_t)fmin(fmax(share, (double)p.least_steps), (double)INT32_MAX);
    }
    if (tid == 0) {
        found[0] = -1;
    }
    int base = 0;
    for (int s0 = 0; s0 < p.sequences; s0 += S::THREADS) {
        const int s = s0 + tid;
        int units = 0;
        if (s < p.sequences) {
            if (p.targets == 0 || p.sequences > S::THREADS) { // else it has this one's already
                w = work_of<S>(p, s);
            }
            units = w.tiles * (int)((w.steps + steps - 1) / steps);
        }
        int total;
        const int before = base + scan<S::WAVES, int>(units, total, int_waves);
        if (of_head >= before && of_head - before < units) {
            found[0] = s, found[1] = before, found[2] = (int)((w.steps + steps - 1) / steps);
        }
        base += total;
        if (of_head < base) {
            break;
        }
    }
    __syncthreads();
    const int s = found[0];
    if (s < 0) {
        return false;
    }
    w = work_of<S>(p, s);
    const int shares = found[2], in_sequence = of_head - found[1], tile = in_sequence / shares;
    const int total_rows = (w.tokens.end - w.tokens.first) * (int)p.group.d;
    u.table = p.page_table + s * p.page_table_ld;
    u.prefix = p.joined ? p.prefix_length : 0, u.keys = w.keys;
    u.token0 = w.tokens.first, u.row0 = (w.tiles - 1 - tile) * S::ROWS, u.rows = min(S::ROWS, total_rows - u.row0), u.head = index - of_head * p.kv_heads;
    u.limit0 = w.own - (w.tokens.end - w.tokens.first) + 1; // it has a token: no overflow
    u.share = in_sequence - tile * shares, u.shares = shares, u.unit = index, u.first = index - u.share * p.kv_heads;
    const int per_share = (w.steps + shares - 1) / shares;
    u.begin = (int)min((int64_t)u.share * per_share * S::STEP, (int64_t)w.keys);
    u.end = (int)min((int64_t)(u.share + 1) * per_share * S::STEP, (int64_t)w.keys);
    return true;
}

// entries that a row sees, of the unit's
__device__ __forceinline__ int limit_of(const AttentionParams &p, const Unit &u, int row)
{
    if (!p.causal || u.limit0 == INT32_MAX) {
        return u.keys;
    }
    const int64_t own = (int64_t)u.limit0 + (int)p.group.quotient((uint32_t)(u.row0 + row));
    return (int)min(max(own, (int64_t)0) + u.prefix, (int64_t)u.keys);
}

template <int D, int QB, int RW, int KW, int KT, bool FP8>
__global__ __launch_bounds__(64 * RW * KW, QB == 1 && D <= 128 ? 2 : 1) void cached_attention_kernel(const AttentionParams p)
{
    using S = Shape<D, QB, RW, KW, KT, FP8>;
    constexpr bool FINE = KW > 1; // 16 bits of the weights
    extern __shared__ __align__(16) char lds[];
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int rw = wave % RW, kw = wave / RW, half = lane >> 5;

    Unit u;
    const bool shared_prefix = (int)blockIdx.x < p.prefix_units;
    if (shared_prefix) {
        // a tile's shares and heads are neighbours, those of the next tile as far on as there are: where that is a multiple of 8 they read the same entries on the same XCD
        const int per_tile = p.prefix_splits * p.kv_heads, tile = (int)blockIdx.x / per_tile, in_tile = (int)blockIdx.x - tile * per_tile;
        u.table = nullptr, u.prefix = u.keys = p.prefix_length;
        u.token0 = 0, u.row0 = tile * S::ROWS, u.rows = min(S::ROWS, p.tokens * (int)p.group.d - u.row0), u.limit0 = INT32_MAX;
        u.share = in_tile / p.kv_heads, u.head = in_tile - u.share * p.kv_heads, u.shares = p.prefix_splits, u.unit = (int)blockIdx.x, u.first = 0;
        u.begin = u.share * p.prefix_steps * S::STEP, u.end = min(u.begin + p.prefix_steps * S::STEP, u.keys);
    } else if (!find_unit<S>(p, (int)blockIdx.x - p.prefix_units, u)) {
        return;
    }
    const int first_limit = limit_of(p, u, 0), last_limit = limit_of(p, u, u.rows - 1);
    const int end = min(u.end, last_limit), steps = max((end - u.begin + S::STEP - 1) / S::STEP, 0);

    // ---- this wave's rows ----
    bf16x8 q[QB][D / 16];
    int limit[QB];
    const int wave_row = 32 * QB * rw;
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        const int row = wave_row + 32 * b + (lane & 31);
        const bool there = row < u.rows;
        const uint32_t of = (uint32_t)(u.row0 + (there ? row : 0)), token = p.group.quotient(of);
        const bf16_t *from = p.q + (int64_t)(u.token0 + (int)token) * p.q_token + (int64_t)(u.head * (int)p.group.d + (int)(of - token * p.group.d)) * p.q_head;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const int at = 16 * i + 8 * half;
            uint4 piece = zero_u4();
            if (there && at < p.size) {
                __builtin_memcpy(&piece, from + at, 16);
            }
            q[b][i] = as_bf16x8(piece);
        }
        limit[b] = there ? limit_of(p, u, row) : u.keys;
    }
    const int wave_last_limit = limit_of(p, u, min(wave_row + 32 * QB, u.rows) - 1);
    const bool wave_idle = wave_row >= u.rows;

    f32x16 o[QB][D / 32];
    float m[QB], sum[QB];
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        m[b] = -INFINITY, sum[b] = 0.f;
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
            o[b][d] = zero16();
        }
    }
    // an unscaled logit's factor in powers of two; as good as zero at its smallest, and not so that -inf times it is no number
    const float factor = fmaxf(p.scale_log2 * (FP8 ? p.k_scales[u.head] : 1.f), 0x1p-100f);

    // ---- entries on their way ----
    const char *k_head = p.k + u.head * p.k_head, *v_head = p.v + u.head * p.v_head;
    const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_char *)lds;
    int page = -1, slot = 0; // of entry `lane` of this wave's next tile
    const auto ask_pages = [&](int step) {
        const int at = u.begin + step * S::STEP + kw * KT + lane;
        page = -1, slot = 0;
        if (lane < KT && at < end) {
            const bool shared = at < u.prefix;
            const uint32_t entry = (uint32_t)(shared ? at : at - u.prefix), column = p.page_size.quotient(entry);
            slot = (int)(entry - column * p.page_size.d);
            page = (shared ? p.prefix_pages : u.table)[column];
        }
    };
    uint64_t there = 0, there_next = 0; // entries of a tile that are there
    constexpr int BYTE_LOADS = FP8 ? S::BYTE_LOADS : 1;
    uint4 k_bytes[BYTE_LOADS], v_bytes[BYTE_LOADS];
    const auto ask = [&](int stage) {
        page = (uint32_t)page < (uint32_t)p.pages ? page : -1;
        there_next = __ballot(page >= 0);
        if constexpr (FP8) {
#pragma unroll
            for (int i = 0; i < S::BYTE_LOADS; ++i) {
                const int row = ((rw * S::BYTE_LOADS + i) * 64 + lane) / (D / 16), piece = lane % (D / 16);
                const int pg = __shfl(page, row, 64), sl = __shfl(slot, row, 64);
                const bool ok = pg >= 0 && 16 * piece < p.size;
                const char *kf = ok ? k_head + pg * p.k_page + sl * p.k_token + 16 * piece : (const char *)&NOTHING;
                const char *vf = ok ? v_head + pg * p.v_page + sl * p.v_token + 16 * piece : (const char *)&NOTHING;
                k_bytes[i] = *(const uint4 *)kf, v_bytes[i] = *(const uint4 *)vf;
            }
        } else {
            const uint32_t to = __builtin_amdgcn_readfirstlane(lds_at + (uint32_t)(stage * S::STAGE + kw * 2 * S::TILE + rw * S::LOADS * 1024));
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i) {
                const int row = ((rw * S::LOADS + i) * 64 + lane) / S::CHUNKS, piece = lane % S::CHUNKS;
                const int pg = __shfl(page, row, 64), sl = __shfl(slot, row, 64);
                const int kp = piece ^ S::key_swizzle(row), vp = piece ^ S::value_swizzle(row);
                const char *kf = pg >= 0 && 8 * kp < p.size ? k_head + pg * p.k_page + sl * p.k_token + 16 * kp : (const char *)&NOTHING;
                const char *vf = pg >= 0 && 8 * vp < p.size ? v_head + pg * p.v_page + sl * p.v_token + 16 * vp : (const char *)&NOTHING;
                load_to_lds_from(to + 1024 * i, kf);
                load_to_lds_from(to + S::TILE + 1024 * i, vf);
            }
        }
    };
    const auto place_bytes = [&](int stage) { // e4m3 as bf16, which holds every one of its values
        if constexpr (FP8) {
            char *to = lds + stage * S::STAGE + kw * 2 * S::TILE;
#pragma unroll
            for (int i = 0; i < S::BYTE_LOADS; ++i) {
                const int row = ((rw * S::BYTE_LOADS + i) * 64 + lane) / (D / 16), piece = lane % (D / 16);
                const auto put = [&](uint4 bytes, char *at, int swizzle) {
                    const uint32_t words[4] = {bytes.x, bytes.y, bytes.z, bytes.w};
                    bf16x2 v[8];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[2 * j] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(words[j], 1.0f, false);
                        v[2 * j + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(words[j], 1.0f, true);
                    }
                    uint4 pieces[2];
                    __builtin_memcpy(pieces, v, sizeof(pieces));
                    *(uint4 *)(at + row * S::PITCH + 16 * ((2 * piece) ^ swizzle)) = pieces[0];
                    *(uint4 *)(at + row * S::PITCH + 16 * ((2 * piece + 1) ^ swizzle)) = pieces[1];
                };
                put(k_bytes[i], to, S::key_swizzle(row));
                put(v_bytes[i], to + S::TILE, S::value_swizzle(row));
            }
        }
    };

    // one tile of this wave's keys; LIMITED: not all rows of the workgroup see all of its entries
    const auto compute = [&](int step, int stage, auto limited) {
        constexpr bool LIMITED = decltype(limited)::value;
        const int tile0 = u.begin + step * S::STEP + kw * KT;
        if (wave_idle || there == 0 || (LIMITED && tile0 >= wave_last_limit)) {
            return;
        }
        const char *keys = lds + stage * S::STAGE + kw * 2 * S::TILE, *values = keys + S::TILE;
        constexpr uint64_t ALL = KT == 64 ? ~(uint64_t)0 : ((uint64_t)1 << (KT & 63)) - 1;

        f32x16 s[QB][KT / 32];
#pragma unroll
        for (int kb = 0; kb < KT / 32; ++kb) {
#pragma unroll
            for (int b = 0; b < QB; ++b) {
                s[b][kb] = zero16();
            }
            const int row = 32 * kb + (lane & 31);
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                const bf16x8 k = as_bf16x8(*(const uint4 *)(keys + row * S::PITCH + 16 * ((2 * i + half) ^ S::key_swizzle(row))));
#pragma unroll
                for (int b = 0; b < QB; ++b) {
                    s[b][kb] = mfma(k, q[b][i], s[b][kb]);
                }
            }
        }
        if (LIMITED || there != ALL) {
#pragma unroll
            for (int kb = 0; kb < KT / 32; ++kb) {
                const uint32_t entries = (uint32_t)(there >> (32 * kb)) >> (4 * half); // of this lane, entry 8 (i / 4) + (i & 3) is logit i
#pragma unroll
                for (int b = 0; b < QB; ++b) {
                    uint32_t seen = entries;
                    if constexpr (LIMITED) {
                        const int count = min(max(limit[b] - tile0 - 32 * kb - 4 * half, 0), 31); // its last one is entry 27
                        seen &= ((uint32_t)1 << count) - 1;
                    }
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[b][kb][i] = (seen & ((uint32_t)1 << (8 * (i / 4) + (i & 3)))) != 0 ? s[b][kb][i] : -INFINITY;
                    }
                }
            }
        }
        bf16x8 w[QB][KT / 16], rest[QB][FINE ? KT / 16 : 1];
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            float most = s[b][0][0];
#pragma unroll
            for (int kb = 0; kb < KT / 32; ++kb) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    most = fmaxf(most, s[b][kb][i]);
                }
            }
            most = fmaxf(m[b], half_swap_max(most));
            const float base = (most == -INFINITY ? 0.f : most) * factor; // nothing seen yet: weights of zero
            const float keep = __builtin_amdgcn_exp2f(fmaf(m[b], factor, -base));
            m[b] = most;
            float add = 0.f;
#pragma unroll
            for (int kb = 0; kb < KT / 32; ++kb) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[b][kb][i] = __builtin_amdgcn_exp2f(fmaf(s[b][kb][i], factor, -base));
                    add += s[b][kb][i];
                }
            }
            sum[b] = fmaf(sum[b], keep, add); // of this lane's half of the keys
#pragma unroll
            for (int i = 0; i < KT / 16; ++i) {
                w[b][i] = pack8(s[b][i / 2], 8 * (i & 1));
                if constexpr (FINE) {
                    f32x16 left = s[b][i / 2];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        left[8 * (i & 1) + e] -= (float)w[b][i][e];
                    }
                    rest[b][i] = pack8(left, 8 * (i & 1));
                }
            }
            if (__any(keep != 1.f)) {
#pragma unroll
                for (int d = 0; d < D / 32; ++d) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        o[b][d][i] *= keep;
                    }
                }
            }
        }
        // values of 16 keys and 32 channels, transposed: lane -> channel lane & 31, keys 4 half .. + 3 and 8 further on, as the logits have them
        const int in16 = lane & 15, from_row = 4 * half + (in16 >> 2), piece0 = 2 * ((lane >> 4) & 1) + ((in16 & 3) >> 1);
        const lds_char *values_at = (const lds_char *)values + from_row * S::PITCH + 8 * (in16 & 1);
        const auto value_fragment = [&](int i, int d) {
            const lds_char *at = values_at + 16 * i * S::PITCH + 16 * ((4 * d + piece0) ^ S::value_swizzle(from_row));
            return lds_transposed_fragment(at, at + 8 * S::PITCH);
        };
        uint32_t wild = 0; // an infinity or no number among values that a row must not see: its weight of zero would not keep it out
#pragma unroll
        for (int i = 0; i < KT / 16; ++i) {
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
                bf16x8 v = value_fragment(i, d);
                if constexpr (LIMITED) {
                    v = finite_part(v, wild);
                }
#pragma unroll
                for (int b = 0; b < QB; ++b) {
                    o[b][d] = mfma(v, w[b][i], o[b][d]);
                    if constexpr (FINE) {
                        o[b][d] = mfma(v, rest[b][i], o[b][d]);
                    }
                }
            }
        }
        if (LIMITED && __any(wild != 0)) { // added where they are seen, as they are: whatever their weight, they are what comes of it
#pragma unroll 1
            for (int key = 0; key < KT; ++key) {
#pragma unroll
                for (int d = 0; d < D / 32; ++d) {
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const int piece = 4 * d + a;
                        bf16x4 v;
                        __builtin_memcpy(&v, values + key * S::PITCH + 16 * (piece ^ S::value_swizzle(key)) + 8 * half, 8);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = (float)v[e];
#pragma unroll
                            for (int b = 0; b < QB; ++b) {
                                o[b][d][4 * a + e] += tile0 + key < limit[b] && !(fabsf(x) < INFINITY) ? x : 0.f;
                            }
                        }
                    }
                }
            }
        }
    };

    // ---- the pass ----
    if (steps > 0) {
        ask_pages(0);
        ask(0);
        ask_pages(1);
    }
    const auto pass = [&](int from, int to, auto limited) {
        for (int step = from; step < to; ++step) {
            const int stage = step & 1;
            there = there_next;
            if constexpr (FP8) {
                place_bytes(stage);
            } else {
                wait_for_loads<0>();
            }
            if constexpr (RW == 1) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // what was read of the other stage has come, too
            } else {
                __syncthreads(); // this stage is there for all, and nobody reads the other any more
            }
            if (step + 1 < steps) {
                ask(stage ^ 1);
                ask_pages(step + 2);
            }
            compute(step, stage, limited);
        }
    };
    // entries up to the first row's limit are every row's; with none past it, the last step is whole, too
    const int whole_steps = first_limit >= end ? steps : max(first_limit - u.begin, 0) / S::STEP;
    pass(0, whole_steps, std::false_type{});
    pass(whole_steps, steps, std::true_type{});

    // ---- the end: results of this unit's rows ----
    const bool direct = !p.combined || (!shared_prefix && u.shares == 1 && p.prefix_units == 0 && p.prefix_partial == nullptr);
    const float v_scale = FP8 ? p.v_scales[u.head] : 1.f;
    float *partial = shared_prefix ? p.prefix_partial : p.partial;
    float2 *sums = shared_prefix ? p.prefix_sums : p.sums;
    const auto place_of = [&](int row, int &token, int &query_head) {
        const uint32_t of = (uint32_t)(u.row0 + row), t = p.group.quotient(of);
        token = u.token0 + (int)t, query_head = u.head * (int)p.group.d + (int)(of - t * p.group.d);
    };
    const auto finish_row = [&](int row, float most, float total) { // most in powers of two
        int token, query_head;
        place_of(row, token, query_head);
        if (direct) {
            if (p.lse != nullptr) {
                p.lse[(int64_t)token * p.heads + query_head] = total > 0.f ? (most + __log2f(total)) * LN2 : total == 0.f ? -INFINITY : total;
            }
        } else {
            sums[(int64_t)u.unit * S::ROWS + row] = make_float2(most, total);
        }
        if (p.combined && !shared_prefix && u.share == 0) {
            p.rows[(int64_t)token * p.heads + query_head] = make_int4(u.first, direct ? 0 : u.shares, row, 0);
        }
    };
    const auto store4 = [&](int row, int at, float (&v)[4], float total) { // channels at .. at + 3
        if (at >= p.size) {
            return;
        }
        if (direct) {
            int token, query_head;
            place_of(row, token, query_head);
            const float over = total == 0.f ? 0.f : v_scale / total;
            bf16x4 r;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                r[e] = (bf16_t)(v[e] * over);
            }
            __builtin_memcpy(p.out + token * p.out_token + query_head * p.out_head + at, &r, 8);
        } else {
            *(float4 *)(partial + ((int64_t)u.unit * S::ROWS + row) * D + at) = make_float4(v[0] * v_scale, v[1] * v_scale, v[2] * v_scale, v[3] * v_scale);
        }
    };
#pragma unroll
    for (int b = 0; b < QB; ++b) {
        sum[b] = half_swap_sum(sum[b]);
        m[b] = m[b] == -INFINITY ? m[b] : m[b] * factor;
    }
    if constexpr (KW == 1) {
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            const int row = wave_row + 32 * b + (lane & 31);
            if (row < u.rows) {
                if (half == 0) {
                    finish_row(row, m[b], sum[b]);
                }
#pragma unroll
                for (int d = 0; d < D / 32; ++d) {
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        float v[4] = {o[b][d][4 * a], o[b][d][4 * a + 1], o[b][d][4 * a + 2], o[b][d][4 * a + 3]};
                        store4(row, 32 * d + 8 * a + 4 * half, v, sum[b]);
                    }
                }
            }
        }
    } else {
        static_assert(QB == 1, "");
        constexpr int P = D + 4; // floats from row to row
        float *shares = (float *)lds;
        float2 *share_sums = (float2 *)(lds + KW * S::ROWS * P * 4);
        __syncthreads();
        const int row = wave_row + (lane & 31);
        if (row < u.rows) {
            if (half == 0) {
                share_sums[kw * S::ROWS + row] = make_float2(m[0], sum[0]);
            }
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    *(float4 *)(shares + (kw * S::ROWS + row) * P + 32 * d + 8 * a + 4 * half) =
                        make_float4(o[0][d][4 * a], o[0][d][4 * a + 1], o[0][d][4 * a + 2], o[0][d][4 * a + 3]);
                }
            }
        }
        __syncthreads();
        for (int i = (int)threadIdx.x; i < u.rows * (D / 4); i += S::THREADS) {
            const int r = i / (D / 4), at = 4 * (i % (D / 4));
            float most = -INFINITY, total = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
            float2 of[KW];
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                of[w] = share_sums[w * S::ROWS + r];
                most = fmaxf(most, of[w].x);
            }
            const float base = most == -INFINITY ? 0.f : most;
#pragma unroll
            for (int w = 0; w < KW; ++w) {
                const float weight = __builtin_amdgcn_exp2f(of[w].x - base);
                const float4 add = *(const float4 *)(shares + (w * S::ROWS + r) * P + at);
                total = fmaf(weight, of[w].y, total);
                v[0] = fmaf(weight, add.x, v[0]), v[1] = fmaf(weight, add.y, v[1]), v[2] = fmaf(weight, add.z, v[2]), v[3] = fmaf(weight, add.w, v[3]);
            }
            if (at == 0) {
                finish_row(r, most, total);
            }
            store4(r, at, v, total);
        }
    }
}

// The shares of a row, of the prefix's units and of its sequence's, by a wave: those of the prefix in order, then the sequence's.
struct CombineParams {
    const float *prefix_partial, *partial;
    const float2 *prefix_sums, *sums;
    const int4 *rows;
    int prefix_splits, prefix_rows, own_rows; // rows of their tiles
    int tokens, heads, kv_heads, size, sequences, most_units;
    Divisor group;
    const int32_t *query_starts;
    bf16_t *out;
    int64_t out_token, out_head;
    float *lse;
};

template <int D>
__global__ __launch_bounds__(256) void combine_kernel(const CombineParams p)
{
    const int lane = (int)threadIdx.x & 63;
    const int64_t index = (int64_t)blockIdx.x * 4 + ((int)threadIdx.x >> 6);
    const int token = (int)(index / p.heads), head = (int)(index - (int64_t)token * p.heads);
    if (token >= p.tokens || token < p.query_starts[0] || token >= p.query_starts[p.sequences]) {
        return;
    }
    const int4 own = p.rows[index];
    const int own_units = own.x >= 0 && own.z >= 0 && own.z < p.own_rows && own.y > 0 && (int64_t)own.x + (int64_t)(own.y - 1) * p.kv_heads < p.most_units ? own.y : 0;
    const int units = p.prefix_splits + own_units;
    if (units == 0) {
        return; // its one unit has written it
    }
    const int kv_head = (int)p.group.quotient((uint32_t)head);
    const uint32_t stacked = (uint32_t)token * p.group.d + (uint32_t)(head - kv_head * (int)p.group.d);
    const uint32_t tile = p.prefix_splits > 0 ? stacked / (uint32_t)p.prefix_rows : 0;
    const auto place = [&](int i) { // of share i: a row of one of the two
        return i < p.prefix_splits ? ((int64_t)tile * p.prefix_splits * p.kv_heads + (int64_t)i * p.kv_heads + kv_head) * p.prefix_rows + (int64_t)(stacked - tile * (uint32_t)p.prefix_rows)
                                   : ((int64_t)own.x + (int64_t)(i - p.prefix_splits) * p.kv_heads) * p.own_rows + own.z;
    };
    const auto sums_of = [&](int i) { return i < p.prefix_splits ? p.prefix_sums[place(i)] : p.sums[place(i)]; };
    float most = -INFINITY;
    for (int i = lane; i < units; i += 64) {
        most = fmaxf(most, sums_of(i).x);
    }
    most = wave_max(most);
    const float base = most == -INFINITY ? 0.f : most;
    constexpr int V = D / 64;
    float v[V] = {}, total = 0.f;
    for (int i0 = 0; i0 < units; i0 += 64) {
        float weight = 0.f;
        if (i0 + lane < units) {
            const float2 s = sums_of(i0 + lane);
            weight = __builtin_amdgcn_exp2f(s.x - base);
            total = fmaf(weight, s.y, total);
        }
        const int count = min(64, units - i0);
        for (int i = 0; i < count; ++i) {
            const float w = __shfl(weight, i, 64);
            const float *from = (i0 + i < p.prefix_splits ? p.prefix_partial : p.partial) + place(i0 + i) * D + V * lane;
            float add[V];
            __builtin_memcpy(add, from, sizeof(add));
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[e] = fmaf(w, add[e], v[e]);
            }
        }
    }
    total = wave_sum(total);
    const float over = total == 0.f ? 0.f : 1.f / total;
    bf16_t *to = p.out + token * p.out_token + head * p.out_head;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if (V * lane + e < p.size) {
            to[V * lane + e] = (bf16_t)(v[e] * over);
        }
    }
    if (p.lse != nullptr && lane == 0) {
        p.lse[index] = total > 0.f ? (most + __log2f(total)) * LN2 : total == 0.f ? -INFINITY : total;
    }
}

// ---- which kernels, how many units ----

template <int D_, int QB_, int RW_, int KW_, int KT_>
struct Variant {
    static constexpr int D = D_, QB = QB_, RW = RW_, KW = KW_, KT = KT_;
    static constexpr int ROWS = 32 * QB * RW, STEP = KW * KT;
};

// a tile's rows by those that there are, and the channels that they take in registers
template <typename F>
auto by_rows(int64_t rows, int64_t size, F f)
{
    if (size <= 64) {
        return rows <= 32 ? f(Variant<64, 1, 1, 4, 64>{}) : rows <= 64 ? f(Variant<64, 1, 2, 2, 64>{}) : f(Variant<64, 1, 4, 1, 64>{});
    }
    if (size <= 128) {
        return rows <= 32 ? f(Variant<128, 1, 1, 4, 32>{}) : rows <= 64 ? f(Variant<128, 1, 2, 2, 32>{}) : f(Variant<128, 1, 4, 1, 64>{});
    }
    return rows <= 32 ? f(Variant<256, 1, 1, 2, 32>{}) : rows <= 64 ? f(Variant<256, 1, 2, 2, 32>{}) : f(Variant<256, 1, 4, 1, 32>{});
}

struct Plan {
    int64_t own_rows_hint, prefix_rows_hint; // rows that choose the variants
    bool shared;                             // the prefix is read once for all, by units of its own
    int prefix_tile, prefix_splits, prefix_steps, own_tile, targets, least_steps, d;
    int64_t prefix_units, own_units;
    bool combined;
    int64_t prefix_partial, partial, prefix_sums, sums, rows, bytes; // offsets in the workspace, and its size
};

Plan plan_of(const kutacc_hip_cached_attention_args_t &a)
{
    const kutacc_hip_cache_batch_t &b = a.batch;
    const int64_t group = a.q_heads / a.cache.kv_heads, kv_heads = a.cache.kv_heads, cus = kutacc_cu_count();
    Plan p = {};
    const int64_t average = (b.tokens * group + std::min(b.sequences, b.tokens) - 1) / std::min(b.sequences, b.tokens);
    p.shared = b.prefix_length > 0 && b.sequences > 1 && average <= 64;
    p.own_rows_hint = average, p.prefix_rows_hint = b.tokens * group;
    p.d = a.cache.head_size <= 64 ? 64 : a.cache.head_size <= 128 ? 128 : 256;
    const int64_t wanted = 2 * cus; // workgroups
    if (p.shared) {
        by_rows(p.prefix_rows_hint, a.cache.head_size, [&](auto variant) {
            using V = decltype(variant);
            const int64_t tiles = (p.prefix_rows_hint + V::ROWS - 1) / V::ROWS, steps = (b.prefix_length + V::STEP - 1) / V::STEP;
            const int64_t splits = std::max<int64_t>(1, std::min(std::min<int64_t>(wanted / (tiles * kv_heads), (steps + 1) / 2), (int64_t)64));
            p.prefix_steps = (int)((steps + splits - 1) / splits);
            p.prefix_splits = (int)((steps + p.prefix_steps - 1) / p.prefix_steps);
            p.prefix_tile = V::ROWS, p.prefix_units = tiles * kv_heads * p.prefix_splits;
            return 0;
        });
    }
    by_rows(p.own_rows_hint, a.cache.head_size, [&](auto variant) {
        using V = decltype(variant);
        const int64_t full = b.tokens * group / V::ROWS, tiles = full + std::min(b.sequences, b.tokens);
        p.own_tile = V::ROWS, p.least_steps = 2;
        p.targets = std::max<int64_t>(full, 1) * kv_heads >= wanted ? 0 : (int)wanted;
        p.own_units = tiles * kv_heads + p.targets;
        return 0;
    });
    p.combined = p.shared || p.targets > 0;
    int64_t at = 0;
    const auto take = [&](int64_t bytes) {
        const int64_t from = at;
        at += (bytes + 255) / 256 * 256;
        return from;
    };
    if (p.combined) {
        p.rows = take(b.tokens * a.q_heads * (int64_t)sizeof(int4));
        p.prefix_sums = take(p.prefix_units * p.prefix_tile * (int64_t)sizeof(float2));
        p.sums = take(p.own_units * p.own_tile * (int64_t)sizeof(float2));
        p.prefix_partial = take(p.prefix_units * p.prefix_tile * p.d * (int64_t)sizeof(float));
        p.partial = take(p.own_units * p.own_tile * p.d * (int64_t)sizeof(float));
    }
    p.bytes = at;
    return p;
}

template <typename V, bool FP8>
int launch_units(const AttentionParams &p, int64_t units, double flops, hipStream_t stream)
{
    using S = Shape<V::D, V::QB, V::RW, V::KW, V::KT, FP8>;
    if (!kutacc_grid_fits(units, S::THREADS)) {
        return KUTACC_HIP_EUNSUPPORTED;
    }
    const auto kernel = cached_attention_kernel<V::D, V::QB, V::RW, V::KW, V::KT, FP8>;
    static size_t opted[KUTACC_DEVICE_SLOTS] = {};
    if (const hipError_t e = kutacc_opt_in_lds((const void *)kernel, S::LDS, opted)) {
        return kutacc_hip_status(e);
    }
    kutacc_prof::KernelTimer timer("cached_attention_kernel", flops, stream);
    kernel<<<dim3((unsigned)units), S::THREADS, S::LDS, stream>>>(p);
    return kutacc_hip_status(hipGetLastError());
}

} // namespace

namespace kutacc_launch {

int64_t cached_attention_workspace(const kutacc_hip_cached_attention_args_t &a) { return plan_of(a).bytes; }

int cached_attention(const kutacc_hip_cached_attention_args_t &a, hipStream_t stream)
{
    const kutacc_hip_cache_t &c = a.cache;
    const kutacc_hip_cache_batch_t &b = a.batch;
    const Plan plan = plan_of(a);
    const int64_t e = c.dtype == KUTACC_DTYPE_E4M3 ? 1 : 2;
    AttentionParams p = {};
    p.q = (const bf16_t *)a.q.data, p.q_token = a.q.token_stride, p.q_head = a.q.head_stride;
    p.out = (bf16_t *)a.out.data, p.out_token = a.out.token_stride, p.out_head = a.out.head_stride, p.lse = a.lse;
    p.k = (const char *)c.k, p.k_page = e * c.k_page_stride, p.k_token = e * c.k_token_stride, p.k_head = e * c.k_head_stride;
    p.v = (const char *)c.v, p.v_page = e * c.v_page_stride, p.v_token = e * c.v_token_stride, p.v_head = e * c.v_head_stride;
    p.k_scales = c.k_scales, p.v_scales = c.v_scales;
    p.query_starts = b.query_starts, p.lengths = b.lengths, p.page_table = b.page_table, p.prefix_pages = b.prefix_pages, p.page_table_ld = b.page_table_ld;
    p.sequences = (int)b.sequences, p.tokens = (int)b.tokens, p.heads = (int)a.q_heads, p.kv_heads = (int)c.kv_heads, p.size = (int)c.head_size;
    p.pages = (int)c.pages, p.own_limit = (int)(b.columns * c.page_size), p.prefix_length = (int)b.prefix_length;
    p.joined = b.prefix_length > 0 && !plan.shared, p.causal = a.causal, p.scale_log2 = a.scale * LOG2E;
    p.page_size = Divisor::of((uint32_t)c.page_size), p.group = Divisor::of((uint32_t)(a.q_heads / c.kv_heads));
    p.prefix_splits = plan.prefix_splits, p.prefix_steps = plan.prefix_steps, p.targets = plan.targets, p.least_steps = plan.least_steps, p.combined = plan.combined;
    char *workspace = (char *)a.workspace;
    if (plan.combined) {
        p.rows = (int4 *)(workspace + plan.rows), p.sums = (float2 *)(workspace + plan.sums), p.partial = (float *)(workspace + plan.partial);
        if (plan.shared) {
            p.prefix_sums = (float2 *)(workspace + plan.prefix_sums), p.prefix_partial = (float *)(workspace + plan.prefix_partial);
        }
    }
    const double flops = 4.0 * (double)c.head_size * (double)a.q_heads * (double)b.tokens;
    const auto launch = [&](auto variant, const AttentionParams &of, int64_t units, double work) {
        using V = decltype(variant);
        return c.dtype == KUTACC_DTYPE_E4M3 ? launch_units<V, true>(of, units, work, stream) : launch_units<V, false>(of, units, work, stream);
    };
    if (plan.shared) {
        AttentionParams of = p;
        of.prefix_units = (int)plan.prefix_units;
        const int rc = by_rows(plan.prefix_rows_hint, c.head_size, [&](auto variant) { return launch(variant, of, plan.prefix_units, flops * (double)b.prefix_length); });
        if (rc != 0) {
            return rc;
        }
    }
    const int rc = by_rows(plan.own_rows_hint, c.head_size, [&](auto variant) { return launch(variant, p, plan.own_units, flops); });
    if (rc != 0 || !plan.combined) {
        return rc;
    }
    const CombineParams join = {p.prefix_partial, p.partial, p.prefix_sums, p.sums, p.rows, plan.shared ? plan.prefix_splits : 0, plan.prefix_tile, plan.own_tile, p.tokens, p.heads,
                                p.kv_heads, p.size, p.sequences, (int)plan.own_units, p.group, p.query_starts, p.out, p.out_token, p.out_head, p.lse};
    const int64_t groups = (b.tokens * a.q_heads + 3) / 4;
    if (!kutacc_grid_fits(groups, 256)) {
        return KUTACC_HIP_EUNSUPPORTED;
    }
    kutacc_prof::KernelTimer timer("combine_kernel", (double)b.tokens * (double)a.q_heads * (double)c.head_size, stream);
    const dim3 grid((unsigned)groups);
    if (plan.d == 64) {
        combine_kernel<64><<<grid, 256, 0, stream>>>(join);
    } else if (plan.d == 128) {
        combine_kernel<128><<<grid, 256, 0, stream>>>(join);
    } else {
        combine_kernel<256><<<grid, 256, 0, stream>>>(join);
    }
    return kutacc_hip_status(hipGetLastError());
}

} // namespace kutacc_launch
