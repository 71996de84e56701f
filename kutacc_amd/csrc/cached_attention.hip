// Attention over a cache of keys and values in pages, behind a prefix that the sequences share.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^-8 exp(scale q k_j - m),  m close to max_j scale q k_j
//
// m is the largest logit of the first keys, and follows the larger ones of later keys only when they leave it behind by more than 8 powers of two: the results are
// multiplied with exp(m - m') for few tiles instead of most.  With the 2^-8 no weight is above one all the same, and sums of weighted values leave fp32 only where those of a softmax
// with the exact maximum do.
//
// A row is one token's query head; the rows of a tile share a kv head: the tokens of one sequence times the heads of its group, or, over the shared prefix, all of the
// batch's.  A pass over the keys holds m, the sum and a wave's results in registers, by the transposed products of the matrix instructions: K Q^T leaves a row's
// logits in two lanes or four, so that maximum and sum need an exchange or two, and P^T is in registers as the second product's operand
// wants it, V^T P^T, when V is read from the LDS transposed in the same order of keys.  K and V go straight into the LDS, double buffered, 16 bytes a lane from any
// page; rows that are not there come from a line of zeros.
//
// Few rows, up to 16 a tile: memory bounds them.  The waves of a workgroup all have the same rows and in turn a tile of keys, and join at the end.  A wave has a tile at hand
// and one on its way in registers; K is there as the matrix instructions take it, V goes through LDS of the wave's own.  More rows: the matrix cores and the softmax bound
// them.  Each wave has 32 of 128, and the four share K and V in the LDS.
//
// The work of a kv head, in steps of keys, is split into equal shares, one for each workgroup, as many as the chip holds at a time; a workgroup whose
// share goes over the end of a tile goes on with the next one.  The lengths are on the device: every wave sums them up and finds its share by itself.  The pieces of a row
// meet in a second kernel, in one order.  Where there are tiles enough, or few keys, a workgroup has a tile, and writes its results.
//
// 32 heads over 8 of 128, bf16: a token after 131071 entries 103 us, 5.2 TB/s (a large copy: 4.9); 8 after 1 to 1500 14.3 us; 64 after 1 to 1000 behind 8192 52 us (34 at the
// copy's rate); 4500 tokens of three prompts behind 2000 239 us, 890 TFLOP/s (a large library product: 1200).  256 after 100 to 2000 behind 16384, e4m3: 187 us (119).
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
    int joined;       // the sequences' tiles walk the prefix too
    int causal;
    float scale_log2; // scale log2(e)
    Divisor page_size, group;
    // workgroups: of the prefix, then of the sequences, kv heads in turn
    int prefix_shares, prefix_tiles, prefix_steps, prefix_per; // of a head: shares, tiles, steps of a tile, steps of a share
    int shares, most_tiles;                                    // of a head: shares of the sequences' work, 0: a workgroup has a tile; what bounds the number of tiles
    int step_log2, prefix_step_log2;                           // keys of a step: such that a head's work is counted in 32 bits
    Divisor by_share, by_prefix_step, by_prefix_per;
    int least;                                                 // steps of a share
    int combined;                                              // whether a second kernel joins pieces
    float *prefix_partial, *partial;                           // [kv head][tile + share][row of the tile][D]
    float2 *prefix_sums, *sums;                                // [kv head][tile + share][row]: m log2(e), sum
    int4 *rows;                                                // [token][head]: first piece, pieces (0: done), row of the tile
};

// The parameters once more, for what is done once a piece: those that are read through here are read when they are needed, and take no scalar registers in the loops
__device__ __forceinline__ const AttentionParams &again()
{
    auto p = (const __attribute__((address_space(4))) AttentionParams *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const AttentionParams *)p;
}

__device__ const uint4 NOTHING[32] = {}; // what is read for entries that are not there: the longest one's bytes

// what a workgroup does at a time: rows row0 .. row0 + rows - 1 of a sequence (or of the batch) over entries begin .. end - 1
struct Piece {
    const int32_t *table;
    int prefix, keys; // entries on the prefix's pages, and all
    int token0, row0, rows;
    int limit0; // entries that token 0 sees (causal)
    int begin, end;
    int at, first, share, shares; // its place among the pieces, that of its tile's first one, its number among these and theirs
};

__device__ __forceinline__ void load_to_lds_from(uint32_t to, const char *from)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(from) : "memory");
}

__device__ __forceinline__ bool wild_pair(uint32_t pair) { return (pair & 0x7f80u) == 0x7f80u || (pair & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ bool wild_piece(uint4 v) { return wild_pair(v.x) || wild_pair(v.y) || wild_pair(v.z) || wild_pair(v.w); }

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

// D channels; tiles of ROWS rows and, of a wave, KT keys; a workgroup's keys in steps of STEP
template <int D_, int WAVES_, bool FP8_>
struct FewRows {
    static constexpr int D = D_, WAVES = WAVES_, THREADS = 64 * WAVES, ROWS = 16, KT = D == 64 ? 64 : 32, STEP = WAVES * KT;
    static constexpr bool FP8 = FP8_, FEW = true;
    static constexpr int PITCH = 2 * D, CHUNKS = D / 8; // bytes and 16-byte pieces of an entry in the LDS
    static constexpr int TILE = KT * PITCH;
    static constexpr int LOADS = TILE / (FP8 ? 2048 : 1024);  // of values
    static constexpr int JOIN = WAVES * ROWS * ((D + 4) * 4 + 8);
    static constexpr int LDS = WAVES * TILE > JOIN ? WAVES * TILE : JOIN;
    // the two pieces that a transposing read takes of each of 8 entries stand in different banks
    static __device__ __forceinline__ int value_swizzle(int row) { return D >= 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3); }
};
template <int D_, bool FP8_>
struct ManyRows {
    static constexpr int D = D_, WAVES = 4, THREADS = 256, ROWS = 128, KT = D == 256 ? 32 : 64, STEP = KT;
    static constexpr bool FP8 = FP8_, FEW = false;
    static constexpr int PITCH = 2 * D, CHUNKS = D / 8;
    static constexpr int TILE = KT * PITCH, STAGE = 2 * TILE;
    static constexpr int LOADS = TILE / (FP8 ? 8192 : 4096); // of a wave, keys and values each
    static constexpr int LDS = 2 * STAGE;
    // a piece of 16 entries' keys and four pieces of four entries' values stand in different banks
    static __device__ __forceinline__ int key_swizzle(int row) { return D >= 128 ? row & 15 : (row >> 1) & 7; }
    static __device__ __forceinline__ int value_swizzle(int row) { return D >= 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }
};

// sum over the lanes up to this one: along rows of 16, then their last lanes' onto the rows behind
__device__ __forceinline__ int scan(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false); // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false); // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false); // row_bcast:31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ int uniform(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

struct Work {
    int first, tokens, own; // own: its entries as the array has them
    int tiles, keys, steps;
};
template <typename S>
__device__ __forceinline__ Work work_of(const AttentionParams &p, int s)
{
    Work w = {};
    if (s < p.sequences) {
        const TokenRange r = tokens_of(p.query_starts, s, p.tokens);
        w.first = r.first, w.tokens = r.end - r.first, w.own = max(p.lengths[s], 0);
        w.tiles = (w.tokens * (int)p.group.d + S::ROWS - 1) / S::ROWS;
        w.keys = min(w.own, p.own_limit) + (p.joined ? p.prefix_length : 0);
        w.steps = max((w.keys + (1 << p.step_log2) - 1) >> p.step_log2, 1);
    }
    return w;
}

// The piece of share `share` of kv head `head` that starts at `at` of the head's work (below zero: the share's first; no shares: tile `share`), and where the next one does, below zero: nowhere.
// False: there is none.  Sequences in order, of one its tiles from the last one on, which sees the most entries.
template <typename S>
__device__ __forceinline__ bool find_piece(const AttentionParams &p, int head, int share, int &at, int &next, Piece &u)
{
    const bool split = p.shares > 0;
    const int lane = (int)threadIdx.x & 63;
    Work w = work_of<S>(p, lane);
    int per = 1, end = INT32_MAX; // steps of a share; where this one's end
    bool whole = false;           // whether a share stays in a tile: those of a tile are multiples of `per` then
    const auto steps_in = [&](const Work &w) { return whole ? (int)(((uint32_t)w.steps + per - 1) / (uint32_t)per) * per : w.steps; };
    if (split) {
        int all = 0, all_tiles = 0;
        Work more = w;
        for (int s0 = 64;; s0 += 64) {
            all += uniform(scan(more.tiles * more.steps), 63), all_tiles += uniform(scan(more.tiles), 63);
            if (s0 >= p.sequences) {
                break;
            }
            more = work_of<S>(p, s0 + lane);
        }
        // A second piece costs its workgroup as much as some steps: with few tiles each piece has a workgroup of its own, all / per + tiles of them at most (8 sequences of 1 to
        // 1500 entries, 64 tiles: 14.6 us, with even shares 19.9; with more than a quarter as many tiles as shares these are the better ones, 123 us instead of 157 for 128 of 10000)
        whole = 4 * all_tiles <= p.shares;
        per = max((int)(whole ? (uint32_t)(all + p.shares - all_tiles - 1) / (uint32_t)(p.shares - all_tiles) : p.by_share.quotient((uint32_t)(all + p.shares - 1))), p.least);
        const int64_t most = whole ? INT32_MAX : all;
        at = at < 0 ? (int)min((int64_t)share * per, most) : at;
        end = (int)min((int64_t)(share + 1) * per, most);
        if (at >= end) {
            return false;
        }
    } else {
        at = share;
    }
    int work_before = 0, tiles_before = 0;
    for (int s0 = 0;;) {
        const int padded = steps_in(w), work = scan(split ? w.tiles * padded : w.tiles), tiles = split ? scan(w.tiles) : work; // up to this sequence
        const uint64_t behind = __ballot(at - work_before < work);
        if (behind != 0) {
            const int l = __builtin_ctzll(behind);
            const int first = uniform(w.first, l), tokens = uniform(w.tokens, l), own = uniform(w.own, l), keys = uniform(w.keys, l), steps = uniform(w.steps, l);
            const int its_tiles = uniform(w.tiles, l), room = uniform(padded, l), from = work_before + uniform(work, l) - (split ? its_tiles * room : its_tiles); // the sequence's first
            const int tile = !split ? at - from : its_tiles == 1 ? 0 : (int)((uint32_t)(at - from) / (uint32_t)room);
            const int number = tiles_before + uniform(tiles, l) - its_tiles + tile; // of the tile
            if ((uint32_t)tile >= (uint32_t)its_tiles || (uint32_t)number >= (uint32_t)p.most_tiles) {
                return false; // more tokens than there are: query_starts that fall
            }
            const int tile_at = split ? from + tile * room : at, step = at - tile_at, count = min(steps - step, split ? end - at : steps);
            u.table = p.page_table + (int64_t)(s0 + l) * p.page_table_ld;
            u.prefix = p.joined ? p.prefix_length : 0, u.keys = keys;
            u.token0 = first, u.row0 = (its_tiles - 1 - tile) * S::ROWS, u.rows = min(S::ROWS, tokens * (int)p.group.d - u.row0);
            u.limit0 = own - tokens + 1; // it has a token: no overflow
            u.begin = min(step << p.step_log2, keys), u.end = (int)min((int64_t)(step + count) << p.step_log2, (int64_t)keys);
            int share0 = share;
            u.shares = 1;
            if (split && count < steps) {
                share0 = (int)((uint32_t)tile_at / (uint32_t)per);
                u.shares = (int)((uint32_t)(tile_at + steps - 1) / (uint32_t)per) - share0 + 1;
            }
            u.first = head * (p.most_tiles + p.shares) + number + (split ? share0 : 0), u.share = share - share0, u.at = u.first + u.share;
            next = split && !whole && at + count < end ? at + count : -1;
            return true;
        }
        work_before += uniform(work, 63), tiles_before += uniform(tiles, 63);
        s0 += 64;
        if (s0 >= p.sequences) {
            return false;
        }
        w = work_of<S>(p, s0 + lane);
    }
}

// the same over the prefix, whose rows are those of the whole batch
template <typename S>
__device__ __forceinline__ bool find_prefix_piece(const AttentionParams &p, int head, int share, int &at, int &next, Piece &u)
{
    const int all = p.prefix_tiles * p.prefix_steps;
    at = at < 0 ? (int)min((int64_t)share * p.prefix_per, (int64_t)all) : at;
    const int end = (int)min((int64_t)(share + 1) * p.prefix_per, (int64_t)all);
    if (at >= end) {
        return false;
    }
    const int tile = (int)p.by_prefix_step.quotient((uint32_t)at);
    const int step = at - tile * p.prefix_steps, count = min(p.prefix_steps - step, end - at);
    u.table = nullptr, u.prefix = u.keys = p.prefix_length;
    u.token0 = 0, u.row0 = tile * S::ROWS, u.rows = min(S::ROWS, p.tokens * (int)p.group.d - u.row0), u.limit0 = INT32_MAX;
    u.begin = step << p.prefix_step_log2, u.end = (int)min((int64_t)(step + count) << p.prefix_step_log2, (int64_t)u.keys);
    u.at = head * (p.prefix_tiles + p.prefix_shares) + tile + share, u.first = 0, u.share = 0, u.shares = 1;
    next = at + count < end ? at + count : -1;
    return true;
}

// entries that a row sees, of the piece's
__device__ __forceinline__ int limit_of(const AttentionParams &p, const Piece &u, int row)
{
    if (!p.causal || u.limit0 == INT32_MAX) {
        return u.keys;
    }
    const int64_t own = (int64_t)u.limit0 + (int)p.group.quotient((uint32_t)(u.row0 + row));
    return (int)min(max(own, (int64_t)0) + u.prefix, (int64_t)u.keys);
}

// e4m3 as bf16, which holds every one of its values
__device__ __forceinline__ bf16x8 from_bytes(uint32_t lo, uint32_t hi)
{
    bf16x8 v;
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1], v[4] = c[0], v[5] = c[1], v[6] = d[0], v[7] = d[1];
    return v;
}

__device__ __forceinline__ int64_t from_lane(int64_t v, int lane)
{
    return (int64_t)((uint64_t)(uint32_t)__shfl((int)(uint32_t)v, lane, 64) | (uint64_t)(uint32_t)__shfl((int)(v >> 32), lane, 64) << 32);
}

// an unscaled logit's factor in powers of two; as good as zero at its smallest, and not so that -inf times it is no number
template <bool FP8>
__device__ __forceinline__ float logit_factor(const AttentionParams &p, int head)
{
    return fmaxf(p.scale_log2 * (FP8 ? p.k_scales[head] : 1.f), 0x1p-100f);
}

// 16 bytes of global memory: of a pointer that may be NOTHING's, which the compiler takes for one to anywhere
__device__ __forceinline__ uint4 load16(const char *from)
{
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    const words w = *(const __attribute__((address_space(1))) words *)from;
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// where the entries of a tile are, one in each of the first KT lanes
struct Entries {
    int page = -1, slot = 0; // of the tile after the next
    int64_t k = 0, v = 0;    // bytes from the head's first, of the next tile
    uint64_t next = 0;       // which of that are there

    template <int KT>
    __device__ __forceinline__ void ask(const AttentionParams &p, const Piece &u, int tile0, int end, int lane)
    {
        const int at = tile0 + lane;
        page = -1, slot = 0;
        if (lane < KT && at < end) {
            const bool shared = at < u.prefix;
            const uint32_t entry = (uint32_t)(shared ? at : at - u.prefix), column = p.page_size.quotient(entry);
            slot = (int)(entry - column * p.page_size.d);
            page = (shared ? p.prefix_pages : u.table)[column];
        }
    }
    __device__ __forceinline__ void place(const AttentionParams &p)
    {
        const bool ok = (uint32_t)page < (uint32_t)p.pages;
        next = __ballot(ok);
        k = page * p.k_page + slot * p.k_token, v = page * p.v_page + slot * p.v_token;
    }
};

// The same where pages are whole blocks of 16 entries, which start where one of the tile's does.  Where 64 of them are is found at a time, a block a lane, and their pages are
// read long before: waiting for a load is waiting for all that were asked for before it.
template <int BLOCKS, int STEP>
struct PagedBlocks {
    static constexpr int TILES = 64 / BLOCKS; // that are found at a time
    int pages;                                // of the tiles after those
    int64_t k, v;                             // bytes from the head's first to a block's first entry,
    int count;                                // and how many there are of it
    uint64_t whole;                           // blocks of which all are

    __device__ __forceinline__ int at(int begin, int tile) const
    {
        const int lane = (int)threadIdx.x & 63;
        return begin + (int)min((int64_t)(tile + lane / BLOCKS) * STEP, (int64_t)1 << 30) + 16 * (lane % BLOCKS);
    }
    __device__ __forceinline__ void read(const AttentionParams &p, const Piece &u, int begin, int end, int tile)
    {
        const int entry = min(at(begin, tile), (end - 1) & ~15);
        const bool shared = entry < u.prefix;
        pages = (shared ? p.prefix_pages : u.table)[p.page_size.quotient((uint32_t)(shared ? entry : entry - u.prefix))];
    }
    // the tiles from `tile` on, every TILES of them
    __device__ __forceinline__ void find(const AttentionParams &p, const Piece &u, int begin, int end, int tile)
    {
        const int here = at(begin, tile);
        const uint32_t entry = (uint32_t)(here < u.prefix ? here : here - u.prefix), slot = entry - p.page_size.quotient(entry) * p.page_size.d;
        const bool ok = here < end && (uint32_t)pages < (uint32_t)p.pages;
        const int64_t page = ok ? pages : 0;
        k = page * p.k_page + (ok ? slot : 0) * p.k_token, v = page * p.v_page + (ok ? slot : 0) * p.v_token;
        count = ok ? min(end - here, 16) : 0;
        whole = __ballot(count == 16);
        if (begin + (int64_t)(tile + TILES) * STEP < end) {
            read(p, u, begin, end, tile + TILES);
        }
    }
    static __device__ __forceinline__ int64_t of_lane(int64_t v, int lane)
    {
        return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane) | (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32);
    }
    __device__ __forceinline__ int64_t key(int tile, int block) const { return of_lane(k, tile % TILES * BLOCKS + block); }
    __device__ __forceinline__ int64_t value(int tile, int block) const { return of_lane(v, tile % TILES * BLOCKS + block); }
    __device__ __forceinline__ int entries(int tile, int block) const { return __builtin_amdgcn_readlane(count, tile % TILES * BLOCKS + block); }
    // which entries of a tile are there
    __device__ __forceinline__ uint64_t there(int tile) const
    {
        constexpr uint64_t ALL = BLOCKS == 4 ? ~(uint64_t)0 : ((uint64_t)1 << (16 * BLOCKS & 63)) - 1;
        const uint32_t blocks = (1u << BLOCKS) - 1;
        if (((uint32_t)(whole >> (tile % TILES * BLOCKS)) & blocks) == blocks) {
            return ALL;
        }
        uint64_t some = 0;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            some |= (((uint64_t)1 << entries(tile, b)) - 1) << (16 * b);
        }
        return some;
    }
};

// 16 bytes `at` bytes from a block's first entry, zeros from `size` on
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer_of(const char *from, int64_t size) { return __builtin_amdgcn_make_buffer_rsrc((void *)from, 0, (int)size, 0x00027000); }
__device__ __forceinline__ uint4 load16(Buffer from, uint32_t at, uint32_t further)
{
    const auto w = __builtin_amdgcn_raw_buffer_load_b128(from, (int)(at + further), 0, 0);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
constexpr uint32_t PAST_BLOCKS = 1u << 30; // no block is as long

// Powers of two by which m may stay behind the largest logit.  Weights are 2^-BEHIND of what they are to m, at most one, and so are the sums that a piece leaves.
constexpr float BEHIND = 8.f;
__device__ __forceinline__ float lse_of(float most, float total) // most in powers of two
{
    return total > 0.f ? (most + __log2f(total * 0x1p8f)) * LN2 : total == 0.f ? -INFINITY : total;
}

// results of a piece's rows: to where they belong, or as a share of them into the workspace
template <typename S>
struct Results {
    const AttentionParams &p;
    const Piece &u;
    int head;
    bool shared_prefix, direct;
    float v_scale;

    __device__ __forceinline__ Results(const AttentionParams &p_, const Piece &u_, int head_, bool shared_prefix_)
        : p(p_), u(u_), head(head_), shared_prefix(shared_prefix_), direct(!p_.combined || (!shared_prefix_ && u_.shares == 1 && p_.prefix_partial == nullptr)),
          v_scale(S::FP8 ? p_.v_scales[head_] : 1.f)
    {
    }
    __device__ __forceinline__ void place_of(int row, int &token, int &query_head) const
    {
        const uint32_t of = (uint32_t)(u.row0 + row), t = p.group.quotient(of);
        token = u.token0 + (int)t, query_head = head * (int)p.group.d + (int)(of - t * p.group.d);
    }
    // most in powers of two
    __device__ __forceinline__ void sums(int row, float most, float total) const
    {
        int token, query_head;
        place_of(row, token, query_head);
        if (direct) {
            if (p.lse != nullptr) {
                p.lse[(int64_t)token * p.heads + query_head] = lse_of(most, total);
            }
        } else {
            (shared_prefix ? p.prefix_sums : p.sums)[(int64_t)u.at * S::ROWS + row] = make_float2(most, total);
        }
        if (p.combined && !shared_prefix && u.share == 0) {
            p.rows[(int64_t)token * p.heads + query_head] = make_int4(u.first, direct ? 0 : u.shares, row, 0);
        }
    }
    // four channels from `at` on of a row, `get(e)` each
    template <int STRIDE, typename F>
    __device__ __forceinline__ void row(int row, int at0, float total, int count, F get) const
    {
        if (direct) {
            int token, query_head;
            place_of(row, token, query_head);
            const float over = total == 0.f ? 0.f : v_scale / total;
            bf16_t *to = p.out + token * p.out_token + query_head * p.out_head;
#pragma unroll
            for (int i = 0; i < count; ++i) {
                if (at0 + STRIDE * i < p.size) {
                    bf16x4 r;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        r[e] = (bf16_t)(get(i, e) * over);
                    }
                    __builtin_memcpy(to + at0 + STRIDE * i, &r, 8);
                }
            }
        } else {
            float *to = (shared_prefix ? p.prefix_partial : p.partial) + ((int64_t)u.at * S::ROWS + row) * S::D;
#pragma unroll
            for (int i = 0; i < count; ++i) {
                *(float4 *)(to + at0 + STRIDE * i) = make_float4(get(i, 0) * v_scale, get(i, 1) * v_scale, get(i, 2) * v_scale, get(i, 3) * v_scale);
            }
        }
    }
};

// COUNT groups of N operands, each read from the LDS while the products of the one before it are formed.  Left to itself the compiler reads one operand, waits, and goes on
// with its product.
template <int N, int COUNT, typename R, typename F>
__device__ __forceinline__ void ahead(R read, F use)
{
    bf16x8 x[2][N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        x[0][i] = read(i);
    }
#pragma unroll
    for (int g = 0; g < COUNT; ++g) {
        if (g + 1 < COUNT) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                x[(g + 1) & 1][i] = read(N * (g + 1) + i);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            use(N * g + i, x[g & 1][i]);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Loads have come, here and not in a loop that follows: there the compiler would wait in each round, for all loads that the last one has asked for
template <int N>
__device__ __forceinline__ void arrived(bf16x8 (&x)[N])
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        asm volatile("" : "+v"(x[i]));
    }
}

// Up to 16 rows by a workgroup, its waves with a tile of keys each in turn.  Lane l has row l & 15; of 16 keys their logits 4 (l >> 4) .. + 3, of 16 channels such results.
template <typename S, bool PAGED_BLOCKS>
__device__ __forceinline__ void attend_few(const AttentionParams &p, const Piece &u, int head, bool shared_prefix, char *lds)
{
    constexpr int D = S::D, KT = S::KT, BLOCKS = KT / 16;
    constexpr bool FP8 = S::FP8;
    constexpr int PIECES = D / (FP8 ? 64 : 32); // 16-byte pieces of a key in a lane
    constexpr uint64_t ALL = KT == 64 ? ~(uint64_t)0 : ((uint64_t)1 << (KT & 63)) - 1;
    const int lane = (int)threadIdx.x & 63, row = lane & 15, quarter = lane >> 4, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int first_limit = limit_of(p, u, 0), end = min(u.end, limit_of(p, u, u.rows - 1)), begin = u.begin + wave * KT; // of this wave, then every STEP keys
    const int steps = max((end - begin + S::STEP - 1) / S::STEP, 0);
    const bool has_row = row < u.rows;
    char *mine = lds + wave * S::TILE; // values of the tile at hand

    Entries entries;
    PagedBlocks<BLOCKS, S::STEP> blocks;
    if (steps > 0) {
        if constexpr (PAGED_BLOCKS) {
            blocks.read(p, u, begin, end, 0);
        } else {
            entries.ask<KT>(p, u, begin, end, lane);
        }
    }
    // channels of a fragment in this lane, the same for keys: 16 bytes of e4m3 are two fragments'
    const auto channel = [&](int i) { return FP8 ? 64 * (i / 2) + 16 * quarter + 8 * (i & 1) : 32 * i + 8 * quarter; };
    bf16x8 q[D / 32];
    {
        const uint32_t of = (uint32_t)(u.row0 + (has_row ? row : 0)), token = p.group.quotient(of);
        const bf16_t *from = p.q + (int64_t)(u.token0 + (int)token) * p.q_token + (int64_t)(head * (int)p.group.d + (int)(of - token * p.group.d)) * p.q_head;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            uint4 piece = zero_u4();
            if (has_row && channel(i) < p.size) {
                __builtin_memcpy(&piece, from + channel(i), 16);
            }
            q[i] = as_bf16x8(piece);
        }
        arrived(q);
    }
    const int limit = has_row ? limit_of(p, u, row) : u.keys;
    const float factor = logit_factor<FP8>(p, head);
    f32x4 o[D / 16];
    float m = -INFINITY, sum = 0.f;
#pragma unroll
    for (int d = 0; d < D / 16; ++d) {
        o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // the tile on its way: keys as the matrix instructions take them, lane -> entry lane & 15 of 16, values by whole entries
    const char *k_head = p.k + head * p.k_head, *v_head = p.v + head * p.v_head;
    constexpr int ACROSS = FP8 ? D / 16 : S::CHUNKS, PER_LOAD = 64 / ACROSS; // pieces of an entry, entries of a load
    uint4 k[BLOCKS][PIECES], v[S::LOADS];
    uint64_t there = 0;
    const auto ask = [&](int step) {
        int l = lane;
        asm volatile("" : "+v"(l)); // what follows from it is formed anew for each tile: kept, it would take the registers that the tiles need
        const int row = l & 15, k_byte = 16 * (l >> 4), in_load = l / ACROSS, v_byte = 16 * (l % ACROSS), bytes = (FP8 ? 1 : 2) * p.size; // piece i of a key is at k_byte + 64 i
        if constexpr (PAGED_BLOCKS) {
            if (step % blocks.TILES == 0) {
                blocks.find(again(), u, begin, end, step);
            }
            there = blocks.there(step);
            const uint32_t k_lane = (uint32_t)(row * (int)p.k_token + k_byte), v_lane = v_byte < bytes ? (uint32_t)(in_load * (int)p.v_token + v_byte) : PAST_BLOCKS;
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
                const Buffer from = buffer_of(k_head + blocks.key(step, b), blocks.entries(step, b) * p.k_token);
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    k[b][i] = load16(from, k_byte + 64 * i < bytes ? k_lane : PAST_BLOCKS, 64 * i);
                }
            }
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
                const Buffer from = buffer_of(v_head + blocks.value(step, b), blocks.entries(step, b) * p.v_token);
#pragma unroll
                for (int i = 0; i < 16 / PER_LOAD; ++i) {
                    v[b * (16 / PER_LOAD) + i] = load16(from, v_lane, i * PER_LOAD * (uint32_t)p.v_token);
                }
            }
        } else {
            entries.place(p);
            there = entries.next;
            entries.ask<KT>(p, u, begin + (step + 1) * S::STEP, end, lane);
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
                const int64_t at = from_lane(entries.k, 16 * b + row);
                const bool ok = ((entries.next >> (16 * b + row)) & 1) != 0;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    k[b][i] = load16(ok && k_byte + 64 * i < bytes ? k_head + at + (k_byte + 64 * i) : (const char *)NOTHING);
                }
            }
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i) {
                const int of = i * PER_LOAD + in_load;
                const int64_t at = from_lane(entries.v, of);
                const bool ok = ((entries.next >> of) & 1) != 0 && v_byte < bytes;
                v[i] = load16(ok ? v_head + at + v_byte : (const char *)NOTHING);
            }
        }
    };
    const auto tile = [&](int step) {
        const int tile0 = begin + step * S::STEP;
        const uint64_t seen = there;
        const bool limited = first_limit < min(tile0 + KT, end); // not all rows see all of its entries
        int l = lane;
        asm volatile("" : "+v"(l)); // as above
        const int in_load = l / ACROSS, piece = l % ACROSS;
#pragma unroll
        for (int i = 0; i < S::LOADS; ++i) {
            const int of = i * PER_LOAD + in_load;
            char *to = mine + of * S::PITCH;
            if constexpr (FP8) {
                *(uint4 *)(to + 16 * ((2 * piece) ^ S::value_swizzle(of))) = as_uint4(from_bytes(v[i].x, v[i].y));
                *(uint4 *)(to + 16 * ((2 * piece + 1) ^ S::value_swizzle(of))) = as_uint4(from_bytes(v[i].z, v[i].w));
            } else {
                *(uint4 *)(to + 16 * (piece ^ S::value_swizzle(of))) = v[i];
            }
        }
        f32x4 s[BLOCKS];
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
            s[b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                bf16x8 key;
                if constexpr (FP8) {
                    key = (i & 1) == 0 ? from_bytes(k[b][i / 2].x, k[b][i / 2].y) : from_bytes(k[b][i / 2].z, k[b][i / 2].w);
                } else {
                    key = as_bf16x8(k[b][i]);
                }
                s[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(key, q[i], s[b], 0, 0, 0);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        ask(step + 1); // past the end: nothing.  Without a condition, so that how many loads are on their way is known
        if (seen == 0) {
            return;
        }
        if (limited || seen != ALL) {
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
                const uint32_t mask = ((uint32_t)(seen >> (16 * b)) >> (4 * quarter)) & (((uint32_t)1 << min(max(limit - tile0 - 16 * b - 4 * quarter, 0), 4)) - 1);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[b][i] = (mask & (1u << i)) != 0 ? s[b][i] : -INFINITY;
                }
            }
        }
        float most = s[0][0];
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                most = fmaxf(most, s[b][i]);
            }
        }
        most = quarter_swap_max(half_swap_max(most));
        const bool follow = (most - m) * factor > BEHIND; // also where nothing has been seen yet; each row for itself, so that none's bits depend on its neighbours
        if (__any(follow)) {
            const float next = follow ? most : m, keep = __builtin_amdgcn_exp2f((m - (next == -INFINITY ? 0.f : next)) * factor);
            m = next, sum *= keep;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) {
                o[d] *= keep;
            }
        }
        const float base = fmaf(m == -INFINITY ? 0.f : m, factor, BEHIND); // nothing seen yet: weights of zero
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[b][i] = __builtin_amdgcn_exp2f(fmaf(s[b][i], factor, -base));
                sum += s[b][i]; // of this lane's quarter of the keys
            }
        }
        if (limited) {
            bool wild = false; // an infinity or no number among values that a row must not see: its weight of zero would not keep it out
#pragma unroll 1
            for (int i = lane; i < KT * S::CHUNKS; i += 64) {
                wild = wild || wild_piece(*(const uint4 *)(mine + 16 * i));
            }
            if (__any(wild)) { // added where they are seen, as they are: whatever their weight, they are what comes of it; then zeros
#pragma unroll 1
                for (int key = 0; key < KT; ++key) {
#pragma unroll
                    for (int d = 0; d < D / 16; ++d) {
                        bf16x4 x;
                        __builtin_memcpy(&x, mine + key * S::PITCH + 16 * ((2 * d + (quarter >> 1)) ^ S::value_swizzle(key)) + 8 * (quarter & 1), 8);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            o[d][e] += tile0 + key < limit && !(fabsf((float)x[e]) < INFINITY) ? (float)x[e] : 0.f;
                        }
                    }
                }
#pragma unroll 1
                for (int i = lane; i < KT * S::CHUNKS; i += 64) {
                    uint32_t any = 0;
                    uint4 *at = (uint4 *)(mine + 16 * i);
                    *at = as_uint4(finite_part(as_bf16x8(*at), any));
                }
            }
        }
        // values of 32 keys and 16 channels, transposed: lane -> channel lane & 15, keys 4 quarter .. + 3 and 16 further on, as the logits have them
        const int from_row = 4 * quarter + (row >> 2);
        uint32_t lane_at = (uint32_t)(from_row * S::PITCH + 16 * (((row & 3) >> 1) ^ S::value_swizzle(from_row)) + 8 * (row & 1));
        asm volatile("" : "+v"(lane_at)); // as above
        // 16 bits of the weights: the second product is no cost here.  Both parts have the weight's sign, and the rest, 2^-30 of the weight larger than it is, is no zero where the
        // weight is none: an infinite value stays one.
        bf16x8 w[KT / 32], rest[KT / 32];
#pragma unroll
        for (int t = 0; t < KT / 32; ++t) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = s[2 * t + e / 4][e & 3];
                const float cut = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
                w[t][e] = (bf16_t)cut;
                rest[t][e] = (bf16_t)fmaf(x, 0x1p-30f, x - cut);
            }
        }
        constexpr int OF_32 = D / 16, GROUP = 4, GROUPS = KT / 32 * OF_32 / GROUP;
        ahead<GROUP, GROUPS>(
            [&](int i) {
                const lds_char *at = (const lds_char *)mine + 32 * (i / OF_32) * S::PITCH + (lane_at ^ (32 * (i % OF_32))); // pieces 2 d and 2 d + 1
                return lds_transposed_fragment(at, at + 16 * S::PITCH);
            },
            [&](int i, bf16x8 x) {
                f32x4 &to = o[i % OF_32];
                to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, w[i / OF_32], to, 0, 0, 0);
                to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, rest[i / OF_32], to, 0, 0, 0);
            });
    };

    if (steps > 0) {
        ask(0);
        for (int step = 0; step < steps; ++step) {
            tile(step);
        }
    }

    // the waves join
    constexpr int P = D + 4; // floats from row to row
    float *joined = (float *)lds;
    float2 *joined_sums = (float2 *)(lds + S::WAVES * S::ROWS * P * 4);
    sum = quarter_swap_sum(half_swap_sum(sum));
    __syncthreads();
    if (has_row) {
        if (quarter == 0) {
            joined_sums[wave * S::ROWS + row] = make_float2(m == -INFINITY ? m : m * factor, sum);
        }
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
            *(f32x4 *)(joined + (wave * S::ROWS + row) * P + 16 * d + 4 * quarter) = o[d];
        }
    }
    __syncthreads();
    const Results<S> results(again(), u, head, shared_prefix);
    for (int i = (int)threadIdx.x; i < u.rows * (D / 4); i += S::THREADS) {
        const int r = i / (D / 4), at = 4 * (i % (D / 4));
        float most = -INFINITY, total = 0.f, x[4] = {0.f, 0.f, 0.f, 0.f};
        float2 of[S::WAVES];
#pragma unroll
        for (int w = 0; w < S::WAVES; ++w) {
            of[w] = joined_sums[w * S::ROWS + r];
            most = fmaxf(most, of[w].x);
        }
        const float base = most == -INFINITY ? 0.f : most;
#pragma unroll
        for (int w = 0; w < S::WAVES; ++w) {
            const float weight = __builtin_amdgcn_exp2f(of[w].x - base);
            const float4 add = *(const float4 *)(joined + (w * S::ROWS + r) * P + at);
            total = fmaf(weight, of[w].y, total);
            x[0] = fmaf(weight, add.x, x[0]), x[1] = fmaf(weight, add.y, x[1]), x[2] = fmaf(weight, add.z, x[2]), x[3] = fmaf(weight, add.w, x[3]);
        }
        if (at == 0) {
            results.sums(r, most, total);
        }
        results.template row<4>(r, at, total, 1, [&](int, int e) { return x[e]; });
    }
    __syncthreads(); // the LDS is free for the next piece
}

// Up to 128 rows by a workgroup, 32 a wave.  Lane l has row l & 31; of 32 keys their logits 8 i + 4 (l >> 5) .. + 3, of 32 channels such results.
template <typename S, bool PAGED_BLOCKS>
__device__ __forceinline__ void attend_many(const AttentionParams &p, const Piece &u, int head, bool shared_prefix, char *lds)
{
    constexpr int D = S::D, KT = S::KT;
    constexpr bool FP8 = S::FP8;
    constexpr uint64_t ALL = KT == 64 ? ~(uint64_t)0 : ((uint64_t)1 << (KT & 63)) - 1;
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), half = lane >> 5;
    const int first_limit = limit_of(p, u, 0), last_limit = limit_of(p, u, u.rows - 1);
    const int end = min(u.end, last_limit), steps = max((end - u.begin + KT - 1) / KT, 0);

    bf16x8 q[D / 16];
    const int wave_row = 32 * wave, row = wave_row + (lane & 31);
    const bool has_row = row < u.rows;
    {
        const uint32_t of = (uint32_t)(u.row0 + (has_row ? row : 0)), token = p.group.quotient(of);
        const bf16_t *from = p.q + (int64_t)(u.token0 + (int)token) * p.q_token + (int64_t)(head * (int)p.group.d + (int)(of - token * p.group.d)) * p.q_head;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            const int at = 16 * i + 8 * half;
            uint4 piece = zero_u4();
            if (has_row && at < p.size) {
                __builtin_memcpy(&piece, from + at, 16);
            }
            q[i] = as_bf16x8(piece);
        }
        arrived(q);
    }
    const int limit = has_row ? limit_of(p, u, row) : u.keys;
    const int wave_last_limit = limit_of(p, u, min(wave_row + 32, u.rows) - 1);
    const bool wave_idle = wave_row >= u.rows;

    f32x16 o[D / 32];
    float m = -INFINITY, sum = 0.f; // of this lane's half of the keys
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
        o[d] = zero16();
    }
    const float factor = logit_factor<FP8>(p, head);

    // ---- entries on their way ----
    const char *k_head = p.k + head * p.k_head, *v_head = p.v + head * p.v_head;
    const uint32_t lds_at = (uint32_t)(uintptr_t)(lds_char *)lds;
    Entries entries;
    constexpr int BYTE_LOADS = FP8 ? S::LOADS : 1;
    uint4 k_bytes[BYTE_LOADS], v_bytes[BYTE_LOADS];
    constexpr int LOADS = S::LOADS, ACROSS = FP8 ? D / 16 : S::CHUNKS, PER_LOAD = 64 / ACROSS; // pieces of an entry, entries of a load
    PagedBlocks<KT / 16, KT> blocks;
    uint64_t there = 0, there_next = 0; // entries of the tile at hand and of the next that are there
    const auto ask = [&](int stage, int step) {
        constexpr int OF_WAVE = LOADS * PER_LOAD; // entries, all of one block
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds_at + (uint32_t)(stage * S::STAGE + wave * S::LOADS * 1024));
        const int in_load = lane / ACROSS, piece = lane % ACROSS, bytes = (FP8 ? 1 : 2) * p.size;
        if constexpr (PAGED_BLOCKS) {
            if (step % blocks.TILES == 0) {
                blocks.find(again(), u, u.begin, end, step);
            }
            there_next = blocks.there(step);
            const int block = wave * OF_WAVE / 16, count = blocks.entries(step, block);
            const char *k = k_head + blocks.key(step, block), *v = v_head + blocks.value(step, block);
            const int first = wave * OF_WAVE & 15; // of the block
            if constexpr (FP8) {
                const Buffer k_from = buffer_of(k, count * p.k_token), v_from = buffer_of(v, count * p.v_token);
                const uint32_t past = 16 * piece < bytes ? 0 : PAST_BLOCKS;
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    k_bytes[i] = load16(k_from, past | (uint32_t)(in_load * (int)p.k_token + 16 * piece), (uint32_t)((first + i * PER_LOAD) * (int)p.k_token));
                    v_bytes[i] = load16(v_from, past | (uint32_t)(in_load * (int)p.v_token + 16 * piece), (uint32_t)((first + i * PER_LOAD) * (int)p.v_token));
                }
            } else if (count == 16 && p.size == D) {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int of = wave * OF_WAVE + i * PER_LOAD + in_load;
                    load_to_lds(to + 1024 * i, k + (first + i * PER_LOAD) * p.k_token, (uint32_t)(in_load * (int)p.k_token + 16 * (piece ^ S::key_swizzle(of))));
                    load_to_lds(to + S::TILE + 1024 * i, v + (first + i * PER_LOAD) * p.v_token, (uint32_t)(in_load * (int)p.v_token + 16 * (piece ^ S::value_swizzle(of))));
                }
            } else {
#pragma unroll
                for (int i = 0; i < LOADS; ++i) {
                    const int of = wave * OF_WAVE + i * PER_LOAD + in_load, in_block = of & 15, kp = piece ^ S::key_swizzle(of), vp = piece ^ S::value_swizzle(of);
                    load_to_lds_from(to + 1024 * i, in_block < count && 16 * kp < bytes ? k + in_block * p.k_token + 16 * kp : (const char *)NOTHING);
                    load_to_lds_from(to + S::TILE + 1024 * i, in_block < count && 16 * vp < bytes ? v + in_block * p.v_token + 16 * vp : (const char *)NOTHING);
                }
            }
        } else {
            entries.place(p);
            there_next = entries.next;
            entries.ask<KT>(p, u, u.begin + (step + 1) * KT, end, lane);
#pragma unroll
            for (int i = 0; i < LOADS; ++i) {
                const int of = wave * OF_WAVE + i * PER_LOAD + in_load;
                const bool ok = ((there_next >> of) & 1) != 0;
                const int kp = FP8 ? piece : piece ^ S::key_swizzle(of), vp = FP8 ? piece : piece ^ S::value_swizzle(of);
                const int64_t k_at = from_lane(entries.k, of), v_at = from_lane(entries.v, of);
                const char *kf = ok && 16 * kp < bytes ? k_head + k_at + 16 * kp : (const char *)NOTHING;
                const char *vf = ok && 16 * vp < bytes ? v_head + v_at + 16 * vp : (const char *)NOTHING;
                if constexpr (FP8) {
                    k_bytes[i] = load16(kf), v_bytes[i] = load16(vf);
                } else {
                    load_to_lds_from(to + 1024 * i, kf);
                    load_to_lds_from(to + S::TILE + 1024 * i, vf);
                }
            }
        }
    };
    const auto place_bytes = [&](int stage) {
        if constexpr (FP8) {
            char *to = lds + stage * S::STAGE;
#pragma unroll
            for (int i = 0; i < S::LOADS; ++i) {
                const int of = ((wave * S::LOADS + i) * 64 + lane) / (D / 16), piece = lane % (D / 16);
                const auto put = [&](uint4 bytes, char *at, int swizzle) {
                    *(uint4 *)(at + of * S::PITCH + 16 * ((2 * piece) ^ swizzle)) = as_uint4(from_bytes(bytes.x, bytes.y));
                    *(uint4 *)(at + of * S::PITCH + 16 * ((2 * piece + 1) ^ swizzle)) = as_uint4(from_bytes(bytes.z, bytes.w));
                };
                put(k_bytes[i], to, S::key_swizzle(of));
                put(v_bytes[i], to + S::TILE, S::value_swizzle(of));
            }
        }
    };

    // one tile of keys; LIMITED: not all rows of the workgroup see all of its entries
    const auto compute = [&](int step, int stage, auto limited) {
        constexpr bool LIMITED = decltype(limited)::value;
        const int tile0 = u.begin + step * KT;
        if (wave_idle || there == 0 || (LIMITED && tile0 >= wave_last_limit)) {
            return;
        }
        const char *keys = lds + stage * S::STAGE, *values = keys + S::TILE;
        f32x16 s[KT / 32];
#pragma unroll
        for (int kb = 0; kb < KT / 32; ++kb) {
            s[kb] = zero16();
        }
        // the lane's part of an address, formed anew for each tile: kept, those of all pieces would take registers
        uint32_t key_at = (uint32_t)((lane & 31) * S::PITCH + 16 * (half ^ S::key_swizzle(lane & 31)));
        asm volatile("" : "+v"(key_at));
        constexpr int GROUP = LIMITED ? 2 : 4; // fewer registers, where there are others to keep
        ahead<GROUP, KT / 32 * D / 16 / GROUP>(
            [&](int i) { return as_bf16x8(*(const uint4 *)(keys + 32 * (i % (KT / 32)) * S::PITCH + (key_at ^ (32 * (i / (KT / 32)))))); }, // piece 2 i + half
            [&](int i, bf16x8 k) { s[i % (KT / 32)] = mfma(k, q[i / (KT / 32)], s[i % (KT / 32)]); });
        if (LIMITED || there != ALL) {
#pragma unroll
            for (int kb = 0; kb < KT / 32; ++kb) {
                uint32_t seen = (uint32_t)(there >> (32 * kb)) >> (4 * half); // of this lane, entry 8 (i / 4) + (i & 3) is logit i
                if constexpr (LIMITED) {
                    const int count = min(max(limit - tile0 - 32 * kb - 4 * half, 0), 31); // its last one is entry 27
                    seen &= ((uint32_t)1 << count) - 1;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[kb][i] = (seen & ((uint32_t)1 << (8 * (i / 4) + (i & 3)))) != 0 ? s[kb][i] : -INFINITY;
                }
            }
        }
        float most = s[0][0];
#pragma unroll
        for (int kb = 0; kb < KT / 32; ++kb) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                most = fmaxf(most, s[kb][i]);
            }
        }
        most = half_swap_max(most);
        const bool follow = (most - m) * factor > BEHIND; // also where nothing has been seen yet; each row for itself, so that none's bits depend on its neighbours
        if (__any(follow)) {
            const float next = follow ? most : m, keep = __builtin_amdgcn_exp2f((m - (next == -INFINITY ? 0.f : next)) * factor);
            m = next, sum *= keep;
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    o[d][i] *= keep;
                }
            }
        }
        const float base = fmaf(m == -INFINITY ? 0.f : m, factor, BEHIND); // nothing seen yet: weights of zero
        bf16x8 w[KT / 16];
#pragma unroll
        for (int i = 0; i < KT / 16; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int at = 8 * (i & 1) + e;
                s[i / 2][at] = __builtin_amdgcn_exp2f(fmaf(s[i / 2][at], factor, -base));
                sum += s[i / 2][at];
                w[i][e] = (bf16_t)s[i / 2][at]; // the one rounding, as an operand: 2^-8 of each at most
            }
        }
        // values of 16 keys and 32 channels, transposed: lane -> channel lane & 31, keys 4 half .. + 3 and 8 further on, as the logits have them
        const int in16 = lane & 15, from_row = 4 * half + (in16 >> 2);
        uint32_t value_at = (uint32_t)(from_row * S::PITCH + 16 * ((2 * ((lane >> 4) & 1) + ((in16 & 3) >> 1)) ^ S::value_swizzle(from_row)) + 8 * (in16 & 1));
        asm volatile("" : "+v"(value_at));
        uint32_t wild = 0; // an infinity or no number among values that a row must not see: its weight of zero would not keep it out
        ahead<GROUP, KT / 16 * D / 32 / GROUP>(
            [&](int i) {
                const lds_char *at = (const lds_char *)values + 16 * (i / (D / 32)) * S::PITCH + (value_at ^ (64 * (i % (D / 32)))); // from piece 4 d on
                return lds_transposed_fragment(at, at + 8 * S::PITCH);
            },
            [&](int i, bf16x8 v) {
                if constexpr (LIMITED) {
                    v = finite_part(v, wild);
                }
                o[i % (D / 32)] = mfma(v, w[i / (D / 32)], o[i % (D / 32)]);
            });
        if (LIMITED && __any(wild != 0)) { // as above
#pragma unroll 1
            for (int key = 0; key < KT; ++key) {
#pragma unroll
                for (int d = 0; d < D / 32; ++d) {
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        bf16x4 v;
                        __builtin_memcpy(&v, values + key * S::PITCH + 16 * ((4 * d + a) ^ S::value_swizzle(key)) + 8 * half, 8);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = (float)v[e];
                            o[d][4 * a + e] += tile0 + key < limit && !(fabsf(x) < INFINITY) ? x : 0.f;
                        }
                    }
                }
            }
        }
    };

    // ---- the pass ----
    if (steps > 0) {
        if constexpr (PAGED_BLOCKS) {
            blocks.read(p, u, u.begin, end, 0);
        } else {
            entries.ask<KT>(p, u, u.begin, end, lane);
        }
        ask(0, 0);
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
            __syncthreads(); // this stage is there for all, and nobody reads the other any more
            if (step + 1 < steps) {
                ask(stage ^ 1, step + 1);
            }
            compute(step, stage, limited);
        }
    };
    // entries up to the first row's limit are every row's; with none past it, the last step is whole, too
    const int whole_steps = first_limit >= end ? steps : max(first_limit - u.begin, 0) / KT;
    pass(0, whole_steps, std::false_type{});
    pass(whole_steps, steps, std::true_type{});

    const Results<S> results(again(), u, head, shared_prefix);
    sum = half_swap_sum(sum);
    if (has_row) {
        if (half == 0) {
            results.sums(row, m == -INFINITY ? m : m * factor, sum);
        }
        results.template row<8>(row, 4 * half, sum, D / 8, [&](int i, int e) { return o[i / 4][4 * (i % 4) + e]; });
    }
    __syncthreads(); // the LDS is free for the next piece
}

template <typename S, bool PAGED_BLOCKS>
__device__ __forceinline__ void attend_all(const AttentionParams &p, int block, bool shared_prefix, char *lds)
{
    const int share = block / p.kv_heads, head = block - share * p.kv_heads;
    int at = -1;
    do {
        int next = -1;
        Piece u;
        if (!(shared_prefix ? find_prefix_piece<S>(again(), head, share, at, next, u) : find_piece<S>(again(), head, share, at, next, u))) {
            break;
        }
        if constexpr (S::FEW) {
            attend_few<S, PAGED_BLOCKS>(p, u, head, shared_prefix, lds);
        } else {
            attend_many<S, PAGED_BLOCKS>(p, u, head, shared_prefix, lds);
        }
        at = next;
    } while (at >= 0);
}

// OWN: of the sequences' tiles, PREFIX: of the prefix's
template <typename OWN, typename PREFIX, bool PAGED_BLOCKS>
__global__ __launch_bounds__(OWN::THREADS, OWN::D <= 128 ? 2 : 1) void cached_attention_kernel(const AttentionParams p)
{
    static_assert(OWN::THREADS == PREFIX::THREADS, "");
    extern __shared__ __align__(16) char lds[];
    const int prefix_blocks = p.prefix_shares * p.kv_heads;
    const bool shared_prefix = (int)blockIdx.x < prefix_blocks;
    const int block = (int)blockIdx.x - (shared_prefix ? 0 : prefix_blocks);
    if constexpr (std::is_same_v<OWN, PREFIX>) {
        attend_all<OWN, PAGED_BLOCKS>(p, block, shared_prefix, lds);
    } else if (shared_prefix) {
        attend_all<PREFIX, PAGED_BLOCKS>(p, block, true, lds);
    } else {
        attend_all<OWN, PAGED_BLOCKS>(p, block, false, lds);
    }
}

// The pieces of a row, those of the prefix in order, then its sequence's: WAVES waves of a row's side by side, where there are few rows, or ROWS rows in a wave, as a row is one
// read after the other, of its place, its sums, its results (3 sequences of 700 tokens, 67000 rows: 167 us with the products, 196 with a wave for each row).
struct CombineParams {
    const float *prefix_partial, *partial;
    const float2 *prefix_sums, *sums;
    const int4 *rows;
    int prefix_shares, prefix_tiles, prefix_steps, prefix_per, prefix_rows; // prefix_rows, own_rows: of a tile
    int own_rows, most_pieces;
    int tokens, heads, size, sequences;
    Divisor group, by_prefix_per;
    const int32_t *query_starts;
    bf16_t *out;
    int64_t out_token, out_head;
    float *lse;
};

template <int D, int WAVES, int ROWS>
__global__ __launch_bounds__(256) void combine_kernel(const CombineParams p)
{
    static_assert(WAVES == 1 || (WAVES == 4 && ROWS == 1), "");
    constexpr int PER_GROUP = 4 / WAVES * ROWS, LANES = 64 / ROWS, V = D / LANES, AHEAD = V > 8 ? 4 : 8, STORED = V < 8 ? V : 8;
    __shared__ float shared[WAVES > 1 ? WAVES * (D + 2) : 1];
    const int lane = (int)threadIdx.x & (LANES - 1), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), part = WAVES > 1 ? wave : 0;
    const int64_t count = (int64_t)p.tokens * p.heads;
    const int from = p.query_starts[0], to = p.query_starts[p.sequences];
    for (int64_t index = (int64_t)blockIdx.x * PER_GROUP + (WAVES > 1 ? 0 : (int)threadIdx.x / LANES); index < count; index += (int64_t)gridDim.x * PER_GROUP) {
        const int token = (int)(index / p.heads), head = (int)(index - (int64_t)token * p.heads);
        const int4 own = p.rows[index];
        if (token < from || token >= to) {
            continue;
        }
        const bool valid = own.x >= 0 && own.z >= 0 && own.z < p.own_rows && own.y > 0 && (int64_t)own.x + own.y <= p.most_pieces;
        const int own_pieces = valid ? own.y : 0;
        int64_t prefix_place = 0; // of the first piece's row
        int prefix_pieces = 0;
        if (p.prefix_shares > 0) {
            const int kv_head = (int)p.group.quotient((uint32_t)head);
            const uint32_t stacked = (uint32_t)token * p.group.d + (uint32_t)(head - kv_head * (int)p.group.d), tile = stacked / (uint32_t)p.prefix_rows;
            const uint32_t start = tile * (uint32_t)p.prefix_steps;
            const int first = (int)p.by_prefix_per.quotient(start);
            prefix_pieces = (int)p.by_prefix_per.quotient(start + (uint32_t)p.prefix_steps - 1) - first + 1;
            prefix_place = ((int64_t)kv_head * (p.prefix_tiles + p.prefix_shares) + tile + first) * p.prefix_rows + (stacked - tile * (uint32_t)p.prefix_rows);
        }
        const int pieces = prefix_pieces + own_pieces;
        if (pieces == 0) {
            continue; // its one workgroup has written it
        }
        const int64_t own_place = (int64_t)own.x * p.own_rows + own.z;
        const auto place = [&](int i) { return i < prefix_pieces ? prefix_place + (int64_t)i * p.prefix_rows : own_place + (int64_t)(i - prefix_pieces) * p.own_rows; };
        const auto sums_of = [&](int i) { return (i < prefix_pieces ? p.prefix_sums : p.sums)[place(i)]; };
        // the first ones of each wave without a wait between them
        float v[V] = {}, total = 0.f, most = -INFINITY;
        const int mine = (pieces - part + WAVES - 1) / WAVES; // of this wave: part, part + WAVES, ..
        for (int i0 = 0; i0 < mine; i0 += AHEAD) {
            float2 s[AHEAD];
            float x[AHEAD][V];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int at = part + WAVES * min(i0 + i, mine - 1);
                s[i] = sums_of(at);
                __builtin_memcpy(x[i], (at < prefix_pieces ? p.prefix_partial : p.partial) + place(at) * D + V * lane, sizeof(x[i]));
            }
            float now = most;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                now = fmaxf(now, s[i].x);
            }
            const float base = now == -INFINITY ? 0.f : now, keep = __builtin_amdgcn_exp2f(most - base);
            most = now, total *= keep;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[e] *= keep;
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                if (i0 + i < mine) {
                    const float w = __builtin_amdgcn_exp2f(s[i].x - base);
                    total = fmaf(w, s[i].y, total);
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        v[e] = fmaf(w, x[i][e], v[e]);
                    }
                }
            }
        }
        if constexpr (WAVES > 1) {
            __syncthreads(); // the last row's have been read
#pragma unroll
            for (int e = 0; e < V; ++e) {
                shared[wave * (D + 2) + V * lane + e] = v[e];
            }
            if (lane == 0) {
                shared[wave * (D + 2) + D] = most, shared[wave * (D + 2) + D + 1] = total;
            }
            __syncthreads();
            if (wave != 0) {
                continue;
            }
            float now = -INFINITY;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                now = fmaxf(now, shared[w * (D + 2) + D]);
            }
            const float base = now == -INFINITY ? 0.f : now;
            total = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[e] = 0.f;
            }
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const float weight = __builtin_amdgcn_exp2f(shared[w * (D + 2) + D] - base);
                total = fmaf(weight, shared[w * (D + 2) + D + 1], total);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    v[e] = fmaf(weight, shared[w * (D + 2) + V * lane + e], v[e]);
                }
            }
            most = now;
        }
        const float over = total == 0.f ? 0.f : 1.f / total;
        bf16_t *out = p.out + token * p.out_token + head * p.out_head;
#pragma unroll
        for (int at = 0; at < V; at += STORED) {
            if (V * lane + at < p.size) { // a multiple of 8
                bf16_t r[STORED];
#pragma unroll
                for (int e = 0; e < STORED; ++e) {
                    r[e] = (bf16_t)(v[at + e] * over);
                }
                __builtin_memcpy(out + V * lane + at, r, sizeof(r));
            }
        }
        if (p.lse != nullptr && lane == 0) {
            p.lse[index] = lse_of(most, total);
        }
    }
}

// ---- which kernels, how many workgroups ----

template <typename F>
auto by_size(int64_t size, F f)
{
    return size <= 64 ? f(std::integral_constant<int, 64>{}) : size <= 128 ? f(std::integral_constant<int, 128>{}) : f(std::integral_constant<int, 256>{});
}

struct Plan {
    bool few, prefix_few; // rows, of the sequences' tiles and of the prefix's
    int waves;            // of a workgroup
    bool shared;          // the prefix is read once for all, by workgroups of its own
    bool combined;
    int d, tile, prefix_tile; // channels in registers, rows of a tile
    int64_t most_tiles, shares, least, prefix_tiles, prefix_shares, prefix_steps, prefix_per; // of a kv head, as in the kernel's parameters
    int step_log2, prefix_step_log2;
    int64_t blocks, pieces, prefix_pieces;
    int64_t prefix_partial, partial, prefix_sums, sums, rows, bytes; // offsets in the workspace, and its size
};

// Whether the keys of the sequences' tiles are split among workgroups: pieces cost a second kernel, 4 us, and their way through memory.  8 kv heads, 4 rows a token:
// Tiles of many rows: where there are fewer of them than half of what the chip holds, and enough keys for as many; of 512 workgroups 14 keys for each tile (split and not, us: 48
// tiles of 500 keys 22 and 22, of 700 24 and 27; 72 of 700 29 and 27, of 1000 31 and 32, of 2000 38 and 53; 144 of 1000 43 and 31, of 2000 53 and 53; 120 of 6000 79 split; 450 of 4000
// 164 and 136), and more than 512 (8 of 500: 20 and 21, of 700: 19 and 24).
// Tiles of few rows: where there are fewer than four times what the chip holds, as long sequences among short ones leave the chip to a few workgroups (64 of 1 to 10000 entries:
// 242 us split, 298 not; all of 3000: 143 and 139), and more than 2048 keys (24 of 1500: 40 and 34; of 1 to 3000: 41 and 48).  With an eighth of the chip's tiles more than 1024
// (8 of 700: 14.5 and 14.1; of 1 to 1500: 14.6 and 18.5: to one CU the keys come with 45 bytes a ns).  Behind a shared prefix, where pieces are joined anyway, more than 256, unless
// there are more tiles than the chip holds (32 of 1 to 900: 35 and 37; 200 of 1 to 200: 84 and 71, of 1 to 900: 130 and 120).
template <typename S>
bool splits(int64_t tiles, int64_t keys, int64_t groups, bool shared)
{
    if (!S::FEW) {
        return 2 * tiles < groups && keys > 512 && keys * groups > 14 * 512 * tiles;
    }
    return tiles < 4 * groups && keys > (shared && tiles < groups ? 256 : tiles <= groups / 8 ? 1024 : 2048);
}

// Steps of a share of the prefix, of 64 keys or 128: fewer are more pieces to join, more are a longer wait for one (us with 2, 4, 8: 64 sequences of 1 to 200 behind 1024 entries 24.2, 20.0, 23.5;
// 2 of 1 to 300 behind 800 12.6, 13.7, 16.4; 8 of 1 to 900 behind 2000 14.9, 15.0, 18.7; 5 x 4 behind 1000, heads of 64, 14.9, 14.8, 15.2; with 1 19.8)
constexpr int64_t LEAST_PREFIX = 4;

Plan plan_of(const kutacc_hip_cached_attention_args_t &a)
{
    const kutacc_hip_cache_batch_t &b = a.batch;
    const int64_t group = a.q_heads / a.cache.kv_heads, kv_heads = a.cache.kv_heads;
    const int64_t with_tokens = std::min(b.sequences, b.tokens), average = (b.tokens * group + with_tokens - 1) / with_tokens, stacked = b.tokens * group;
    Plan p = {};
    p.few = average <= 16, p.prefix_few = stacked <= 16;
    by_size(a.cache.head_size, [&](auto d) {
        constexpr int D = decltype(d)::value;
        const int64_t groups = (D <= 128 ? 2 : 1) * (int64_t)kutacc_cu_count(); // workgroups that are on the chip at a time
        const int64_t own_tiles = std::max(stacked / (p.few ? 16 : 128), with_tokens) * kv_heads;
        // A prefix that each sequence's tiles walk by themselves needs no second kernel (short sequences, 8 kv heads, us shared and by themselves: 16 behind 512 entries 14.5 and
        // 11.9, behind 1024 15.0 and 16.5; 64 behind 256 16.7 and 13.0, behind 512 17.0 and 18.1; 248 behind 16 35 and 29, behind 256 34 and 44).  A length that is no multiple of 16,
        // which those tiles read entry by entry, moves the border by little (1 to 200 of their own: 64 behind 300 21 and 17, behind 500 19 and 21; 248 behind 33 42 and 41, behind 100 42 and
        // 46, behind 200 42 and 52).
        p.shared = b.sequences > 1 && average <= 64 && (b.prefix_length > 768 || b.prefix_length * own_tiles > 500 * groups);
        // The prefix's workgroups and the sequences' share the CUs, the ones bound by the matrix cores, the others by memory: they are best done at the same time.  Few of the prefix
        // leave room for the sequences' and have few pieces to join (64 sequences of 1 to 1000 behind 8192 entries: 256 of them 59 us, 128 53, 64 65); where those would be long, every
        // CU has one (256 behind 16384, e4m3: 256 of them 191 us, 320 209), and where the sequences' tiles are short beside them, of 128 keys at most and what each costs anyway (64 of
        // 1 to 200 behind 16000: 128 of them 61 us, 256 46, 512 53; 200 of 1 to 200 behind 3000, which is the other side: 52, 54 and 60).
        const int64_t steps = p.prefix_few ? 0 : (stacked + 127) / 128 * ((b.prefix_length + 63) / 64) * kv_heads;
        const int64_t own_steps = own_tiles * (1 + (b.columns * a.cache.page_size + 127) / 128);
        const int64_t prefix_groups = !p.shared ? 0 : steps <= 32 * (groups / 4) && 10 * steps <= 7 * own_steps ? groups / 4 : groups / 2;
        p.d = D;
        // steps of a tile's keys, and so few of them that those of all tiles are counted in 29 bits, of whole shares in 30
        const auto steps_of = [](int64_t tiles, int64_t keys, int step, int &log2) {
            for (log2 = 0; 1 << log2 < step; ++log2) {
            }
            const auto steps = [&] { return std::max<int64_t>((keys + ((int64_t)1 << log2) - 1) >> log2, 1); };
            while (log2 < 30 && tiles * steps() >= (int64_t)1 << 29) {
                ++log2;
            }
            return steps();
        };
        const auto tiles_of = [&](auto shape) {
            using S = decltype(shape);
            const int64_t keys = b.columns * a.cache.page_size + (p.shared ? 0 : b.prefix_length); // at most
            const int64_t tiles = (S::FEW ? std::max(stacked / S::ROWS, with_tokens) : std::max<int64_t>(stacked / S::ROWS, 1)) * kv_heads;
            p.tile = S::ROWS, p.waves = S::WAVES;
            p.least = S::WAVES == 8 ? 1 : 2; // of 256 keys and of 128 or 64 (8 sequences of 1 to 1500: 14.6 us, 16.0 with 2 of 256)
            p.most_tiles = stacked / S::ROWS + with_tokens;
            p.shares = splits<S>(tiles, keys, groups, p.shared) ? std::max<int64_t>(1, (groups - p.prefix_shares * kv_heads) * 4 / S::WAVES / kv_heads) : 0;
            p.blocks = (p.prefix_shares + (p.shares > 0 ? p.shares : p.most_tiles)) * kv_heads;
            (void)steps_of(p.most_tiles, keys, S::STEP, p.step_log2);
        };
        const auto prefix_of = [&](auto shape) {
            using S = decltype(shape);
            p.prefix_tile = S::ROWS;
            p.prefix_tiles = (stacked + S::ROWS - 1) / S::ROWS, p.prefix_steps = steps_of(p.prefix_tiles, b.prefix_length, S::STEP, p.prefix_step_log2);
            const int64_t all = p.prefix_tiles * p.prefix_steps, shares = std::max<int64_t>(1, prefix_groups / kv_heads);
            p.prefix_per = std::max<int64_t>((all + shares - 1) / shares, LEAST_PREFIX);
            p.prefix_shares = (all + p.prefix_per - 1) / p.prefix_per;
        };
        if (p.shared) {
            p.prefix_few ? prefix_of(FewRows<D, 4, false>{}) : prefix_of(ManyRows<D, false>{});
        }
        if (!p.few) {
            tiles_of(ManyRows<D, false>{});
        } else if (D <= 128 && !p.shared && std::max(stacked / 16, with_tokens) * kv_heads <= groups / 2) { // a workgroup a CU: of eight waves
            tiles_of(FewRows<D, D <= 128 ? 8 : 4, false>{});
        } else {
            tiles_of(FewRows<D, 4, false>{});
        }
        return 0;
    });
    p.combined = p.shared || p.shares > 0;
    p.pieces = (p.most_tiles + p.shares) * kv_heads, p.prefix_pieces = p.shared ? (p.prefix_tiles + p.prefix_shares) * kv_heads : 0;
    const auto take = [&](int64_t bytes) {
        const int64_t from = p.bytes;
        p.bytes += (bytes + 255) / 256 * 256;
        return from;
    };
    if (p.combined) {
        p.rows = take(b.tokens * a.q_heads * (int64_t)sizeof(int4));
        p.prefix_sums = take(p.prefix_pieces * p.prefix_tile * (int64_t)sizeof(float2));
        p.sums = take(p.pieces * p.tile * (int64_t)sizeof(float2));
        p.prefix_partial = take(p.prefix_pieces * p.prefix_tile * p.d * (int64_t)sizeof(float));
        p.partial = take(p.pieces * p.tile * p.d * (int64_t)sizeof(float));
    }
    return p;
}

template <typename OWN, typename PREFIX, bool PAGED_BLOCKS>
int launch_kernel(const AttentionParams &p, int64_t blocks, hipStream_t stream)
{
    constexpr int LDS = OWN::LDS > PREFIX::LDS ? OWN::LDS : PREFIX::LDS;
    const auto kernel = cached_attention_kernel<OWN, PREFIX, PAGED_BLOCKS>;
    static size_t opted[KUTACC_DEVICE_SLOTS] = {};
    if (const hipError_t e = kutacc_opt_in_lds((const void *)kernel, LDS, opted)) {
        return kutacc_hip_status(e);
    }
    kutacc_prof::KernelTimer timer("cached_attention_kernel", 0.0, stream); // how many keys there are is known on the device alone
    kernel<<<dim3((unsigned)blocks), OWN::THREADS, LDS, stream>>>(p);
    return kutacc_hip_status(hipGetLastError());
}
template <typename OWN, typename PREFIX>
int launch(const AttentionParams &p, bool paged_blocks, int64_t blocks, hipStream_t stream)
{
    return paged_blocks ? launch_kernel<OWN, PREFIX, true>(p, blocks, stream) : launch_kernel<OWN, PREFIX, false>(p, blocks, stream);
}

} // namespace

namespace kutacc_launch {

int64_t cached_attention_workspace(const kutacc_hip_cached_attention_args_t &a) { return plan_of(a).bytes; }

int cached_attention(const kutacc_hip_cached_attention_args_t &a, hipStream_t stream)
{
    const kutacc_hip_cache_t &c = a.cache;
    const kutacc_hip_cache_batch_t &b = a.batch;
    const Plan plan = plan_of(a);
    if (!kutacc_grid_fits(plan.blocks, 64 * plan.waves) || plan.pieces > INT32_MAX || plan.prefix_pieces > INT32_MAX || plan.prefix_tiles * plan.prefix_steps > INT32_MAX) {
        return KUTACC_HIP_EUNSUPPORTED;
    }
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
    p.joined = b.prefix_length > 0 && !plan.shared;
    const auto near = [](int64_t stride) { return stride < 1 << 26; }; // 16 entries within 2^30 bytes
    // Entry by entry otherwise, with a shuffle and an address for each load: prompts behind 2001 entries 299 us, behind 2000 248; 64 single tokens of 1 to 200 behind 500 21, behind 496 20; pages of
    // one entry 72, of 16 66 (64 of 100 to 2000)
    const bool paged_blocks = c.page_size % 16 == 0 && (!p.joined || b.prefix_length % 16 == 0) && near(p.k_token) && near(p.v_token);
    p.causal = a.causal, p.scale_log2 = a.scale * LOG2E;
    p.page_size = Divisor::of((uint32_t)c.page_size), p.group = Divisor::of((uint32_t)(a.q_heads / c.kv_heads));
    p.prefix_shares = (int)plan.prefix_shares, p.prefix_tiles = (int)plan.prefix_tiles, p.prefix_steps = (int)plan.prefix_steps, p.prefix_per = (int)plan.prefix_per;
    p.shares = (int)plan.shares, p.most_tiles = (int)plan.most_tiles, p.least = (int)plan.least, p.combined = plan.combined;
    p.step_log2 = plan.step_log2, p.prefix_step_log2 = plan.prefix_step_log2, p.by_share = Divisor::of((uint32_t)std::max<int64_t>(plan.shares, 1));
    p.by_prefix_step = Divisor::of((uint32_t)std::max<int64_t>(plan.prefix_steps, 1)), p.by_prefix_per = Divisor::of((uint32_t)std::max<int64_t>(plan.prefix_per, 1));
    char *workspace = (char *)a.workspace;
    if (plan.combined) {
        p.rows = (int4 *)(workspace + plan.rows), p.sums = (float2 *)(workspace + plan.sums), p.partial = (float *)(workspace + plan.partial);
        if (plan.shared) {
            p.prefix_sums = (float2 *)(workspace + plan.prefix_sums), p.prefix_partial = (float *)(workspace + plan.prefix_partial);
        }
    }
    const int rc = by_size(c.head_size, [&](auto d) {
        constexpr int D = decltype(d)::value;
        const auto of_type = [&](auto fp8) {
            using Few = FewRows<D, 4, decltype(fp8)::value>;
            using Wide = FewRows<D, D <= 128 ? 8 : 4, decltype(fp8)::value>;
            using Many = ManyRows<D, decltype(fp8)::value>;
            return !plan.few                           ? launch<Many, Many>(p, paged_blocks, plan.blocks, stream)
                   : plan.shared && !plan.prefix_few ? launch<Few, Many>(p, paged_blocks, plan.blocks, stream)
                   : plan.waves == 8                 ? launch<Wide, Wide>(p, paged_blocks, plan.blocks, stream)
                                                     : launch<Few, Few>(p, paged_blocks, plan.blocks, stream);
        };
        return c.dtype == KUTACC_DTYPE_E4M3 ? of_type(std::true_type{}) : of_type(std::false_type{});
    });
    if (rc != 0 || !plan.combined) {
        return rc;
    }
    const CombineParams join = {p.prefix_partial, p.partial, p.prefix_sums, p.sums, p.rows, p.prefix_shares, p.prefix_tiles, p.prefix_steps, p.prefix_per, plan.prefix_tile,
                                plan.tile, (int)plan.pieces, p.tokens, p.heads, p.size, p.sequences, p.group, p.by_prefix_per, p.query_starts, p.out, p.out_token, p.out_head, p.lse};
    const int64_t rows = b.tokens * a.q_heads;
    const bool side_by_side = rows <= 4 * kutacc_cu_count(); // four waves a row
    const dim3 grid((unsigned)std::min<int64_t>(side_by_side ? rows : (rows + 15) / 16, 1 << 20));
    kutacc_prof::KernelTimer timer("combine_kernel", 0.0, stream); // nor how many pieces
    return by_size(c.head_size, [&](auto d) {
        if (side_by_side) {
            combine_kernel<decltype(d)::value, 4, 1><<<grid, 256, 0, stream>>>(join);
        } else {
            combine_kernel<decltype(d)::value, 1, 4><<<grid, 256, 0, stream>>>(join);
        }
        return kutacc_hip_status(hipGetLastError());
    });
}

} // namespace kutacc_launch
