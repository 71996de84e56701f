// Rotary positions, by themselves and on the way of new keys into a cache in pages.
//
//   a' = m (a cos(t f_j) - b sin(t f_j)),  b' = m (b cos(t f_j) + a sin(t f_j))
//
// Memory bounds both: a value is read once and written once.  The sines and cosines of a token are the same for all of its heads: a workgroup takes a few tokens (one, with
// few of them in the call), forms theirs once into the LDS, m included, and turns 2 V channels of a head a thread.  The angle is formed in turns in 64 bits -- at a
// position of 10^6 a 32-bit product is off by 0.06 radians -- and its whole turns are dropped there.
//
// 8191 tokens of 40 heads of 128 in bf16: 38.9 us, 4.32 TB/s (a large copy: 4.9); prompts of 9800 tokens into a cache: 48.9 us, 4.1 TB/s.  16 tokens: 4.2 us, as a kernel that does
// nothing.  Tried and not kept: the next two pieces loaded ahead of the turns and of the ones at hand (38.4 us, but 14.1 in place of 11.9 for 3000 tokens into 8 bits: the
// workgroups of a CU cover one another's waits as well, and more of them fit).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "launch_internal.h"
#include "paged_cache.h"
#include "profiler.h"
#include "row_chunks.h"

namespace {
using namespace kutacc_dev;

constexpr int THREADS = 256;
constexpr int MOST_TOKENS = 8; // of a workgroup
constexpr int MOST_GROUPS = 1 << 16; // of a launch, which then go on to the next tokens
constexpr double TURN = 0.15915494309189533576888376337251;

struct HeadsIn {
    const void *data;
    int64_t token_stride, head_stride;
};
struct HeadsOut {
    void *data;
    int64_t token_stride, head_stride;
};

struct RotaryParams {
    HeadsIn q, k, v;
    HeadsOut q_out, k_out;
    const int32_t *positions;
    const float *inv_freq;
    int tokens, q_heads, k_heads, v_heads; // v_heads: of a cache, else 0
    int size, rotated, first, per_group;   // per_group: tokens of a workgroup
    float magnitude, sign;
    Divisor per_token, per_head, per_value;  // items of a token, of a turned head and of one of values
    // a cache
    uint8_t *k_cache, *v_cache;
    int64_t k_page, k_token, k_head, v_page, v_token, v_head; // strides
    const float *k_scales, *v_scales;
    const int32_t *query_starts, *lengths, *page_table;
    int64_t page_table_ld;
    int sequences, columns, pages, prefix_length;
    Divisor page_size;
};

constexpr int NOWHERE = -1, PADDING = -2; // in the place of a page: a token that is not kept, one that is nobody's

template <int V, typename T>
__device__ __forceinline__ void load(float (&x)[V], const T *from)
{
    T raw[V];
    __builtin_memcpy(raw, from, sizeof(raw));
#pragma unroll
    for (int e = 0; e < V; ++e) {
        x[e] = to_f32(raw[e]);
    }
}
template <int V, typename T>
__device__ __forceinline__ void store(T *to, const float (&x)[V])
{
    T raw[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        raw[e] = from_f32<T>(x[e]);
    }
    __builtin_memcpy(to, raw, sizeof(raw));
}

// Quotients by one scale: x times the rounded 1 / scale, put right by what is left over, is x / scale as rounded (Markstein 1990), in fewer instructions
// (3000 tokens of 12 heads of 64: 10.7 us, 11.9 with divisions).  Not for scales whose quotients or rests leave the range, and not from where they are saturated on, infinities
// among them.
struct Over {
    float scale, inverse;
    bool plain;
    __device__ __forceinline__ explicit Over(float s) : scale(s), inverse(1.f / s), plain(!(s >= 0x1p-60f && s <= 0x1p60f)) {}
    template <bool PLAIN>
    __device__ __forceinline__ float quotient(float x) const
    {
        if (PLAIN) {
            return x / scale;
        }
        const float q = x * inverse, better = copysignf(fmaf(fmaf(-q, scale, x), inverse, q), x); // of -0, too
        return fabsf(q) < 2.f * FP8_LARGEST ? better : q;
    }
};
// as the cache in 8 bits holds them: saturated (a NaN stays one)
template <bool PLAIN, int V>
__device__ __forceinline__ void store_fp8(uint8_t *to, const float (&x)[V], const Over &over)
{
    uint8_t raw[V < 4 ? 4 : V];
#pragma unroll
    for (int e = 0; e < V; e += 4) {
        float q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            q[i] = e + i < V ? __builtin_elementwise_maximum(__builtin_elementwise_minimum(over.quotient<PLAIN>(x[e + i]), FP8_LARGEST), -FP8_LARGEST) : 0.f;
        }
        int word = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
        word = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], word, true);
        __builtin_memcpy(raw + e, &word, 4);
    }
    __builtin_memcpy(to, raw, V);
}

// T: of the inputs and of q_out; CACHE: of what keys and values go into (uint8_t: e4m3), void: k_out.  An item is two pieces of V channels: V pairs,
// or two pieces that are copied.
template <typename T, typename CACHE, int V, bool INTERLEAVED>
__global__ __launch_bounds__(THREADS) void rotary_kernel(const RotaryParams p)
{
    constexpr bool CACHED = !std::is_same_v<CACHE, void>, FP8 = std::is_same_v<CACHE, uint8_t>;
    extern __shared__ float2 turns[]; // [per_group][rotated / 2]
    __shared__ int place_page[MOST_TOKENS], place_slot[MOST_TOKENS];
    __shared__ int64_t place_position[MOST_TOKENS]; // a length may be such that they pass 32 bits
    const int tid = (int)threadIdx.x, pairs = p.rotated / 2;
    for (int token0 = (int)blockIdx.x * p.per_group; token0 < p.tokens; token0 += (int)gridDim.x * p.per_group) {
        const int count = min(p.per_group, p.tokens - token0);
        __syncthreads(); // the last tokens' turns and places have been read
        if (CACHED) {
            if (tid < MOST_TOKENS) {
                place_page[tid] = PADDING, place_position[tid] = 0, place_slot[tid] = 0;
            }
            __syncthreads();
            for (int s = tid; s < p.sequences; s += THREADS) {
                const TokenRange r = tokens_of(p.query_starts, s, p.tokens);
                const int from = max(r.first, token0), to = min(r.end, token0 + count);
                if (from < to) {
                    const int64_t at0 = (int64_t)max(p.lengths[s], 0) - (r.end - r.first) - r.first; // of token 0, among the sequence's own entries
                    for (int t = from; t < to; ++t) {
                        const int64_t at = at0 + t;
                        int page = NOWHERE, slot = 0;
                        if (at >= 0 && at < (int64_t)p.columns * p.page_size.d) {
                            const uint32_t column = p.page_size.quotient((uint32_t)at);
                            slot = (int)((uint32_t)at - column * p.page_size.d);
                            page = p.page_table[s * p.page_table_ld + column];
                            page = (uint32_t)page < (uint32_t)p.pages ? page : NOWHERE;
                        }
                        place_page[t - token0] = page, place_slot[t - token0] = slot;
                        place_position[t - token0] = p.prefix_length + at;
                    }
                }
            }
            __syncthreads();
        }
        for (int i = tid; i < count * pairs; i += THREADS) {
            const int t = i / pairs, j = i - t * pairs;
            const int64_t position = p.positions != nullptr ? p.positions[token0 + t] : CACHED ? place_position[t] : token0 + t;
            double angle = (double)position * (double)p.inv_freq[j] * TURN;
            angle -= rint(angle);
            float s, c;
            sincospif((float)(2.0 * angle), &s, &c);
            turns[i] = make_float2(c * p.magnitude, s * p.magnitude * p.sign);
        }
        __syncthreads();

        const int turned = p.q_heads + p.k_heads;
        const uint32_t items = p.per_token.d * (uint32_t)count;
        for (uint32_t i = (uint32_t)blockIdx.y * THREADS + (uint32_t)tid; i < items; i += gridDim.y * THREADS) {
            const uint32_t t = p.per_token.quotient(i), in_token = i - t * p.per_token.d;
            const int token = token0 + (int)t;
            const int page = CACHED ? place_page[t] : 0;
            if (CACHED && page == PADDING) {
                continue;
            }
            const bool value = CACHED && in_token >= (uint32_t)turned * p.per_head.d;
            const uint32_t of = value ? in_token - (uint32_t)turned * p.per_head.d : in_token;
            int head = (int)(value ? p.per_value : p.per_head).quotient(of);
            const int piece = (int)(of - (uint32_t)head * (value ? p.per_value : p.per_head).d);
            const bool key = !value && head >= p.q_heads;
            if (CACHED && (key || value) && page == NOWHERE) {
                continue;
            }
            head -= key ? p.q_heads : 0;
            const HeadsIn in = value ? p.v : key ? p.k : p.q;
            const T *from = (const T *)in.data + token * in.token_stride + head * in.head_stride;

            const bool pair = !value && piece * V < pairs;
            int at_a, at_b; // channels of the pieces
            if (pair) {
                at_a = p.first + (INTERLEAVED ? 2 * V * piece : V * piece), at_b = INTERLEAVED ? at_a + V : at_a + pairs;
            } else { // the channels beside the turned ones, in order
                at_a = value ? 2 * V * piece : 2 * (V * piece - pairs);
                at_b = at_a + V;
                at_a += !value && at_a >= p.first ? p.rotated : 0, at_b += !value && at_b >= p.first ? p.rotated : 0;
            }
            const bool two = at_b < p.size;
            float a[V], b[V];
            load<V>(a, from + at_a);
            load<V>(b, from + (two ? at_b : at_a));
            if (pair) {
                const float2 *turn = turns + t * pairs + piece * V;
                if (INTERLEAVED) {
                    if (V == 1) {
                        const float x = a[0], y = b[0];
                        a[0] = fmaf(x, turn[0].x, -(y * turn[0].y)), b[0] = fmaf(y, turn[0].x, x * turn[0].y);
                    } else {
#pragma unroll
                        for (int e = 0; e < V; e += 2) {
                            const float x = a[e], y = a[e + (V > 1)], z = b[e], w = b[e + (V > 1)];
                            const float2 u = turn[e / 2], v = turn[(V + e) / 2];
                            a[e] = fmaf(x, u.x, -(y * u.y)), a[e + (V > 1)] = fmaf(y, u.x, x * u.y);
                            b[e] = fmaf(z, v.x, -(w * v.y)), b[e + (V > 1)] = fmaf(w, v.x, z * v.y);
                        }
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float x = a[e], y = b[e];
                        a[e] = fmaf(x, turn[e].x, -(y * turn[e].y)), b[e] = fmaf(y, turn[e].x, x * turn[e].y);
                    }
                }
            }
            if (CACHED && (key || value)) {
                using C = std::conditional_t<FP8, uint8_t, T>;
                const int64_t at = value ? page * p.v_page + place_slot[t] * p.v_token + head * p.v_head : page * p.k_page + place_slot[t] * p.k_token + head * p.k_head;
                C *to = (C *)(value ? p.v_cache : p.k_cache) + at;
                if constexpr (FP8) {
                    const Over over((value ? p.v_scales : p.k_scales)[head]);
                    const auto both = [&](auto plain) {
                        store_fp8<decltype(plain)::value>(to + at_a, a, over);
                        if (two) {
                            store_fp8<decltype(plain)::value>(to + at_b, b, over);
                        }
                    };
                    over.plain ? both(std::true_type{}) : both(std::false_type{});
                } else {
                    store<V>(to + at_a, a);
                    if (two) {
                        store<V>(to + at_b, b);
                    }
                }
            } else {
                const HeadsOut out = key ? p.k_out : p.q_out;
                T *to = (T *)out.data + token * out.token_stride + head * out.head_stride;
                store<V>(to + at_a, a);
                if (two) {
                    store<V>(to + at_b, b);
                }
            }
        }
    }
}

HeadsIn in_of(const kutacc_hip_heads_t &x) { return {x.data, x.token_stride, x.head_stride}; }
HeadsOut out_of(const kutacc_hip_heads_t &x) { return {x.data, x.token_stride, x.head_stride}; }

// Channels of a piece: the turned channels and the others have to be whole pieces, and the halves of the turned ones.
int piece_of(int64_t size, const kutacc_hip_rotation_t &r)
{
    for (const int v : {8, 4}) {
        const int turned = r.interleaved ? 2 * v : v; // a half has to be whole pieces, or the pairs of two pieces
        if (size % v == 0 && r.first % v == 0 && (r.interleaved ? r.rotated : r.rotated / 2) % turned == 0) {
            return v;
        }
    }
    return 1;
}

template <typename T, typename CACHE>
int launch(RotaryParams &p, const kutacc_hip_rotation_t &r, hipStream_t stream)
{
    p.inv_freq = r.inv_freq, p.rotated = r.rotated, p.first = r.first, p.magnitude = r.magnitude, p.sign = r.inverse ? -1.f : 1.f;
    const int v = piece_of(p.size, r), pairs = p.rotated / 2;
    const int per_head = pairs / v + (p.size - p.rotated + 2 * v - 1) / (2 * v), per_value = (p.size + 2 * v - 1) / (2 * v);
    const int64_t per_token = (int64_t)(p.q_heads + p.k_heads) * per_head + (int64_t)p.v_heads * per_value;
    if (per_token * MOST_TOKENS > INT32_MAX) {
        return KUTACC_HIP_EUNSUPPORTED;
    }
    p.per_token = Divisor::of((uint32_t)per_token), p.per_head = Divisor::of((uint32_t)per_head), p.per_value = Divisor::of((uint32_t)per_value);
    const int cus = kutacc_cu_count();
    // four workgroups for each CU, before each gets more tokens: 3000 tokens of 12 heads of 64 11.8 us, with two 13.7, with eight 13.4; 2000 of 40 of 128 9.0, 9.6 and 9.0
    p.per_group = (int)std::min<int64_t>(MOST_TOKENS, std::max<int64_t>(1, p.tokens / (4 * cus)));
    const int64_t groups = (p.tokens + p.per_group - 1) / p.per_group;
    const int64_t parts = std::max<int64_t>(1, std::min((per_token * p.per_group + THREADS - 1) / THREADS, 4 * cus / groups));
    kutacc_prof::KernelTimer timer("rotary_kernel", 3.0 * (double)p.tokens * (p.q_heads + p.k_heads) * p.rotated, stream);
    const dim3 grid((unsigned)std::min<int64_t>(groups, MOST_GROUPS), (unsigned)parts);
    const size_t lds = (size_t)p.per_group * pairs * sizeof(float2);
    const auto go = [&](auto piece) {
        constexpr int V = decltype(piece)::value;
        if (r.interleaved) {
            rotary_kernel<T, CACHE, V, true><<<grid, THREADS, lds, stream>>>(p);
        } else {
            rotary_kernel<T, CACHE, V, false><<<grid, THREADS, lds, stream>>>(p);
        }
        return kutacc_hip_status(hipGetLastError());
    };
    return v == 8 ? go(std::integral_constant<int, 8>{}) : v == 4 ? go(std::integral_constant<int, 4>{}) : go(std::integral_constant<int, 1>{});
}

} // namespace

namespace kutacc_launch {

int rotary(const kutacc_hip_rotary_args_t &a, hipStream_t stream)
{
    RotaryParams p = {};
    p.q = in_of(a.q), p.q_out = out_of(a.q_out), p.q_heads = a.q.data != nullptr ? (int)a.q_heads : 0;
    p.k = in_of(a.k), p.k_out = out_of(a.k_out), p.k_heads = a.k.data != nullptr ? (int)a.k_heads : 0;
    p.positions = a.positions, p.tokens = (int)a.tokens, p.size = (int)a.head_size;
    return a.dtype == KUTACC_DTYPE_BF16 ? launch<bf16_t, void>(p, a.rotation, stream) : launch<float, void>(p, a.rotation, stream);
}

int cache_append(const kutacc_hip_cache_append_args_t &a, hipStream_t stream)
{
    const kutacc_hip_cache_t &c = a.cache;
    const kutacc_hip_cache_batch_t &b = a.batch;
    RotaryParams p = {};
    p.q = in_of(a.q), p.q_out = out_of(a.q_out), p.q_heads = a.q.data != nullptr ? (int)a.q_heads : 0;
    p.k = in_of(a.k), p.v = in_of(a.v), p.k_heads = p.v_heads = (int)c.kv_heads;
    p.positions = a.positions, p.tokens = (int)b.tokens, p.size = (int)c.head_size;
    p.k_cache = (uint8_t *)c.k, p.k_page = c.k_page_stride, p.k_token = c.k_token_stride, p.k_head = c.k_head_stride;
    p.v_cache = (uint8_t *)c.v, p.v_page = c.v_page_stride, p.v_token = c.v_token_stride, p.v_head = c.v_head_stride;
    p.k_scales = c.k_scales, p.v_scales = c.v_scales;
    p.query_starts = b.query_starts, p.lengths = b.lengths, p.page_table = b.page_table, p.page_table_ld = b.page_table_ld;
    p.sequences = (int)b.sequences, p.columns = (int)b.columns, p.pages = (int)c.pages, p.prefix_length = (int)b.prefix_length;
    p.page_size = Divisor::of((uint32_t)c.page_size);
    return c.dtype == KUTACC_DTYPE_BF16 ? launch<bf16_t, bf16_t>(p, a.rotation, stream) : launch<bf16_t, uint8_t>(p, a.rotation, stream);
}

} // namespace kutacc_launch
