// extern "C" layer of the attention half of a transformer block: rotary positions, the cache of keys and values in pages, and the attention that reads
// it.  None of them has a counterpart in the reference.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>

#include "api_internal.h"
#include "kutacc_hip.h"
#include "launch_internal.h"

namespace {
constexpr int64_t MAX_INDEX = INT32_MAX / 2; // extents that the kernels count in 32 bits
constexpr int64_t MAX_HEAD = 256;            // of a cache
constexpr int32_t MAX_ROTATED = 512;
constexpr int64_t MAX_STRIDE = INT64_MAX / 4 / MAX_INDEX; // so that no offset passes 64 bits

bool extent(int64_t v) { return v > 0 && v <= MAX_INDEX; }
bool stride(int64_t v) { return v >= 0 && v <= MAX_STRIDE; }
bool readable(const kutacc_hip_heads_t &x) { return x.data != nullptr && stride(x.token_stride) && stride(x.head_stride); }
// `inner` rows of `size` elements within each of `outer`
bool nested(int64_t outer, int64_t outer_stride, int64_t inner, int64_t inner_stride, int64_t size)
{
    return (inner == 1 || inner_stride >= size) && (outer == 1 || outer_stride >= (inner - 1) * inner_stride + size);
}
bool writable(const kutacc_hip_heads_t &x, int64_t tokens, int64_t heads, int64_t size)
{
    return readable(x) && (nested(tokens, x.token_stride, heads, x.head_stride, size) || nested(heads, x.head_stride, tokens, x.token_stride, size));
}
// from x into out, or within x
bool mapped(const kutacc_hip_heads_t &x, const kutacc_hip_heads_t &out, int64_t tokens, int64_t heads, int64_t size)
{
    return extent(heads) && readable(x) && writable(out, tokens, heads, size) &&
           (x.data != out.data || ((tokens == 1 || x.token_stride == out.token_stride) && (heads == 1 || x.head_stride == out.head_stride)));
}
bool rotation_of(const kutacc_hip_rotation_t &r, int64_t head_size)
{
    return r.rotated >= 0 && r.rotated <= MAX_ROTATED && r.rotated % 2 == 0 && r.first >= 0 && (int64_t)r.first + r.rotated <= head_size &&
           (r.rotated == 0 || (r.inv_freq != nullptr && std::isfinite(r.magnitude)));
}

bool sizes_of(const kutacc_hip_cache_t &c, const kutacc_hip_cache_batch_t &b)
{
    return extent(c.pages) && extent(c.page_size) && c.pages <= MAX_INDEX / c.page_size && extent(c.kv_heads) && extent(c.head_size) &&
           (c.dtype == KUTACC_DTYPE_BF16 || c.dtype == KUTACC_DTYPE_E4M3) && b.sequences >= 0 && b.sequences <= MAX_INDEX && b.tokens >= 0 && b.tokens <= MAX_INDEX &&
           b.columns >= 0 && b.columns <= MAX_INDEX / c.page_size && b.prefix_length >= 0 && b.prefix_length <= MAX_INDEX - b.columns * c.page_size;
}
bool batch_of(const kutacc_hip_cache_batch_t &b)
{
    return b.query_starts != nullptr && b.lengths != nullptr && (b.columns == 0 || b.page_table != nullptr) && (b.sequences == 1 || b.page_table_ld >= b.columns) &&
           b.page_table_ld <= MAX_INDEX && (b.prefix_length == 0 || b.prefix_pages != nullptr);
}
// pages, slots and heads in any order of nesting, each apart from the next
bool entries_apart(const kutacc_hip_cache_t &c, int64_t page, int64_t token, int64_t head)
{
    if (!stride(page) || !stride(token) || !stride(head)) {
        return false;
    }
    int64_t count[3] = {c.pages, c.page_size, c.kv_heads}, step[3] = {page, token, head};
    for (int i = 0; i < 2; ++i) { // by stride
        for (int j = 0; j < 2 - i; ++j) {
            if (step[j] > step[j + 1]) {
                const int64_t s = step[j], n = count[j];
                step[j] = step[j + 1], count[j] = count[j + 1], step[j + 1] = s, count[j + 1] = n;
            }
        }
    }
    int64_t reach = c.head_size;
    for (int i = 0; i < 3; ++i) {
        if (count[i] > 1) {
            if (step[i] < reach) {
                return false;
            }
            reach += (count[i] - 1) * step[i];
        }
    }
    return true;
}
bool cache_of(const kutacc_hip_cache_t &c)
{
    const bool scaled = c.dtype == KUTACC_DTYPE_E4M3;
    return c.k != nullptr && c.v != nullptr && (c.k_scales != nullptr) == scaled && (c.v_scales != nullptr) == scaled &&
           entries_apart(c, c.k_page_stride, c.k_token_stride, c.k_head_stride) && entries_apart(c, c.v_page_stride, c.v_token_stride, c.v_head_stride);
}
// what the kernels read and write in pieces of 16 bytes
bool cache_in_pieces(const kutacc_hip_cache_t &c)
{
    const int64_t piece = c.dtype == KUTACC_DTYPE_E4M3 ? 16 : 8;
    const auto whole = [&](int64_t step, int64_t count) { return count == 1 || step % piece == 0; };
    return c.head_size % piece == 0 && c.head_size <= MAX_HEAD && kutacc_hip_aligned16(c.k) && kutacc_hip_aligned16(c.v) && whole(c.k_page_stride, c.pages) &&
           whole(c.k_token_stride, c.page_size) && whole(c.k_head_stride, c.kv_heads) && whole(c.v_page_stride, c.pages) && whole(c.v_token_stride, c.page_size) &&
           whole(c.v_head_stride, c.kv_heads);
}
bool attention_sizes(const kutacc_hip_cached_attention_args_t &a)
{
    return sizes_of(a.cache, a.batch) && extent(a.q_heads) && a.q_heads % a.cache.kv_heads == 0 && (a.batch.tokens == 0 || a.q_heads <= MAX_INDEX / a.batch.tokens);
}
} // namespace

extern "C" {

int kutacc_hip_rotary_frequencies(float *inv_freq, int32_t rotated, int32_t scaling, double base, double factor, double original_length, double fast, double slow)
{
    const bool mixed = scaling == KUTACC_HIP_ROTARY_BY_PAIRS || scaling == KUTACC_HIP_ROTARY_BY_TURNS;
    if (inv_freq == nullptr || rotated <= 0 || rotated % 2 != 0 || rotated > MAX_ROTATED || scaling < KUTACC_HIP_ROTARY_PLAIN || scaling > KUTACC_HIP_ROTARY_BY_TURNS || !(base > 1.0) ||
        !std::isfinite(base) || !(factor >= 1.0) || !std::isfinite(factor) ||
        (mixed && (!(original_length > 0.0) || !std::isfinite(original_length) || !(slow > 0.0) || !(fast > slow) || !std::isfinite(fast))) ||
        (scaling == KUTACC_HIP_ROTARY_BASE && rotated == 2)) {
        return KUTACC_HIP_EINVAL;
    }
    const double two_pi = 6.283185307179586476925286766559;
    if (scaling == KUTACC_HIP_ROTARY_BASE) {
        base *= std::pow(factor, (double)rotated / (rotated - 2));
    }
    // the pair, no whole number, that turns `turns` times over the original length
    const auto pair_of = [&](double turns) { return rotated * std::log(original_length / (turns * two_pi)) / (2.0 * std::log(base)); };
    for (int j = 0; j < rotated / 2; ++j) {
        double f = std::pow(base, -2.0 * j / rotated);
        double stretched = scaling == KUTACC_HIP_ROTARY_LINEAR ? 1.0 : 0.0; // the share of f / factor
        if (scaling == KUTACC_HIP_ROTARY_BY_PAIRS) {
            const double from = std::fmax(std::floor(pair_of(fast)), 0.0), to = std::fmin(std::ceil(pair_of(slow)), rotated - 1.0);
            stretched = from < to ? (j - from) / (to - from) : j >= pair_of(slow) ? 1.0 : 0.0; // to <= 0: all pairs are slow; from >= rotated - 1: all are fast
        } else if (scaling == KUTACC_HIP_ROTARY_BY_TURNS) {
            stretched = (fast - original_length * f / two_pi) / (fast - slow);
        }
        stretched = std::fmin(std::fmax(stretched, 0.0), 1.0);
        inv_freq[j] = (float)(f / factor * stretched + f * (1.0 - stretched));
    }
    return 0;
}

int kutacc_hip_rotary(const kutacc_hip_rotary_args_t *args, void *stream)
{
    if (args == nullptr) {
        return KUTACC_HIP_EINVAL;
    }
    const kutacc_hip_rotary_args_t &a = *args;
    if (a.tokens < 0 || a.tokens > MAX_INDEX || !extent(a.head_size) || (a.dtype != KUTACC_DTYPE_BF16 && a.dtype != KUTACC_DTYPE_FP32) || !rotation_of(a.rotation, a.head_size)) {
        return KUTACC_HIP_EINVAL;
    }
    if (a.tokens == 0) { // tensors of no element may have no address
        return 0;
    }
    if ((a.q.data == nullptr && a.k.data == nullptr) || (a.q.data != nullptr && !mapped(a.q, a.q_out, a.tokens, a.q_heads, a.head_size)) || (a.k.data != nullptr && !mapped(a.k, a.k_out, a.tokens, a.k_heads, a.head_size))) {
        return KUTACC_HIP_EINVAL;
    }
    return kutacc_launch::rotary(a, kutacc_api::stream_or_default(stream));
}

int kutacc_hip_cache_append(const kutacc_hip_cache_append_args_t *args, void *stream)
{
    if (args == nullptr) {
        return KUTACC_HIP_EINVAL;
    }
    const kutacc_hip_cache_append_args_t &a = *args;
    if (!sizes_of(a.cache, a.batch) || !rotation_of(a.rotation, a.cache.head_size)) {
        return KUTACC_HIP_EINVAL;
    }
    if (a.batch.tokens == 0 || a.batch.sequences == 0) {
        return 0;
    }
    if (!batch_of(a.batch) || !cache_of(a.cache) || !readable(a.k) || !readable(a.v) || (a.q.data != nullptr && !mapped(a.q, a.q_out, a.batch.tokens, a.q_heads, a.cache.head_size))) {
        return KUTACC_HIP_EINVAL;
    }
    if (!cache_in_pieces(a.cache)) {
        return KUTACC_HIP_EUNSUPPORTED;
    }
    return kutacc_launch::cache_append(a, kutacc_api::stream_or_default(stream));
}

int64_t kutacc_hip_cached_attention_workspace(const kutacc_hip_cached_attention_args_t *args)
{
    if (args == nullptr || !attention_sizes(*args)) {
        return KUTACC_HIP_EINVAL;
    }
    return args->batch.tokens == 0 || args->batch.sequences == 0 || args->cache.head_size > MAX_HEAD ? 0 : kutacc_launch::cached_attention_workspace(*args);
}

int kutacc_hip_cached_attention(const kutacc_hip_cached_attention_args_t *args, void *stream)
{
    if (args == nullptr) {
        return KUTACC_HIP_EINVAL;
    }
    const kutacc_hip_cached_attention_args_t &a = *args;
    if (!attention_sizes(a) || !(a.scale > 0.f) || !std::isfinite(a.scale) || (a.causal != 0 && a.causal != 1)) {
        return KUTACC_HIP_EINVAL;
    }
    if (a.batch.tokens == 0 || a.batch.sequences == 0) {
        return 0;
    }
    if (!batch_of(a.batch) || !cache_of(a.cache) || !mapped(a.q, a.out, a.batch.tokens, a.q_heads, a.cache.head_size)) {
        return KUTACC_HIP_EINVAL;
    }
    if (!cache_in_pieces(a.cache)) {
        return KUTACC_HIP_EUNSUPPORTED;
    }
    const int64_t needed = kutacc_launch::cached_attention_workspace(a);
    if (needed > 0 && (a.workspace == nullptr || a.workspace_bytes < needed || (reinterpret_cast<uintptr_t>(a.workspace) & 255u) != 0)) {
        return KUTACC_HIP_EINVAL;
    }
    return kutacc_launch::cached_attention(a, kutacc_api::stream_or_default(stream));
}

} // extern "C"
