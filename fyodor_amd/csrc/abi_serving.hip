// extern "C" entry points of libfyodor_hip.so declared in include/fyodor_hip_serving.h.
#include "serving_checks.h"

namespace {

bool cache_ok(const nya_hip_kv8 *c)
{
    return geometry_ok(c) && c->keys && c->values && !((c->keys | c->values) & 15u) && vec(c->key_scales) &&
           vec(c->value_scales);
}

Kv8 cache_of(const nya_hip_kv8 *c)
{
    return {(int8_t *)c->keys, (int8_t *)c->values, (float *)c->key_scales, (float *)c->value_scales, (int)c->pages,
            (int)c->page_tokens, (int)c->kv_heads, (int)c->width};
}

}  // namespace

extern "C" {

NYA_HIP_EXPORT int nya_hip_page_step(uintptr_t lengths, uintptr_t counts, size_t requests, size_t page_tokens,
    uintptr_t table, size_t table_stride, uintptr_t held, uintptr_t free_pages, size_t pages, uintptr_t free_count,
    uintptr_t starts, uintptr_t positions, uintptr_t slots, size_t max_tokens, uintptr_t stream)
{
    if (!vec(lengths) || !vec(counts) || !vec(table) || !vec(held) || !vec(free_pages) || !vec(free_count) ||
        !vec(starts) || !vec(positions) || !vec(slots) || !requests || requests > 65536 || !page_ok(page_tokens) ||
        !some(table_stride) || table_stride > (size_t)INT_MAX / requests ||
        table_stride > (size_t)INT_MAX / page_tokens || !some(pages) || pages > (size_t)INT_MAX / page_tokens ||
        !rows_fit(max_tokens))
        return 1;
    return status(launch_page_step({(const int *)lengths, (const int *)counts, (int)requests, (int)page_tokens,
                                    (int *)table, (int)table_stride, (int *)held, (int *)free_pages, (int)pages,
                                    (int *)free_count, (int *)starts, (int *)positions, (int *)slots,
                                    (int)max_tokens}, (hipStream_t)stream));
}

NYA_HIP_EXPORT int nya_hip_rope_frequencies(float *out, size_t rotated, double base, const float *factors,
    unsigned scaling, double factor, double original, double low, double high, float *magnitude)
{
    if (!out || !magnitude || !rotated || rotated % 2 || rotated > (size_t)INT_MAX || !(base > 1) || !isfinite(base) ||
        scaling > NYA_HIP_ROPE_RAMP)
        return 1;
    const bool bands = scaling == NYA_HIP_ROPE_BANDS || scaling == NYA_HIP_ROPE_RAMP;
    if (scaling != NYA_HIP_ROPE_NONE && (!(factor >= 1) || !isfinite(factor))) return 1;
    if (bands && (!(original > 0) || !isfinite(original) || !(low >= 0) || !(high > low) || !isfinite(high))) return 1;
    if (scaling == NYA_HIP_ROPE_RAMP && !(low > 0)) return 1;
    for (size_t j = 0; factors && j < rotated / 2; ++j)
        if (!isfinite(factors[j]) || factors[j] == 0) return 1;
    const double turn = 2 * M_PI, r = (double)rotated;
    // The pair that turns n times within `original` positions: base^(-2j/r) original / 2 pi = n.
    const auto pair_of = [&](double n) { return r * log(original / (turn * n)) / (2 * log(base)); };
    double from = 0, to = 0;
    if (scaling == NYA_HIP_ROPE_RAMP) {
        from = fmin(fmax(floor(pair_of(high)), 0), r - 1);
        to = fmin(fmax(ceil(pair_of(low)), 0), r - 1);
    }
    for (size_t j = 0; j < rotated / 2; ++j) {
        double f = pow(base, -2 * (double)j / r);
        if (factors) f /= (double)factors[j];
        double keep = scaling == NYA_HIP_ROPE_NONE ? 1 : 0;
        if (scaling == NYA_HIP_ROPE_BANDS) keep = (original * f / turn - low) / (high - low);
        if (scaling == NYA_HIP_ROPE_RAMP) keep = 1 - ((double)j - from) / fmax(to - from, 1e-3);
        keep = fmin(fmax(keep, 0), 1);
        out[j] = (float)(keep == 1 ? f : keep * f + (1 - keep) * f / factor);
    }
    *magnitude = scaling == NYA_HIP_ROPE_RAMP ? (float)(1 + 0.1 * log(factor)) : 1.f;
    return 0;
}

NYA_HIP_EXPORT int nya_hip_rope_angles(uintptr_t positions, size_t count, uintptr_t frequencies, size_t rotated,
    float magnitude, uintptr_t angles, uintptr_t stream)
{
    if (!vec(positions) || !vec(frequencies) || !angles || (angles & 7u) || !rows_fit(count) || !rotated ||
        rotated % 2 || rotated > 1024 || !isfinite(magnitude))
        return 1;
    return status(launch_rope_angles((const int *)positions, (int)count, (const float *)frequencies,
                                     (int)(rotated / 2), magnitude, (float2 *)angles, (hipStream_t)stream));
}

NYA_HIP_EXPORT int nya_hip_rope(uintptr_t q, size_t q_stride, uintptr_t q_out, size_t q_out_stride, size_t heads,
    uintptr_t k, size_t k_stride, uintptr_t k_out, size_t k_out_stride, size_t kv_heads, size_t width, size_t count,
    uintptr_t angles, size_t rotated, unsigned layout, uintptr_t stream)
{
    if (!rows_fit(count) || !heads_ok(heads, width) || !rows_ok(q, q_stride, q_out, q_out_stride, heads * width, count) ||
        !rotation_ok(angles, rotated, width, layout))
        return 1;
    // No row that is written is another's input or output.
    const size_t n = heads * width, kn = kv_heads * width;
    if (k && (!heads_ok(kv_heads, width) || !rows_ok(k, k_stride, k_out, k_out_stride, kn, count) ||
              !apart(q_out, q_out_stride, n, k, k_stride, kn, count) ||
              !apart(q_out, q_out_stride, n, k_out, k_out_stride, kn, count) ||
              !apart(k_out, k_out_stride, kn, q, q_stride, n, count)))
        return 1;
    const Rows qr = {(const float *)q, (float *)q_out, (int64_t)q_stride, (int64_t)q_out_stride, (int)heads};
    const Rows kr = {(const float *)k, (float *)k_out, (int64_t)k_stride, (int64_t)k_out_stride,
                     k ? (int)kv_heads : 0};
    return status(launch_rope(qr, kr, (int)width, (int)count, (const float2 *)angles, (int)rotated,
                              layout == NYA_HIP_ROPE_HALVES, (hipStream_t)stream));
}

NYA_HIP_EXPORT int nya_hip_kv8_bytes(const nya_hip_kv8 *cache, size_t *codes, size_t *scales)
{
    if (!geometry_ok(cache) || !codes || !scales) return 1;
    *codes = cache->pages * cache->page_tokens * cache->kv_heads * cache->width;
    *scales = cache->pages * cache->kv_heads * sizeof(float);
    return 0;
}

NYA_HIP_EXPORT int nya_hip_kv8_store(const nya_hip_kv8 *cache, uintptr_t slots, size_t count, uintptr_t k,
    size_t k_stride, uintptr_t v, size_t v_stride, uintptr_t angles, size_t rotated, unsigned layout, uintptr_t q,
    size_t q_stride, uintptr_t q_out, size_t q_out_stride, size_t heads, uintptr_t stream)
{
    if (!cache_ok(cache) || !vec(slots) || !pairs_fit(cache, count) || !vec(k) || !vec(v)) return 1;
    const size_t n = cache->kv_heads * cache->width;
    if (k_stride < n || v_stride < n || k_stride > (size_t)INT_MAX || v_stride > (size_t)INT_MAX) return 1;
    if (angles && !rotation_ok(angles, rotated, cache->width, layout)) return 1;
    // Without angles there is nothing to do for q.
    if (q && (!angles || !heads_ok(heads, cache->width) ||
              !rows_ok(q, q_stride, q_out, q_out_stride, heads * cache->width, count) ||
              !apart(q_out, q_out_stride, heads * cache->width, k, k_stride, n, count) ||
              !apart(q_out, q_out_stride, heads * cache->width, v, v_stride, n, count)))
        return 1;
    const Rows qr = {(const float *)q, (float *)q_out, (int64_t)q_stride, (int64_t)q_out_stride, q ? (int)heads : 0};
    return status(launch_kv8_store(cache_of(cache), (const int *)slots, (int)count, (const float *)k,
                                   (int64_t)k_stride, (const float *)v, (int64_t)v_stride, (const float2 *)angles,
                                   angles ? (int)rotated : 0, layout == NYA_HIP_ROPE_HALVES, qr,
                                   (hipStream_t)stream));
}

NYA_HIP_EXPORT int nya_hip_kv8_load(const nya_hip_kv8 *cache, uintptr_t slots, size_t count, uintptr_t k,
    size_t k_stride, uintptr_t v, size_t v_stride, uintptr_t stream)
{
    if (!cache_ok(cache) || !vec(slots) || !pairs_fit(cache, count) || !vec(k) || !vec(v)) return 1;
    const size_t n = cache->kv_heads * cache->width;
    if (k_stride < n || v_stride < n || k_stride > (size_t)INT_MAX || v_stride > (size_t)INT_MAX ||
        !apart(k, k_stride, n, v, v_stride, n, count))
        return 1;
    return status(launch_kv8_load(cache_of(cache), (const int *)slots, (int)count, (float *)k, (int64_t)k_stride,
                                  (float *)v, (int64_t)v_stride, (hipStream_t)stream));
}

NYA_HIP_EXPORT int nya_hip_kv8_attention_bytes(const nya_hip_kv8 *cache, size_t count, size_t requests,
    size_t max_tokens, size_t max_length, size_t heads, size_t window, size_t *bytes)
{
    if (!bytes || !attention_ok(cache, count, requests, max_tokens, max_length, heads, window)) return 1;
    Kv8Attention a = {};
    a.cache = cache_of(cache);
    a.count = (int)count;
    a.requests = (int)requests;
    a.max_tokens = (int)max_tokens;
    a.max_length = (int)max_length;
    a.heads = (int)heads;
    a.window = (int)window;
    *bytes = kv8_attention_workspace(a);
    return 0;
}

NYA_HIP_EXPORT int nya_hip_kv8_attention(const nya_hip_kv8 *cache, uintptr_t q, size_t q_stride, uintptr_t out,
    size_t out_stride, size_t count, uintptr_t starts, uintptr_t lengths, uintptr_t table, size_t table_stride,
    size_t requests, size_t max_tokens, size_t max_length, size_t heads, size_t window, float scale,
    uintptr_t workspace, size_t workspace_bytes, uintptr_t stream)
{
    if (!cache_ok(cache) || !attention_ok(cache, count, requests, max_tokens, max_length, heads, window) || !vec(q) ||
        !vec(out) || !vec(starts) || !vec(lengths) || !vec(table) || !some(table_stride) ||
        table_stride > (size_t)INT_MAX / requests || (workspace & 15u) || !isfinite(scale))
        return 1;
    const size_t n = heads * cache->width;
    if (q_stride < n || out_stride < n || q_stride > (size_t)INT_MAX || out_stride > (size_t)INT_MAX ||
        !apart(q, q_stride, n, out, out_stride, n, count))
        return 1;
    const Kv8Attention a = {cache_of(cache), (const float *)q, (int64_t)q_stride, (float *)out, (int64_t)out_stride,
                            (int)count, (const int *)starts, (const int *)lengths, (const int *)table,
                            (int)table_stride, (int)requests, (int)max_tokens, (int)max_length, (int)heads,
                            (int)window, scale};
    return status(launch_kv8_attention(a, (void *)workspace, workspace ? workspace_bytes : 0, (hipStream_t)stream));
}

}  // extern "C"
