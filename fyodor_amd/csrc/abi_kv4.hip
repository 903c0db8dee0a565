// extern "C" entry points of libfyodor_hip.so declared in include/fyodor_hip_kv4.h.
#include "../../include/fyodor_hip_kv4.h"
#include "serving_checks.h"

namespace {

bool cache_ok(const nya_hip_kv4 *c)
{
    return geometry_ok(c) && c->keys && c->values && c->key_steps && c->value_steps &&
           !((c->keys | c->values | c->key_steps | c->value_steps) & 15u);
}

Kv4 cache_of(const nya_hip_kv4 *c)
{
    return {(uint8_t *)c->keys, (uint8_t *)c->values, (uint16_t *)c->key_steps, (uint16_t *)c->value_steps,
            (int)c->pages, (int)c->page_tokens, (int)c->kv_heads, (int)c->width};
}

}  // namespace

extern "C" {

NYA_HIP_EXPORT int nya_hip_kv4_bytes(const nya_hip_kv4 *cache, size_t *codes, size_t *steps)
{
    if (!geometry_ok(cache) || !codes || !steps) return 1;
    const size_t elements = cache->pages * cache->page_tokens * cache->kv_heads * cache->width;
    *codes = elements / 2;
    *steps = elements / 32 * sizeof(uint16_t);
    return 0;
}

NYA_HIP_EXPORT int nya_hip_kv4_store(const nya_hip_kv4 *cache, uintptr_t slots, size_t count, uintptr_t k,
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
    return status(launch_kv4_store(cache_of(cache), (const int *)slots, (int)count, (const float *)k,
                                   (int64_t)k_stride, (const float *)v, (int64_t)v_stride, (const float2 *)angles,
                                   angles ? (int)rotated : 0, layout == NYA_HIP_ROPE_HALVES, qr,
                                   (hipStream_t)stream));
}

NYA_HIP_EXPORT int nya_hip_kv4_load(const nya_hip_kv4 *cache, uintptr_t slots, size_t count, uintptr_t k,
    size_t k_stride, uintptr_t v, size_t v_stride, uintptr_t stream)
{
    if (!cache_ok(cache) || !vec(slots) || !pairs_fit(cache, count) || !vec(k) || !vec(v)) return 1;
    const size_t n = cache->kv_heads * cache->width;
    if (k_stride < n || v_stride < n || k_stride > (size_t)INT_MAX || v_stride > (size_t)INT_MAX ||
        !apart(k, k_stride, n, v, v_stride, n, count))
        return 1;
    return status(launch_kv4_load(cache_of(cache), (const int *)slots, (int)count, (float *)k, (int64_t)k_stride,
                                  (float *)v, (int64_t)v_stride, (hipStream_t)stream));
}

NYA_HIP_EXPORT int nya_hip_kv4_attention_bytes(const nya_hip_kv4 *cache, size_t count, size_t requests,
    size_t max_tokens, size_t max_length, size_t heads, size_t window, size_t *bytes)
{
    if (!bytes || !attention_ok(cache, count, requests, max_tokens, max_length, heads, window)) return 1;
    Kv4Attention a = {};
    a.cache = cache_of(cache);
    a.count = (int)count;
    a.requests = (int)requests;
    a.max_tokens = (int)max_tokens;
    a.max_length = (int)max_length;
    a.heads = (int)heads;
    a.window = (int)window;
    *bytes = kv4_attention_workspace(a);
    return 0;
}

NYA_HIP_EXPORT int nya_hip_kv4_attention(const nya_hip_kv4 *cache, uintptr_t q, size_t q_stride, uintptr_t out,
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
    const Kv4Attention a = {cache_of(cache), (const float *)q, (int64_t)q_stride, (float *)out, (int64_t)out_stride,
                            (int)count, (const int *)starts, (const int *)lengths, (const int *)table,
                            (int)table_stride, (int)requests, (int)max_tokens, (int)max_length, (int)heads,
                            (int)window, scale};
    return status(launch_kv4_attention(a, (void *)workspace, workspace ? workspace_bytes : 0, (hipStream_t)stream));
}

}  // extern "C"
