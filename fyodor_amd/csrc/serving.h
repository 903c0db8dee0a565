// Launchers of the serving kernels (serving.hip, attention_kv8.hip; kv4.hip, attention_kv4.hip), called by
// abi_serving.hip and abi_kv4.hip.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace fy {

// An 8-bit paged cache (include/fyodor_hip_serving.h).
struct Kv8 {
    int8_t *keys, *values;
    float *key_scales, *value_scales;
    int pages, page_tokens, kv_heads, width;
};

// Rows of one tensor: heads of a common width, rows `stride` floats apart.
struct Rows {
    const float *x;
    float *out;
    int64_t stride, out_stride;
    int heads;
};

struct PageStep {
    const int *lengths, *counts;
    int requests, page_tokens;
    int *table;
    int table_stride;
    int *held, *free_pages;
    int pages;
    int *free_count, *starts, *positions, *slots;
    int max_tokens;
};
hipError_t launch_page_step(const PageStep &p, hipStream_t s);

hipError_t launch_rope_angles(const int *positions, int count, const float *frequencies, int pairs, float magnitude,
    float2 *angles, hipStream_t s);
// k.heads 0: q only.
hipError_t launch_rope(const Rows &q, const Rows &k, int width, int count, const float2 *angles, int rotated,
    bool halves, hipStream_t s);

// angles null: no rotation; q.heads 0: no q.
hipError_t launch_kv8_store(const Kv8 &cache, const int *slots, int count, const float *k, int64_t k_stride,
    const float *v, int64_t v_stride, const float2 *angles, int rotated, bool halves, const Rows &q, hipStream_t s);
hipError_t launch_kv8_load(const Kv8 &cache, const int *slots, int count, float *k, int64_t k_stride, float *v,
    int64_t v_stride, hipStream_t s);

struct Kv8Attention {
    static constexpr float kLess = 0x1p-18f;   // sums of weights are held this much smaller
    Kv8 cache;
    const float *q;
    int64_t q_stride;
    float *out;
    int64_t out_stride;
    int count;
    const int *starts, *lengths, *table;
    int table_stride, requests, max_tokens, max_length, heads, window;
    float scale;
};
// Of the arguments' sizes alone.
size_t kv8_attention_workspace(const Kv8Attention &a);
hipError_t launch_kv8_attention(const Kv8Attention &a, void *workspace, size_t workspace_bytes, hipStream_t s);

// A 4-bit paged cache (include/fyodor_hip_kv4.h).
struct Kv4 {
    uint8_t *keys, *values;
    uint16_t *key_steps, *value_steps;
    int pages, page_tokens, kv_heads, width;
};

// As the 8-bit cache's.
hipError_t launch_kv4_store(const Kv4 &cache, const int *slots, int count, const float *k, int64_t k_stride,
    const float *v, int64_t v_stride, const float2 *angles, int rotated, bool halves, const Rows &q, hipStream_t s);
hipError_t launch_kv4_load(const Kv4 &cache, const int *slots, int count, float *k, int64_t k_stride, float *v,
    int64_t v_stride, hipStream_t s);

struct Kv4Attention {
    static constexpr float kLess = 1.f;
    Kv4 cache;
    const float *q;
    int64_t q_stride;
    float *out;
    int64_t out_stride;
    int count;
    const int *starts, *lengths, *table;
    int table_stride, requests, max_tokens, max_length, heads, window;
    float scale;
};
size_t kv4_attention_workspace(const Kv4Attention &a);
hipError_t launch_kv4_attention(const Kv4Attention &a, void *workspace, size_t workspace_bytes, hipStream_t s);

}  // namespace fy
