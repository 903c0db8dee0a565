// Checks of the arguments that the serving entry points share (abi_serving.hip, abi_kv4.hip).
#pragma once
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include "../../include/fyodor_hip_serving.h"
#include "serving.h"

namespace {

using namespace fy;

inline int status(hipError_t e)
{
    return e == hipSuccess ? 0 : -(int)(e > 0 ? e : 1);
}

// Device arrays of 4-byte elements: non-null and aligned.
inline bool vec(uintptr_t p) { return p && !(p & 3u); }
inline bool some(size_t n) { return n && n <= (size_t)INT_MAX; }
// Rows of a step, and floats of a row: launches stay within 2^32 threads.
inline bool rows_fit(size_t n) { return n && n <= (size_t)1 << 22; }
constexpr size_t kMaxRow = (size_t)1 << 22;

// `count` rows of a_n and of b_n floats share nothing: the whole ranges, or
// (parts of common rows) the same stride and other columns.
inline bool apart(uintptr_t a, size_t a_stride, size_t a_n, uintptr_t b, size_t b_stride, size_t b_n, size_t count)
{
    if (a_stride == b_stride) {
        const size_t d = a <= b ? (b - a) / 4 % a_stride : a_stride - ((a - b + 3) / 4 - 1) % a_stride - 1;
        if (d >= a_n && d + b_n <= a_stride) return true;
    }
    const uintptr_t a_end = a + 4 * ((count - 1) * a_stride + a_n), b_end = b + 4 * ((count - 1) * b_stride + b_n);
    return a_end <= b || b_end <= a;
}

// Rows in, rows out: the same ones, or apart.
inline bool rows_ok(uintptr_t x, size_t stride, uintptr_t out, size_t out_stride, size_t n, size_t count)
{
    return vec(x) && vec(out) && stride >= n && out_stride >= n && stride <= (size_t)INT_MAX &&
           out_stride <= (size_t)INT_MAX && ((x == out && stride == out_stride) ||
                                             apart(x, stride, n, out, out_stride, n, count));
}

inline bool heads_ok(size_t heads, size_t width)
{
    return heads && heads <= 65535 && width && width <= kMaxRow && heads <= kMaxRow / width;
}

inline bool rotation_ok(uintptr_t angles, size_t rotated, size_t width, unsigned layout)
{
    return angles && !(angles & 7u) && rotated && rotated % 2 == 0 && rotated <= width &&
           layout <= NYA_HIP_ROPE_HALVES;
}

inline bool page_ok(size_t n) { return n == 16 || n == 32 || n == 64 || n == 128; }

// A cache's geometry (C: nya_hip_kv8 or nya_hip_kv4).
template <class C>
bool geometry_ok(const C *c)
{
    return c && some(c->pages) && page_ok(c->page_tokens) &&
           (c->width == 64 || c->width == 128 || c->width == 256 || c->width == 512) &&
           c->kv_heads <= 16384 && heads_ok(c->kv_heads, c->width) &&
           c->pages <= (size_t)INT_MAX / c->page_tokens && c->pages <= (size_t)INT_MAX / c->kv_heads;
}

// (Row, KV head) pairs of a store or load: launches stay within 2^32 threads.
template <class C>
bool pairs_fit(const C *c, size_t count) { return rows_fit(count) && count <= ((size_t)1 << 25) / c->kv_heads; }

// What both attention entries ask of the sizes.
template <class C>
bool attention_ok(const C *cache, size_t count, size_t requests, size_t max_tokens, size_t max_length,
    size_t heads, size_t window)
{
    return geometry_ok(cache) && rows_fit(count) && requests && requests <= 65535 && max_tokens && max_tokens <= count &&
           some(max_length) && heads_ok(heads, cache->width) && heads % cache->kv_heads == 0 &&
           count <= ((size_t)1 << 27) / heads && requests <= ((size_t)1 << 21) / cache->kv_heads && window <= (size_t)INT_MAX;
}

}  // namespace
