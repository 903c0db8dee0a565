// The rotary step of rows of heads, as a kernel of its own (serving.hip) and beside
// the rows that go into a cache (serving.hip, kv4.hip).
#pragma once
#include "serving.h"

#pragma clang fp contract(off)

namespace fy {
namespace {

// Element d of a head's rotated vector: products of fp32 values are exact in
// 64 bits, so the sum is rounded once there and once to fp32. What is stored
// in 8 bits next is then the code of the defined value.
__device__ __forceinline__ float rotated_at(const float *x, int d, const float2 *angles, int rotated, bool halves)
{
    if (d >= rotated) return x[d];
    const int half = rotated / 2;
    const int j = halves ? (d < half ? d : d - half) : d >> 1;
    const bool second = halves ? d >= half : d & 1;
    const double a = x[halves ? j : 2 * j], b = x[halves ? j + half : 2 * j + 1];
    const double c = angles[j].x, s = angles[j].y;
    return (float)(second ? a * s + b * c : a * c - b * s);
}

// (a, b) by the angle of (c, s).
__device__ __forceinline__ void rotate_pair(float &a, float &b, double c, double s)
{
    const double x = a, y = b;
    a = (float)(x * c - y * s);
    b = (float)(x * s + y * c);
}

// Heads head, head + step, ... of one row: their elements 4 quad .. + 3 (as
// HALVES the pairs' other halves with them), 16 bytes at a time. What does not
// turn is copied, or stays where it is in place.
__device__ __forceinline__ void rotate_quads(const float *x, float *out, int head, int step, int heads,
    int width, int quad, const float2 *__restrict__ angles, int rotated, bool halves)
{
    const int d = 4 * quad, half = rotated / 2;
    const bool turns = halves ? d < half : d < rotated;
    if (!turns && ((halves && d < rotated) || x == out)) return;
    x += d;
    out += d;
    if (!turns) {
#pragma unroll 4
        for (int h = head; h < heads; h += step)
            *(float4 *)(out + (size_t)h * width) = *(const float4 *)(x + (size_t)h * width);
    } else if (halves) {
        const float4 *a4 = (const float4 *)(angles + d);
        const float4 p = a4[0], q = a4[1];
        const double c0 = p.x, s0 = p.y, c1 = p.z, s1 = p.w, c2 = q.x, s2 = q.y, c3 = q.z, s3 = q.w;
#pragma unroll 2
        for (int h = head; h < heads; h += step) {
            float4 u = *(const float4 *)(x + (size_t)h * width), v = *(const float4 *)(x + (size_t)h * width + half);
            rotate_pair(u.x, v.x, c0, s0);
            rotate_pair(u.y, v.y, c1, s1);
            rotate_pair(u.z, v.z, c2, s2);
            rotate_pair(u.w, v.w, c3, s3);
            *(float4 *)(out + (size_t)h * width) = u;
            *(float4 *)(out + (size_t)h * width + half) = v;
        }
    } else {
        const float4 p = *(const float4 *)(angles + d / 2);
        const double c0 = p.x, s0 = p.y, c1 = p.z, s1 = p.w;
#pragma unroll 4
        for (int h = head; h < heads; h += step) {
            float4 u = *(const float4 *)(x + (size_t)h * width);
            rotate_pair(u.x, u.y, c0, s0);
            rotate_pair(u.z, u.w, c1, s1);
            *(float4 *)(out + (size_t)h * width) = u;
        }
    }
}

// Heads [first, last) of one row by the workgroup's 256 threads: 16 bytes a
// thread where everything allows it, else a pair or a kept element.
__device__ __forceinline__ void rotate_heads(const Rows &t, int row, int first, int last, int width,
    const float2 *__restrict__ angles, int rotated, bool halves, bool quads)
{
    const float *x = t.x + row * t.stride;
    float *out = t.out + row * t.out_stride;
    angles += (size_t)row * (rotated / 2);
    const int tid = threadIdx.x;
    if (quads) {
        const int n = width / 4, step = 256 / n, head = tid / n;
        if (head < step) rotate_quads(x, out, first + head, step, last, width, tid - head * n, angles, rotated, halves);
        return;
    }
    const int half = rotated / 2, n = width - half;
    for (int i = tid; i < (last - first) * n; i += 256) {
        const int h = first + i / n, e = i % n;
        const float *xh = x + (size_t)h * width;
        float *oh = out + (size_t)h * width;
        if (e >= half) {
            oh[half + e] = xh[half + e];
            continue;
        }
        const int d0 = halves ? e : 2 * e, d1 = halves ? e + half : 2 * e + 1;
        const float u = rotated_at(xh, d0, angles, rotated, halves), v = rotated_at(xh, d1, angles, rotated, halves);
        oh[d0] = u;
        oh[d1] = v;
    }
}

inline bool quads_ok(const Rows &t, int width, int rotated, bool halves, const float2 *angles)
{
    return !t.heads || (width % 4 == 0 && width <= 1024 && rotated % (halves ? 8 : 4) == 0 && t.stride % 4 == 0 &&
                        t.out_stride % 4 == 0 && (((uintptr_t)t.x | (uintptr_t)t.out | (uintptr_t)angles) & 15) == 0);
}

// Heads of a row per workgroup: few where there are few rows, so that there
// are workgroups for the chip; more where a thread can then use its angles for
// several heads.
inline int heads_each(int count, int heads, int width)
{
    const int at_once = width <= 1024 ? 1024 / width : 1;
    int each = at_once;
    while (each < heads && (int64_t)count * ((heads + each - 1) / each) > 4096) each += at_once;
    return each;
}

}  // namespace
}  // namespace fy
