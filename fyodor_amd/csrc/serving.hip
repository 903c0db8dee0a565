// The steps around attention over a paged 8-bit cache
// (include/fyodor_hip_serving.h): page tables from request lengths, rotary
// positions, and the cache's store and load.
#include <math.h>

#include "device.h"
#include "serving.h"

#pragma clang fp contract(off)

namespace fy {
namespace {

// ---- pages ----------------------------------------------------------------

constexpr int kPageThreads = 1024;

// Exclusive prefix sums over the workgroup's threads, saturating at `most`
// (a + b of two values up to INT_MAX fits 32 bits); *total over all of them.
// `parts`: one word per wavefront.
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t most, uint32_t *parts, uint32_t *total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t s = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t o = (uint32_t)__shfl_up((int)s, d, 64);
        if (lane >= d) s = min(s + o, most);
    }
    __syncthreads();   // the last call's parts are read
    if (lane == 63) parts[wave] = s;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPageThreads / 64; ++w) {
        if (w == wave) before = all;
        all = min(all + parts[w], most);
    }
    *total = all;
    const uint32_t own = (uint32_t)__shfl_up((int)s, 1, 64);
    return min(before + (lane ? own : 0), most);
}

__device__ __forceinline__ int clamped(int v, int most) { return v < 0 ? 0 : v > most ? most : v; }

// The largest i < n with first[i] <= at (first[0] = 0 <= at), first ascending.
__device__ __forceinline__ int last_from(const uint32_t *first, int n, uint32_t at)
{
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= at) lo = mid;
        else hi = mid;
    }
    return lo;
}

// One workgroup: the page stack is one thing. Requests go 1024 at a time, a
// thread each; the moved pages of such a chunk are spread over all threads.
__global__ __launch_bounds__(kPageThreads) void page_tables(PageStep p)
{
    __shared__ uint32_t parts[kPageThreads / 64], first[kPageThreads];
    __shared__ int base[kPageThreads];
    const int tid = threadIdx.x;
    const int chunks = (p.requests + kPageThreads - 1) / kPageThreads;
    uint32_t top = (uint32_t)clamped(p.free_count[0], p.pages);
    auto need_of = [&](int r, bool *beyond) {
        const int length = max(p.lengths[r], 0), need = (int)(((uint32_t)length + p.page_tokens - 1) / p.page_tokens);
        *beyond = need > p.table_stride;
        return need;
    };
    // 1. Pages past the need, back on the stack.
    for (int c = 0; c < chunks; ++c) {
        const int r = c * kPageThreads + tid;
        uint32_t back = 0;
        int need = 0;
        if (r < p.requests) {
            bool beyond;
            need = need_of(r, &beyond);
            const int held = clamped(p.held[r], p.table_stride);
            if (!beyond && held > need) {
                back = (uint32_t)(held - need);
                p.held[r] = need;
            }
        }
        uint32_t total;
        first[tid] = block_prefix(back, INT_MAX, parts, &total);
        base[tid] = need;
        __syncthreads();
        for (uint32_t i = tid; i < total; i += kPageThreads) {
            const int k = last_from(first, kPageThreads, i);
            int *entry = p.table + (size_t)(c * kPageThreads + k) * p.table_stride + base[k] + (i - first[k]);
            if (top + i < (uint32_t)p.pages) p.free_pages[top + i] = *entry;
            *entry = -1;
        }
        top = min(top + total, (uint32_t)p.pages);
        __syncthreads();
    }
    // 2. Pages for the requests that grow, from the top.
    uint32_t asked = 0, given = 0, refused = 0;
    for (int c = 0; c < chunks; ++c) {
        const int r = c * kPageThreads + tid;
        uint32_t grow = 0;
        int held = 0;
        bool beyond = false;
        if (r < p.requests) {
            const int need = need_of(r, &beyond);
            held = clamped(p.held[r], p.table_stride);
            if (!beyond && need > held) grow = (uint32_t)(need - held);
        }
        uint32_t total, served;
        const uint32_t before = min(asked + block_prefix(grow, INT_MAX, parts, &total), (uint32_t)INT_MAX);
        const bool fits = before + grow <= top;
        const uint32_t mine = fits ? grow : 0;
        // A request that is not served, and with it every later one that
        // needs pages, takes nothing: those served are a prefix.
        first[tid] = block_prefix(mine, INT_MAX, parts, &served);
        base[tid] = held;
        if (mine) p.held[r] = held + (int)mine;
        __syncthreads();
        for (uint32_t i = tid; i < served; i += kPageThreads) {
            const int k = last_from(first, kPageThreads, i);
            p.table[(size_t)(c * kPageThreads + k) * p.table_stride + base[k] + (i - first[k])] =
                p.free_pages[top - 1 - given - i];
        }
        asked = min(asked + total, (uint32_t)INT_MAX);
        given += served;
        uint32_t left;
        block_prefix(beyond || (grow && !fits) ? 1 : 0, INT_MAX, parts, &left);
        refused += left;
    }
    // 3. The rows' starts.
    uint32_t rows = 0;
    for (int c = 0; c < chunks; ++c) {
        const int r = c * kPageThreads + tid;
        const uint32_t n = r < p.requests ? (uint32_t)clamped(p.counts[r], p.max_tokens) : 0;
        uint32_t total;
        const uint32_t before = block_prefix(n, (uint32_t)p.max_tokens, parts, &total);
        if (r < p.requests) p.starts[r] = (int)min(rows + before, (uint32_t)p.max_tokens);
        rows = min(rows + total, (uint32_t)p.max_tokens);
    }
    if (tid == 0) {
        p.starts[p.requests] = (int)rows;
        p.free_count[0] = (int)(top - given);
        p.free_count[1] = (int)refused;
    }
}

__global__ __launch_bounds__(256) void page_rows(PageStep p)
{
    const int row = blockIdx.x * 256 + threadIdx.x;
    if (row >= p.max_tokens) return;
    int position = -1, slot = -1;
    if (row < p.starts[p.requests]) {
        const int r = last_from((const uint32_t *)p.starts, p.requests, (uint32_t)row);
        // 64 bits: the lengths are the caller's.
        const int64_t at = (int64_t)max(p.lengths[r], 0) - clamped(p.counts[r], p.max_tokens) + (row - p.starts[r]);
        position = (int)at;
        if (at >= 0) {
            const int64_t j = at / p.page_tokens;
            if (j < clamped(p.held[r], p.table_stride)) {
                const int page = p.table[(size_t)r * p.table_stride + j];
                if ((unsigned)page < (unsigned)p.pages) slot = page * p.page_tokens + (int)(at % p.page_tokens);
            }
        }
    }
    p.positions[row] = position;
    p.slots[row] = slot;
}

// ---- rotary positions -----------------------------------------------------

__global__ __launch_bounds__(256) void rope_angles(const int *__restrict__ positions, int64_t n,
    const float *__restrict__ frequencies, int pairs, float magnitude, float2 *__restrict__ angles)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const double turns = (double)positions[i / pairs] * (double)frequencies[i % pairs] * (1 / M_PI);
    double s, c;
    sincospi(turns, &s, &c);
    angles[i] = make_float2((float)(c * magnitude), (float)(s * magnitude));
}

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

// Thread (row, head, pair or kept element).
__global__ __launch_bounds__(256) void rope_rows(Rows q, Rows k, int width, const float2 *__restrict__ angles,
    int rotated, bool halves)
{
    const int row = blockIdx.x, half = rotated / 2, per_head = width - half;
    const int i = blockIdx.y * 256 + threadIdx.x, head = i / per_head, e = i % per_head;
    if (head >= q.heads + k.heads) return;
    const Rows &t = head < q.heads ? q : k;
    const int h = head < q.heads ? head : head - q.heads;
    const float *x = t.x + row * t.stride + (int64_t)h * width;
    float *out = t.out + row * t.out_stride + (int64_t)h * width;
    if (e >= half) {
        out[half + e] = x[half + e];
        return;
    }
    const int d0 = halves ? e : 2 * e, d1 = halves ? e + half : 2 * e + 1;
    const float2 *a = angles + (size_t)row * half;
    const float u = rotated_at(x, d0, a, rotated, halves), v = rotated_at(x, d1, a, rotated, halves);
    out[d0] = u;
    out[d1] = v;
}

// ---- the 8-bit cache ------------------------------------------------------

constexpr float kScaleFloor = 0x1p-100f;

__device__ __forceinline__ int key_at(int t, int d, int page_tokens) { return ((d >> 4) * page_tokens + t) * 16 + (d & 15); }
__device__ __forceinline__ int value_at(int t, int d, int width) { return ((t >> 4) * width + d) * 16 + (t & 15); }

// round(x / scale), ties to even: the remainder x - n scale of the nearest
// guess is exact (a multiple of scale's last bit, below scale), so comparing it
// with half a step settles the guesses next to a border.
__device__ __forceinline__ int8_t code_of(float x, float scale, float inverse)
{
    float n = rintf(x * inverse);
    const float r = __builtin_fmaf(-n, scale, x), half = 0.5f * scale;
    const bool odd = (int)n & 1;
    if (r > half || (r == half && odd)) n += 1.f;
    else if (r < -half || (r == -half && odd)) n -= 1.f;
    return (int8_t)(int)fminf(fmaxf(n, -127.f), 127.f);
}

// Workgroup (row, KV head): the run of rows that begins at this one, if one
// does; (row, kv_heads + part): a part of this row's q.
__global__ __launch_bounds__(256) void kv8_store(Kv8 c, const int *__restrict__ slots, int count,
    const float *__restrict__ k, int64_t k_stride, const float *__restrict__ v, int64_t v_stride,
    const float2 *__restrict__ angles, int rotated, bool halves, Rows q)
{
    __shared__ uint32_t top[2][4];
    const int row = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, width = c.width, page_tokens = c.page_tokens;
    if (head >= c.kv_heads) {
        const int half = rotated / 2, per_head = width - half;
        const int i = (head - c.kv_heads) * 256 + tid, h = i / per_head, e = i % per_head;
        if (h >= q.heads) return;
        const float *x = q.x + row * q.stride + (int64_t)h * width;
        float *out = q.out + row * q.out_stride + (int64_t)h * width;
        if (e >= half) {
            out[half + e] = x[half + e];
            return;
        }
        const int d0 = halves ? e : 2 * e, d1 = halves ? e + half : 2 * e + 1;
        const float2 *a = angles + (size_t)row * half;
        const float u = rotated_at(x, d0, a, rotated, halves), w = rotated_at(x, d1, a, rotated, halves);
        out[d0] = u;
        out[d1] = w;
        return;
    }
    const int slot = slots[row], at = slot % page_tokens;
    if (slot < 0 || slot >= c.pages * page_tokens) return;
    if (at && row && slots[row - 1] == slot - 1) return;
    int n = 1;
    while (row + n < count && at + n < page_tokens && slots[row + n] == slot + n) ++n;
    const size_t place = (size_t)(slot / page_tokens) * c.kv_heads + head;
    int8_t *codes[2] = {c.keys + place * page_tokens * width, c.values + place * page_tokens * width};
    float *scales[2] = {c.key_scales + place, c.value_scales + place};
    auto key = [&](int t, int d) {
        return rotated_at(k + (row + t) * k_stride + (int64_t)head * width, d,
                          angles + (size_t)(row + t) * (rotated / 2), rotated, halves);
    };
    auto value = [&](int t, int d) { return v[(row + t) * v_stride + (int64_t)head * width + d]; };
    // The largest magnitude by its bits: NaN above infinity above the rest.
    uint32_t big[2] = {0, 0};
    for (int i = tid; i < n * width; i += 256) {
        big[0] = max(big[0], __builtin_bit_cast(uint32_t, key(i / width, i % width)) & 0x7FFFFFFFu);
        big[1] = max(big[1], __builtin_bit_cast(uint32_t, value(i / width, i % width)) & 0x7FFFFFFFu);
    }
    const float old[2] = {*scales[0], *scales[1]};
    for (int kind = 0; kind < 2; ++kind) {
        for (int o = 32; o; o >>= 1) big[kind] = max(big[kind], (uint32_t)__shfl_xor((int)big[kind], o, 64));
        if ((tid & 63) == 0) top[kind][tid >> 6] = big[kind];
    }
    __syncthreads();
    for (int kind = 0; kind < 2; ++kind) {
        const uint32_t b = max(max(top[kind][0], top[kind][1]), max(top[kind][2], top[kind][3]));
        const float amax = __builtin_bit_cast(float, b);
        float scale = amax / 127.f;
        if (scale < kScaleFloor) scale = kScaleFloor;
        if (at) {
            if (scale <= old[kind] || old[kind] != old[kind]) {
                scale = old[kind];
            } else {
                for (int i = tid; i < page_tokens * width; i += 256)
                    codes[kind][i] = (int8_t)(int)fmin(fmax(rint((double)codes[kind][i] * old[kind] / scale), -127.0), 127.0);
                __syncthreads();
            }
        }
        const float inverse = 1.f / scale;
        for (int i = tid; i < n * width; i += 256) {
            const int t = i / width, d = i % width;
            if (kind == 0) codes[0][key_at(at + t, d, page_tokens)] = code_of(key(t, d), scale, inverse);
            else codes[1][value_at(at + t, d, width)] = code_of(value(t, d), scale, inverse);
        }
        if (tid == 0) *scales[kind] = scale;
    }
}

__global__ __launch_bounds__(256) void kv8_load(Kv8 c, const int *__restrict__ slots, float *__restrict__ k,
    int64_t k_stride, float *__restrict__ v, int64_t v_stride)
{
    const int row = blockIdx.x, i = blockIdx.y * 256 + threadIdx.x, head = i / c.width, d = i % c.width;
    const int slot = slots[row];
    if (head >= c.kv_heads || slot < 0 || slot >= c.pages * c.page_tokens) return;
    const int t = slot % c.page_tokens;
    const size_t place = (size_t)(slot / c.page_tokens) * c.kv_heads + head, codes = place * c.page_tokens * c.width;
    k[row * k_stride + i] = (float)c.keys[codes + key_at(t, d, c.page_tokens)] * c.key_scales[place];
    v[row * v_stride + i] = (float)c.values[codes + value_at(t, d, c.width)] * c.value_scales[place];
}

}  // namespace

hipError_t launch_page_step(const PageStep &p, hipStream_t s)
{
    hipLaunchKernelGGL(page_tables, dim3(1), dim3(kPageThreads), 0, s, p);
    hipLaunchKernelGGL(page_rows, dim3((unsigned)((p.max_tokens + 255ll) / 256)), dim3(256), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_rope_angles(const int *positions, int count, const float *frequencies, int pairs, float magnitude,
    float2 *angles, hipStream_t s)
{
    const int64_t n = (int64_t)count * pairs;
    hipLaunchKernelGGL(rope_angles, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, s, positions, n, frequencies,
                       pairs, magnitude, angles);
    return hipGetLastError();
}

hipError_t launch_rope(const Rows &q, const Rows &k, int width, int count, const float2 *angles, int rotated,
    bool halves, hipStream_t s)
{
    const int64_t n = (int64_t)(q.heads + k.heads) * (width - rotated / 2);
    hipLaunchKernelGGL(rope_rows, dim3((unsigned)count, (unsigned)((n + 255) / 256)), dim3(256), 0, s, q, k, width,
                       angles, rotated, halves);
    return hipGetLastError();
}

hipError_t launch_kv8_store(const Kv8 &cache, const int *slots, int count, const float *k, int64_t k_stride,
    const float *v, int64_t v_stride, const float2 *angles, int rotated, bool halves, const Rows &q, hipStream_t s)
{
    const int64_t n = (int64_t)q.heads * (cache.width - rotated / 2);
    hipLaunchKernelGGL(kv8_store, dim3((unsigned)count, (unsigned)(cache.kv_heads + (n + 255) / 256)), dim3(256), 0, s,
                       cache, slots, count, k, k_stride, v, v_stride, angles, rotated, halves, q);
    return hipGetLastError();
}

hipError_t launch_kv8_load(const Kv8 &cache, const int *slots, int count, float *k, int64_t k_stride, float *v,
    int64_t v_stride, hipStream_t s)
{
    hipLaunchKernelGGL(kv8_load, dim3((unsigned)count, (unsigned)(((int64_t)cache.kv_heads * cache.width + 255) / 256)),
                       dim3(256), 0, s, cache, slots, k, k_stride, v, v_stride);
    return hipGetLastError();
}

}  // namespace fy
