// The 4-bit paged cache's store and load (include/fyodor_hip_kv4.h).
//
// A thread has 4 elements of a head's key and of its value, 8 lanes a block of
// 32 of each: the block's extremes by lane moves, its step, and the codes,
// which are fixed by the defined quotients (64-bit rotations rounded once, the
// quotient's side of a border from its exact remainder). A block's lanes are
// neighbours, so its extremes are three lane moves and no LDS, and a word of a
// key's codes one more.
//
// Many rows are bound by their bytes: the store of three prompts of up to 1601
// tokens (32 heads over 4 of 64, q rotated in the same launch) moves 72 MB in 15.4
// us, 4.7 TB/s, three quarters of it q; the load of five prefixes (8 heads
// of 256) 85 MB in 18.3 us, 4.7 TB/s. Few rows are a launch and one chain of waits
// (slot, row): 61 of 8 heads of 128 4.2 us stored, 2.9 loaded.
#include <math.h>

#include "device.h"

#pragma clang fp contract(off)

#include "rotary.h"

namespace fy {
namespace {

constexpr int kBlock = 32;           // elements that share a step
constexpr float kMostStep = 8160.f;  // 8 of them are the largest multiple of a step in fp16

// Lanes of a head, each with kQuads groups of 4 elements, 4 kHeadLanes apart.
template <int W> struct Lanes {
    static constexpr int kHead = W / 4 < 64 ? W / 4 : 64, kQuads = W / 4 / kHead;
};

struct Store4 {
    Kv4 c;
    const int *slots;
    int count;
    const float *k, *v;
    int64_t k_stride, v_stride;
    const float2 *angles;
    int rotated;
    bool halves, quads_k, quads_v, quads_q;
    Rows q;
    int each, parts;      // q heads per workgroup, workgroups per row of q
    unsigned stores;      // workgroups that store
};

// round(x / step) of a step above 0, ties to even, within [-8, 7]: the remainder
// x - n step of the nearest guess is exact (a multiple of x's last bit, at most
// a step), so comparing it with half a step settles the guesses next to a border.
__device__ __forceinline__ int code_of(float x, float step, float inverse)
{
    float n = fminf(fmaxf(rintf(x * inverse), -9.f), 8.f);
    const float r = __builtin_fmaf(-n, step, x), half = 0.5f * step;
    const bool odd = (int)n & 1;
    if (r > half || (r == half && odd)) n += 1.f;
    else if (r < -half || (r == -half && odd)) n -= 1.f;
    return (int)fminf(fmaxf(n, -8.f), 7.f);
}

// A block's step from its extremes: m / -8 to 8 bits, as fp16.
__device__ __forceinline__ float step_of(float low, float high)
{
    const float m = -low >= high ? low : high;
    uint32_t b = __builtin_bit_cast(uint32_t, m * -0.125f);
    b = (b + 0x7FFFu + (b >> 16 & 1u)) & 0xFFFF0000u;
    return (float)(_Float16)fminf(fmaxf(__builtin_bit_cast(float, b), -kMostStep), kMostStep);
}

__device__ __forceinline__ float block_max(float v)
{
    v = fmaxf(v, row_lane<0xB1>(v));
    v = fmaxf(v, row_lane<0x4E>(v));
    return fmaxf(v, row_lane<0x141>(v));
}

// The codes (0 .. 15) of a thread's four elements, and the block's step.
__device__ __forceinline__ float quantise(const float (&x)[4], uint32_t (&n)[4])
{
    const float high = block_max(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    const float low = -block_max(fmaxf(fmaxf(-x[0], -x[1]), fmaxf(-x[2], -x[3])));
    const float step = step_of(low, high), size = fabsf(step), inverse = 1.f / size;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        n[e] = size > 0.f ? (uint32_t)(code_of(step < 0.f ? -x[e] : x[e], size, inverse) + 8) : 8u;
    return step;
}

__device__ __forceinline__ void load4(const float *x, bool whole, float (&out)[4])
{
    if (whole) {
        *(float4 *)out = *(const float4 *)x;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = x[e];
    }
}

// Elements d .. d + 3 of a rotated head.
__device__ __forceinline__ void key_quad(const Store4 &s, int row, int head, int d, int width, float (&x)[4])
{
    const float *k = s.k + row * s.k_stride + (int64_t)head * width;
    const int half = s.rotated / 2;
    const float2 *angles = s.angles + (size_t)row * half;
    if (!s.quads_k) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = rotated_at(k, d + e, angles, s.rotated, s.halves);
        return;
    }
    load4(k + d, true, x);
    if (d >= s.rotated) return;
    if (!s.halves) {
        const float4 a = *(const float4 *)(angles + d / 2);
        rotate_pair(x[0], x[1], a.x, a.y);
        rotate_pair(x[2], x[3], a.z, a.w);
        return;
    }
    const bool second = d >= half;
    const int j = second ? d - half : d;
    float o[4];
    load4(k + (second ? j : d + half), true, o);
    const float4 a0 = *(const float4 *)(angles + j), a1 = *(const float4 *)(angles + j + 2);
    const float c[4] = {a0.x, a0.z, a1.x, a1.z}, sn[4] = {a0.y, a0.w, a1.y, a1.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float u = second ? o[e] : x[e], w = second ? x[e] : o[e];
        rotate_pair(u, w, c[e], sn[e]);
        x[e] = second ? w : u;
    }
}

__device__ __forceinline__ bool finite4(const float (&x)[4])
{
    // (0 of each: NaN where one is not finite.)
    const float z = (x[0] * 0.f + x[1] * 0.f) + (x[2] * 0.f + x[3] * 0.f);
    return z == 0.f;
}

// Workgroup: 256 threads of (row, head, quad) from number blockIdx.x * 256 on;
// from workgroup `stores` on, (row, part): a part of a row's q.
template <int W>
__global__ __launch_bounds__(256) void kv4_store(Store4 s)
{
    if (blockIdx.x >= s.stores) {
        const int i = blockIdx.x - s.stores, first = i % s.parts * s.each;
        rotate_heads(s.q, i / s.parts, first, min(first + s.each, s.q.heads), W, s.angles, s.rotated, s.halves,
                     s.quads_q);
        return;
    }
    constexpr int kHead = Lanes<W>::kHead, kQuads = Lanes<W>::kQuads, kBlocks = W / kBlock;
    const Kv4 &c = s.c;
    const unsigned pair = (blockIdx.x * 256u + threadIdx.x) / kHead;   // (row, head)
    const int lane = threadIdx.x & 63, within = threadIdx.x % kHead;
    const int row = min(pair / c.kv_heads, (unsigned)s.count - 1), head = pair % c.kv_heads;
    const int slot = s.slots[row], t = slot & (c.page_tokens - 1);
    float k[kQuads][4], v[kQuads][4];
    bool fine = true;
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
        const int d = 4 * (within + kHead * i);
        key_quad(s, row, head, d, W, k[i]);
        load4(s.v + row * s.v_stride + (int64_t)head * W + d, s.quads_v, v[i]);
        fine = fine && finite4(k[i]) && finite4(v[i]);
    }
    // A head with an element that is not finite: marked by NaN steps of its key.
    const uint64_t bad = __builtin_amdgcn_ballot_w64(!fine);
    const bool marked = bad >> (lane & ~(kHead - 1)) & (~0ull >> (64 - kHead));
    const size_t place = (size_t)((unsigned)slot / c.page_tokens) * c.kv_heads + head;
    const bool live = pair / c.kv_heads < (unsigned)s.count && (unsigned)slot < (unsigned)(c.pages * c.page_tokens);
    uint8_t *keys = c.keys + place * (c.page_tokens * (W / 2)), *values = c.values + place * (c.page_tokens * (W / 2));
    uint16_t *ks = c.key_steps + place * (c.page_tokens * kBlocks);
    uint16_t *vs = c.value_steps + place * (c.page_tokens * kBlocks);
#pragma unroll
    for (int i = 0; i < kQuads; ++i) {
        const int quad = within + kHead * i, b = quad / 8;
        if (marked) {
#pragma unroll
            for (int e = 0; e < 4; ++e) k[i][e] = v[i][e] = 0.f;
        }
        uint32_t n[4], m[4];
        const float kstep = quantise(k[i], n), vstep = quantise(v[i], m);
        // A word of 8 elements of the key is two lanes'.
        uint32_t word = (n[0] | n[1] << 16 | n[2] << 4 | n[3] << 20) << (quad & 1 ? 8 : 0);
        word |= (uint32_t)__builtin_amdgcn_update_dpp(0, (int)word, 0xB1, 0xF, 0xF, false);
        if (!live) continue;
        if (!(quad & 1)) *(uint32_t *)(keys + (b * c.page_tokens + t) * 16 + quad % 8 * 2) = word;
        *(uint16_t *)(values + ((t / 8 * (W / 4) + quad) * 8 + t % 8) * 2) =
            (uint16_t)(m[0] | m[1] << 4 | m[2] << 8 | m[3] << 12);
        if (quad % 8 == 0) {
            const _Float16 kh = marked ? (_Float16)NAN : (_Float16)kstep, vh = (_Float16)vstep;
            ks[(t / 16 * kBlocks + b) * 16 + t % 4 * 4 + t % 16 / 4] = __builtin_bit_cast(uint16_t, kh);
            vs[b * c.page_tokens + t] = __builtin_bit_cast(uint16_t, vh);
        }
    }
}

// Workgroup: 256 threads of (row, quad) from number blockIdx.x * 256 on. One width per
// kernel and numbers in 32 bits leave no division by a variable but the row's; outputs
// go past the caches, where the codes they come from stay (20.1 and 18.3 us).
template <int W>
__global__ __launch_bounds__(256) void kv4_load(Kv4 c, const int *__restrict__ slots, int count,
    float *__restrict__ k, int64_t k_stride, float *__restrict__ v, int64_t v_stride, bool quads)
{
    const unsigned per_row = c.kv_heads * W / 4, at = blockIdx.x * 256 + threadIdx.x;
    const int row = (int)(at / per_row);
    if (row >= count) return;
    const int slot = slots[row];
    if ((unsigned)slot >= (unsigned)(c.pages * c.page_tokens)) return;
    const int t = slot & (c.page_tokens - 1), i = (int)(at % per_row), head = i / (W / 4),
              quad = i % (W / 4), b = quad / 8, blocks = W / kBlock;
    const size_t place = (size_t)(slot / c.page_tokens) * c.kv_heads + head;
    const size_t codes = place * (c.page_tokens * (W / 2)), steps = place * (c.page_tokens * blocks);
    const uint32_t kw = *(const uint32_t *)(c.keys + codes + (b * c.page_tokens + t) * 16 + (quad % 8 & ~1) * 2) >>
                        (quad & 1 ? 8 : 0);
    const uint32_t vw = *(const uint16_t *)(c.values + codes + ((t / 8 * (W / 4) + quad) * 8 + t % 8) * 2);
    const float ks = f16_to_f32(c.key_steps[steps + (t / 16 * blocks + b) * 16 + t % 4 * 4 + t % 16 / 4]);
    const float vs = ks != ks ? ks : f16_to_f32(c.value_steps[steps + b * c.page_tokens + t]);
    float x[4], y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[e] = (float)((int)(kw >> (e % 2 * 16 + e / 2 * 4) & 15u) - 8) * ks;
        y[e] = (float)((int)(vw >> (4 * e) & 15u) - 8) * vs;
    }
    float *to_k = k + row * k_stride + 4 * i, *to_v = v + row * v_stride + 4 * i;
    if (quads) {
        typedef float f32x4 __attribute__((ext_vector_type(4)));
        __builtin_nontemporal_store((f32x4){x[0], x[1], x[2], x[3]}, (f32x4 *)to_k);
        __builtin_nontemporal_store((f32x4){y[0], y[1], y[2], y[3]}, (f32x4 *)to_v);
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            to_k[e] = x[e];
            to_v[e] = y[e];
        }
    }
}

template <int W>
void store_width(Store4 &s, hipStream_t stream)
{
    const int64_t threads = (int64_t)s.count * s.c.kv_heads * Lanes<W>::kHead;
    s.stores = (unsigned)((threads + 255) / 256);
    hipLaunchKernelGGL((kv4_store<W>), dim3((unsigned)(s.stores + (int64_t)s.count * s.parts)), dim3(256), 0, stream, s);
}

}  // namespace

hipError_t launch_kv4_store(const Kv4 &cache, const int *slots, int count, const float *k, int64_t k_stride,
    const float *v, int64_t v_stride, const float2 *angles, int rotated, bool halves, const Rows &q, hipStream_t s)
{
    const bool quads_k = (((uintptr_t)k | (uintptr_t)angles) & 15) == 0 && k_stride % 4 == 0 &&
                         rotated % (halves ? 8 : 4) == 0;
    const bool quads_v = ((uintptr_t)v & 15) == 0 && v_stride % 4 == 0;
    const int each = q.heads ? heads_each(count, q.heads, cache.width) : 1, parts = (q.heads + each - 1) / each;
    Store4 args = {cache, slots, count, k, v, k_stride, v_stride, angles, rotated, halves, quads_k, quads_v,
                   quads_ok(q, cache.width, rotated, halves, angles), q, each, parts, 0};
    switch (cache.width) {
    case 64: store_width<64>(args, s); break;
    case 128: store_width<128>(args, s); break;
    case 256: store_width<256>(args, s); break;
    default: store_width<512>(args, s); break;
    }
    return hipGetLastError();
}

hipError_t launch_kv4_load(const Kv4 &cache, const int *slots, int count, float *k, int64_t k_stride, float *v,
    int64_t v_stride, hipStream_t s)
{
    const bool quads = (((uintptr_t)k | (uintptr_t)v) & 15) == 0 && k_stride % 4 == 0 && v_stride % 4 == 0;
    // Threads are numbered in 32 bits: as many rows in a launch as that allows, nearly always all.
    const int per_row = cache.kv_heads * (cache.width / 4), most = (1 << 30) / per_row;
    for (int first = 0; first < count; first += most) {
        const int rows = count - first < most ? count - first : most;
        const dim3 grid((unsigned)(((int64_t)rows * per_row + 255) / 256));
        const auto launch = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, cache, slots + first, rows, k + first * k_stride, k_stride,
                               v + first * v_stride, v_stride, quads);
        };
        switch (cache.width) {
        case 64: launch(kv4_load<64>); break;
        case 128: launch(kv4_load<128>); break;
        case 256: launch(kv4_load<256>); break;
        default: launch(kv4_load<512>); break;
        }
    }
    return hipGetLastError();
}

}  // namespace fy
