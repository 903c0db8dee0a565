// What attention over a paged cache is made of whatever the cache holds
// (attention_kv8.hip, attention_kv4.hip: A is its arguments): operands in fp16
// pieces, reductions over a score's column, which workgroup takes what, and the
// join of shares.
#pragma once
#include <float.h>
#include <math.h>

#include "device.h"
#include "kv8_shares.h"

namespace fy {
namespace {

typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// x as two fp16 pieces, hi + lo = x to 2^-22; the remainder x - hi is exact.
__device__ __forceinline__ void split_f16(const float *x, half8 &hi, half8 &lo)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    union { half8 v; half2 p[4]; } h, l;
    float minus = -1.f;
    asm("" : "+s"(minus));   // keeps the product: one v_fma_mix_f32 instead of a conversion and a subtraction
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x2 v = {x[2 * i], x[2 * i + 1]};
        h.p[i] = __builtin_convertvector(v, half2);
        const f32x2 r = {__builtin_fmaf((float)h.p[i].x, minus, v.x), __builtin_fmaf((float)h.p[i].y, minus, v.y)};
        l.p[i] = __builtin_convertvector(r, half2);
    }
    hi = h.v;
    lo = l.v;
}

// max / sum over lanes l and l ^ 32 (and l ^ 16), in all of them.
__device__ __forceinline__ float halves_max(float v)
{
    const int b = __builtin_bit_cast(int, v);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return fmaxf(__builtin_bit_cast(float, (int)r[0]), __builtin_bit_cast(float, (int)r[1]));
}
__device__ __forceinline__ float halves_sum(float v)
{
    const int b = __builtin_bit_cast(int, v);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __builtin_bit_cast(float, (int)r[0]) + __builtin_bit_cast(float, (int)r[1]);
}
__device__ __forceinline__ float column_max(float v)
{
    const int b = __builtin_bit_cast(int, v);
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    return halves_max(fmaxf(__builtin_bit_cast(float, (int)r[0]), __builtin_bit_cast(float, (int)r[1])));
}
__device__ __forceinline__ float column_sum(float v)
{
    const int b = __builtin_bit_cast(int, v);
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    return halves_sum(__builtin_bit_cast(float, (int)r[0]) + __builtin_bit_cast(float, (int)r[1]));
}

// A score times its scale less the maximum, rounded once at the end, may be above
// 0 by half the last place of the maximum. From this maximum on that is more than
// weights in fp16, up to 2^15 of the 2^16 they hold, have room for.
constexpr float kFar = 0x1p22f;
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) >= kFar && m != -INFINITY; }

// What a row's sum of weights makes of its outputs (times A::kLess, by which sums are
// held smaller). Without weights the row saw nothing (no maximum) and gives zeros,
// or its scores were beyond fp32.
__device__ __forceinline__ float inverse_of(float total, float top)
{
    return total == 0.f ? (top == -INFINITY ? 0.f : NAN) : 1.f / total;
}

// The request and the tile of kTile rows of number `index` over the requests
// of more than most_rows rows, in order (request < 0: past the last). Later
// tokens see more: a request's last tile comes first.
struct TileOf {
    int request, tile;
};

template <int kTile, class A>
__device__ __forceinline__ TileOf tile_of(const A &a, int most_rows, int index)
{
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < a.requests; base += 64) {
        const int r = base + lane, rows = r < a.requests ? request_of(a, r).rows : 0;
        const int tiles = rows > most_rows ? (rows + kTile - 1) / kTile : 0;
        int sum = tiles;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int v = __shfl_up(sum, o, 64);
            if (lane >= o) sum += v;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(sum > index);
        if (past) {
            const int at = __builtin_ctzll(past);
            return {base + at, __builtin_amdgcn_readlane(sum, at) - 1 - index};
        }
        index -= __builtin_amdgcn_readlane(sum, 63);
    }
    return {-1, 0};
}

// The item of number `index` over the requests of a few rows, in order (request
// < 0: past the last). The shares that its tile does not have are no work.
struct ItemOf {
    int request;
    Item item;
};

template <class A>
__device__ __forceinline__ ItemOf item_of(const A &a, const Split &split, int most_rows, int index)
{
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < a.requests; base += 64) {
        const int r = base + lane;
        const Items items = r < a.requests ? items_of(a, split, request_of(a, r), most_rows) : Items{0, 0};
        int sum = items.tiles * items.shares;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int v = __shfl_up(sum, o, 64);
            if (lane >= o) sum += v;
        }
        const uint64_t past = __builtin_amdgcn_ballot_w64(sum > index);
        if (past) {
            const int at = __builtin_ctzll(past);
            return {base + at, item_at(__builtin_amdgcn_readlane(items.tiles, at),
                                       __builtin_amdgcn_readlane(sum, at) - 1 - index)};
        }
        index -= __builtin_amdgcn_readlane(sum, 63);
    }
    return {-1, {0, 0}};
}

// LDS writes and reads of the workgroup up to here; global loads stay in flight.
__device__ __forceinline__ void lds_barrier()
{
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
    __builtin_amdgcn_sched_barrier(0);
}

// The same among a wavefront's lanes, where others are not waited for: what lanes wrote may be read by the
// wavefront's others after it, and what they read overwritten. (Its LDS operations are in order, so this
// costs nothing; it keeps the compiler from moving one before the other.)
__device__ __forceinline__ void lds_wave()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// out = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M) over a row's shares.
// Requests of a few rows: workgroup (place, row of a KV head).
template <int W, class A>
__device__ __forceinline__ void join_row(const A &a, const Split &split, int most_rows, int index)
{
    const auto &c = a.cache;
    const int group = a.heads / c.kv_heads, place = index / (split.tile * c.kv_heads), kvh = index % c.kv_heads,
              within = index / c.kv_heads % split.tile;
    int r = place, row = within;
    if constexpr (W > 256) {
        if (split.listed) {
            const TileOf at = tile_of<kRows>(a, 0, place);
            if (at.request < 0) return;
            r = at.request;
            row += kRows * at.tile;
        }
    }
    const Request rq = request_of(a, r);
    if (row >= rq.rows || rq.rows > most_rows) return;
    const Range g = range_of(a, rq, row / kRows, kRows, split.most, split.least);
    if (g.active <= 1) return;
    const Share from = split.share(c.kv_heads, place, kvh, within, 0, W);
    constexpr int kCols = W / 4, kParts = 256 / kCols;
    __shared__ f32x4 po[kParts][kCols];
    __shared__ float fs[kMostSplits];
    const int lane = threadIdx.x & 63, col = threadIdx.x % kCols, part = threadIdx.x / kCols;
    // Shares' outputs are requested before their weights are known; lane s forms
    // the weight of share s.
    const f32x4 *po_at = (const f32x4 *)from.o + col;
    constexpr int kOnce = kMostSplits / kParts;
    f32x4 v[kOnce];
#pragma unroll
    for (int k = 0; k < kOnce; ++k) v[k] = po_at[(size_t)min(part + kParts * k, g.active - 1) * kCols];
    const float2 mine = lane < g.active ? from.ml[lane] : make_float2(-INFINITY, 0.f);
    const float top = wave_reduce<true>(mine.x), base = top == -INFINITY ? 0.f : top;
    const float f = __builtin_amdgcn_exp2f(mine.x - base), total = wave_sum(mine.y * f);
    if (threadIdx.x < kMostSplits) fs[lane] = f;
    __syncthreads();
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kOnce; ++k) o += v[k] * fs[part + kParts * k];   // (shares past the last weigh 0)
    po[part][col] = o;
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int k = 1; k < kParts; ++k) o += po[k][col];
    float *out = a.out + (rq.begin + row / group) * a.out_stride + (int64_t)(kvh * group + row % group) * W + 4 * col;
    const float inverse = inverse_of(total, top);
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = o[k] * A::kLess * inverse;
}

// Wide tiles: workgroup (tile, 16 of its rows, KV head), a wavefront every
// fourth row.
constexpr int kJoinParts = kWideRows / 16;
template <int W, class A>
__device__ __forceinline__ void join_wide(const A &a, const Split &split, int most_rows, int index)
{
    const auto &c = a.cache;
    const int kvh = index % c.kv_heads, lane = threadIdx.x & 63, group = a.heads / c.kv_heads;
    const int part = index / c.kv_heads % kJoinParts, place = index / c.kv_heads / kJoinParts;
    const TileOf at = tile_of<kWideRows>(a, most_rows, place);
    if (at.request < 0) return;
    const Request rq = request_of(a, at.request);
    const Range g = range_of(a, rq, at.tile, kWideRows, split.most, split.least);
    if (g.active <= 1) return;
    constexpr int kCols = W / 64;   // columns per lane
    const int first_row = kWideRows * at.tile + 16 * part;
    for (int row = first_row + (threadIdx.x >> 6); row < min(first_row + 16, rq.rows); row += 4) {
        const Share from = split.share(c.kv_heads, place, kvh, row - kWideRows * at.tile, 0, W);
        const float2 mine = lane < g.active ? from.ml[lane] : make_float2(-INFINITY, 0.f);
        const float top = wave_reduce<true>(mine.x), base = top == -INFINITY ? 0.f : top;
        const float f = __builtin_amdgcn_exp2f(mine.x - base), total = wave_sum(mine.y * f);
        float o[kCols] = {};
        for (int s = 0; s < g.active; s += 4) {
            float v[4][kCols];
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int e = 0; e < kCols; ++e) v[n][e] = from.o[min(s + n, g.active - 1) * W + 64 * e + lane];
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                const float weight = lane_value(f, s + n);   // 0 past the last share
#pragma unroll
                for (int e = 0; e < kCols; ++e) o[e] += v[n][e] * weight;
            }
        }
        float *out = a.out + (rq.begin + row / group) * a.out_stride + (int64_t)(kvh * group + row % group) * W + lane;
        const float inverse = inverse_of(total, top);
#pragma unroll
        for (int e = 0; e < kCols; ++e) out[64 * e] = o[e] * A::kLess * inverse;
    }
}

}  // namespace
}  // namespace fy
