// Causal attention over a paged 8-bit cache (include/fyodor_hip_serving.h).
#include <math.h>

#include "device.h"
#include "serving.h"

namespace fy {
namespace {

typedef _Float16 half2 __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kStep = 64;   // positions per step of a wavefront
constexpr int kRows = 16;   // query rows per tile
constexpr int kWaves = 4;

// The positions that a tile of query rows sees and how they are split: steps
// [begin, end) of 64 positions in `active` shares of `chunk`.
struct Range {
    int lowest, highest;   // positions, highest < 0: none
    int begin, chunk, active, end;
};

// Request r's rows, the first position and whether it brings any.
struct Request {
    int begin, rows;   // first row; rows of one KV head: tokens x group
    int64_t first;     // position of its first token
};

__device__ __forceinline__ Request request_of(const Kv8Attention &a, int r)
{
    const int start = a.starts[r], stop = a.starts[r + 1];
    const int begin = max(start, 0), end = min(stop, a.count), tokens = min(end - begin, a.max_tokens);
    return {begin, tokens > 0 ? tokens * (a.heads / a.cache.kv_heads) : 0,
            (int64_t)a.lengths[r] - ((int64_t)stop - begin)};
}

__device__ __forceinline__ Range range_of(const Kv8Attention &a, const Request &q, int tile, int rows, int splits,
    int least)
{
    const int group = a.heads / a.cache.kv_heads;
    // Positions of a whole step past the last one still fit 31 bits.
    const int64_t most = min((int64_t)a.table_stride * a.cache.page_tokens - 1, (int64_t)INT32_MAX - 2 * kStep);
    const int64_t low = q.first + rows * tile / group, high = q.first + (min(rows * tile + rows, q.rows) - 1) / group;
    Range g;
    g.highest = (int)(high < 0 ? -1 : high < most ? high : most);
    g.lowest = (int)(a.window && low >= a.window ? (low - a.window < most ? low - a.window + 1 : most) : 0);
    g.begin = g.lowest / kStep;
    g.end = g.highest < 0 ? g.begin : g.highest / kStep + 1;
    const int steps = g.end - g.begin;
    g.chunk = max(least, (steps + splits - 1) / splits);
    g.active = steps > 0 ? (steps + g.chunk - 1) / g.chunk : 1;
    return g;
}

// 8 codes as fp16, exactly: the byte with its sign bit flipped under the
// exponent of 1024 is 1152 + code.
__device__ __forceinline__ half8 codes_f16(uint32_t lo, uint32_t hi)
{
    lo ^= 0x80808080u;
    hi ^= 0x80808080u;
    const half2 bias = {(_Float16)1152.f, (_Float16)1152.f};
    union { half8 v; half2 p[4]; } u;
    u.p[0] = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u)) - bias;
    u.p[1] = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u)) - bias;
    u.p[2] = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u)) - bias;
    u.p[3] = __builtin_bit_cast(half2, __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u)) - bias;
    return u.v;
}

// x as two fp16 pieces, hi + lo = x to 2^-22.
__device__ __forceinline__ void split_f16(const float *x, half8 &hi, half8 &lo)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    union { half8 v; half2 p[4]; } h, l;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f32x2 v = {x[2 * i], x[2 * i + 1]};
        h.p[i] = __builtin_convertvector(v, half2);
        const f32x2 r = {v.x - (float)h.p[i].x, v.y - (float)h.p[i].y};
        l.p[i] = __builtin_convertvector(r, half2);
    }
    hi = h.v;
    lo = l.v;
}

// The largest over lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float column_max(float v)
{
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float column_sum(float v)
{
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

template <int W>
__global__ __launch_bounds__(64 * kWaves, W <= 128 ? 2 : 1) void kv8_rows(Kv8Attention a, int splits, int least,
    float *__restrict__ partials)
{
    constexpr int C = W / 64, D = W / 16;
    const Kv8 &c = a.cache;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, part = lane >> 4;
    const int group = a.heads / c.kv_heads, r = blockIdx.y;
    int x = blockIdx.x;
    const int kvh = x % c.kv_heads;
    x /= c.kv_heads;
    const int sp = x % splits, tile = x / splits;
    const Request rq = request_of(a, r);
    if (kRows * tile >= rq.rows) return;
    const Range g = range_of(a, rq, tile, kRows, splits, least);
    if (sp >= g.active) return;

    const int row = kRows * tile + col, row_in = min(row, rq.rows - 1), token = row_in / group;
    const int head = kvh * group + row_in % group;
    const int64_t p = rq.first + token;
    const int last = row < rq.rows ? (int)(p < g.highest ? p : g.highest) : -1;
    const int first = (int)(a.window && p >= a.window ? (p - a.window < g.highest ? p - a.window + 1 : g.highest + 1) : 0);

    // The row's q in two pieces, scaled by a power of two.
    half8 qh[2 * C], ql[2 * C];
    float qscale;
    {
        const float *q = a.q + (rq.begin + token) * a.q_stride + (int64_t)head * W + 16 * part;
        float v[16 * C];
        if (((uintptr_t)a.q & 15) == 0 && a.q_stride % 4 == 0) {
#pragma unroll
            for (int i = 0; i < C; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) *(float4 *)(v + 16 * i + 4 * e) = *(const float4 *)(q + 64 * i + 4 * e);
        } else {
#pragma unroll
            for (int i = 0; i < C; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) v[16 * i + e] = q[64 * i + e];
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 16 * C; ++i) top = fmaxf(top, fabsf(v[i]));
        const int e = 14 - __builtin_amdgcn_frexp_expf(column_max(top));
#pragma unroll
        for (int i = 0; i < 16 * C; ++i) v[i] = ldexpf(v[i], e);
#pragma unroll
        for (int i = 0; i < 2 * C; ++i) split_f16(v + 8 * i, qh[i], ql[i]);
        // exp(s) = exp2(s log2 e), q back to its size.
        qscale = ldexpf(a.scale * 1.44269504f, -e);
    }

    const int *table = a.table + (size_t)r * a.table_stride;
    const int shift = 31 - __builtin_clz(c.page_tokens), within = c.page_tokens - 1;
    // Lane l reads keys of the granule of 16 positions (l % 16) / 4 of a step and
    // holds scores and values of granule l / 16.
    auto page_of = [&](int at) {
        const int j = at >> shift;
        int page = -1;
        if (at <= g.highest && j < a.table_stride) page = table[j];
        return (unsigned)page < (unsigned)c.pages ? page : -1;
    };
    auto place_of = [&](int page) { return (size_t)max(page, 0) * c.kv_heads + kvh; };
    const size_t plane = (size_t)c.page_tokens * W;

    f32x4 O[D];
#pragma unroll
    for (int d = 0; d < D; ++d) O[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const int stop = min(g.begin + (sp + 1) * g.chunk, g.end);
    for (int step = g.begin + sp * g.chunk + wave; step < stop; step += kWaves) {
        const int kat = kStep * step + 16 * (col >> 2), vat = kStep * step + 16 * part;
        const int kpage = page_of(kat), vpage = page_of(vat);
        const int8_t *kb = c.keys + place_of(kpage) * plane + (part * c.page_tokens + (kat & within) + (col & 3)) * 16;
        const int8_t *vb = c.values + place_of(vpage) * plane + ((vat & within) * W + 16 * col);
        uint4 kr[4][C], vr[D];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < C; ++i) kr[t][i] = *(const uint4 *)(kb + (size_t)64 * c.page_tokens * i + 64 * t);
#pragma unroll
        for (int d = 0; d < D; ++d) vr[d] = *(const uint4 *)(vb + 256 * d);
        float ks = 0.f, vs = 0.f;
        if (vpage >= 0) {
            ks = c.key_scales[place_of(vpage)];
            vs = c.value_scales[place_of(vpage)];
        }
        f32x4 S[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            S[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const half8 k0 = codes_f16(kr[t][i].x, kr[t][i].y), k1 = codes_f16(kr[t][i].z, kr[t][i].w);
                S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qh[2 * i], S[t], 0, 0, 0);
                S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql[2 * i], S[t], 0, 0, 0);
                S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qh[2 * i + 1], S[t], 0, 0, 0);
                S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql[2 * i + 1], S[t], 0, 0, 0);
            }
        }
        // Scores in powers of two with the exponent of the page's value scale
        // added, so that weights times that scale are what is normalised.
        const int e = __builtin_amdgcn_frexp_expf(vs);
        float mant = __builtin_amdgcn_frexp_mantf(vs);
        if (!__builtin_isfinite(vs)) mant = NAN;
        const float scale = __builtin_isfinite(ks) ? ks * qscale : NAN;
        const int from = vpage >= 0 ? first - vat : 16, to = vpage >= 0 ? last - vat : -1;
        float w[16];
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float s = S[i >> 2][i & 3] * scale;
            w[i] = i >= from && i <= to ? s : -INFINITY;
            top = fmaxf(top, w[i]);
        }
        const float next = fmaxf(m, ceilf(column_max(top + e)));
        const float base = next == -INFINITY ? 0.f : next;
        const float alpha = __builtin_amdgcn_exp2f(m - base);
        m = next;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float s = __builtin_fmaf(S[i >> 2][i & 3], scale, e - base + 15.f);
            const bool seen = i >= from && i <= to;
            const float v = seen ? __builtin_amdgcn_exp2f(s) : 0.f;
            sum += v;
            w[i] = seen ? v * mant : 0.f;
        }
        l = l * alpha + ldexpf(sum, -e);
        half8 ph[2], pl[2];
        split_f16(w, ph[0], pl[0]);
        split_f16(w + 8, ph[1], pl[1]);
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const half8 v0 = codes_f16(vr[d].x, vr[d].y), v1 = codes_f16(vr[d].z, vr[d].w);
            f32x4 o = O[d] * alpha;
            o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, ph[0], o, 0, 0, 0);
            o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pl[0], o, 0, 0, 0);
            o = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, ph[1], o, 0, 0, 0);
            O[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pl[1], o, 0, 0, 0);
        }
    }
    l = column_sum(l);

    // The wavefronts' partial softmaxes meet in LDS, 64 columns at a time.
    __shared__ float ml[2][kWaves][kRows];
    __shared__ __align__(16) float po[kWaves][kRows][64 + 4];
    if (part == 0) {
        ml[0][wave][col] = m;
        ml[1][wave][col] = l;
    }
    const int mrow = threadIdx.x >> 4, mcol = 4 * (threadIdx.x & 15);   // this thread's output: 4 columns of a row
    const int out_row = kRows * tile + mrow;
    const size_t prow = ((size_t)r * a.max_tokens * group + out_row) * c.kv_heads + kvh;
#pragma unroll
    for (int i = 0; i < C; ++i) {
        if (i) __syncthreads();
#pragma unroll
        for (int d = 0; d < 4; ++d) *(f32x4 *)&po[wave][col][16 * d + 4 * part] = O[4 * i + d];
        __syncthreads();
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[0][w][mrow]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(ml[0][w][mrow] - base);
            total += ml[1][w][mrow] * f;
            o += *(const f32x4 *)&po[w][mrow][mcol] * f;
        }
        if (out_row < rq.rows) {
            if (g.active > 1) {
                *(f32x4 *)(partials + (prow * splits + sp) * W + 64 * i + mcol) = o;
                if (i == 0 && mcol == 0) {
                    float *pm = partials + (size_t)a.requests * a.max_tokens * a.heads * splits * W + 2 * (prow * splits + sp);
                    pm[0] = top;
                    pm[1] = total;
                }
            } else {
                float *out = a.out + (rq.begin + out_row / group) * a.out_stride +
                             (int64_t)(kvh * group + out_row % group) * W + 64 * i + mcol;
#pragma unroll
                for (int k = 0; k < 4; ++k) out[k] = total == 0.f ? 0.f : o[k] / total;
            }
        }
    }
}

// out = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M) over a row's shares.
// Workgroup (row of a KV head and request).
template <int W>
__global__ __launch_bounds__(256) void kv8_join(Kv8Attention a, int splits, int least,
    const float *__restrict__ partials)
{
    const Kv8 &c = a.cache;
    const int group = a.heads / c.kv_heads, r = blockIdx.y, kvh = blockIdx.x % c.kv_heads, row = blockIdx.x / c.kv_heads;
    const Request rq = request_of(a, r);
    if (row >= rq.rows) return;
    const Range g = range_of(a, rq, row / kRows, kRows, splits, least);
    if (g.active <= 1) return;
    const size_t prow = ((size_t)r * a.max_tokens * group + row) * c.kv_heads + kvh;
    const float *pm = partials + (size_t)a.requests * a.max_tokens * a.heads * splits * W + 2 * prow * splits;
    constexpr int kCols = W / 4, kParts = 256 / kCols < 1 ? 1 : 256 / kCols;
    __shared__ f32x4 po[kParts][kCols];
    const int col = threadIdx.x % kCols, part = threadIdx.x / kCols;
    float top = -INFINITY;
    for (int s = 0; s < g.active; ++s) top = fmaxf(top, pm[2 * s]);
    const float base = top == -INFINITY ? 0.f : top;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    float total = 0.f;
    for (int s = part; s < g.active; s += kParts) {
        const float f = __builtin_amdgcn_exp2f(pm[2 * s] - base);
        o += *(const f32x4 *)(partials + (prow * splits + s) * W + 4 * col) * f;
    }
    for (int s = 0; s < g.active; ++s) total += pm[2 * s + 1] * __builtin_amdgcn_exp2f(pm[2 * s] - base);
    po[part][col] = o;
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int k = 1; k < kParts; ++k) o += po[k][col];
    float *out = a.out + (rq.begin + row / group) * a.out_stride + (int64_t)(kvh * group + row % group) * W + 4 * col;
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = total == 0.f ? 0.f : o[k] / total;
}

// How the work is split: `splits` workgroups at most share a tile's
// positions, at least `least` steps each.
struct Plan {
    int splits, least;
};

Plan plan_of(int requests, int max_tokens, int max_length, int heads, int kv_heads, int window)
{
    const int64_t tiles = ((int64_t)max_tokens * (heads / kv_heads) + kRows - 1) / kRows;
    const int64_t groups = tiles * kv_heads * requests;
    int64_t range = max_length;
    if (window && (int64_t)window + max_tokens < range) range = (int64_t)window + max_tokens;
    const int64_t steps = (range + kStep - 1) / kStep + 1;
    int64_t splits = (1024 + groups - 1) / groups;
    if (splits > 64) splits = 64;
    if (splits > (steps + kWaves - 1) / kWaves) splits = (steps + kWaves - 1) / kWaves;
    if (splits < 1) splits = 1;
    return {(int)splits, kWaves};
}

size_t row_bytes(int requests, int max_tokens, int heads, int width)
{
    return (size_t)requests * max_tokens * heads * (width + 2) * sizeof(float);
}

template <int W>
hipError_t launch_rows(const Kv8Attention &a, Plan p, float *partials, hipStream_t s)
{
    const int group = a.heads / a.cache.kv_heads;
    const int64_t tiles = ((int64_t)a.max_tokens * group + kRows - 1) / kRows;
    hipLaunchKernelGGL((kv8_rows<W>), dim3((unsigned)(tiles * p.splits * a.cache.kv_heads), (unsigned)a.requests),
                       dim3(64 * kWaves), 0, s, a, p.splits, p.least, partials);
    if (p.splits > 1)
        hipLaunchKernelGGL((kv8_join<W>), dim3((unsigned)(a.max_tokens * a.heads), (unsigned)a.requests), dim3(256), 0,
                           s, a, p.splits, p.least, partials);
    return hipGetLastError();
}

}  // namespace

size_t kv8_attention_workspace(int requests, int max_tokens, int max_length, int heads, int kv_heads, int width,
    int window)
{
    const Plan p = plan_of(requests, max_tokens, max_length, heads, kv_heads, window);
    return p.splits > 1 ? p.splits * row_bytes(requests, max_tokens, heads, width) : 0;
}

hipError_t launch_kv8_attention(const Kv8Attention &a, void *workspace, size_t workspace_bytes, hipStream_t s)
{
    Plan p = plan_of(a.requests, a.max_tokens, a.max_length, a.heads, a.cache.kv_heads, a.window);
    const size_t each = row_bytes(a.requests, a.max_tokens, a.heads, a.cache.width);
    if (workspace_bytes / each < (size_t)p.splits) p.splits = (int)(workspace_bytes / each);
    if (p.splits < 1) p.splits = 1;
    switch (a.cache.width) {
    case 64: return launch_rows<64>(a, p, (float *)workspace, s);
    case 128: return launch_rows<128>(a, p, (float *)workspace, s);
    case 256: return launch_rows<256>(a, p, (float *)workspace, s);
    default: return launch_rows<512>(a, p, (float *)workspace, s);
    }
}

}  // namespace fy
