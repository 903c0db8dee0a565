// Causal attention over a paged 8-bit cache (include/fyodor_hip_serving.h).
//
// For a KV head, its group's heads and the request's new tokens make the rows
// of one product: row i is token i / group, head i % group of the group. With
// codes K, V and the scales a_t, b_t of position t's page,
//     s_it = (q_i . K_t) a_t scale,   out_i = sum_t e^(s_it) b_t V_t / sum_t e^(s_it).
// One pass over the positions, 64 a step: S^T = K Q^T and O^T = V^T P^T on the
// fp16 matrix cores, with the softmax's running maximum and sum (fp32, like S
// and O) per column, so that a column of S^T is already laid out as the operand
// P^T. The codes are exact in fp16. q and P go in as two fp16 pieces each
// (22 bits, the error of fp32 sums of this length; one piece would be 2^-11),
// which makes two matrix instructions of one: half the fp16 rate is this
// kernel's ceiling. b_t is a power of two times a mantissa: the power joins the
// exponent of e^s and the mantissa multiplies P, so P's fp16 pieces see what
// is summed, not codes of a page of small values. The maximum is rounded up to
// a whole power of two: rescaling by it is exact, and rare. From 2^22 on (kFar)
// the scores are rounded first, and their distances from the maximum taken after.
//
// A call of few rows reads each position once, 2 W bytes per KV head and position,
// and is bound by that; one of many rows by the matrix cores and the
// conversions and the softmax beside them. Hence two kernels, a workgroup of
// 16 rows that loads straight into the operands' lanes (kv8_rows), and one of
// 128 rows that convert each code once, in LDS (kv8_wide). What is too few
// tiles for the chip is split over the positions and joined by a second
// launch (kv8_join).
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

// Sums of weights are held without the exponent e of the value scales (-99 to 122,
// as stored): up to 2^(15 - e) for a position where outputs hold 2^15. Times kLess
// they stay in fp32 at both ends, for up to 2^30 positions; kLess joins the outputs
// at the end.
constexpr int kLessBits = -18;
constexpr float kLess = 0x1p-18f;

// What a row's sum of weights makes of its outputs (times kLess). Without weights the row saw
// nothing (no maximum) and gives zeros, or its scores were beyond fp32.
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

template <int kTile>
__device__ __forceinline__ TileOf tile_of(const Kv8Attention &a, int most_rows, int index)
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

__device__ __forceinline__ ItemOf item_of(const Kv8Attention &a, const Split &split, int most_rows, int index)
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

// Requests of a few rows: 16 rows per workgroup, whose wavefronts take every
// fourth step of its share of the positions and meet in LDS at the end. Keys
// and values go from memory straight into the operands' lanes: K and V of a
// step are requested as soon as the last step's are used up, pages a step
// before that: with a load and its use in one step the wavefronts, two per SIMD,
// waited for memory (64 requests of 500 to 8192 positions, 32 heads over 8 of
// 128, 371 MB: 105 us with the join, so 95; counted shares 86, 4.6 TB/s of the
// 5.1 that a copy reaches; 1 of 32768, 67 MB: 28 us, so 20). Registers for three
// wavefronts per SIMD measured slower.
template <int W>
__device__ __forceinline__ void few_rows(const Kv8Attention &a, int r, int kvh, int sp, int tile, const Split &split,
    int place, int most_rows, float (*ml)[kWaves][kRows], float (*po)[kRows][64 + 4])
{
    constexpr int C = W / 64, D = W / 16;
    constexpr bool kAhead = W <= 256;   // room for a step's K and V in registers
    const Kv8 &c = a.cache;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, part = lane >> 4;
    const int group = a.heads / c.kv_heads;
    const Request rq = request_of(a, r);
    if (kRows * tile >= rq.rows || rq.rows > most_rows) return;
    const Range g = range_of(a, rq, tile, kRows, split.most, split.least);
    if (sp >= g.active) return;

    // Rows past the request's last repeat it and are not written.
    const int row = min(kRows * tile + col, rq.rows - 1), token = row / group, head = kvh * group + row % group;
    const int64_t p = rq.first + token;
    const int last = (int)(p < g.highest ? p : g.highest);
    const int first = (int)(a.window && p >= a.window ? (p - a.window < g.highest ? p - a.window + 1 : g.highest + 1) : 0);
    // Positions that all rows see: up to the first row's last, from the last row's first.
    const int64_t p0 = rq.first + kRows * tile / group, p1 = rq.first + min(kRows * tile + kRows - 1, rq.rows - 1) / group;
    const int all_to = (int)(p0 < g.highest ? p0 : g.highest);
    const int all_from = (int)(a.window && p1 >= a.window ? (p1 - a.window < g.highest ? p1 - a.window + 1 : g.highest + 1) : 0);

    const int *table = a.table + (size_t)r * a.table_stride;
    const int shift = 31 - __builtin_clz(c.page_tokens), within = c.page_tokens - 1;
    const int begin = g.from(sp) + wave, stop = g.until(sp);
    // Lane l reads keys of the granule of 16 positions (l % 16) / 4 of a step and
    // holds scores and values of granule l / 16. Everything is read
    // unconditionally (positions past the last one lead to page 0).
    auto entry_of = [&](int at) {
        const int entry = table[min(at >> shift, a.table_stride - 1)];
        return at <= g.highest ? entry : -1;
    };
    auto place_of = [&](int page) { return (size_t)((unsigned)page < (unsigned)c.pages ? page : 0) * c.kv_heads + kvh; };
    const size_t plane = (size_t)c.page_tokens * W;
    int kpage, vpage;
    auto look = [&](int step) {
        kpage = entry_of(kStep * step + 16 * (col >> 2));
        vpage = entry_of(kStep * step + 16 * part);
    };
    auto keys_at = [&](int step) {
        const int at = kStep * step + 16 * (col >> 2);
        return c.keys + place_of(kpage) * plane + (part * c.page_tokens + (at & within) + (col & 3)) * 16;
    };
    auto values_at = [&](int step) {
        const int at = kStep * step + 16 * part;
        return c.values + place_of(vpage) * plane + ((at & within) * W + 16 * col);
    };
    uint4 kr[4][C], vr[D];
    float ks, vs;
    bool there;
    auto fetch_k = [&](int step) {
        const int8_t *kb = keys_at(step);
#pragma unroll
        for (int i = 0; i < C; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t) kr[t][i] = *(const uint4 *)(kb + (size_t)64 * c.page_tokens * i + 64 * t);
    };
    auto fetch_v = [&](int step) {
        const int8_t *vb = values_at(step);
        ks = c.key_scales[place_of(vpage)];
        vs = c.value_scales[place_of(vpage)];
        there = (unsigned)vpage < (unsigned)c.pages;
        if constexpr (kAhead) {
#pragma unroll
            for (int d = 0; d < D; ++d) vr[d] = *(const uint4 *)(vb + 256 * d);
        }
    };
    look(begin);

    // The row's q in two pieces, scaled by a power of two; the scale's sign goes with it.
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
        if constexpr (kAhead) {
            fetch_k(begin);
            fetch_v(begin);
            look(begin + kWaves);
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 16 * C; ++i) top = fmaxf(top, fabsf(v[i]));
        const int e = 14 - __builtin_amdgcn_frexp_expf(column_max(top));
#pragma unroll
        for (int i = 0; i < 16 * C; ++i) v[i] = ldexpf(a.scale < 0.f ? -v[i] : v[i], e);
#pragma unroll
        for (int i = 0; i < 2 * C; ++i) split_f16(v + 8 * i, qh[i], ql[i]);
        // exp(s) = exp2(s log2 e), q back to its size.
        qscale = ldexpf(fabsf(a.scale) * 1.44269504f, -e);
    }

    f32x4 O[D];
#pragma unroll
    for (int d = 0; d < D; ++d) O[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    bool far = false;
    uint64_t saw = 0;   // lanes that had a score
    for (int step = begin; step < stop; step += kWaves) {
        const int8_t *vb = nullptr;
        if constexpr (!kAhead) {
            fetch_k(step);
            fetch_v(step);
            vb = values_at(step);
            look(step + kWaves);
        }
        f32x4 S[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) S[t] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < C; ++i) {
            half8 k[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) k[t] = codes_f16(kr[t][i].x, kr[t][i].y);
#pragma unroll
            for (int t = 0; t < 4; ++t) S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t], qh[2 * i], S[t], 0, 0, 0);
#pragma unroll
            for (int t = 0; t < 4; ++t) S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t], ql[2 * i], S[t], 0, 0, 0);
#pragma unroll
            for (int t = 0; t < 4; ++t) k[t] = codes_f16(kr[t][i].z, kr[t][i].w);
#pragma unroll
            for (int t = 0; t < 4; ++t) S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t], qh[2 * i + 1], S[t], 0, 0, 0);
#pragma unroll
            for (int t = 0; t < 4; ++t) S[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t], ql[2 * i + 1], S[t], 0, 0, 0);
        }
        if constexpr (kAhead) fetch_k(step + kWaves);
        // Scores in powers of two with the exponent of the page's value scale
        // added, so that weights times that scale are what is normalised, by a
        // whole power of two. A page that reads as NaN makes the rows that see
        // it NaN by their sum alone.
        const int at = kStep * step, pos = at + 16 * part;
        const bool fine = __builtin_isfinite(ks) && __builtin_isfinite(vs);
        float scale = fine ? fmaxf(fabsf(ks) * qscale, 0x1p-126f) : 1.f;   // above 0: keeps minus infinity
        const int e = fine ? __builtin_amdgcn_frexp_expf(vs) : 0;
        const float mant = fine ? __builtin_amdgcn_frexp_mantf(vs) : 1.f;
        if (there && !fine && first <= pos + 15 && last >= pos) l = NAN;
        if (all_from > at || all_to < at + kStep - 1 || __builtin_amdgcn_ballot_w64(!there)) {
            const int from = there ? max(first - pos, 0) : 16, to = min(last - pos, 15);
#pragma unroll
            for (int i = 0; i < 16; ++i) S[i >> 2][i & 3] = i >= from && i <= to ? S[i >> 2][i & 3] : -INFINITY;
        }
        float best = S[0][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) best = fmaxf(best, S[i >> 2][i & 3]);
        saw |= __builtin_amdgcn_ballot_w64(best > -INFINITY);
        const float top = __builtin_fmaf(best, scale, e);
        if (__builtin_amdgcn_ballot_w64(top > m)) {
            const float next = fmaxf(m, ceilf(column_max(top)));
            const float alpha = __builtin_amdgcn_exp2f(m - (next == -INFINITY ? 0.f : next));
            m = next;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < D; ++d) O[d] *= alpha;
            far = __builtin_amdgcn_ballot_w64(is_far(m));
        }
        const float base = m == -INFINITY ? 0.f : m;
        float add = e - base + 15.f;
        if (far) {
#pragma unroll
            for (int i = 0; i < 16; ++i) S[i >> 2][i & 3] = __builtin_fmaf(S[i >> 2][i & 3], scale, e) - base;
            scale = 1.f;
            add = 15.f;
        }
        half8 ph[2], pl[2];
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(S[2 * n + (i >> 2)][i & 3], scale, add));
                sum[i & 1] += v;
                w[i] = v * mant;
            }
            split_f16(w, ph[n], pl[n]);
        }
        l += ldexpf(sum[0] + sum[1], kLessBits - e);
#pragma unroll
        for (int d0 = 0; d0 < D; d0 += 4) {
            uint4 v[4];
#pragma unroll
            for (int d = 0; d < 4; ++d) v[d] = kAhead ? vr[d0 + d] : *(const uint4 *)(vb + 256 * (d0 + d));
            half8 x[4];
#pragma unroll
            for (int d = 0; d < 4; ++d) x[d] = codes_f16(v[d].x, v[d].y);
#pragma unroll
            for (int d = 0; d < 4; ++d) O[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[d], ph[0], O[d0 + d], 0, 0, 0);
#pragma unroll
            for (int d = 0; d < 4; ++d) O[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[d], pl[0], O[d0 + d], 0, 0, 0);
#pragma unroll
            for (int d = 0; d < 4; ++d) x[d] = codes_f16(v[d].z, v[d].w);
#pragma unroll
            for (int d = 0; d < 4; ++d) O[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[d], ph[1], O[d0 + d], 0, 0, 0);
#pragma unroll
            for (int d = 0; d < 4; ++d) O[d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[d], pl[1], O[d0 + d], 0, 0, 0);
        }
        if constexpr (kAhead) {
            fetch_v(step + kWaves);
            look(step + 2 * kWaves);
        }
    }
    l = column_sum(l);
    if (m == -INFINITY && (saw >> col & 0x0001000100010001u)) m = -FLT_MAX;   // scores, none in fp32

    // The wavefronts' partial softmaxes meet in LDS, 64 columns at a time.
    if (part == 0) {
        ml[0][wave][col] = m;
        ml[1][wave][col] = l;
    }
    const int mrow = threadIdx.x >> 4, mcol = 4 * (threadIdx.x & 15);   // this thread's output: 4 columns of a row
    const int out_row = kRows * tile + mrow;
    const Share to = split.share(c.kv_heads, place, kvh, split.listed ? mrow : out_row, sp, W);
    const bool aligned = ((uintptr_t)a.out & 15) == 0 && a.out_stride % 4 == 0;
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
                *(f32x4 *)(to.o + 64 * i + mcol) = o;
                if (i == 0 && mcol == 0) *to.ml = make_float2(top, total);
            } else {
                float *out = a.out + (rq.begin + out_row / group) * a.out_stride +
                             (int64_t)(kvh * group + out_row % group) * W + 64 * i + mcol;
                const float inverse = inverse_of(total, top);
                o = o * kLess * inverse;
                if (aligned) {
                    *(f32x4 *)out = o;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) out[k] = o[k];
                }
            }
        }
    }
}

template <int W>
__global__ __launch_bounds__(64 * kWaves, W <= 128 ? 2 : 1) void kv8_rows(Kv8Attention a, Split split, int most_rows)
{
    __shared__ float ml[2][kWaves][kRows];
    __shared__ __align__(16) float po[kWaves][kRows][64 + 4];
    TileOf at = {(int)blockIdx.y, (int)(blockIdx.x / a.cache.kv_heads)};
    int place = at.request, share = split.most - 1 - (int)blockIdx.z;
    if (split.packed) {
        const ItemOf it = item_of(a, split, most_rows, at.tile);
        if (it.request < 0) return;
        at = {it.request, it.item.tile};
        place = it.request;
        share = it.item.share;
    }
    if constexpr (W > 256) {   // every request runs here, prompts too
        if (split.listed) {
            place = at.tile;
            at = tile_of<kRows>(a, 0, place);
            if (at.request < 0) return;
        }
    }
    few_rows<W>(a, at.request, blockIdx.x % a.cache.kv_heads, share, at.tile, split, place, most_rows, ml, po);
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

// Many rows of one request: 32 per wavefront, 128 per group of four
// wavefronts, which share every step's keys and values, converted to fp16 in
// LDS once. KS groups take every KS-th step of the same rows and meet at the
// end. Two groups run half a step apart: while one is in its MFMAs (last
// step's outputs, this step's scores) the other does its softmax and stages
// its next codes, so that the matrix cores of a SIMD always have one of its two
// wavefronts (1024 tokens at the end of 8192 positions, 32 heads over 8 of 128:
// 345 us with one group, and copies of tiles around conditions, so 245: 528
// TFLOP/s, 1056 as issued, where the library's product of 8192^3 in fp16 reaches
// 1154). Heads of 256 fill the
// registers with one group: 420 to 450 TFLOP/s in long prompts.
template <int W, int KS>
__global__ __launch_bounds__(256 * KS) __attribute__((amdgpu_waves_per_eu(KS, KS)))
void kv8_wide(Kv8Attention a, Split split, int most_rows)
{
    constexpr int M = W / 16;       // MFMA steps of a score
    constexpr int D = W / 32;       // output tiles
    constexpr int N = W / 64;       // 16-byte pieces of K, and of V, per thread and step
    constexpr int kBytes = 2 * kStep * W;
    __shared__ __align__(16) uint8_t smem[KS][2][kBytes];   // [group][K, V]
    __shared__ float2 scales[KS][2][4];
    __shared__ float2 smem_ml[4][32];
    const Kv8 &c = a.cache;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((threadIdx.x >> 6) & 3);
    const int ks = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8), tid = threadIdx.x & 255;
    const int col = lane & 31, h = lane >> 5;
    const int group = a.heads / c.kv_heads;
    int x = blockIdx.x;
    const int kvh = x % c.kv_heads;
    x /= c.kv_heads;
    const int tiles = gridDim.x / (c.kv_heads * split.most), sp = split.most - 1 - x / tiles;
    const TileOf at_tile = tile_of<kWideRows>(a, most_rows, x % tiles);
    const int r = at_tile.request, tile = at_tile.tile;
    if (r < 0) return;
    const Request rq = request_of(a, r);
    const Range g = range_of(a, rq, tile, kWideRows, split.most, split.least);
    if (sp >= g.active) return;

    const int row = kWideRows * tile + 32 * wave + col, row_in = min(row, rq.rows - 1), token = row_in / group;
    const int head = kvh * group + row_in % group;
    const int64_t p = rq.first + token;
    // (Rows past the request's last repeat it and are not written.)
    const int last = (int)(p < g.highest ? p : g.highest);
    const int first = (int)(a.window && p >= a.window ? (p - a.window < g.highest ? p - a.window + 1 : g.highest + 1) : 0);
    // Positions that all of the wavefront's rows see.
    int all_from = first, all_to = last;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        all_from = max(all_from, __shfl_xor(all_from, o, 64));
        all_to = min(all_to, __shfl_xor(all_to, o, 64));
    }
    all_from = __builtin_amdgcn_readfirstlane(all_from);
    all_to = __builtin_amdgcn_readfirstlane(all_to);

    const int *table = a.table + (size_t)r * a.table_stride;
    const int shift = 31 - __builtin_clz(c.page_tokens), within = c.page_tokens - 1;
    // This group's steps: begin, begin + KS, ...
    const int begin = g.from(sp) + ks, stop = g.until(sp);
    const int rounds = (stop - (begin - ks) + KS - 1) / KS;   // the same for every group
    // Table entries are read a round before the codes they lead to, and
    // everything unconditionally (positions past the last one lead to page 0):
    // loads under a condition would be waited for where it ends.
    const int until = min(g.highest, kStep * stop - 1);   // this workgroup's last position
    auto entry_of = [&](int at) {
        const int entry = table[min(at >> shift, a.table_stride - 1)];
        return at <= until ? entry : -1;
    };
    auto place_of = [&](int page) { return (size_t)((unsigned)page < (unsigned)c.pages ? page : 0) * c.kv_heads + kvh; };
    const size_t plane = (size_t)c.page_tokens * W;
    int kpage, vpage[N], spage;
    auto look_k = [&](int step) {
        kpage = entry_of(kStep * step + (lane & 48));
        spage = entry_of(kStep * step + 16 * (tid & 3));
    };
    auto look_v = [&](int step) {
#pragma unroll
        for (int i = 0; i < N; ++i) vpage[i] = entry_of(kStep * step + 16 * ((tid + 256 * i) / W));
    };
    // Codes on their way to LDS: this thread's piece i of K is dims
    // 16 (wave + 4 i).. of position `lane` of the step, of V dim
    // (tid + 256 i) % W of granule (tid + 256 i) / W.
    uint4 kreg[N], vreg[N];
    float2 sreg;
    bool sthere;
    auto fetch_k = [&](int step) {
        const int8_t *kb = c.keys + place_of(kpage) * plane + (wave * c.page_tokens + ((kStep * step + lane) & within)) * 16;
#pragma unroll
        for (int i = 0; i < N; ++i) kreg[i] = *(const uint4 *)(kb + (size_t)64 * c.page_tokens * i);
        sreg = make_float2(c.key_scales[place_of(spage)], c.value_scales[place_of(spage)]);
        sthere = (unsigned)spage < (unsigned)c.pages;
    };
    auto fetch_v = [&](int step) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int piece = tid + 256 * i, vat = kStep * step + 16 * (piece / W);
            const int8_t *vb = c.values + place_of(vpage[i]) * plane + ((vat & within) * W + 16 * (piece % W));
            vreg[i] = *(const uint4 *)vb;
        }
    };
    uint8_t *const ksm = smem[ks][0], *const vsm = smem[ks][1];
    auto stage_k = [&](int buffer) {
        const int t = lane & 31, rho = 8 * ((t & 15) >> 2) + 4 * (t >> 4) + (t & 3);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            uint8_t *to = ksm + (((lane >> 5) * M + wave + 4 * i) * 64 + rho) * 16;
            *(half8 *)to = codes_f16(kreg[i].x, kreg[i].y);
            *(half8 *)(to + 512) = codes_f16(kreg[i].z, kreg[i].w);
        }
        // A value scale below 0: nothing there.
        if (tid < 4) scales[ks][buffer][tid] = make_float2(sreg.x, sthere ? fabsf(sreg.y) : -1.f);
    };
    auto stage_v = [&]() {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int piece = tid + 256 * i, granule = piece / W, d = piece % W;
            uint8_t *to = vsm + ((((granule >> 1) * D + (d >> 5)) * 2) * 64 + 32 * (granule & 1) + (d & 31)) * 16;
            *(half8 *)to = codes_f16(vreg[i].x, vreg[i].y);
            *(half8 *)(to + 1024) = codes_f16(vreg[i].z, vreg[i].w);
        }
    };
    look_k(begin);
    fetch_k(begin);
    look_v(begin);
    look_k(begin + KS);

    half8 qh[M], ql[M];
    float qscale;
    {
        const float *q = a.q + (rq.begin + token) * a.q_stride + (int64_t)head * W + 8 * h;
        const bool aligned = ((uintptr_t)a.q & 15) == 0 && a.q_stride % 4 == 0;
        float v[8 * M];
#pragma unroll
        for (int i = 0; i < M; ++i) {
            if (aligned) {
                *(float4 *)(v + 8 * i) = *(const float4 *)(q + 16 * i);
                *(float4 *)(v + 8 * i + 4) = *(const float4 *)(q + 16 * i + 4);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[8 * i + e] = q[16 * i + e];
            }
        }
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 8 * M; ++i) top = fmaxf(top, fabsf(v[i]));
        const int e = 14 - __builtin_amdgcn_frexp_expf(halves_max(top));
#pragma unroll
        for (int i = 0; i < 8 * M; ++i) v[i] = ldexpf(a.scale < 0.f ? -v[i] : v[i], e);
#pragma unroll
        for (int i = 0; i < M; ++i) split_f16(v + 8 * i, qh[i], ql[i]);
        qscale = ldexpf(fabsf(a.scale) * 1.44269504f, -e);
    }
    f32x16 O[D], S[2];
#pragma unroll
    for (int d = 0; d < D; ++d) O[d] = (f32x16){};
    half8 ph[2][2], pl[2][2];
    float m = -INFINITY, l = 0.f;
    bool far = false;
    uint64_t saw = 0;   // lanes that had a score
    auto outputs = [&]() {
        const uint8_t *vs = vsm + 16 * lane;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                half8 v[D];
#pragma unroll
                for (int d = 0; d < D; ++d) v[d] = *(const half8 *)(vs + ((t * D + d) * 2 + u) * 1024);
#pragma unroll
                for (int d = 0; d < D; ++d)
                    O[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], ph[t][u], O[d], 0, 0, 0);
#pragma unroll
                for (int d = 0; d < D; ++d)
                    O[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[d], pl[t][u], O[d], 0, 0, 0);
            }
    };
    auto scores = [&]() {
        const uint8_t *kp = ksm + 16 * lane;
#pragma unroll
        for (int t = 0; t < 2; ++t) S[t] = (f32x16){};
#pragma unroll
        for (int j = 0; j < M; ++j) {
            const half8 k0 = *(const half8 *)(kp + j * 1024), k1 = *(const half8 *)(kp + (M + j) * 1024);
            S[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, qh[j], S[0], 0, 0, 0);
            S[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, qh[j], S[1], 0, 0, 0);
            S[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, ql[j], S[0], 0, 0, 0);
            S[1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, ql[j], S[1], 0, 0, 0);
        }
    };
    // Between the MFMAs: softmax of the scores, the last codes into LDS.
    auto between = [&](int step, int buffer) {
        stage_v();
        stage_k(buffer ^ 1);
        const int at = kStep * step;
        const bool whole = all_from <= at && all_to >= at + kStep - 1;
        float scale[2], mant[2];
        int e[2];
        bool there[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const float2 s = scales[ks][buffer][2 * t + h];
            there[t] = !(s.y < 0.f);
            const bool fine = __builtin_isfinite(s.x) && __builtin_isfinite(s.y);
            // Above 0, so that it keeps minus infinity. A page that reads as
            // NaN makes the rows that see it NaN by their sum alone.
            scale[t] = fine ? fmaxf(fabsf(s.x) * qscale, 0x1p-126f) : 1.f;
            e[t] = fine ? __builtin_amdgcn_frexp_expf(s.y) : 0;
            mant[t] = fine ? __builtin_amdgcn_frexp_mantf(s.y) : 1.f;
            const int pos = at + 32 * t + 16 * h;
            if (there[t] && !fine && first <= pos + 15 && last >= pos) l = NAN;
        }
        if (!whole || __builtin_amdgcn_ballot_w64(!there[0] || !there[1])) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int from = max(first - (at + 32 * t + 16 * h), 0), to = min(last - (at + 32 * t + 16 * h), 15);
                const uint32_t seen = there[t] && from <= to ? (0xFFFFu >> (15 - to)) & (0xFFFFu << from) : 0;
#pragma unroll
                for (int n = 0; n < 16; ++n) S[t][n] = seen >> n & 1 ? S[t][n] : -INFINITY;
            }
        }
        float top = -INFINITY, any = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float best = S[t][0];
#pragma unroll
            for (int n = 1; n < 16; ++n) best = fmaxf(best, S[t][n]);
            any = fmaxf(any, best);
            top = fmaxf(top, __builtin_fmaf(best, scale[t], e[t]));
        }
        saw |= __builtin_amdgcn_ballot_w64(any > -INFINITY);
        if (__builtin_amdgcn_ballot_w64(top > m)) {
            const float next = fmaxf(m, ceilf(halves_max(top)));
            const float alpha = __builtin_amdgcn_exp2f(m - (next == -INFINITY ? 0.f : next));
            m = next;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < D; ++d) O[d] *= alpha;
            far = __builtin_amdgcn_ballot_w64(is_far(m));
        }
        const float base = m == -INFINITY ? 0.f : m;
        float add[2] = {e[0] - base + 15.f, e[1] - base + 15.f};
        if (far) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int n = 0; n < 16; ++n) S[t][n] = __builtin_fmaf(S[t][n], scale[t], e[t]) - base;
                scale[t] = 1.f;
                add[t] = 15.f;
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int n = 0; n < 16; n += 8) {
                float w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(S[t][n + i], scale[t], add[t]));
                    sum[i & 1] += v;
                    w[i] = v * mant[t];
                }
                split_f16(w, ph[t][n / 8], pl[t][n / 8]);
            }
            l += ldexpf(sum[0] + sum[1], kLessBits - e[t]);
        }
    };
    // The next codes set out before the MFMAs and are there after them. A
    // round past the group's last step is one of positions that are not there.
    auto ahead = [&](int step) {
        fetch_k(step + KS);
        fetch_v(step);
        look_v(step + KS);
        look_k(step + 2 * KS);
    };
    if (rounds > 0) {
        stage_k(0);
        lds_barrier();
        if (KS == 2 && ks) lds_barrier();   // half a step behind
        ahead(begin);
        __builtin_amdgcn_s_setprio(1);
        scores();
        __builtin_amdgcn_s_setprio(0);
        lds_barrier();
        between(begin, 0);
        lds_barrier();
        for (int i = 1; i < rounds; ++i) {
            ahead(begin + KS * i);
            __builtin_amdgcn_s_setprio(1);
            outputs();
            scores();
            __builtin_amdgcn_s_setprio(0);
            lds_barrier();   // this group's tiles are read
            between(begin + KS * i, i & 1);
            lds_barrier();   // the next ones are there
        }
        outputs();
        if (KS == 2 && !ks) lds_barrier();
        __syncthreads();
    }
    l = halves_sum(l);
    if (m == -INFINITY && (saw >> col & 0x0000000100000001u)) m = -FLT_MAX;   // scores, none in fp32
    if constexpr (KS == 2) {
        // The second group's rows through LDS, as they lie in its registers.
        float *po = (float *)&smem[0][0][0] + wave * (16 * D * 64) + lane;
        static_assert(sizeof(smem) >= 4 * 16 * D * 64 * sizeof(float), "the second group's outputs fit");
        if (ks) {
#pragma unroll
            for (int d = 0; d < D; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) po[(16 * d + i) * 64] = O[d][i];
            if (h == 0) smem_ml[wave][col] = make_float2(m, l);
        }
        __syncthreads();
        if (ks) return;
        const float2 other = smem_ml[wave][col];
        const float top = fmaxf(m, other.x), base = top == -INFINITY ? 0.f : top;
        const float f0 = __builtin_amdgcn_exp2f(m - base), f1 = __builtin_amdgcn_exp2f(other.x - base);
        m = top;
        l = l * f0 + other.y * f1;
#pragma unroll
        for (int d = 0; d < D; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) O[d][i] = O[d][i] * f0 + po[(16 * d + i) * 64] * f1;
    }
    if (row >= rq.rows) return;
    if (g.active > 1) {
        const Share to = split.share(c.kv_heads, x % tiles, kvh, row - kWideRows * tile, sp, W);
#pragma unroll
        for (int d = 0; d < D; ++d)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *(float4 *)(to.o + 32 * d + 8 * i + 4 * h) =
                    make_float4(O[d][4 * i], O[d][4 * i + 1], O[d][4 * i + 2], O[d][4 * i + 3]);
        if (h == 0) *to.ml = make_float2(m, l);
        return;
    }
    float *out = a.out + (rq.begin + token) * a.out_stride + (int64_t)head * W + 4 * h;
    const float inverse = inverse_of(l, m);
    const bool aligned = ((uintptr_t)a.out & 15) == 0 && a.out_stride % 4 == 0;
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 o = make_float4(O[d][4 * i] * kLess * inverse, O[d][4 * i + 1] * kLess * inverse,
                                         O[d][4 * i + 2] * kLess * inverse, O[d][4 * i + 3] * kLess * inverse);
            if (aligned) {
                *(float4 *)(out + 32 * d + 8 * i) = o;
            } else {
                out[32 * d + 8 * i] = o.x;
                out[32 * d + 8 * i + 1] = o.y;
                out[32 * d + 8 * i + 2] = o.z;
                out[32 * d + 8 * i + 3] = o.w;
            }
        }
}

// out = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M) over a row's shares.
// Requests of a few rows: workgroup (place, row of a KV head).
template <int W>
__device__ __forceinline__ void join_row(const Kv8Attention &a, const Split &split, int most_rows, int index)
{
    const Kv8 &c = a.cache;
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
    for (int k = 0; k < 4; ++k) out[k] = o[k] * kLess * inverse;
}

// Wide tiles: workgroup (tile, 16 of its rows, KV head), a wavefront every
// fourth row.
constexpr int kJoinParts = kWideRows / 16;
template <int W>
__device__ __forceinline__ void join_wide(const Kv8Attention &a, const Split &split, int most_rows, int index)
{
    const Kv8 &c = a.cache;
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
        for (int e = 0; e < kCols; ++e) out[64 * e] = o[e] * kLess * inverse;
    }
}

// Both in one launch: `wide_blocks` workgroups of wide tiles, then those of few rows.
template <int W>
__global__ __launch_bounds__(256) void kv8_join(Kv8Attention a, Split few, Split wide, int most_rows, int wide_blocks)
{
    const int index = blockIdx.x;
    if (index >= wide_blocks) join_row<W>(a, few, most_rows, index - wide_blocks);
    else join_wide<W>(a, wide, most_rows, index);
}

template <int W>
hipError_t launch_width(const Kv8Attention &a, const Plan &p, hipStream_t s)
{
    const unsigned requests = a.requests, kv_heads = a.cache.kv_heads;
    if (p.any_few) {
        const bool listed = p.few.listed;
        const unsigned tiles = listed ? (unsigned)p.few.places : (unsigned)((p.few.tile + kRows - 1) / kRows);
        const unsigned most = p.few.most, packed = p.few.packed ? tiles * requests * most : 0;
        hipLaunchKernelGGL((kv8_rows<W>), packed ? dim3(packed * kv_heads) : dim3(tiles * kv_heads, listed ? 1 : requests, most),
                           dim3(64 * kWaves), 0, s, a, p.few, p.most_rows);
    }
    int64_t wide_blocks = 0;
    if constexpr (W <= 256) {
        if (p.any_wide) {
            constexpr int KS = W <= 128 ? 2 : 1;
            const int64_t tiles = p.wide.places;
            hipLaunchKernelGGL((kv8_wide<W, KS>), dim3((unsigned)(tiles * p.wide.most * kv_heads)), dim3(256 * KS), 0, s, a,
                               p.wide, p.most_rows);
            if (p.wide.most > 1) wide_blocks = tiles * kJoinParts * kv_heads;
        }
    }
    const int64_t blocks = wide_blocks + (p.any_few && p.few.most > 1 ? (int64_t)p.few.tile * kv_heads * p.few.places : 0);
    if (blocks)
        hipLaunchKernelGGL((kv8_join<W>), dim3((unsigned)blocks), dim3(256), 0, s, a, p.few, p.wide, p.most_rows,
                           (int)wide_blocks);
    return hipGetLastError();
}

}  // namespace

size_t kv8_attention_workspace(const Kv8Attention &a)
{
    const Plan p = plan_of(a, nullptr, SIZE_MAX);
    return (p.few.most > 1 ? p.few.most * share_bytes(a, p.few) : 0) +
           (p.wide.most > 1 ? p.wide.most * share_bytes(a, p.wide) : 0);
}

hipError_t launch_kv8_attention(const Kv8Attention &a, void *workspace, size_t workspace_bytes, hipStream_t s)
{
    const Plan p = plan_of(a, (float *)workspace, workspace ? workspace_bytes : 0);
    switch (a.cache.width) {
    case 64: return launch_width<64>(a, p, s);
    case 128: return launch_width<128>(a, p, s);
    case 256: return launch_width<256>(a, p, s);
    default: return launch_width<512>(a, p, s);
    }
}

}  // namespace fy
