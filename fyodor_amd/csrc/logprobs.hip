// Log probabilities of given tokens, entropies and the most likely tokens of
// rows of logits, and their entry points (include/fyodor_hip_logprobs.h).
//
// With M the largest logit that is not masked, d_j = x_j - M and
// S = sum_j e^(scale d_j): ln p_j = scale d_j - ln S, and the entropy is
// ln S - scale sum_j d_j e^(scale d_j) / S. One pass over the logits, a tile of
// them in registers at a time, with a running maximum and sums per thread. The
// terms of the maximum itself are counted, not added: of S = 1 + s a likely
// token's ln p is -ln(1 + s), which 1 + s in fp32 would leave without its last
// bits.
//
// The most likely tokens are a sorted list in LDS. A tile has at least `top`
// logits not below the top-th largest of 64 maxima of its parts, and few more
// (24 of 20 in random order): those, or the ones above the list's last, are put
// in order by counting, each against all.
//
// Bound by reading the logits for many rows; a few rows are split into shares,
// which a second launch joins.
#include <float.h>
#include <limits.h>
#include <math.h>

#include "../../include/fyodor_hip_logprobs.h"
#include "device.h"
#include "kernels.h"

namespace fy {
namespace {

constexpr int kMostShares = 64;
constexpr int kMostTop = NYA_HIP_LOGPROBS_TOP;
static_assert(kMostTop <= 64, "a tile's 64 maxima bound its most likely");

// What is known of a part of a row: its largest logit, how many are that, the
// sums of the others' terms, and how many come before the given token.
struct Part {
    float m;
    int rank;
    double count, s, t;
};
static_assert(sizeof(Part) % 16 == 0, "lists follow");

// Order of tokens: the larger logit, of equal ones (zeros of both signs among
// them) the lower id. 0 is no token.
__device__ __forceinline__ uint32_t ordered(float x)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
    return b ^ ((int)b < 0 ? ~0u : 0x80000000u);
}
__device__ __forceinline__ float of_order(uint32_t o) { return __builtin_bit_cast(float, o ^ ((int)o < 0 ? 0x80000000u : ~0u)); }
__device__ __forceinline__ uint64_t key_of(float x, int id) { return (uint64_t)ordered(x) << 32 | ~(uint32_t)id; }
__device__ __forceinline__ float logit_of(uint64_t key) { return of_order((uint32_t)(key >> 32)); }
__device__ __forceinline__ int id_of(uint64_t key) { return (int)~(uint32_t)key; }

// The first float above x, or below it (of 0 the one below both zeros); finite ones.
__device__ __forceinline__ float above(float x) { return of_order(ordered(x) + 1); }
__device__ __forceinline__ float below(float x)
{
    const uint32_t o = ordered(x) - 1;
    return of_order(o == 0x7FFFFFFFu ? o - 1 : o);   // (0x7FFFFFFF is -0)
}

// A workgroup's list, in front of what may join it.
template <int T> struct List {
    static constexpr int kRoom = T + kMostTop > 1024 ? T + kMostTop : 1024;
    uint64_t keys[kRoom], next[kMostTop];
    float maxima[T];
    unsigned n;
};

// Puts keys[0 .. n) in order and keeps the first `top`; how many there are.
template <int T>
__device__ int settle(List<T> &list, int top)
{
    const int n = min(list.n, (unsigned)List<T>::kRoom), held = min(n, top);
    for (int i = threadIdx.x; i < n; i += T) {
        const uint64_t key = list.keys[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += list.keys[j] > key;
        if (rank < top) list.next[rank] = key;
    }
    __syncthreads();
    if ((int)threadIdx.x < held) list.keys[threadIdx.x] = list.next[threadIdx.x];
    if (threadIdx.x == 0) list.n = held;
    __syncthreads();
    return held;
}

// N tokens of each thread into the list (held of them so far); `most`: the thread's largest
// logit. In order: none of them comes before one in the list of the same logit.
template <int T, int N, class X, class Id>
__device__ __forceinline__ int join_list(List<T> &list, int held, int top, float most, const X &x, const Id &id)
{
    const int tid = threadIdx.x, lane = tid & 63;
    float from;
    if (held == top) {
        from = above(logit_of(list.keys[top - 1]));
        if (!__syncthreads_or(most >= from)) return held;
    } else {
        list.maxima[tid] = most;
        __syncthreads();
        float u = list.maxima[lane];
#pragma unroll
        for (int w = 1; w < T / 64; ++w) u = fmaxf(u, list.maxima[64 * w + lane]);
        // Distinct by the lane, in place of the last bits: rounded down, it still bounds them.
        const uint32_t o = (ordered(u) & ~63u) | lane;
        int rank = 0;
#pragma unroll 16
        for (int j = 0; j < 64; ++j) rank += (uint32_t)__builtin_amdgcn_readlane((int)o, j) > o;
        const int at = __builtin_ctzll(__builtin_amdgcn_ballot_w64(rank == top - 1));
        // Minus infinity is no token.
        from = fmaxf(of_order((uint32_t)__builtin_amdgcn_readlane((int)o, at) & ~63u), -FLT_MAX);
    }
    if (most >= from) {
        int mine = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) mine += x(i) >= from;
        unsigned at = atomicAdd(&list.n, (unsigned)mine);
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (x(i) >= from) {
                if (at < (unsigned)List<T>::kRoom) list.keys[at] = key_of(x(i), id(i));
                ++at;
            }
    }
    __syncthreads();
    if (list.n <= (unsigned)List<T>::kRoom) return settle(list, top);
    // More than there is room for (many equal or ascending logits): a token of each thread at a time.
    __syncthreads();
    if (tid == 0) list.n = held;
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < N; ++i) {
        float v = 0.f;
        int k = 0;
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (j == i) {
                v = x(j);
                k = id(j);
            }
        const uint64_t key = key_of(v, k);
        if (v >= -FLT_MAX && (held < top || key > list.keys[top - 1])) list.keys[atomicAdd(&list.n, 1u)] = key;
        __syncthreads();
        held = settle(list, top);
    }
    return held;
}

// What the threads know, together, in all of them. c: scale in powers of two.
template <int T>
__device__ __forceinline__ Part together(const Part &p, float c)
{
    __shared__ double sums[4][T / 64];
    __shared__ float tops[T / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float top = wave_reduce<true>(p.m);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    Part all = {tops[0], 0, 0, 0, 0};
#pragma unroll
    for (int w = 1; w < T / 64; ++w) all.m = fmaxf(all.m, tops[w]);
    const float d = p.m - all.m, f = p.m == all.m ? 1.f : __builtin_amdgcn_exp2f(d * c);
    const bool most = p.m == all.m;
    const double count = wave_sum(most ? p.count : 0.0), s = wave_sum(p.s * f + (most ? 0.0 : p.count * f)),
                 t = wave_sum(f == 0.f ? 0.0 : most ? p.t : (p.t + (p.count + p.s) * d) * f), rank = wave_sum((double)p.rank);
    if (lane == 0) {
        sums[0][wave] = count;
        sums[1][wave] = s;
        sums[2][wave] = t;
        sums[3][wave] = rank;
    }
    __syncthreads();
    double ranks = 0;
#pragma unroll
    for (int w = 0; w < T / 64; ++w) {
        all.count += sums[0][w];
        all.s += sums[1][w];
        all.t += sums[2][w];
        ranks += sums[3][w];
    }
    all.rank = (int)ranks;
    return all;
}

// The given token of a row, and its logit (minus infinity where it is masked).
struct Given {
    int id;
    bool there;
    float x;
};

__device__ __forceinline__ Given given_of(const Logprobs &a, int row)
{
    Given g = {a.tokens ? a.tokens[row] : -1, false, -INFINITY};
    g.there = (unsigned)g.id < (unsigned)a.n;
    const int id = g.there ? g.id : 0;
    const float x = a.logits[row * a.stride + id];
    if (g.there && !(a.mask && (a.mask[id >> 5] >> (id & 31) & 1u))) g.x = x;
    return g;
}

// A row's results.
template <int T>
__device__ __forceinline__ void finish(const Logprobs &a, int row, const Given &g, const Part &p, const List<T> *list, int held)
{
    __shared__ double log_s;
    // NaN leaves a sum NaN; plus infinity is the maximum.
    const bool none = !(p.m > -INFINITY && p.m < INFINITY) || !(p.s >= 0);
    if (threadIdx.x == 0) {
        log_s = log1p((p.count - 1) + p.s);
        if (a.tokens) {
            const bool ranked = g.there && !none && g.x > -INFINITY;
            a.logprobs[row] = !g.there ? 0.f : none ? NAN : (float)(((double)g.x - p.m) * a.scale - log_s);
            if (a.ranks) a.ranks[row] = ranked ? p.rank : -1;
        }
        if (a.entropies) a.entropies[row] = none ? NAN : (float)(log_s - p.t / (p.count + p.s) * a.scale);
    }
    if (!list) return;
    __syncthreads();
    for (int k = threadIdx.x; k < a.top; k += T) {
        const uint64_t key = k < held ? list->keys[k] : 0;
        const size_t at = (size_t)row * a.top + k;
        a.top_ids[at] = none || !key ? -1 : id_of(key);
        a.top_logprobs[at] = none ? NAN : !key ? -INFINITY : (float)(((double)logit_of(key) - p.m) * a.scale - log_s);
    }
}

// Workgroup (row, share of its tiles) of T threads, V times 4 logits each a tile.
// Positions begin at the 16 bytes that the row begins in.
template <int T, int V, bool kTop>
__global__ __launch_bounds__(T) void logprobs_rows(Logprobs a, int shares, int tiles_each, Part *parts, uint64_t *lists)
{
    __shared__ List<kTop ? T : 64> list;
    constexpr int kTile = 4 * T * V;
    const int row = blockIdx.x / shares, share = blockIdx.x % shares, tid = threadIdx.x;
    const float *x0 = a.logits + row * a.stride;
    const int shift = (int)((uintptr_t)x0 >> 2 & 3), end = a.n + shift;
    x0 -= shift;
    const int from = share * tiles_each * kTile, to = min(end, from + tiles_each * kTile);
    const Given g = given_of(a, row);
    const float c = a.scale * 1.44269504f;
    Part p = {-INFINITY, 0, 0, 0, 0};
    float s = 0.f, t = 0.f;
    int count = 0, held = 0;
    if (kTop) {
        if (tid == 0) list.n = 0;
        __syncthreads();
    }
    for (int tile = from; tile < to; tile += kTile) {
        float x[4 * V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int at = tile + 4 * (T * v + tid);
            if (at >= shift && at + 3 < end) {
                const float4 q = *(const float4 *)(x0 + at);
                x[4 * v] = q.x;
                x[4 * v + 1] = q.y;
                x[4 * v + 2] = q.z;
                x[4 * v + 3] = q.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * v + e] = at + e >= shift && at + e < end ? x0[at + e] : -INFINITY;
            }
        }
        if (a.mask) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int id = tile + 4 * (T * v + tid) - shift;
                const int last = (a.n - 1) >> 5, first = max(id, 0) >> 5;
                const uint64_t both = (uint64_t)a.mask[min(max(id + 3, 0) >> 5, last)] << 32 | a.mask[min(first, last)];
                // (Of one word twice, the low one has the bits.)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int bit = id + e - 32 * first;
                    if (bit >= 0 && (both >> (bit & 63) & 1u)) x[4 * v + e] = -INFINITY;
                }
            }
        }
        float most = x[0];
#pragma unroll
        for (int i = 1; i < 4 * V; ++i) most = fmaxf(most, x[i]);
        if (most > p.m) {
            // (The thread's first tile: there is nothing to rescale.)
            const float d = p.m - most, f = __builtin_amdgcn_exp2f(d * c);
            t = f == 0.f ? 0.f : (t + ((float)count + s) * d) * f;
            s = s * f + (float)count * f;
            count = 0;
            p.m = most;
        }
        const float m = p.m == -INFINITY ? 0.f : p.m;
#pragma unroll
        for (int i = 0; i < 4 * V; ++i) {
            const float d = x[i] - m, e = __builtin_amdgcn_exp2f(d * c);
            const bool at_most = x[i] == m;
            count += at_most;
            s += at_most ? 0.f : e;
            t = __builtin_fmaf(fmaxf(d, -FLT_MAX), e, t);
        }
        // Which logits come before the given one goes by the id where they are equal.
        if (g.there) {
            const int id = tile - shift;
            if (g.id >= id && g.id < id + kTile) {
#pragma unroll
                for (int i = 0; i < 4 * V; ++i) {
                    const int mine = id + 4 * (T * (i / 4) + tid) + i % 4;
                    p.rank += x[i] > g.x || (x[i] == g.x && mine < g.id);
                }
            } else {
                const float bar = g.id < id || !(g.x > -INFINITY) ? g.x : below(g.x);
#pragma unroll
                for (int i = 0; i < 4 * V; ++i) p.rank += x[i] > bar;
            }
        }
        if constexpr (kTop)
            held = join_list<T, 4 * V>(list, held, a.top, most, [&](int i) { return x[i]; },
                                       [&](int i) { return tile - shift + 4 * (T * (i / 4) + tid) + i % 4; });
    }
    p.count = count;
    p.s = s;
    p.t = t;
    p = together<T>(p, c);
    if (shares == 1) {
        if constexpr (kTop) finish<T>(a, row, g, p, &list, held);
        else finish<T>(a, row, g, p, nullptr, 0);
        return;
    }
    if (tid == 0) parts[blockIdx.x] = p;
    if constexpr (kTop)
        for (int k = tid; k < a.top; k += T) lists[(size_t)blockIdx.x * a.top + k] = k < held ? list.keys[k] : 0;
}

// Workgroup: a row, from its shares.
template <bool kTop>
__global__ __launch_bounds__(256) void logprobs_join(Logprobs a, int shares, const Part *parts, const uint64_t *lists)
{
    __shared__ List<kTop ? 256 : 64> list;
    const int row = blockIdx.x, tid = threadIdx.x;
    const Given g = given_of(a, row);
    Part p = {-INFINITY, 0, 0, 0, 0};
    if (tid < shares) p = parts[(size_t)row * shares + tid];
    int held = 0;
    if constexpr (kTop) {
        if (tid == 0) list.n = 0;
        __syncthreads();
        constexpr int kEach = 4;
        const int n = shares * a.top;
        lists += (size_t)row * n;
        // Share after share, so that of equal logits the lower ids come first.
        for (int at = 0; at < n; at += 256 * kEach) {
            uint64_t key[kEach];
            float most = -INFINITY;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int k = at + 256 * i + tid;
                key[i] = k < n ? lists[k] : 0;
                if (!key[i]) key[i] = key_of(-INFINITY, 0);
                most = fmaxf(most, logit_of(key[i]));
            }
            held = join_list<256, kEach>(list, held, a.top, most, [&](int i) { return logit_of(key[i]); },
                                         [&](int i) { return id_of(key[i]); });
        }
    }
    p = together<256>(p, a.scale * 1.44269504f);
    if constexpr (kTop) finish<256>(a, row, g, p, &list, held);
    else finish<256>(a, row, g, p, nullptr, 0);
}

// How a call's rows are read: `threads` per workgroup, a row's tiles in `shares` of `each`.
struct Reading {
    int threads, shares, each;
};

constexpr int kFew = 1024, kFewTile = 4 * kFew * 8, kManyTile = 4 * 256 * 4;

Reading reading_of(int n, int count, int top, size_t bytes)
{
    const int span = n + 3;   // a row may begin 3 floats into its 16 bytes
    const auto tiles = [&](int tile) { return (span + tile - 1) / tile; };
    // Rows of two large tiles: what a second launch costs is more.
    if (count <= 256 && tiles(kFewTile) <= 2) return {kFew, 1, tiles(kFewTile)};
    const int all = tiles(kManyTile);
    int shares = count >= 1024 ? 1 : (2048 + count - 1) / count;
    shares = shares < kMostShares ? shares : kMostShares;
    const size_t each = (sizeof(Part) + sizeof(uint64_t) * top) * count;
    if (bytes / each < (size_t)shares) shares = (int)(bytes / each);
    if (shares > all) shares = all;
    if (shares < 2) return {256, 1, all};
    const int tiles_each = (all + shares - 1) / shares;
    return {256, (all + tiles_each - 1) / tiles_each, tiles_each};
}

}  // namespace

size_t logprobs_workspace(int n, int count, int top)
{
    const Reading r = reading_of(n, count, top, SIZE_MAX);
    return r.shares == 1 ? 0 : (sizeof(Part) + sizeof(uint64_t) * top) * count * r.shares;
}

hipError_t launch_logprobs(const Logprobs &a, void *workspace, size_t workspace_bytes, hipStream_t s)
{
    const Reading r = reading_of(a.n, a.count, a.top, workspace ? workspace_bytes : 0);
    Part *parts = (Part *)workspace;
    uint64_t *lists = (uint64_t *)(parts + (size_t)a.count * r.shares);
    const dim3 grid((unsigned)((int64_t)a.count * r.shares));
    if (r.threads == kFew) {
        if (a.top) hipLaunchKernelGGL((logprobs_rows<kFew, 8, true>), grid, dim3(kFew), 0, s, a, 1, r.each, parts, lists);
        else hipLaunchKernelGGL((logprobs_rows<kFew, 8, false>), grid, dim3(kFew), 0, s, a, 1, r.each, parts, lists);
        return hipGetLastError();
    }
    if (a.top) hipLaunchKernelGGL((logprobs_rows<256, 4, true>), grid, dim3(256), 0, s, a, r.shares, r.each, parts, lists);
    else hipLaunchKernelGGL((logprobs_rows<256, 4, false>), grid, dim3(256), 0, s, a, r.shares, r.each, parts, lists);
    if (r.shares > 1) {
        if (a.top) hipLaunchKernelGGL((logprobs_join<true>), dim3(a.count), dim3(256), 0, s, a, r.shares, parts, lists);
        else hipLaunchKernelGGL((logprobs_join<false>), dim3(a.count), dim3(256), 0, s, a, r.shares, parts, lists);
    }
    return hipGetLastError();
}

}  // namespace fy

namespace {

using namespace fy;

bool sizes_ok(size_t n, size_t count, size_t top)
{
    return n && n <= (size_t)1 << 24 && count && count <= (size_t)1 << 22 && top <= NYA_HIP_LOGPROBS_TOP;
}

// Arrays of 4-byte elements (0: none): a start and an end.
struct Array {
    uintptr_t from;
    size_t n;
    bool ok() const { return !(from & 3u); }
    bool apart(const Array &o) const { return !from || !o.from || from + 4 * n <= o.from || o.from + 4 * o.n <= from; }
};

}  // namespace

extern "C" {

NYA_HIP_EXPORT int nya_hip_logprobs_bytes(size_t n, size_t count, size_t top, size_t *bytes)
{
    if (!bytes || !sizes_ok(n, count, top)) return 1;
    *bytes = logprobs_workspace((int)n, (int)count, (int)top);
    return 0;
}

NYA_HIP_EXPORT int nya_hip_logprobs(uintptr_t logits, size_t stride, size_t n, size_t count, uintptr_t mask, float scale,
    uintptr_t tokens, uintptr_t logprobs, uintptr_t ranks, uintptr_t entropies, size_t top, uintptr_t top_ids,
    uintptr_t top_logprobs, uintptr_t workspace, size_t workspace_bytes, uintptr_t stream)
{
    if (!sizes_ok(n, count, top) || !logits || stride < n || stride > (size_t)INT_MAX || !(scale >= 0x1p-20f) ||
        !(scale <= 0x1p20f) || (workspace & 15u) || (!tokens && !entropies && !top) || (tokens && !logprobs) ||
        (top && (!top_ids || !top_logprobs)))
        return 1;
    const Array in[] = {{logits, (count - 1) * stride + n}, {mask, (n + 31) / 32}, {tokens, count}};
    const Array out[] = {{tokens ? logprobs : 0, count}, {tokens ? ranks : 0, count}, {entropies, count},
                         {top ? top_ids : 0, count * top}, {top ? top_logprobs : 0, count * top}};
    for (const Array &o : out) {
        if (!o.ok()) return 1;
        for (const Array &i : in)
            if (!i.ok() || !o.apart(i)) return 1;
        for (const Array &p : out)
            if (&p != &o && !o.apart(p)) return 1;
    }
    const Logprobs a = {(const float *)logits, (int64_t)stride, (int)n, (int)count, (const uint32_t *)mask, scale,
                        (const int *)tokens, (float *)logprobs, tokens ? (int *)ranks : nullptr, (float *)entropies,
                        (int)top, (int *)top_ids, (float *)top_logprobs};
    const hipError_t e = launch_logprobs(a, (void *)workspace, workspace ? workspace_bytes : 0, (hipStream_t)stream);
    return e == hipSuccess ? 0 : -(int)(e > 0 ? e : 1);
}

}  // extern "C"
