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
// The pass keeps the maximum of every group of 32 logits as well. The top-th
// largest of 256 maxima (of groups together) is not above the top-th logit,
// and only the groups that reach it, about as many as are asked for, are read
// again: a list of little more than `top` tokens is put in order by counting,
// each against all. (Choosing in every tile as it passes cost nearly as much as the
// pass: 64 rows of 128256 17 us with 20 alternatives, 10 without.)
//
// Bound by reading the logits for many rows (2047 of 50257 without alternatives
// 77 us, 5.4 TB/s; with 20 of them 94: the choice at a row's end is waits, and its LDS
// leaves five workgroups on a CU for eight). A few rows are split into shares,
// which a second launch joins (64 of 128256 with 20: 11.0 us and 7.2, masked 12.2 and
// 7.4; 1 of 32000 with 5: 3.8 and 5.0): chains of waits, of which the join has four:
// the shares with the maxima, the bound with the sums beside it, the logits, their
// order. (The maxima read twice, the logits one after another, the sums first:
// 11.8 for 7.4.)
#include <float.h>
#include <limits.h>
#include <math.h>

#include "../../include/fyodor_hip_logprobs.h"
#include "device.h"
#include "kernels.h"

namespace fy {
namespace {

constexpr int kMostShares = 64;
constexpr int kSplitRows = 1024;   // from so many rows on they are whole; shares are for so many workgroups
constexpr int kMostTop = NYA_HIP_LOGPROBS_TOP;
static_assert(kMostTop <= 64, "a tile's 64 maxima bound its most likely");

// What is known of a part of a row: its largest logit, how many are that, the
// sums of the others' terms, and how many come before the given token.
struct Part {
    float m;
    int rank;
    double count, s, t;
};
static_assert(sizeof(Part) % 16 == 0, "maxima follow");

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

// The first float below x (of 0 the one below both zeros); finite ones.
__device__ __forceinline__ float below(float x)
{
    const uint32_t o = ordered(x) - 1;
    return of_order(o == 0x7FFFFFFFu ? o - 1 : o);   // (0x7FFFFFFF is -0)
}

// The sums by a maximum m, added to those by another that is not below it.
__device__ __forceinline__ void add_to(Part &p, float m, double count, double s, double t, float c)
{
    const float d = m - p.m, f = m == p.m ? 1.f : __builtin_amdgcn_exp2f(d * c);
    if (m == p.m) {
        p.count += count;
        p.s += s;
        p.t += t;
    } else {
        p.s += (s + count) * f;
        if (f != 0.f) p.t += (t + (s + count) * d) * f;
    }
}

__device__ __forceinline__ bool is_masked(const Logprobs &a, int id) { return a.mask && (a.mask[id >> 5] >> (id & 31) & 1u); }

constexpr int kThreads = 256;
constexpr int kV = 2;                    // 4 kV logits of a thread in a tile (four: 2047 rows of 50257 79 us, two 77)
constexpr int kTile = 4 * kThreads * kV;
constexpr int kRoom = 1024 + kMostTop;   // a list, and what may join it before it is put in order
constexpr int kListed = 512;             // groups that are read again, by number
constexpr int kMostGroups = 64 * 64;     // of a row

struct List {
    __align__(16) uint64_t keys[kRoom];
    uint64_t next[kMostTop];
    float maxima[kThreads], bound;
    int groups[kListed];
    uint32_t reach[2][kThreads / 64];
    unsigned n, listed;
    unsigned equal[kMostGroups / 64];   // groups of each set whose maximum is the bound
};

// Leaves, of more keys than are worth comparing with each other (634 rows of 984, 33 of them: 34 us without
// this, 13 with it), the ones above a bound that at least `top` of them reach and few more do: as bound_of, with
// every thread's keys in registers, and their ids where logits are equal.
__device__ void narrow(List &list, int top)
{
    constexpr int kEach = (kRoom + kThreads - 1) / kThreads;
    const int n = list.n, tid = threadIdx.x, wave = tid >> 6;
    uint64_t key[kEach];
    uint32_t least = ~0u, most = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int k = tid + i * kThreads;
        key[i] = k < n ? list.keys[k] : 0;
        const uint32_t o = (uint32_t)(key[i] >> 32);
        if (key[i]) least = min(least, o);
        most = max(most, o);
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        least = min(least, (uint32_t)__shfl_xor((int)least, d, 64));
        most = max(most, (uint32_t)__shfl_xor((int)most, d, 64));
    }
    if ((tid & 63) == 0) {
        list.reach[0][wave] = least;
        list.reach[1][wave] = most;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
        least = min(least, list.reach[0][w]);
        most = max(most, list.reach[1][w]);
    }
    __syncthreads();
    // (Ids are below 2^31, so keys above that of the last one.)
    uint64_t from = (uint64_t)least << 32 | 0x80000000u, to = (uint64_t)most << 32 | 0xFFFFFFFFu;
    for (int turn = 0; to > from + 1 && turn < 64; ++turn) {
        const uint64_t middle = from + (to - from) / 2;
        int mine = 0, reach = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            mine += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[i] >= middle));
        if ((tid & 63) == 0) list.reach[turn & 1][wave] = mine;
        __syncthreads();   // (the other half is written next: one wait a turn)
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) reach += (int)list.reach[turn & 1][w];
        if (reach < top) {
            to = middle;
        } else {
            from = middle;
            if (reach <= top + 8) break;
        }
    }
    __syncthreads();
    if (tid == 0) list.n = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        if (key[i] >= from) list.keys[atomicAdd(&list.n, 1u)] = key[i];
    __syncthreads();
}

// Puts keys[0 .. n) in order, each against all, and keeps the first `top`; how many there are.
__device__ int settle(List &list, int top)
{
    if (list.n > 256 && (int)list.n > top) narrow(list, top);
    const int n = list.n, held = min(n, top), lane = threadIdx.x & 63;
    if (n <= 64) {
        // One wavefront, the keys in its lanes.
        if (threadIdx.x < 64) {
            const uint64_t key = lane < n ? list.keys[lane] : 0;
            int rank = 0;
            for (int j = 0; j < n; j += 4)
#pragma unroll
                for (int i = j; i < j + 4; ++i) {   // (0 past the last)
                    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)key, i),
                                   hi = __builtin_amdgcn_readlane((int)(uint32_t)(key >> 32), i);
                    rank += ((uint64_t)hi << 32 | lo) > key;
                }
            if (lane < n && rank < top) list.keys[rank] = key;
            if (lane == 0) list.n = held;
        }
        __syncthreads();
        return held;
    }
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t key = list.keys[i];
        int rank = 0, j = 0;
        for (; j + 8 <= n; j += 8)
#pragma unroll
            for (int k = 0; k < 8; ++k) rank += list.keys[j + k] > key;
        for (; j < n; ++j) rank += list.keys[j] > key;
        if (rank < top) list.next[rank] = key;
    }
    __syncthreads();
    if ((int)threadIdx.x < held) list.keys[threadIdx.x] = list.next[threadIdx.x];
    if (threadIdx.x == 0) list.n = held;
    __syncthreads();
    return held;
}

// A bound that at least `top` of the 256 maxima reach and not many more, by halving the range
// between the least and the largest, in their order as whole numbers; one of the maxima, where too
// many are equal.
__device__ __forceinline__ float bound_of(const List &list, int top)
{
    const int lane = threadIdx.x & 63;
    uint32_t u[4];
    float low, high;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v = list.maxima[64 * i + lane];
        u[i] = ordered(v);
        low = i ? fminf(low, v) : v;
        high = i ? fmaxf(high, v) : v;
    }
    // Minus infinity is no token.
    uint32_t from = ordered(fmaxf(-wave_reduce<true>(-low), -FLT_MAX)), to = ordered(wave_reduce<true>(high)) + 1;
    for (int k = 0; k < 32 && to > from + 1; ++k) {
        const uint32_t middle = from + (to - from) / 2;
        int reach = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) reach += __builtin_popcountll(__builtin_amdgcn_ballot_w64(u[i] >= middle));
        if (reach < top) {
            to = middle;
        } else {
            from = middle;
            if (reach <= top + 2 + k) break;   // (equal maxima: a few groups more, not every turn)
        }
    }
    return of_order(__builtin_amdgcn_readfirstlane((int)from));
}

// How a row is read: `shares` of `sets` x `per_set` tiles. A set's group g of 64
// has the 16 logits from 16 g on of each 1024.
struct Reading {
    int shares, sets, per_set;
    __host__ __device__ int each() const { return sets * per_set; }
};

// A thread's maxima of a row's groups (a multiple of 64 of them, in the order of shares and sets).
struct Maxima {
    static constexpr int kChunks = 4;
    float4 v[kChunks];

    // Four side by side while 256 threads have some each.
    static __device__ __forceinline__ bool wide(int groups) { return groups >= 4 * kThreads; }
    static __device__ __forceinline__ int number(bool wide, int i, int e)
    {
        return wide ? 4 * (i * kThreads + (int)threadIdx.x) + e : e * kThreads + (int)threadIdx.x;
    }
    __device__ __forceinline__ void load(const float *maxima, int groups)
    {
        const bool is_wide = wide(groups);
#pragma unroll
        for (int i = 0; i < kChunks; ++i) {
            v[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (i * 4 * kThreads >= groups) continue;
            const int g = number(is_wide, i, 0);
            if (is_wide) {
                if (g < groups) v[i] = *(const float4 *)(maxima + g);
            } else {
                if (g < groups) v[i].x = maxima[g];
                if (g + kThreads < groups) v[i].y = maxima[g + kThreads];
                if (g + 2 * kThreads < groups) v[i].z = maxima[g + 2 * kThreads];
                if (g + 3 * kThreads < groups) v[i].w = maxima[g + 3 * kThreads];
            }
        }
    }
    __device__ __forceinline__ float most() const
    {
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < kChunks; ++i) m = fmaxf(fmaxf(fmaxf(m, v[i].x), fmaxf(v[i].y, v[i].z)), v[i].w);
        return m;
    }
};
static_assert(4 * kThreads * Maxima::kChunks >= kMostGroups, "every group of a row");

// Lists the groups of a row anew where too many reach the bound, as they do in a row of equal logits (a batch's
// padding: with all of its groups gone through, 64 rows of 128256 with 20 alternatives, half of them zeros,
// took 306 us, so 33): those above it, and of those with just it the first sets' until there are `top`. A set's ids
// are below the next one's, so no other group has a token that comes as early.
__device__ void list_first(List &list, int top, float from, bool wide, const Maxima &mine)
{
    static_assert(kMostGroups / 64 == 64, "a lane each");
    const int tid = threadIdx.x, lane = tid & 63;
    __syncthreads();   // the count is read
    if (tid < 64) list.equal[tid] = 0;
    if (tid == 0) list.listed = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < Maxima::kChunks; ++i) {
        const float v[4] = {mine.v[i].x, mine.v[i].y, mine.v[i].z, mine.v[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (v[e] == from) atomicAdd(&list.equal[Maxima::number(wide, i, e) / 64], 1u);
    }
    __syncthreads();
    int sum = (int)list.equal[lane];
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const int v = __shfl_up(sum, o, 64);
        if (lane >= o) sum += v;
    }
    const uint64_t past = __builtin_amdgcn_ballot_w64(sum >= top);
    const int end = past ? 64 * (__builtin_ctzll(past) + 1) : kMostGroups;
#pragma unroll
    for (int i = 0; i < Maxima::kChunks; ++i) {
        const float v[4] = {mine.v[i].x, mine.v[i].y, mine.v[i].z, mine.v[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int g = Maxima::number(wide, i, e);
            if (!(v[e] > from || (v[e] == from && g < end))) continue;
            const unsigned at = atomicAdd(&list.listed, 1u);
            if (at < (unsigned)kListed) list.groups[at] = g;
        }
    }
    __syncthreads();
}

// The first `top` tokens of a row, in order, from its groups' maxima (a thread's are `mine`); how many
// there are. `beside` is done by the second wavefront, while the first looks for the bound.
template <class F>
__device__ __forceinline__ int choose(const Logprobs &a, int row, int shift, const Reading &r, const Maxima &mine,
    const float *maxima, int groups, List &list, const F &beside)
{
    const int tid = threadIdx.x, top = a.top;
    if (tid == 0) list.n = list.listed = 0;
    const float most = mine.most();
    list.maxima[tid] = most;
    __syncthreads();
    if (tid < 64) {
        const float bound = bound_of(list, top);
        if (tid == 0) list.bound = bound;
    } else if (tid < 128) {
        beside();
    }
    __syncthreads();
    const float from = list.bound;
    const bool wide = Maxima::wide(groups);
    if (most >= from) {
        unsigned n = 0;
#pragma unroll
        for (int i = 0; i < Maxima::kChunks; ++i)
            n += (mine.v[i].x >= from) + (mine.v[i].y >= from) + (mine.v[i].z >= from) + (mine.v[i].w >= from);
        unsigned at = atomicAdd(&list.listed, n);
#pragma unroll
        for (int i = 0; i < Maxima::kChunks; ++i) {
            const float4 q = mine.v[i];
            const float v[4] = {q.x, q.y, q.z, q.w};
            if (fmaxf(fmaxf(q.x, q.y), fmaxf(q.z, q.w)) < from) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v[e] >= from) {
                    if (at < (unsigned)kListed) list.groups[at] = Maxima::number(wide, i, e);
                    ++at;
                }
        }
    }
    __syncthreads();
    if (list.listed > (unsigned)kListed) list_first(list, top, from, wide, mine);
    // (More groups than are listed all the same: all of them are gone through.)
    const bool all = list.listed > (unsigned)kListed;
    const int n = all ? groups : (int)list.listed;
    const float *x = a.logits + row * a.stride;
    // 32 threads a group of 32 logits of each of its tiles, 32 groups at a time.
    constexpr int kAtOnce = 4 * kThreads / 32;
    static_assert(kV == 2, "32 logits");
    int held = 0;
    for (int base = 0, tile = 0;;) {
        // All of a thread's loads set out together (of what is no candidate, the row's first).
        int id[4];
        bool is[4];
        float logit[4];
        uint32_t word[4] = {};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = base + i * (kThreads / 32) + tid / 32;
            is[i] = k < n;
            const int g = !is[i] ? 0 : all ? k : list.groups[k];
            if (all && is[i]) is[i] = maxima[g] >= from;
            id[i] = ((g / 64 * r.per_set + tile) * kV + (tid >> 4 & 1)) * 1024 + 16 * (g % 64) + tid % 16 - shift;
            is[i] = is[i] && id[i] >= 0 && id[i] < a.n;
            id[i] = is[i] ? id[i] : 0;
            logit[i] = x[id[i]];
        }
        if (a.mask) {
#pragma unroll
            for (int i = 0; i < 4; ++i) word[i] = a.mask[id[i] >> 5];
        }
        const uint64_t bar = held == top ? list.keys[top - 1] + 1 : key_of(from, 0x7FFFFFFF);
        uint64_t key[4];
        unsigned joins = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            key[i] = key_of(logit[i], id[i]);
            is[i] = is[i] && logit[i] >= -FLT_MAX && !(word[i] >> (id[i] & 31) & 1u) && key[i] >= bar;
            joins += is[i];
        }
        if (joins) {
            unsigned to = atomicAdd(&list.n, joins);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (is[i]) list.keys[to++] = key[i];
        }
        __syncthreads();
        const unsigned now = list.n;
        __syncthreads();   // read by all before the next ones join
        if (++tile == r.per_set) {
            tile = 0;
            base += kAtOnce;
        }
        const bool last = base >= n;
        if (last || now > (unsigned)(kRoom - 4 * kThreads)) held = settle(list, top);
        if (last) return held;
    }
}

// What the threads know, together, in all of them. c: scale in powers of two.
__device__ __forceinline__ Part together(float m, float count, float s, float t, int rank, float c)
{
    __shared__ float sums[3][kThreads / 64], tops[kThreads / 64];
    __shared__ int ranks[kThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // A wavefront's sums by its own maximum. (Whole numbers up to 2^24 are exact.)
    const float top = wave_reduce<true>(m), d = m - top;
    const bool most = m == top;
    const float f = most ? 1.f : __builtin_amdgcn_exp2f(d * c);
    t = f == 0.f ? 0.f : most ? t : (t + (count + s) * d) * f;
    s = s * f + (most ? 0.f : count * f);
    s = wave_sum(s);
    t = wave_sum(t);
    count = wave_sum(most ? count : 0.f);
    rank = (int)wave_sum((float)rank);
    if (lane == 0) {
        tops[wave] = top;
        sums[0][wave] = count;
        sums[1][wave] = s;
        sums[2][wave] = t;
        ranks[wave] = rank;
    }
    __syncthreads();
    Part all = {tops[0], 0, 0, 0, 0};
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) all.m = fmaxf(all.m, tops[w]);
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
        add_to(all, tops[w], sums[0][w], sums[1][w], sums[2][w], c);
        all.rank += ranks[w];
    }
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
    if (g.there && !is_masked(a, id)) g.x = x;
    return g;
}

// ln S. The exponentials were formed with scale log2 e rounded to fp32, scale (1 + off): to the first order in
// `off` (at most 2^-23) ln S is larger by off times the mean of scale d.
__device__ __forceinline__ double log_sum(const Logprobs &a, const Part &p)
{
    const float c = a.scale * 1.44269504f;
    const double off = c / (a.scale * 1.4426950408889634) - 1;
    return log1p((p.count - 1) + p.s) - off * a.scale * (p.t / (p.count + p.s));
}

// NaN leaves a sum NaN; plus infinity is the maximum.
__device__ __forceinline__ bool has_none(const Part &p) { return !(p.m > -INFINITY && p.m < INFINITY) || !(p.s >= 0); }

// A row's results beside its first tokens, by one thread; ln S.
__device__ __forceinline__ double finish(const Logprobs &a, int row, const Given &g, const Part &p)
{
    const bool none = has_none(p);
    const double log_s = log_sum(a, p);
    if (a.tokens) {
        const bool ranked = g.there && !none && g.x > -INFINITY;
        a.logprobs[row] = !g.there ? 0.f : none ? NAN : (float)(((double)g.x - p.m) * a.scale - log_s);
        if (a.ranks) a.ranks[row] = ranked ? p.rank : -1;
    }
    if (a.entropies) a.entropies[row] = none ? NAN : (float)(log_s - p.t / (p.count + p.s) * a.scale);
    return log_s;
}

__device__ __forceinline__ void put_top(const Logprobs &a, int row, const Part &p, double log_s, const List &list, int held)
{
    const int k = threadIdx.x;
    if (k >= a.top) return;
    const bool none = has_none(p);
    const uint64_t key = k < held ? list.keys[k] : 0;
    const size_t at = (size_t)row * a.top + k;
    a.top_ids[at] = none || !key ? -1 : id_of(key);
    a.top_logprobs[at] = none ? NAN : !key ? -INFINITY : (float)(((double)logit_of(key) - p.m) * a.scale - log_s);
}

// Workgroup (row, share), 4 kV logits a thread and tile. Positions begin at the 16
// bytes that the row begins in. kWhole: the row is one share.
template <bool kTop, bool kWhole>
__global__ __launch_bounds__(kThreads) void logprobs_rows(Logprobs a, Reading r, Part *parts, float *all_maxima)
{
    __shared__ __align__(16) float maxima[kTop && kWhole ? kMostGroups : 4];
    const int row = kWhole ? blockIdx.x : blockIdx.x / r.shares, share = kWhole ? 0 : blockIdx.x % r.shares, tid = threadIdx.x;
    const float *x0 = a.logits + row * a.stride;
    const int shift = (int)((uintptr_t)x0 >> 2 & 3), end = a.n + shift;
    x0 -= shift;
    float *to_maxima = kWhole ? maxima : all_maxima + (size_t)blockIdx.x * r.sets * 64;
    const Given g = given_of(a, row);
    const float c = a.scale * 1.44269504f;
    float m = -INFINITY, s = 0.f, t = 0.f;
    int count = 0, rank = 0;
    float highest = -INFINITY;
    int set = 0, in_set = 0;
    // A set's maxima, of four threads each.
    auto put = [&]() {
        highest = fmaxf(highest, row_lane<0xB1>(highest));
        highest = fmaxf(highest, row_lane<0x4E>(highest));
        if (tid % 4 == 0) to_maxima[set * 64 + tid / 4] = highest;
        highest = -INFINITY;
        in_set = 0;
        ++set;
    };
    const int from = share * r.each() * kTile, to = min(end, from + r.each() * kTile);
    for (int tile = from; tile < to; tile += kTile) {
        float x[4 * kV];
#pragma unroll
        for (int v = 0; v < kV; ++v) {
            const int at = tile + 4 * (kThreads * v + tid);
            if (at >= shift && at + 3 < end) {
                *(float4 *)(x + 4 * v) = *(const float4 *)(x0 + at);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * v + e] = at + e >= shift && at + e < end ? x0[at + e] : -INFINITY;
            }
        }
        if (a.mask) {
#pragma unroll
            for (int v = 0; v < kV; ++v) {
                const int id = tile + 4 * (kThreads * v + tid) - shift;
                const int last = (a.n - 1) >> 5, first = max(id, 0) >> 5;
                uint32_t off = a.mask[min(first, last)];
                if (shift) {
                    // The four may lie in two words, or before the row's first.
                    const uint64_t both = (uint64_t)a.mask[min(max(id + 3, 0) >> 5, last)] << 32 | off;
                    off = id < 0 ? off << -id : (uint32_t)(both >> (id & 31));
                } else {
                    off >>= id & 31;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (off >> e & 1u) x[4 * v + e] = -INFINITY;
            }
        }
        float most = x[0];
#pragma unroll
        for (int i = 1; i < 4 * kV; ++i) most = fmaxf(most, x[i]);
        highest = fmaxf(highest, most);
        if (most > m) {
            // (The thread's first tile: there is nothing to rescale.)
            const float d = m - most, f = __builtin_amdgcn_exp2f(d * c);
            t = f == 0.f ? 0.f : (t + ((float)count + s) * d) * f;
            s = s * f + (float)count * f;
            count = 0;
            m = most;
        }
        const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int i = 0; i < 4 * kV; ++i) {
            // (NaN stays NaN in e, minus infinity is 0 there.)
            const float d = x[i] - base, low = fmaxf(d, -FLT_MAX);
            const float e = __builtin_amdgcn_exp2f(d * c);
            const bool at_most = x[i] == base;
            count += at_most;
            s += at_most ? 0.f : e;
            t = __builtin_fmaf(low, e, t);
        }
        // Which logits come before the given one goes by the id where they are equal.
        if (g.there) {
            const int id = tile - shift;
            if (g.id >= id && g.id < id + kTile) {
#pragma unroll
                for (int i = 0; i < 4 * kV; ++i) {
                    const int mine = id + 4 * (kThreads * (i / 4) + tid) + i % 4;
                    rank += x[i] > g.x || (x[i] == g.x && mine < g.id);
                }
            } else {
                const float bar = g.id < id || !(g.x > -INFINITY) ? g.x : below(g.x);
#pragma unroll
                for (int i = 0; i < 4 * kV; ++i) rank += x[i] > bar;
            }
        }
        if constexpr (kTop)
            if (++in_set == r.per_set) put();
    }
    if constexpr (kTop)
        while (set < r.sets) put();
    const Part p = together(m, (float)count, s, t, rank, c);
    if constexpr (!kWhole) {
        if (tid == 0) parts[blockIdx.x] = p;
    } else if constexpr (kTop) {
        __shared__ List list;
        __shared__ double log_s;
        Maxima mine;
        mine.load(maxima, r.sets * 64);
        const int held = choose(a, row, shift, r, mine, maxima, r.sets * 64, list, [&]() {
            if (tid == 64) log_s = finish(a, row, g, p);
        });
        put_top(a, row, p, log_s, list, held);
    } else if (tid == 0) {
        finish(a, row, g, p);
    }
}

// Workgroup: a row, from its shares.
template <bool kTop>
__global__ __launch_bounds__(kThreads) void logprobs_join(Logprobs a, Reading r, const Part *parts, const float *all_maxima)
{
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, groups = r.shares * r.sets * 64;
    Part p = {-INFINITY, 0, 0, 0, 0};
    if (lane < r.shares) p = parts[(size_t)row * r.shares + lane];
    const Given g = given_of(a, row);
    const float c = a.scale * 1.44269504f;
    // The shares' sums, in a wavefront.
    auto sums = [&]() {
        Part q = {wave_reduce<true>(p.m), 0, 0, 0, 0};
        add_to(q, p.m, p.count, p.s, p.t, c);
        q.count = wave_sum(q.count);
        q.s = wave_sum(q.s);
        q.t = wave_sum(q.t);
        q.rank = (int)wave_sum((float)p.rank);
        return q;
    };
    if constexpr (kTop) {
        __shared__ List list;
        __shared__ double log_s;
        __shared__ Part all;
        const float *maxima = all_maxima + (size_t)row * groups;
        Maxima mine;
        mine.load(maxima, groups);
        const int shift = (int)((uintptr_t)(a.logits + row * a.stride) >> 2 & 3);
        const int held = choose(a, row, shift, r, mine, maxima, groups, list, [&]() {
            const Part q = sums();
            if (lane != 0) return;
            all = q;
            log_s = finish(a, row, g, q);
        });
        put_top(a, row, all, log_s, list, held);
    } else if (tid < 64) {
        const Part q = sums();
        if (lane == 0) finish(a, row, g, q);
    }
}

size_t share_bytes(const Reading &r, int top) { return sizeof(Part) + (top ? (size_t)r.sets * 64 * sizeof(float) : 0); }

Reading reading_of(int n, int count, int top, size_t bytes)
{
    const int all = (n + 3 + kTile - 1) / kTile;   // a row may begin 3 floats into its 16 bytes
    // Four workgroups for each CU: 64 rows of 128256, 8, 16 and 32 shares 13.0, 10.6 and 11.5 us, the join 7;
    // from 1024 rows on, whole ones (2047 of 50257 77 us, in 4 shares 85 and 5 for the join).
    int shares = count >= kSplitRows ? 1 : (kSplitRows + count - 1) / count;
    shares = shares < kMostShares ? shares : kMostShares;
    for (;; --shares) {
        if (shares > all) shares = all;
        if (shares < 1) shares = 1;
        // Tiles of a share, in sets so that a row has at most 64 of them.
        const int each = (all + shares - 1) / shares, most = kMostGroups / 64 / shares, per_set = (each + most - 1) / most;
        Reading r = {shares, (each + per_set - 1) / per_set, per_set};
        r.shares = (all + r.each() - 1) / r.each();
        if (r.shares == 1 || share_bytes(r, top) * r.shares * count <= bytes) return r;
    }
}

}  // namespace

size_t logprobs_workspace(int n, int count, int top)
{
    // Fewer rows are split into more shares, and may want more: of the counts with the same shares the largest.
    size_t most = 0;
    for (int shares = 1; shares <= kMostShares; ++shares) {
        const int rows = shares == 1 || count < (kSplitRows - 1) / (shares - 1) ? count : (kSplitRows - 1) / (shares - 1);
        const Reading r = reading_of(n, rows, top, SIZE_MAX);
        const size_t bytes = r.shares == 1 ? 0 : share_bytes(r, top) * r.shares * rows;
        most = bytes > most ? bytes : most;
    }
    return most;
}

hipError_t launch_logprobs(const Logprobs &a, void *workspace, size_t workspace_bytes, hipStream_t s)
{
    const Reading r = reading_of(a.n, a.count, a.top, workspace ? workspace_bytes : 0);
    Part *parts = (Part *)workspace;
    float *maxima = (float *)(parts + (size_t)a.count * r.shares);
    const dim3 grid((unsigned)((int64_t)a.count * r.shares)), threads(kThreads);
    if (r.shares == 1) {
        if (a.top) hipLaunchKernelGGL((logprobs_rows<true, true>), grid, threads, 0, s, a, r, parts, maxima);
        else hipLaunchKernelGGL((logprobs_rows<false, true>), grid, threads, 0, s, a, r, parts, maxima);
        return hipGetLastError();
    }
    if (a.top) {
        hipLaunchKernelGGL((logprobs_rows<true, false>), grid, threads, 0, s, a, r, parts, maxima);
        hipLaunchKernelGGL((logprobs_join<true>), dim3(a.count), threads, 0, s, a, r, parts, maxima);
    } else {
        hipLaunchKernelGGL((logprobs_rows<false, false>), grid, threads, 0, s, a, r, parts, maxima);
        hipLaunchKernelGGL((logprobs_join<false>), dim3(a.count), threads, 0, s, a, r, parts, maxima);
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
