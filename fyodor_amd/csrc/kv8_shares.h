// How attention over a paged cache (attention_kv8.hip, attention_kv4.hip: A is its
// arguments) is divided: the positions that a tile of query rows sees, their
// shares, and the grids of a call. Plain arithmetic, the same on the host and
// in the kernels.
#pragma once
#include "serving.h"

namespace fy {
namespace {

constexpr int kStep = 64;   // positions per step of a wavefront
constexpr int kRows = 16;   // query rows per tile of a few
constexpr int kWaves = 4;
constexpr int kMostSplits = 64;   // a lane each where they are joined
constexpr int kWideRows = 32 * kWaves;   // query rows per tile of many

// The positions that a tile of query rows sees and how they are split: steps
// [begin, end) of 64 positions in `active` shares of `chunk`.
struct Range {
    int lowest, highest;   // positions, highest < 0: none
    int begin, chunk, active, end;

    // Steps of share sp. The first one has what is left over: the grids begin
    // with the last shares, so the shorter ones come where others have ended.
    __host__ __device__ __forceinline__ int until(int sp) const { return end - (active - 1 - sp) * chunk; }
    __host__ __device__ __forceinline__ int from(int sp) const { return max(begin, until(sp) - chunk); }
};

// How the positions of tiles are shared out: among `most` workgroups, at least
// `least` steps each, which leave their rows (and each row's maximum and sum)
// in the workspace: room for `places` places of `tile` rows, for every KV head.
// A place is a request, or (listed) a tile of the requests' rows by tile_of.
// Packed: the grid counts the shares there are, by item_of.
struct Share {
    float *o;
    float2 *ml;
};
struct Split {
    int most, least, tile, places;
    bool listed, packed;
    float *partials;

    __host__ __device__ __forceinline__ Share share(int kv_heads, int place, int kvh, int row, int sp, int width) const
    {
        const size_t at = (((size_t)place * kv_heads + kvh) * tile + row) * most + sp;
        return {partials + at * width, (float2 *)(partials + (size_t)places * kv_heads * tile * most * width) + at};
    }
};

// Request r's rows, the first position and whether it brings any.
struct Request {
    int begin, rows;   // first row; rows of one KV head: tokens x group
    int64_t first;     // position of its first token
};

template <class A>
__host__ __device__ __forceinline__ Request request_of(const A &a, int r)
{
    const int start = a.starts[r], stop = a.starts[r + 1];
    const int begin = max(start, 0), end = max(min(stop, a.count), 0), tokens = min(end - begin, a.max_tokens);
    return {begin, tokens > 0 ? tokens * (a.heads / a.cache.kv_heads) : 0,
            (int64_t)a.lengths[r] - ((int64_t)stop - begin)};
}

template <class A>
__host__ __device__ __forceinline__ Range range_of(const A &a, const Request &q, int tile, int rows, int splits,
    int least)
{
    const int group = a.heads / a.cache.kv_heads;
    // Positions of the steps looked up past the last one still fit 31 bits.
    const int64_t most = min((int64_t)a.table_stride * a.cache.page_tokens - 1, (int64_t)INT32_MAX - 64 * kStep);
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

// How the counted grid takes a request of a few rows: its tiles, each with as
// many shares as the one that has most. (Not as the last tile has: under a
// window, or where a tile's steps divide otherwise, an earlier one may have more.)
struct Items {
    int tiles, shares;
};

template <class A>
__host__ __device__ __forceinline__ Items items_of(const A &a, const Split &split, const Request &q,
    int most_rows)
{
    Items items = {0, 0};
    if (q.rows <= 0 || q.rows > most_rows) return items;
    items.tiles = (q.rows + kRows - 1) / kRows;
    for (int tile = 0; tile < items.tiles; ++tile) {
        const int active = range_of(a, q, tile, kRows, split.most, split.least).active;
        items.shares = active > items.shares ? active : items.shares;
    }
    return items;
}

// Item `left` < tiles x shares of them.
struct Item {
    int tile, share;
};

__host__ __device__ __forceinline__ Item item_at(int tiles, int left) { return {left % tiles, left / tiles}; }

// Tiles of `tile` rows that a step can have: every request's last one may be short.
inline int64_t most_tiles(int requests, int max_tokens, int count, int group, int tile)
{
    const int64_t each = ((int64_t)max_tokens * group + tile - 1) / tile * requests;
    const int64_t all = (int64_t)count * group / tile + requests;
    return each < all ? each : all;
}

// Requests of more than most_rows rows (of one KV head) run in wide tiles.
struct Plan {
    int most_rows;
    bool any_few, any_wide;
    Split few, wide;
};

template <class A>
inline size_t share_bytes(const A &a, const Split &s)
{
    return (size_t)s.places * s.tile * a.cache.kv_heads * (a.cache.width + 2) * sizeof(float);
}

template <class A>
inline Plan plan_of(const A &a, float *workspace, size_t bytes)
{
    const int group = a.heads / a.cache.kv_heads, width = a.cache.width;
    const int64_t rows = (int64_t)a.max_tokens * group;
    int64_t range = a.max_length;
    if (a.window && (int64_t)a.window + a.max_tokens < range) range = (int64_t)a.window + a.max_tokens;
    const int64_t steps = (range + kStep - 1) / kStep + 1;
    Plan p = {INT32_MAX, true, false, {1, kWaves, 0, 0, false, false, nullptr}, {1, 4, kWideRows, 0, true, false, nullptr}};
    if (width <= 256 && rows > 64) {
        // Up to 64 rows are fewer keys read again than wide tiles leave empty (8
        // requests of 5 tokens of 32 heads over 4 of 64: 12 us, wide 18 to 23). In
        // a batch with longer ones, which pays for every place of a tile that
        // a request of a few rows might have, the tiles that one token takes (a
        // prompt of 512 among 64 requests, 32 heads over 8 of 128: 176 us, with
        // two tiles 188; 64 over 2 of 64: 107 with the two tiles of a token, 149
        // with it in wide ones); a single request is all wide. It loses where single
        // tokens are many and take many tiles: 130 requests with a prompt among
        // them, 32 heads over 1 of 128: 83, in wide tiles 67.
        p.most_rows = a.requests == 1 ? 0 : group > 64 ? kRows : (group + kRows - 1) / kRows * kRows;
        p.any_wide = true;
        p.any_few = a.requests > 1;
    }
    if (p.any_few) {
        p.few.tile = (int)(rows < p.most_rows ? rows : p.most_rows);
        p.few.places = a.requests;
        if (!p.any_wide && rows > 64) {
            // Prompts of heads of 512: as many tiles as the rows make.
            p.few.listed = true;
            p.few.tile = kRows;
            p.few.places = (int)most_tiles(a.requests, a.max_tokens, a.count, group, kRows);
        }
        // In a mixed batch most of these requests bring a token each.
        const int64_t tiles = (p.any_wide ? (int64_t)(group + kRows - 1) / kRows * a.requests
                                          : most_tiles(a.requests, a.max_tokens, a.count, group, kRows)) *
                              a.cache.kv_heads;
        // Fewer tiles than CUs: shares for three workgroups per CU (one at widths
        // that fill a CU's registers), at least a step per wavefront. Enough
        // tiles: none, sharing costs about 6 us (32 requests of 2048 positions, 8
        // heads of 128, us: whole 25, halves 31, quarters 34), but in long contexts,
        // where the requests' lengths differ by more (64 of 500 to 8192: whole 105,
        // 2048 shares were they all long 97). The border, 96 steps, is on the side of
        // whole ones (64 requests of 300 to n positions, whole and in shares: n 1500
        // 25 and 37, 3000 46 and 50, 4500 63 and 59, 5900 77 and 68).
        const int64_t wanted = tiles < 256 ? (width <= 128 ? 768 : 256) : steps >= 96 ? 2048 : 0;
        const int64_t share = wanted ? (tiles * steps + wanted - 1) / wanted : steps;
        if (share > p.few.least) p.few.least = (int)share;
        const int64_t most = (steps + p.few.least - 1) / p.few.least;
        p.few.most = most > kMostSplits ? kMostSplits : (int)most;
        // Requests of unequal lengths leave gaps in a grid of all their shares,
        // and the CUs get unequal work; counting them costs a look at
        // every request, one for up to 64 (32 and 64 of 500 to 8192 positions: 53
        // and 98 us, counted 50 and 91; 16, with 128 tiles, 28 and 29; past 64
        // it gains nothing: 65 requests 94 both, 96 128 and 130, 192 of up to
        // 6500 209 and 213).
        p.few.packed = p.few.most > 1 && tiles >= 256 && a.requests <= 64 && !p.few.listed;
    }
    if (p.any_wide) {
        // Wide tiles fill a CU each, so they are split while they leave CUs idle: as
        // many tiles as the rows make, short last ones left out (24 requests, two
        // of them prompts of 256 tokens, 32 heads over 8 of 128: 65 us whole, 42 and 9
        // for the join in halves).
        p.wide.places = (int)most_tiles(a.requests, a.max_tokens, a.count, group, kWideRows);
        const double tiles = (double)a.count * group / kWideRows * a.cache.kv_heads;
        int64_t most = (int64_t)(256 / (tiles < 1 ? 1 : tiles) + 0.4);
        if (most > steps / 4) most = steps / 4;
        // Places that stay empty are launched and have their share of the workspace, too.
        const int64_t places = (int64_t)p.wide.places * a.cache.kv_heads;
        if (most > 16384 / places) most = 16384 / places;
        p.wide.most = most < 1 ? 1 : most > kMostSplits ? kMostSplits : (int)most;
    }
    size_t taken = 0;
    for (Split *s : {&p.wide, &p.few}) {
        if (s->most == 1) continue;
        const size_t each = share_bytes(a, *s);
        if (bytes / each < (size_t)s->most) s->most = bytes / each < 2 ? 1 : (int)(bytes / each);
        if (s->most == 1) continue;
        if (workspace) s->partials = workspace + taken;
        taken += s->most * each / sizeof(float);
        bytes -= s->most * each;
    }
    return p;
}

}  // namespace
}  // namespace fy
