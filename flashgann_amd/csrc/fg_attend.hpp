// fg_attend.hpp -- what the attention kernels over the paged cache share.
//
// The work is a list of items.  An item is a block of query rows (rows of one
// request that read the same keys and values: the query heads of a group, for
// each new token) against its request's visible tokens.  Each item has a weight
// near its cost, the weights of all items are laid end to end, and that length
// is dealt out evenly: workgroup w takes [w * share, (w + 1) * share) of it, and
// of an item that a cut goes through the tokens in proportion.  A ragged batch, a
// causal triangle and one long context fill the device the same way, and the
// host needs no lengths.
// A workgroup writes the rows of an item that it holds whole; of one that it
// holds in part it leaves the sum, the maximum and the weighted values in the
// workspace, and the join kernel adds the parts in their order, so the result
// doesn't depend on timing.
#ifndef FG_ATTEND_HPP
#define FG_ATTEND_HPP

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "fg_cache.hpp"

namespace fgk {

struct AttendParams {
    CacheView cache;
    const char *q;
    char *out;
    float *lse;
    int64_t q_token, q_head, out_token, out_head;  // bytes
    const int32_t *table, *q_starts, *kv_lens;
    const uint32_t *ids;
    int64_t table_row;
    float *part;         // kParts x rows x dim
    float2 *part_ml;     // kParts x rows: maximum (base 2), sum
    struct Join *joins;  // one a workgroup
    uint32_t table_width, requests, tokens, heads;
    uint32_t lists;      // items side by side: key/value heads, or id lists
    uint32_t list_heads; // lists a key/value head
    uint32_t nids, window, sinks;  // window 0xFFFFFFFF: none
    uint32_t join;       // whether the join kernel follows
    uint64_t least;      // weight that a workgroup takes at least
    FastDiv group;       // query heads that share a list
    float scale2;        // scale * log2(e)
};

// What the join kernel needs of an item in parts; pieces 0: nothing to do.
struct Join {
    uint32_t pieces, row0, rows, q0, list;
};

// One request as the kernels see it.
struct Request {
    int32_t q0, rows;     // first row of q, query rows of a list (new tokens * group)
    int32_t kv, limit;    // tokens of the request, and of those how many the table can name
    int32_t fresh;        // new tokens
    uint32_t blocks;      // of rows
    // Weight of the first b blocks of a list: b * base + b (b + 1) / 2 * step, in
    // (token, query head of the group) pairs.  Without a window the tokens that
    // block b sees grow by a block's tokens from block to block.
    uint64_t base, step;
    __device__ __forceinline__ uint64_t weight_of(uint64_t b) const { return b * base + b * (b + 1) / 2 * step; }
};

// An item's own cost beside its tokens: its prologue and its rows' output, in
// tokens.  Not zero: an item without tokens still writes its rows.
constexpr uint32_t kItemTokens = 32;

// The tokens that the rows row0 .. of a block see between them: 0 .. first - 1, then
// from `from` on, then the ids.  Token number t of them is at position_of(t).
struct Span {
    int32_t first, from, dense, total;
    int32_t pos0;  // position of the block's first row's token less that token's number
};

// Whole-wave exchanges without LDS: x from the lane whose bit 4 (5) differs.
__device__ __forceinline__ float max_other16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_other32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_other16(float x) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_other32(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ int32_t clampi(int32_t v, int32_t lo, int32_t hi) { return min(max(v, lo), hi); }

template <bool FOUND, uint32_t ROWS>
__device__ __forceinline__ Request request_of(const AttendParams &P, uint32_t r) {
    Request q;
    const int32_t T = static_cast<int32_t>(P.tokens);
    if constexpr (FOUND) {
        q.q0 = static_cast<int32_t>(r);
        q.fresh = 1;
    } else {
        q.q0 = clampi(P.q_starts[r], 0, T);
        q.fresh = clampi(P.q_starts[r + 1], q.q0, T) - q.q0;
    }
    q.kv = max(P.kv_lens[r], 0);
    const uint64_t room = static_cast<uint64_t>(P.table_width) * P.cache.page_size.d;
    q.limit = static_cast<int32_t>(min(static_cast<uint64_t>(q.kv), room));
    q.rows = q.fresh * static_cast<int32_t>(P.group.d);
    q.blocks = (static_cast<uint32_t>(q.rows) + ROWS - 1) / ROWS;
    q.base = static_cast<uint64_t>(kItemTokens + max(q.kv - q.fresh, 0)) * P.group.d;
    q.step = ROWS;
    if (FOUND || P.window != 0xFFFFFFFFu) {
        // every block sees about as much (the first ones of a context less)
        uint64_t seen = min(static_cast<uint64_t>(q.limit), static_cast<uint64_t>(P.sinks) + P.window + ROWS / P.group.d);
        if constexpr (FOUND) seen += P.nids;
        q.base = (kItemTokens + seen) * P.group.d;
        q.step = 0;
    }
    return q;
}

template <bool FOUND, uint32_t ROWS>
__device__ __forceinline__ Span span_of(const AttendParams &P, const Request &q, uint32_t block) {
    const int32_t row0 = static_cast<int32_t>(block * ROWS), row1 = min(row0 + static_cast<int32_t>(ROWS), q.rows) - 1;
    const int32_t t0 = P.group.div(row0), t1 = P.group.div(row1);
    Span s;
    s.pos0 = q.kv - q.fresh;
    const int32_t end = clampi(s.pos0 + t1 + 1, 0, q.limit);
    s.first = s.from = 0;
    if (P.window != 0xFFFFFFFFu) {
        s.first = static_cast<int32_t>(min(P.sinks, static_cast<uint32_t>(end)));
        s.from = static_cast<int32_t>(max(static_cast<int64_t>(s.first), static_cast<int64_t>(s.pos0) + t0 + 1 - P.window));
    }
    s.dense = s.first + max(end - s.from, 0);
    s.total = s.dense + (FOUND ? static_cast<int32_t>(P.nids) : 0);
    return s;
}

__device__ __forceinline__ int32_t position_of(const Span &s, int32_t t) { return t < s.first ? t : t + s.from - s.first; }

// Page and offset of the token at position j of request r; page -1 where the
// table names none.  j is below the request's limit.
__device__ __forceinline__ int2 place_of(const AttendParams &P, uint32_t r, int32_t j) {
    const uint32_t b = P.cache.page_size.div(j);
    const int32_t page = P.table[r * P.table_row + b];
    return {static_cast<uint32_t>(page) < P.cache.pages ? page : -1, static_cast<int32_t>(j - b * P.cache.page_size.d)};
}

// Where a workgroup's share begins.
struct Start {
    uint64_t all, share;  // weight of all items; of a workgroup
    uint64_t before;      // weight of the requests before `request`
    uint32_t request;
};

// Called by all THREADS threads; every workgroup sums the requests' weights itself.
template <bool FOUND, uint32_t ROWS, uint32_t THREADS>
__device__ Start find_start(const AttendParams &P, uint32_t w, uint32_t workgroups) {
    constexpr uint32_t WAVES = THREADS / 64;
    __shared__ uint64_t wave_sum[WAVES];
    __shared__ uint64_t found_before;
    __shared__ uint32_t found_request;
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const bool once = P.requests <= THREADS;  // one look at the requests gives the sum and the place
    Start s{0, 0, 0, 0};
    for (int pass = once ? 1 : 0; pass < 2; ++pass) {
        uint64_t sum = 0;
        for (uint32_t r0 = 0; r0 < P.requests; r0 += THREADS) {
            const uint32_t r = r0 + tid;
            uint64_t u = 0;
            if (r < P.requests) {
                const Request q = request_of<FOUND, ROWS>(P, r);
                u = q.weight_of(q.blocks) * P.lists;
            }
            uint64_t v = u;
#pragma unroll
            for (uint32_t d = 1; d < 64; d <<= 1) {
                const uint64_t o = __shfl_up(v, d);
                if (lane >= d) v += o;
            }
            if (lane == 63) wave_sum[wave] = v;
            __syncthreads();
            uint64_t base = sum;
#pragma unroll
            for (uint32_t i = 0; i < WAVES; ++i) {
                if (i < wave) base += wave_sum[i];
                sum += wave_sum[i];
            }
            if (once) {
                s.all = sum;
                s.share = max((sum + workgroups - 1) / workgroups, P.least);
            }
            const uint64_t x = w * s.share;
            if (pass == 1 && u && base + v - u <= x && x < base + v) {
                found_before = base + v - u;
                found_request = r;
            }
            __syncthreads();
        }
        if (pass == 0) {
            s.all = sum;
            s.share = max((sum + workgroups - 1) / workgroups, P.least);
        }
    }
    if (w * s.share < s.all) {
        s.before = found_before;
        s.request = found_request;
    }
    return s;
}

// What of an item a workgroup holds.
struct Piece {
    uint32_t list, block;
    uint32_t t_lo, t_hi;      // token numbers of its span, cut between units of UNIT tokens
    uint64_t end;             // where the item's weight ends
    bool begins, ends;        // whether the item's first (last) unit is here
    bool none;                // no unit is, and none came before: another workgroup begins the item
};

// The item that x lies in (x is inside request q, whose weight begins at
// `before`), and its tokens up to x1.  Two neighbours work out the cut between
// them from the same numbers.
template <bool FOUND, uint32_t ROWS, uint32_t UNIT>
__device__ __forceinline__ Piece piece_of(const AttendParams &P, const Request &q, uint64_t before, uint64_t x, uint64_t x1,
                                          Span *span) {
    Piece p;
    const uint64_t list_weight = q.weight_of(q.blocks);
    p.list = static_cast<uint32_t>((x - before) / list_weight);
    const uint64_t start = before + p.list * list_weight, at = x - start;
    uint32_t lo = 0, hi = q.blocks;  // the last block that begins at or before `at`
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (q.weight_of(mid) <= at) lo = mid;
        else hi = mid;
    }
    p.block = lo;
    const uint64_t begin = start + q.weight_of(lo), weight = q.weight_of(lo + 1) - q.weight_of(lo);
    p.end = begin + weight;
    *span = span_of<FOUND, ROWS>(P, q, lo);
    const uint32_t total = span->total, units = max((total + UNIT - 1) / UNIT, 1u);
    // x, and x1 inside the item, fall into units 0 .. units - 1: the workgroup that holds the
    // item's end holds its last unit, and an item of one unit is never cut
    const uint32_t u0 = static_cast<uint32_t>((x - begin) * units / weight);
    const uint32_t u1 = x1 >= p.end ? units : static_cast<uint32_t>((x1 - begin) * units / weight);
    p.begins = u0 == 0;
    p.ends = u1 == units;
    p.none = u1 == 0;
    p.t_lo = min(u0 * UNIT, total);
    p.t_hi = min(u1 * UNIT, total);
    return p;
}

}  // namespace fgk

#endif
