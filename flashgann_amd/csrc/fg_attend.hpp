// fg_attend.hpp -- what the attention kernels over the paged cache share.
//
// The work is a list of items.  An item is a block of query rows (rows of one
// request that read the same keys and values: the query heads of a group, for
// each new token) against its request's visible tokens; these are counted in
// units, and the units of all items, laid end to end, are dealt out evenly:
// workgroup w takes units [w * share, (w + 1) * share).  A ragged batch and one
// long context fill the device the same way, and the host needs no lengths.
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
    uint32_t blocks, units;  // row blocks, units of each (enough for the longest)
};

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

template <bool FOUND, uint32_t ROWS, uint32_t UNIT>
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
    // a block's window spans that many tokens more than one row's
    uint64_t seen = q.limit;
    if (P.window != 0xFFFFFFFFu)
        seen = min(seen, static_cast<uint64_t>(P.sinks) + P.window + (ROWS - 1) / P.group.d + 1);
    if constexpr (FOUND) seen += P.nids;
    q.units = max(1u, static_cast<uint32_t>((seen + UNIT - 1) / UNIT));
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
    uint64_t units, share;  // of all items; of a workgroup
    uint64_t before;        // units of the requests before `request`
    uint32_t request;
};

// Called by all 256 threads; every workgroup sums the requests' units itself.
template <bool FOUND, uint32_t ROWS, uint32_t UNIT>
__device__ Start find_start(const AttendParams &P, uint32_t w, uint32_t workgroups, uint64_t least) {
    __shared__ uint64_t wave_sum[4];
    __shared__ uint64_t found_before;
    __shared__ uint32_t found_request;
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    Start s{0, 0, 0, 0};
    for (int pass = 0; pass < 2; ++pass) {
        uint64_t sum = 0;
        for (uint32_t r0 = 0; r0 < P.requests; r0 += 256) {
            const uint32_t r = r0 + tid;
            uint64_t u = 0;
            if (r < P.requests) {
                const Request q = request_of<FOUND, ROWS, UNIT>(P, r);
                u = static_cast<uint64_t>(q.blocks) * q.units * P.lists;
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
            for (uint32_t i = 0; i < 4; ++i) {
                if (i < wave) base += wave_sum[i];
                sum += wave_sum[i];
            }
            // one chunk of requests: the totals of the first pass serve the second
            if (pass == 1 || P.requests <= 256) {
                if (P.requests <= 256) {
                    s.units = sum;
                    s.share = max((sum + workgroups - 1) / workgroups, least);
                }
                const uint64_t x = w * s.share;
                if (u && base + v - u <= x && x < base + v) {
                    found_before = base + v - u;
                    found_request = r;
                }
            }
            __syncthreads();
        }
        if (P.requests <= 256) break;
        if (pass == 0) {
            s.units = sum;
            s.share = max((sum + workgroups - 1) / workgroups, least);
        }
    }
    if (w * s.share < s.units) {
        s.before = found_before;
        s.request = found_request;
    }
    return s;
}

}  // namespace fgk

#endif
