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
#include <type_traits>

#include "fg_cache.hpp"

namespace fgk {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;

// kTopWeight: the base-2 logarithm that the largest weight of a row may have when it is
// rounded for the product with the values.  bfloat16 has float's exponents; float16 ends
// at 2^-24, so its weights are taken as far up as it goes (2^16 is past its end), or
// those below 2^-25 of the maximum would be lost, which over 65,536 tokens may be 0.2%
// of a row, over a million 3%.
struct BF16 {
    using vec = bf16x8;
    static constexpr uint32_t kExponent = 0x7F80, kMantissa = 0x007F;
    static constexpr int kTopWeight = 0;
    static __device__ __forceinline__ f32x4 mfma16(vec a, vec b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(vec a, vec b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
        return __builtin_bit_cast(uint32_t, v);
    }
};
struct F16 {
    using vec = f16x8;
    static constexpr uint32_t kExponent = 0x7C00, kMantissa = 0x03FF;
    static constexpr int kTopWeight = 15;
    static __device__ __forceinline__ f32x4 mfma16(vec a, vec b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(vec a, vec b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        f16x2 v = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
        return __builtin_bit_cast(uint32_t, v);
    }
};

// Four rows of one column each: lane i of 16 gets column i of the 4 x 16 block
// whose row i / 4, columns 4 (i % 4) .. + 3 lie at lane i's address.
__device__ __forceinline__ s16x4 read_transposed(const char *lds) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(lds));
}

template <class T>
__device__ __forceinline__ bool any_special(u32x4 w) {
    bool s = false;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        s |= ((w[i] & T::kExponent) == T::kExponent) | (((w[i] >> 16) & T::kExponent) == T::kExponent);
    return s;
}

// The same with its infinities and NaNs as zeros.
template <class T>
__device__ __forceinline__ u32x4 finite_part(u32x4 w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if ((w[i] & T::kExponent) == T::kExponent) w[i] &= 0xFFFF0000u;
        if (((w[i] >> 16) & T::kExponent) == T::kExponent) w[i] &= 0x0000FFFFu;
    }
    return w;
}

// An infinity or NaN among a value's 16 bits as a float, 0 for any other.
template <class T>
__device__ __forceinline__ float special_part(uint32_t x) {
    const float inf = x & 0x8000 ? -INFINITY : INFINITY;
    return (x & T::kExponent) != T::kExponent ? 0.0f : x & T::kMantissa ? NAN : inf;
}

struct AttendParams {
    CacheView cache;
    const char *q;
    char *out;
    float *lse;
    int64_t q_token, q_head, out_token, out_head;  // bytes
    const int32_t *table, *q_starts, *kv_lens;
    const uint32_t *ids;
    int64_t table_row;
    float *part;         // two a workgroup x rows x dim
    float2 *part_ml;     // two a workgroup x rows: maximum (base 2), sum
    struct Join *joins;  // one a workgroup
    uint32_t table_width, requests, tokens, heads;
    uint32_t lists;      // items side by side: key/value heads, or id lists
    uint32_t list_heads; // lists a key/value head
    uint32_t nids, window, sinks;  // window 0xFFFFFFFF: none
    uint32_t join;       // whether the join kernel follows
    uint32_t tiles, rows;  // whether the tile kernel runs; query rows of a block
    uint32_t workgroups; // of the attention kernel, a power of two
    FastDiv group;       // query heads that share a list
    FastDiv unit;        // tokens between cuts through an item, a multiple of a tile
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
// tokens.  It is also the weight that a workgroup takes at least.  With 32 of both
// (and 256 at least) four items of few tokens shared a workgroup while most had
// none: 7 requests of up to 24 tokens took 43.7 us against 13.0, 24 mixed chunks 105
// against 85; few rows, 4 requests of 200 to 1,500 tokens, 16.4 against 13.5 (and
// 64 of 500 to 16,000, 475 against 480).
template <uint32_t ROWS>
constexpr uint32_t kItemTokens = ROWS > 16 ? 256 : 128;

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

// A value that all lanes hold alike, into scalar registers: what describes an item
// lives through its whole loop.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int32_t uniform(int32_t x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint64_t uniform(uint64_t x) {
    return static_cast<uint64_t>(uniform(static_cast<uint32_t>(x >> 32))) << 32 | uniform(static_cast<uint32_t>(x));
}

// Lane `from`'s value; `from` is the same in all lanes.
__device__ __forceinline__ int32_t of_lane(int32_t x, uint32_t from) { return __builtin_amdgcn_readlane(x, from); }
__device__ __forceinline__ uint64_t of_lane(uint64_t x, uint32_t from) {
    return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int32_t>(x >> 32), from))) << 32 |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int32_t>(x), from));
}

// Waits for every load from global memory.  Where loads on one path into a loop are
// not known to have landed, the compiler waits for all of them inside it, those
// under way for the next tile with them.
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// The same value, as far as the compiler knows another: what follows from it is
// worked out again instead of being kept in registers through the products.
__device__ __forceinline__ int32_t renewed(int32_t x) {
    asm volatile("" : "+v"(x));
    return x;
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
    q.base = static_cast<uint64_t>(kItemTokens<ROWS> + max(q.kv - q.fresh, 0)) * P.group.d;
    q.step = ROWS;
    if (FOUND || P.window != 0xFFFFFFFFu) {
        // every block sees about as much (the first ones of a context less)
        uint64_t seen = min(static_cast<uint64_t>(q.limit), static_cast<uint64_t>(P.sinks) + P.window + ROWS / P.group.d);
        if constexpr (FOUND) seen += P.nids;
        q.base = (kItemTokens<ROWS> + seen) * P.group.d;
        q.step = 0;
    }
    return q;
}

template <bool FOUND, uint32_t ROWS>
__device__ __forceinline__ Span span_of(const AttendParams &P, const Request &q, uint32_t block) {
    const int32_t row0 = static_cast<int32_t>(block * ROWS), row1 = min(row0 + static_cast<int32_t>(ROWS), q.rows) - 1;
    const int32_t t0 = uniform(static_cast<int32_t>(P.group.div(row0))), t1 = uniform(static_cast<int32_t>(P.group.div(row1)));
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

// The workgroup that weight x falls to.
__device__ __forceinline__ uint32_t workgroup_at(uint64_t x, uint64_t share) {
    uint64_t w = static_cast<uint64_t>(static_cast<double>(x) / static_cast<double>(share));
    w -= w * share > x;
    w += (w + 1) * share <= x;
    return static_cast<uint32_t>(w);
}

// The n lowest bits; none below 0, all from 64 on.
__device__ __forceinline__ uint64_t bits_below(int32_t n) {
    return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1;
}

// x where bit `at` of `bits` is set, else -infinity.
__device__ __forceinline__ float keep_if(uint32_t bits, int at, float x) {
    const uint32_t all = static_cast<int32_t>(bits << (31 - at)) >> 31;
    return __uint_as_float((__float_as_uint(x) & all) | (0xFF800000u & ~all));
}

// Whether the row at `pos` sees the token at position j (pages aside).
__device__ __forceinline__ bool sees(const AttendParams &P, int32_t pos, int32_t j) {
    const int32_t back = pos - j;
    return (back >= 0) & ((static_cast<uint32_t>(back) < P.window) | (static_cast<uint32_t>(j) < P.sinks));
}

// The request of every lane's `r`, which is the same.
template <bool FOUND, uint32_t ROWS>
__device__ __forceinline__ Request uniform_request(const AttendParams &P, uint32_t r) {
    Request q = request_of<FOUND, ROWS>(P, r);
    q.q0 = uniform(q.q0);
    q.fresh = uniform(q.fresh);
    q.rows = uniform(q.rows);
    q.kv = uniform(q.kv);
    q.limit = uniform(q.limit);
    q.blocks = uniform(q.blocks);
    q.base = uniform(q.base);
    return q;
}

// Where a workgroup's share begins.
struct Start {
    uint64_t all, share;  // weight of all items; of a workgroup
    uint64_t before;      // weight of the requests before `request`
    uint32_t request;     // the first of the lane's run that the share begins in: up to requests / 64 before its own
    Request first;        // what that request is
};

// Every wave sums the requests' weights itself, a lane a run of them: nothing is
// waited for but the lengths.  The run that the share begins in is then walked a request
// at a time (65,536 requests: up to 1,023).  One token each over 10, 8 heads over 2: 64
// requests 8 us, 4,096 135 us, 65,536 2,160 us, most of it their items.  workgroups is a
// power of two.
template <bool FOUND, uint32_t ROWS>
__device__ __forceinline__ Start find_start(const AttendParams &P, uint32_t w) {
    const uint32_t lane = threadIdx.x % 64, run = (P.requests + 63) / 64;
    uint64_t mine = 0;
    Request q{};  // the first of the lane's run
    for (uint32_t i = run; i-- > 0;) {
        const uint32_t r = lane * run + i;
        if (r < P.requests) {
            q = request_of<FOUND, ROWS>(P, r);
            mine += q.weight_of(q.blocks) * P.lists;
        }
    }
    uint64_t upto = mine;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint64_t o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
    }
    Start s;
    s.all = of_lane(upto, 63);
    s.share = max((s.all + P.workgroups - 1) >> __builtin_ctz(P.workgroups), static_cast<uint64_t>(kItemTokens<ROWS>) * P.group.d);
    const uint64_t x = w * s.share;
    const uint64_t at = __ballot(upto > x && upto - mine <= x);
    const uint32_t owner = at ? __ffsll(static_cast<unsigned long long>(at)) - 1 : 0;
    s.before = of_lane(upto - mine, owner);
    s.request = owner * run;
    s.first.q0 = of_lane(q.q0, owner);
    s.first.rows = of_lane(q.rows, owner);
    s.first.kv = of_lane(q.kv, owner);
    s.first.limit = of_lane(q.limit, owner);
    s.first.fresh = of_lane(q.fresh, owner);
    s.first.blocks = of_lane(static_cast<int32_t>(q.blocks), owner);
    s.first.base = of_lane(q.base, owner);
    s.first.step = FOUND || P.window != 0xFFFFFFFFu ? 0 : ROWS;
    return s;
}

// What of an item a workgroup holds.
struct Piece {
    uint32_t list, block;
    uint32_t t_lo, t_hi;      // token numbers of its span, cut between units
    uint64_t end;             // where the item's weight ends
    bool begins, ends;        // whether the item's first (last) unit is here
    bool none;                // no unit is, and none came before: another workgroup begins the item
};

// The item that x lies in (x is inside request q, whose weight begins at
// `before`), and its tokens up to x1.  Two neighbours work out the cut between
// them from the same numbers.
template <bool FOUND, uint32_t ROWS>
__device__ __forceinline__ Piece piece_of(const AttendParams &P, const Request &q, uint64_t before, uint64_t x, uint64_t x1,
                                          Span *span) {
    Piece p;
    const uint32_t lane = threadIdx.x % 64;
    // the list and the block by 64 guesses at a time (a division of 64-bit numbers is
    // a hundred instructions in a row)
    const uint64_t list_weight = q.weight_of(q.blocks);
    uint32_t list = 0;
    for (uint32_t n = 64; n == 64; list += 64) {
        const uint32_t guess = list + lane;
        n = __popcll(__ballot(guess < P.lists && guess * list_weight <= x - before));
        if (n < 64) list += n - 1;
        if (n < 64) break;
    }
    p.list = list;
    const uint64_t start = before + list * list_weight, at = x - start;
    uint32_t lo = 0;  // the last block that begins at or before `at`
    for (uint32_t len = q.blocks; len > 1;) {
        const uint32_t stride = (len + 63) / 64, guess = lane * stride;
        const uint32_t n = __popcll(__ballot(guess < len && q.weight_of(lo + guess) <= at)) - 1;
        lo += n * stride;
        len = min(stride, len - n * stride);
    }
    p.block = lo;
    const uint64_t begin = start + q.weight_of(lo), weight = q.weight_of(lo + 1) - q.weight_of(lo);
    p.end = begin + weight;
    *span = span_of<FOUND, ROWS>(P, q, lo);
    const uint32_t total = span->total, units = uniform(max(P.unit.div(total + P.unit.d - 1), 1u));
    // x, and x1 inside the item, fall into units 0 .. units - 1: the workgroup that holds the
    // item's end holds its last unit, and an item of one unit is never cut
    const float per = static_cast<float>(units) * __builtin_amdgcn_rcpf(static_cast<float>(weight));
    const uint32_t u0 = uniform(min(static_cast<uint32_t>(static_cast<float>(x - begin) * per), units - 1));
    const uint32_t u1 = x1 >= p.end ? units : uniform(min(static_cast<uint32_t>(static_cast<float>(x1 - begin) * per), units - 1));
    p.begins = u0 == 0;
    p.ends = u1 == units;
    p.none = u1 == 0;
    p.t_lo = min(u0 * P.unit.d, total);
    p.t_hi = u1 == units ? total : u1 * P.unit.d;
    return p;
}

constexpr uint32_t kRows = 16;         // query rows of a block of the few-rows kernel
constexpr uint32_t kWorkgroups = 512;  // at most: two a CU
constexpr float kLn2 = 0.69314718055994531f;

// The parts of items into their rows.  Workgroup w of the attention kernel began an
// item and did not end it where joins[w] says so; its parts are the second of w and
// the first of w + 1, w + 2, ...  Every workgroup here lists the rows of all such
// items; few rows (one long context, its parts by the hundred) take several workgroups
// each, many (a part or two each) the lanes of one row.  Bound by latency: a part is
// read once, without a look at the maximum before.  4 us for a few rows, 6.5 for 16 rows in
// 512 parts (one token over 131,070), 11 for 25 MB of parts (24 mixed chunks).
template <class T, int D, uint32_t ROWS>
__global__ __launch_bounds__(256) void fg_join_kernel(AttendParams P) {
    constexpr uint32_t QUADS = D / 4, LANES = D <= 64 ? 16 : D <= 128 ? 32 : 64, SETS = 256 / LANES;
    __shared__ uint32_t first[kWorkgroups + 1], wave_sum[4];
    __shared__ f32x4 acc[256];
    __shared__ float2 acc_ml[4];
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = tid / 64, W = P.workgroups;
    uint32_t mine[kWorkgroups / 256], sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < kWorkgroups / 256; ++i) {  // consecutive workgroups in one thread
        const uint32_t w = tid * (kWorkgroups / 256) + i;
        mine[i] = 0;
        if (w < W) {
            const Join j = P.joins[w];
            if (j.pieces) mine[i] = min(ROWS, j.rows - j.row0);
        }
        sum += mine[i];
    }
    uint32_t upto = sum;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
    }
    if (lane == 63) wave_sum[wave] = upto;
    __syncthreads();
    upto -= sum;
    uint32_t all = 0;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
        if (i < wave) upto += wave_sum[i];
        all += wave_sum[i];
    }
#pragma unroll
    for (uint32_t i = 0; i < kWorkgroups / 256; ++i) {
        first[tid * (kWorkgroups / 256) + i] = upto;
        upto += mine[i];
    }
    __syncthreads();

    // a workgroup for every 32 values of a row, for a row, or for every SETS rows
    constexpr uint32_t SLICES = D / 32;
    const bool few = all <= gridDim.x, least = all <= 64;
    const uint32_t lanes = least ? 8 : LANES, sets = 256 / lanes, step = few ? sets : 1;
    const uint32_t tasks = least ? all * SLICES : all;
    for (uint32_t at = blockIdx.x * (few ? 1 : SETS); at < tasks; at += gridDim.x * (few ? 1 : SETS)) {
        const uint32_t set = tid / lanes, quad = (least ? at % SLICES * 8 : 0) + tid % lanes;
        const uint32_t task = least ? at / SLICES : few ? at : at + set;
        uint32_t lo = 0, hi = W;  // the last workgroup whose rows begin at or before `task`
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (first[mid] <= task) lo = mid;
            else hi = mid;
        }
        const uint32_t w = lo, row = task - first[w];
        const Join j = P.joins[w];
        float top = -INFINITY, l = 0.0f;
        f32x4 a = {0, 0, 0, 0};
        if (task < all && quad < QUADS) {
#pragma unroll 8
            for (uint32_t i = few ? set : 0; i < j.pieces; i += step) {
                const uint32_t p = (i == 0 ? 2 * w + 1 : 2 * (w + i)) * ROWS + row;
                const float2 ml = P.part_ml[p];
                const f32x4 v = *reinterpret_cast<const f32x4 *>(P.part + static_cast<uint64_t>(p) * D + 4 * quad);
                const float next = fmaxf(top, ml.x), base = next == -INFINITY ? 0.0f : next;
                const float f = __builtin_amdgcn_exp2f(top - base), g = __builtin_amdgcn_exp2f(ml.x - base);
                a = a * f + v * g;
                l = fmaf(g, ml.y, l * f);
                top = next;
            }
        }
        if (few) {  // the sets of a wave, then the four waves
            for (uint32_t d = lanes; d < 64; d <<= 1) {
                const float next = fmaxf(top, __shfl_xor(top, d)), f = __builtin_amdgcn_exp2f(top - (next == -INFINITY ? 0.0f : next));
                l *= f;
                a *= f;
                l += __shfl_xor(l, d);
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] += __shfl_xor(a[i], d);
                top = next;
            }
            if (lane < lanes) {
                acc[wave * 64 + lane] = a;
                if (lane == 0) acc_ml[wave] = float2{top, l};
            }
            __syncthreads();
            if (set == 0) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) top = fmaxf(top, acc_ml[i].x);
                const float base = top == -INFINITY ? 0.0f : top;
                a = f32x4{0, 0, 0, 0};
                l = 0.0f;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const float f = __builtin_amdgcn_exp2f(acc_ml[i].x - base);
                    a += acc[lane + i * 64] * f;
                    l = fmaf(f, acc_ml[i].y, l);
                }
            }
        }
        if (task < all && quad < QUADS && (!few || set == 0)) {
            const uint32_t r = j.row0 + row, token = P.group.div(r), head = j.list * P.group.d + (r - token * P.group.d);
            const int64_t qrow = static_cast<int64_t>(j.q0) + token;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            *reinterpret_cast<uint2 *>(P.out + qrow * P.out_token + head * P.out_head + 8 * quad) = uint2{T::pack(a[0] * inv, a[1] * inv), T::pack(a[2] * inv, a[3] * inv)};
            if (quad == 0 && P.lse) P.lse[qrow * P.heads + head] = (top + __builtin_amdgcn_logf(l)) * kLn2;
        }
        if (few) __syncthreads();
    }
}
// Eight a CU for blocks of many rows, whose tasks wait for their loads (of 512: 24 mixed
// chunks 94.5 us, 1,024: 87.9, 2,048: 85.4); fewer for few rows, where every one
// sums the list (1,024: 28.1 us for 32 requests with 256 ids, 512: 27.6).
template <uint32_t ROWS>
constexpr uint32_t kJoinWorkgroups = ROWS > 16 ? 2048 : 512;

// Blocks of many rows (fg_attend_tiles.hip): sets rows, unit, workgroups and join for items of up to `seen` tokens; launches.
void plan_tiles(AttendParams &P, uint32_t dim, uint64_t seen);
int launch_tiles(AttendParams &P, int dtype, uint32_t dim, hipStream_t stream);

}  // namespace fgk

#endif
