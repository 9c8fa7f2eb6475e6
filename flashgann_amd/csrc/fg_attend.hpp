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

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(8))) short s16x8;

struct BF16 {
    using vec = bf16x8;
    static constexpr uint32_t kExponent = 0x7F80, kMantissa = 0x007F;
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
__device__ __forceinline__ bool any_special(uint4 w) {
    bool s = false;
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
        s |= (x[i] & T::kExponent) == T::kExponent || ((x[i] >> 16) & T::kExponent) == T::kExponent;
    return s;
}

// The same with its infinities and NaNs as zeros.
template <class T>
__device__ __forceinline__ uint4 finite_part(uint4 w) {
    const auto part = [](uint32_t x) {
        if ((x & T::kExponent) == T::kExponent) x &= 0xFFFF0000u;
        if (((x >> 16) & T::kExponent) == T::kExponent) x &= 0x0000FFFFu;
        return x;
    };
    return {part(w.x), part(w.y), part(w.z), part(w.w)};
}

// An infinity or NaN among a value's 16 bits as a float, 0 for any other.
template <class T>
__device__ __forceinline__ float special_part(uint32_t x) {
    if ((x & T::kExponent) != T::kExponent) return 0.0f;
    return x & T::kMantissa ? NAN : x & 0x8000 ? -INFINITY : INFINITY;
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

// Whether the row at `pos` sees the token at position j (pages aside).
__device__ __forceinline__ bool sees(const AttendParams &P, int32_t pos, int32_t j) {
    const int32_t back = pos - j;
    return (back >= 0) & ((static_cast<uint32_t>(back) < P.window) | (static_cast<uint32_t>(j) < P.sinks));
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

constexpr uint32_t kRows = 16;         // query rows of a block of the few-rows kernel
constexpr uint32_t kWorkgroups = 512;  // at most: two a CU
constexpr float kLn2 = 0.69314718055994531f;

// The parts of an item into its rows: workgroup (w, row) of the item that
// workgroup w of the attention kernel began and did not end.  Its parts are the
// second of w and the first of w + 1, w + 2, ...
template <class T, int D, uint32_t ROWS>
__global__ __launch_bounds__(256) void fg_join_kernel(AttendParams P) {
    constexpr uint32_t QUADS = D / 4, SETS = 256 / QUADS;  // threads across a row, sets of parts side by side
    __shared__ float sum_m[4];
    __shared__ float acc[SETS][D], acc_l[SETS];
    const uint32_t w = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
    const Join j = P.joins[w];
    if (j.pieces == 0 || j.row0 + row >= j.rows) return;
    const auto slot_of = [&](uint32_t i) { return i == 0 ? 2 * w + 1 : 2 * (w + i); };

    float top = -INFINITY;
    for (uint32_t i = tid; i < j.pieces; i += 256) top = fmaxf(top, P.part_ml[slot_of(i) * ROWS + row].x);
#pragma unroll
    for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
    if (tid % 64 == 0) sum_m[tid / 64] = top;
    __syncthreads();
    top = fmaxf(fmaxf(sum_m[0], sum_m[1]), fmaxf(sum_m[2], sum_m[3]));
    const float base = top == -INFINITY ? 0.0f : top;

    const uint32_t set = tid / QUADS, quad = tid % QUADS;
    if (set < SETS) {
        f32x4 a = {0, 0, 0, 0};
        float l = 0.0f;
#pragma unroll 4
        for (uint32_t i = set; i < j.pieces; i += SETS) {
            const uint32_t at = slot_of(i) * ROWS + row;
            const float2 ml = P.part_ml[at];
            const float f = __builtin_amdgcn_exp2f(ml.x - base);
            a += f * *reinterpret_cast<const f32x4 *>(P.part + static_cast<uint64_t>(at) * D + 4 * quad);
            l = fmaf(f, ml.y, l);
        }
        *reinterpret_cast<f32x4 *>(&acc[set][4 * quad]) = a;
        if (quad == 0) acc_l[set] = l;
    }
    __syncthreads();
    const uint32_t all = j.row0 + row, token = P.group.div(all), head = j.list * P.group.d + (all - token * P.group.d);
    const int64_t qrow = static_cast<int64_t>(j.q0) + token;
    float l = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < SETS; ++i) l += acc_l[i];
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (tid < D / 2) {
        float a = 0.0f, b = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < SETS; ++i) {
            a += acc[i][2 * tid];
            b += acc[i][2 * tid + 1];
        }
        *reinterpret_cast<uint32_t *>(P.out + qrow * P.out_token + head * P.out_head + 4 * tid) = T::pack(a * inv, b * inv);
    }
    if (tid == 0 && P.lse) P.lse[qrow * P.heads + head] = (top + __builtin_amdgcn_logf(l)) * kLn2;
}

// Rows of the tile kernel's blocks together over all workgroups: two parts of
// the workspace each.
constexpr uint32_t kTileRows = 256 * 256;

// Blocks of many rows (fg_attend_tiles.hip): launches on `stream`.
int launch_tiles(AttendParams &P, int dtype, uint32_t dim, hipStream_t stream);

}  // namespace fgk

#endif
