// fg_attend_blocks.hip -- attention over selected pages of a paged cache.
//
// Softmax and products are those of fg_attend.hip's few-rows kernel: S' = K Q', then
// O' = V' P', a running maximum and sum.  What differs is
// which tokens a row sees: the first blocks, the last ones and those of its list.  Rows of
// neighbouring tokens share a tile of 16 rows, and the tile reads the union of what its
// tokens see, each block with a mask of the tokens that see it: neighbours ask for much the
// same, and where they do not, the rows that a block is not for cost matrix work only.
#include "fg_blocks.hpp"
#include "fg_pick.hpp"

namespace fgk {
namespace {

constexpr uint32_t kTileRows = 16;
constexpr uint32_t kTokenPlaces = 1024;  // token places resolved at a time
constexpr uint32_t kSplitTokens = 128;   // a part's tokens are a multiple: a tile of each wave
constexpr uint32_t kMostParts = 64;

// What rounding two weights to the values' type left of them, in that type too.  The matrix unit takes
// 16 bits, and outputs are to be off by their own rounding alone: a weight goes in as the sum of two
// such numbers (16 bits of it in bfloat16, 22 in float16), against the same values read once.  A chunk's
// attention takes 6% longer for it, single tokens and drafts do not; the error is that of 32-bit
// weights (0.0017 relative in bfloat16, the output's rounding, against 0.0021 with one part).
template <class T>
__device__ __forceinline__ uint32_t rest_of(float a, float b, uint32_t rounded) {
    return T::pack(a - as_float<T>(rounded & 0xFFFF), b - as_float<T>(rounded >> 16));
}

// Whether an infinity or NaN is among N pieces of 16-bit values: 0 times any other is 0, two values
// an instruction.
__device__ __forceinline__ float plus_zero_times(BF16, uint32_t w, float sum) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), bf16x2{0.0f, 0.0f}, sum, false);
}
__device__ __forceinline__ float plus_zero_times(F16, uint32_t w, float sum) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), f16x2{0, 0}, sum, false);
}
template <class T, int N>
__device__ __forceinline__ bool any_specials(const u32x4 (&w)[N]) {
    float zero[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < N; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) zero[i] = plus_zero_times(T{}, w[k][i], zero[i]);
    const float sum = (zero[0] + zero[1]) + (zero[2] + zero[3]);
    return sum != sum;
}

struct BlocksParams {
    CacheView cache;
    const char *q;
    char *out;
    float *lse;
    int64_t q_token, q_head, out_token, out_head;  // bytes
    const int32_t *table, *q_starts, *kv_lens, *ids;
    int64_t table_row;
    float *part;      // tile, list, head part, part, row: D each
    float2 *part_ml;  // maximum (base 2), sum
    uint32_t table_width, requests, tokens, heads, lists, list_heads;
    uint32_t nids, first, last;
    uint32_t group, head_parts;  // query heads of a list; blocks of 16 that they make
    uint32_t parts;              // workgroups that share a tile's tokens
    uint32_t lanes;              // lists * head_parts
    FastDiv per;                 // rows of a token in a tile
    FastDiv tile;                // tokens of a tile
    float scale2;                // scale * log2(e)
};

// A tile's tokens and what they see.
struct Seen {
    int32_t pos, tokens;         // position of the first; how many
    int32_t top;                 // block of the last token
    int32_t first, dense;        // blocks 0 .. first - 1 and dense .. top are seen by range
    uint32_t listed, entries;    // blocks between them from lists; all
};

// The tokens (a bit each) at or after position j.
__device__ __forceinline__ uint32_t from_position(const Seen &s, int64_t j) {
    const int64_t i = j - s.pos;
    return i <= 0 ? 0xFFFFu : i >= 16 ? 0u : (0xFFFFu << i) & 0xFFFFu;
}

// Where a list's running maxima reach b first, if b itself is on the list.
__device__ __forceinline__ bool on_list(const int32_t *list, uint32_t n, int32_t b) {
    uint32_t lo = 0;
    for (uint32_t len = n; len;) {
        const uint32_t half = len / 2;
        if (list[lo + half] < b) lo += half + 1, len -= half + 1;
        else len = half;
    }
    return lo < n && list[lo] == b;
}

// Bound by the bytes of the union: 48 single tokens over 48 selected pages of 32 and the first and last
// (32 heads over 8, dim 128) 66 us, 4.9 TB/s; of few tokens by latency, lists, union, table and keys one
// after another: 5 requests of 1 to 5 tokens 11.0 us, and 4 to join their parts.
template <class T, int D>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void fg_blocks_kernel(BlocksParams P) {
    using vec = typename T::vec;
    constexpr int STEPS = D / 32, DB = D / 16;
    constexpr uint32_t VROW = 2 * D + 32;  // bytes of a row of V in LDS: 16 rows' 32-byte pieces meet each bank twice
    constexpr uint32_t OROW = D + 4;       // floats of a row of O in LDS
    constexpr float UP = T::kTopWeight, DOWN = 1.0f / (1 << T::kTopWeight);
    static_assert(kTileRows * OROW * 4 <= 32 * VROW);
    __shared__ __attribute__((aligned(16))) char vbuf[4][32 * VROW];
    __shared__ int2 place[kTokenPlaces];
    __shared__ __attribute__((aligned(16))) uint32_t shown[kTokenPlaces];
    __shared__ float wave_m[4][kTileRows], wave_l[4][kTileRows];
    __shared__ uint32_t found[4];
    extern __shared__ int32_t lists[];  // nids a token; then the union's blocks, then their masks

    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = uniform(tid / 64), col = lane % 16, quarter = lane / 16;
    const uint32_t lane_of = blockIdx.x % P.lanes, at_tile = blockIdx.x / P.lanes;  // list and head part; tile and part
    const uint32_t tile = at_tile / P.parts, part = at_tile - tile * P.parts;
    const uint32_t list = lane_of / P.head_parts, head0 = (lane_of - list * P.head_parts) * kTileRows;
    const Tile t = tile_of(P.q_starts, P.kv_lens, P.requests, P.tokens, P.tile, tile);
    if (t.rows == 0) return;
    const uint32_t tokens = t.rows, nids = P.nids, page_size = P.cache.page_size.d;
    const int32_t *const table = P.table + t.request * P.table_row;
    int32_t *const blocks = lists + P.tile.d * nids;
    uint32_t *const masks = reinterpret_cast<uint32_t *>(blocks + P.tile.d * nids);

    Seen sn;
    sn.pos = t.pos, sn.tokens = t.rows;
    const int32_t last_pos = t.pos + t.rows - 1;
    sn.top = last_pos < 0 ? -1 : static_cast<int32_t>(P.cache.page_size.div(last_pos));
    const int32_t low = t.pos < 0 ? -1 : static_cast<int32_t>(P.cache.page_size.div(t.pos));
    sn.top = min(sn.top, static_cast<int32_t>(P.table_width) - 1);
    sn.first = static_cast<int32_t>(min(P.first, static_cast<uint32_t>(sn.top + 1)));
    sn.dense = static_cast<int32_t>(min(max(static_cast<int64_t>(low) - P.last + 1, static_cast<int64_t>(sn.first)), static_cast<int64_t>(sn.top) + 1));

    // the tokens' lists as running maxima: an id counts where the maximum rises
    for (uint32_t i = wave; i < tokens; i += 4) {
        const int32_t *src = P.ids + ((t.q0 + static_cast<uint64_t>(i)) * P.lists + list) * nids;
        int32_t most = -1;
        for (uint32_t k0 = 0; k0 < nids; k0 += 64) {
            int32_t x = k0 + lane < nids ? src[k0 + lane] : -1;
#pragma unroll
            for (uint32_t d = 1; d < 64; d <<= 1) {
                const int32_t o = __shfl_up(x, d);
                if (lane >= d) x = max(x, o);
            }
            x = max(x, most);
            if (k0 + lane < nids) lists[i * nids + k0 + lane] = x;
            most = of_lane(x, 63);
        }
    }
    __syncthreads();
    // their union, each block at the first token that has it.  A token has what lies between its
    // first and last blocks; those from sn.dense on are masked where they are read.
    sn.listed = 0;
    for (uint32_t e0 = 0; e0 < tokens * nids; e0 += 256) {
        const uint32_t e = e0 + tid, i = nids ? e / nids : 0, k = e - i * nids;
        bool mine = false;
        int32_t b = -1;
        uint32_t mask = 0;
        if (e < tokens * nids) {
            b = lists[e];
            const int32_t pos = t.pos + static_cast<int32_t>(i);
            const auto has_room = [&](int32_t p) { return p >= 0 && b <= static_cast<int64_t>(P.cache.page_size.div(p)) - P.last; };
            mine = (k ? lists[e - 1] : -1) != b && b >= sn.first && b < sn.dense && has_room(pos);
            if (mine) mask = 1u << i;
            for (uint32_t o = 0; o < tokens && mine; ++o) {
                if (o == i || !on_list(lists + o * nids, nids, b) || !has_room(t.pos + static_cast<int32_t>(o))) continue;
                if (o < i) mine = false;
                mask |= 1u << o;
            }
        }
        const uint64_t which = __ballot(mine);
        if (lane == 0) found[wave] = __popcll(which);
        __syncthreads();
        uint32_t at = sn.listed + __popcll(which & ((1ull << lane) - 1));
#pragma unroll
        for (uint32_t w = 0; w < 4; ++w) {
            if (w < wave) at += found[w];
            sn.listed += found[w];
        }
        if (mine) blocks[at] = b, masks[at] = mask;
        __syncthreads();
    }
    sn.listed = uniform(sn.listed);
    sn.entries = sn.first + sn.listed + static_cast<uint32_t>(sn.top + 1 - sn.dense);
    // (a table names fewer than 2^30 tokens, and no block is in the union twice)
    const uint32_t total = sn.entries * page_size;
    const uint32_t share = P.parts == 1 ? total : ((total + P.parts * kSplitTokens - 1) / (P.parts * kSplitTokens)) * kSplitTokens;
    const int32_t t_lo = static_cast<int32_t>(min(part * share, total)), t_hi = static_cast<int32_t>(min(part * share + share, total));

    // this lane's row: its query, and its token's bit
    const uint32_t rows = tokens * P.per.d, heads = min(P.group - head0, P.per.d);
    const uint32_t token = P.per.div(col), bit = min(token, 15u);
    const bool real = col < rows && col - token * P.per.d < heads;
    const int64_t head = static_cast<int64_t>(list) * P.group + head0 + (col - token * P.per.d);
    vec qv[STEPS];
    {
        const char *src = P.q + (t.q0 + static_cast<int64_t>(token)) * P.q_token + head * P.q_head + quarter * 16;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            u32x4 v = {0, 0, 0, 0};
            if (real) v = *reinterpret_cast<const u32x4 *>(src + 64 * s);
            qv[s] = __builtin_bit_cast(vec, v);
        }
    }
    const uint32_t kv_head = list / P.list_heads;
    const char *const kbase = P.cache.k + kv_head * P.cache.k_head + quarter * 16;
    const char *const vbase = P.cache.v + kv_head * P.cache.v_head + quarter * 16;
    char *const vmine = vbuf[wave];
    const uint32_t everyone = (1u << tokens) - 1;

    float m = -INFINITY, l = 0.0f;
    f32x4 o[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) o[i] = f32x4{0, 0, 0, 0};

    for (int32_t c0 = t_lo; c0 < t_hi; c0 += kTokenPlaces) {
        const int32_t n = min(t_hi - c0, static_cast<int32_t>(kTokenPlaces));
        __syncthreads();
        for (int32_t i = tid; i < ((n + 31) & ~31); i += 256) {
            int2 at = {-1, 0};
            uint32_t mask = 0;
            if (i < n) {
                const uint32_t e = P.cache.page_size.div(c0 + i);
                const int32_t off = static_cast<int32_t>(c0 + i - e * page_size);
                int32_t b;
                if (e < static_cast<uint32_t>(sn.first)) {
                    b = static_cast<int32_t>(e);
                    mask = everyone;
                } else if (e < sn.first + sn.listed) {
                    b = blocks[e - sn.first];
                    mask = masks[e - sn.first];
                } else {
                    b = sn.dense + static_cast<int32_t>(e - sn.first - sn.listed);
                    // among the last blocks of the tokens before position (b + last) * page_size
                    mask = everyone & ~from_position(sn, (static_cast<int64_t>(b) + P.last) * page_size);
                    for (uint32_t others = everyone & ~mask; others; others &= others - 1) {
                        const uint32_t x = __ffs(others) - 1;
                        if (on_list(lists + x * nids, nids, b)) mask |= 1u << x;
                    }
                }
                const int32_t page = table[b];
                mask &= from_position(sn, static_cast<int64_t>(b) * page_size + off);
                if (static_cast<uint32_t>(page) >= P.cache.pages) mask = 0;
                if (mask) at = {page, off};
            }
            place[i] = at;
            shown[i] = mask;
        }
        __syncthreads();

        u32x4 kr[2][STEPS], vr[2][STEPS];
        uint32_t held[2];
        const auto load = [&](int32_t at32) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int2 at = place[at32 * 32 + 16 * b + col];
                held[b] = shown[at32 * 32 + 16 * b + col];
                const int64_t page = max(at.x, 0);
                const char *ks = kbase + page * P.cache.k_page + at.y * P.cache.k_token;
                const char *vs = vbase + page * P.cache.v_page + at.y * P.cache.v_token;
#pragma unroll
                for (int s = 0; s < STEPS; ++s) {
                    kr[b][s] = *reinterpret_cast<const u32x4 *>(ks + 64 * s);
                    vr[b][s] = *reinterpret_cast<const u32x4 *>(vs + 64 * s);
                }
            }
        };
        if (static_cast<int32_t>(wave) * 32 < n) load(wave);
        for (int32_t at32 = wave; at32 * 32 < n; at32 += 4) {
            // scores: register i of s[b] is token 16 b + 4 quarter + i
            f32x4 s[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                s[b] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < STEPS; ++k) s[b] = T::mfma16(__builtin_bit_cast(vec, kr[b][k]), qv[k], s[b]);
            }
            uint32_t odd = 0;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                u32x4 v[STEPS];  // (of a token that no row sees: zeros, whatever was read instead)
#pragma unroll
                for (int k = 0; k < STEPS; ++k) v[k] = held[b] ? vr[b][k] : u32x4{0, 0, 0, 0};
                // 0 * inf is NaN: infinities and NaNs are taken out of the product, whose weights, or
                // parts of them, may be 0 or negative, and added to the rows that see them
                const uint64_t special = __ballot(any_specials<T>(v));
                if (special) {
#pragma unroll
                    for (int k = 0; k < STEPS; ++k) v[k] = finite_part<T>(v[k]);
                    const uint64_t any = special | special >> 32;
                    odd |= static_cast<uint32_t>((any | any >> 16) & 0xFFFF) << (16 * b);
                }
#pragma unroll
                for (int k = 0; k < STEPS; ++k) *reinterpret_cast<u32x4 *>(vmine + (16 * b + col) * VROW + 64 * k + 16 * quarter) = v[k];
            }
            if ((at32 + 4) * 32 < n) load(at32 + 4);

            float p[8];
            float top = -INFINITY;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const u32x4 sees = *reinterpret_cast<const u32x4 *>(shown + at32 * 32 + 16 * b + 4 * quarter);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p[4 * b + i] = (sees[i] >> bit) & 1u ? s[b][i] * P.scale2 : -INFINITY;
                    top = fmaxf(top, p[4 * b + i]);
                }
            }
            top = fmaxf(m, max_other32(max_other16(top)));
            const float base = top == -INFINITY ? 0.0f : top;
            if (__any(top > m)) {
                const float shrink = __builtin_amdgcn_exp2f(m - base);
                l *= shrink;
#pragma unroll
                for (int i = 0; i < DB; ++i) o[i] *= shrink;
                m = top;
            }
            const float zero = base - UP;
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = __builtin_amdgcn_exp2f(p[i] - zero);
            l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            u32x4 pk = {T::pack(p[0], p[1]), T::pack(p[2], p[3]), T::pack(p[4], p[5]), T::pack(p[6], p[7])};
            u32x4 pr;
#pragma unroll
            for (int i = 0; i < 4; ++i) pr[i] = rest_of<T>(p[2 * i], p[2 * i + 1], pk[i]);
            const vec pv = __builtin_bit_cast(vec, pk), rv = __builtin_bit_cast(vec, pr);
            team_sync<1>();  // (the values that other lanes have written)
            const char *vt = vmine + (4 * quarter + col / 4) * VROW + (col % 4) * 8;
#pragma unroll
            for (int i = 0; i < DB; ++i) {
                const s16x4 a0 = read_transposed(vt + 32 * i), a1 = read_transposed(vt + 16 * VROW + 32 * i);
                const s16x8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
                o[i] = T::mfma16(__builtin_bit_cast(vec, a), pv, o[i]);
                o[i] = T::mfma16(__builtin_bit_cast(vec, a), rv, o[i]);
            }
            for (; odd; odd &= odd - 1) {
                const int32_t at = at32 * 32 + __ffs(odd) - 1;
                const int2 where = place[at];
                const char *src = vbase + where.x * P.cache.v_page + where.y * P.cache.v_token - quarter * 8;
                const bool visible = (shown[at] >> bit) & 1u;
#pragma unroll
                for (int i = 0; i < DB; ++i) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(src + 32 * i);
                    o[i][0] += visible ? special_part<T>(v.x & 0xFFFF) : 0.0f;
                    o[i][1] += visible ? special_part<T>(v.x >> 16) : 0.0f;
                    o[i][2] += visible ? special_part<T>(v.y & 0xFFFF) : 0.0f;
                    o[i][3] += visible ? special_part<T>(v.y >> 16) : 0.0f;
                }
            }
        }
    }

    // the four waves' softmaxes into one (each wave writes over its own tile of V)
    l = add_other32(add_other16(l));
    if (quarter == 0) wave_m[wave][col] = m;
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, wave_m[i][col]);
    const float mine = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top)) * DOWN;
    if (quarter == 0) wave_l[wave][col] = l * mine;
    float *omine = reinterpret_cast<float *>(vmine);
#pragma unroll
    for (int i = 0; i < DB; ++i) *reinterpret_cast<f32x4 *>(omine + col * OROW + 16 * i + 4 * quarter) = o[i] * mine;
    __syncthreads();
    const bool whole = P.parts == 1;
    const uint64_t slot = ((static_cast<uint64_t>(tile) * P.lanes + lane_of) * P.parts + part) * kTileRows;
    l = wave_l[0][col] + wave_l[1][col] + wave_l[2][col] + wave_l[3][col];
    if (wave == 0 && quarter == 0 && real) {
        if (!whole) P.part_ml[slot + col] = float2{top, l};
        else if (P.lse) P.lse[(t.q0 + static_cast<int64_t>(token)) * P.heads + head] = (top + __builtin_amdgcn_logf(l)) * kLn2;
    }
#pragma unroll
    for (uint32_t e = 0; e < kTileRows * D / 4; e += 256) {
        const uint32_t at = e + tid, orow = at / (D / 4), quad = at % (D / 4);
        const uint32_t otoken = P.per.div(orow), ohead = orow - otoken * P.per.d;
        if ((kTileRows * D / 4 % 256 == 0 || at < kTileRows * D / 4) && orow < rows && ohead < heads) {
            f32x4 a = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) a += *reinterpret_cast<const f32x4 *>(reinterpret_cast<float *>(vbuf[i]) + orow * OROW + 4 * quad);
            if (whole) {
                const float sum = wave_l[0][orow] + wave_l[1][orow] + wave_l[2][orow] + wave_l[3][orow];
                a *= sum == 0.0f ? 0.0f : 1.0f / sum;
                char *dst = P.out + (t.q0 + static_cast<int64_t>(otoken)) * P.out_token +
                            (static_cast<int64_t>(list) * P.group + head0 + ohead) * P.out_head;
                *reinterpret_cast<uint2 *>(dst + 8 * quad) = uint2{T::pack(a[0], a[1]), T::pack(a[2], a[3])};
            } else {
                *reinterpret_cast<f32x4 *>(P.part + (slot + orow) * D + 4 * quad) = a;
            }
        }
    }
}

// The parts of a tile into its rows, in their order.
template <class T, int D>
__global__ __launch_bounds__(256) void fg_blocks_join_kernel(BlocksParams P) {
    const uint32_t tile = blockIdx.x / P.lanes, lane_of = blockIdx.x - tile * P.lanes, list = lane_of / P.head_parts,
                   head0 = (lane_of - list * P.head_parts) * kTileRows;
    const Tile t = tile_of(P.q_starts, P.kv_lens, P.requests, P.tokens, P.tile, tile);
    if (t.rows == 0) return;
    const uint32_t rows = t.rows * P.per.d, heads = min(P.group - head0, P.per.d);
    for (uint32_t at = threadIdx.x; at < rows * (D / 4); at += 256) {
        const uint32_t row = at / (D / 4), quad = at % (D / 4), token = P.per.div(row), head = row - token * P.per.d;
        if (head >= heads) continue;
        const uint64_t slot = static_cast<uint64_t>(blockIdx.x) * P.parts * kTileRows + row;
        float top = -INFINITY, l = 0.0f;
        f32x4 a = {0, 0, 0, 0};
#pragma unroll 8
        for (uint32_t i = 0; i < P.parts; ++i) {
            const float2 ml = P.part_ml[slot + i * kTileRows];
            const f32x4 v = *reinterpret_cast<const f32x4 *>(P.part + (slot + i * kTileRows) * D + 4 * quad);
            const float next = fmaxf(top, ml.x), base = next == -INFINITY ? 0.0f : next;
            const float f = __builtin_amdgcn_exp2f(top - base), g = __builtin_amdgcn_exp2f(ml.x - base);
            a = a * f + v * g;
            l = fmaf(g, ml.y, l * f);
            top = next;
        }
        const int64_t qrow = t.q0 + static_cast<int64_t>(token), qhead = static_cast<int64_t>(list) * P.group + head0 + head;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        *reinterpret_cast<uint2 *>(P.out + qrow * P.out_token + qhead * P.out_head + 8 * quad) = uint2{T::pack(a[0] * inv, a[1] * inv), T::pack(a[2] * inv, a[3] * inv)};
        if (quad == 0 && P.lse) P.lse[qrow * P.heads + qhead] = (top + __builtin_amdgcn_logf(l)) * kLn2;
    }
}

// ---------------------------------------------------------------- chunks
//
// 32 rows a workgroup, so that what neighbours both select is read once for twice as many tokens,
// on 32 x 32 matrix tiles; as above each of the four waves takes every fourth tile of 32 tokens and
// nothing is waited for but its own loads.  A lane loads the keys of the token whose place it has
// worked out.  The union of the lists is made a window of blocks at a time, a word of
// tokens for each block, so its blocks come in order and none twice.
//
// A chunk of 2,048 tokens after 62,000 (32 heads over 8, dim 128, 16 pages of 64 each) 353 us; its
// tiles of eight tokens read 59 blocks each of the 160 listed, 4 GB in all, of which the L2 has 67%.
// Waves wait for loads 41% of their time, vector issue is 42% of it, the matrix unit 23%.  In tiles
// of 16 rows 689 us; rows of several waves over tiles shared in LDS took 546 us against 354 (a barrier a
// tile, and each wave masks what only the others asked for).
constexpr uint32_t kChunkRows = 32;
constexpr uint32_t kWindow = 1024;  // blocks whose tokens are known at a time

// The tokens (a bit each, the first at position pos) at or after position j.
__device__ __forceinline__ uint32_t tokens_from(int32_t pos, int64_t j) {
    const int64_t i = j - pos;
    return i <= 0 ? ~0u : i >= 32 ? 0u : ~0u << i;
}

template <class T, int D>
__global__ __launch_bounds__(256, 2) void fg_blocks_chunk_kernel(BlocksParams P) {
    using vec = typename T::vec;
    constexpr int STEPS = D / 16, DB = D / 32, CHUNKS = D / 8;
    constexpr uint32_t VROW = 2 * D + (D == 96 ? 128 : 64);  // bytes of a row of V in LDS: eight rows' 64-byte pieces meet every bank equally often
    constexpr uint32_t OROW = D + 4;                         // floats of a row of O in LDS
    constexpr float UP = T::kTopWeight, DOWN = 1.0f / (1 << T::kTopWeight);
    // values of a tile of each wave, the window's blocks and those of its entries; then the waves' outputs
    struct Blocks {
        uint32_t seen[kWindow];                   // the tokens that have a block on their list
        int32_t entry_page[kWindow], entry_block[kWindow];
        uint32_t entry_seen[kWindow];             // of the blocks that some token sees
    };
    constexpr uint32_t VBYTES = 4 * 32 * VROW, OBYTES = 4 * kChunkRows * OROW * 4;
    __shared__ __attribute__((aligned(16))) char lds[VBYTES + sizeof(Blocks) > OBYTES ? VBYTES + sizeof(Blocks) : OBYTES];
    __shared__ float wave_m[4][kChunkRows], wave_l[4][kChunkRows];
    __shared__ uint32_t found[4], next_block;
    __shared__ int64_t value_at[4][2][32];  // where a wave's tile's values lie, from the head's first; of the next one
    Blocks &B = *reinterpret_cast<Blocks *>(lds + VBYTES);

    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = uniform(tid / 64), col = lane % 32, half = lane / 32;
    const uint32_t tile = blockIdx.x / P.lanes, lane_of = blockIdx.x - tile * P.lanes;
    const uint32_t list = lane_of / P.head_parts, head0 = (lane_of - list * P.head_parts) * kChunkRows;
    const Tile t = tile_of(P.q_starts, P.kv_lens, P.requests, P.tokens, P.tile, tile);
    if (t.rows == 0) return;
    const uint32_t tokens = t.rows, nids = P.nids, page_size = P.cache.page_size.d;
    const int32_t *const table = P.table + t.request * P.table_row;
    const auto block_of = [&](int32_t pos) { return pos < 0 ? -1 : static_cast<int32_t>(P.cache.page_size.div(pos)); };
    const uint32_t blocks = static_cast<uint32_t>(min(block_of(t.pos + t.rows - 1), static_cast<int32_t>(P.table_width) - 1) + 1);
    const uint32_t dense = static_cast<uint32_t>(min(max(static_cast<int64_t>(block_of(t.pos)) - P.last + 1, static_cast<int64_t>(0)), static_cast<int64_t>(blocks)));
    const uint32_t everyone = tokens >= 32 ? ~0u : (1u << tokens) - 1;
    const bool by_block = page_size * tokens > 32;  // fewer blocks in a tile of 32 places than tokens

    // this lane's row
    const uint32_t rows = tokens * P.per.d, token = P.per.div(col), heads = min(P.group - head0, P.per.d);
    const bool real = col < rows && col - token * P.per.d < heads;
    const int64_t head = static_cast<int64_t>(list) * P.group + head0 + (col - token * P.per.d);
    vec qv[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        u32x4 v = {0, 0, 0, 0};
        if (real) v = *reinterpret_cast<const u32x4 *>(P.q + (t.q0 + static_cast<int64_t>(token)) * P.q_token + head * P.q_head + half * 16 + 32 * s);
        qv[s] = __builtin_bit_cast(vec, v);
    }
    const uint32_t kv_head = list / P.list_heads;
    const char *const kbase = P.cache.k + kv_head * P.cache.k_head + half * 16, *const vbase = P.cache.v + kv_head * P.cache.v_head;
    char *const vmine = lds + wave * 32 * VROW;

    float m, l;
    f32x16 o[DB];
    bool careful = false;  // whether infinities and NaN are taken out of the products
again:
    m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < DB; ++i) o[i] = f32x16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};

    for (uint32_t w0 = 0; w0 < blocks;) {
        const uint32_t w1 = min(w0 + kWindow, blocks);
        __syncthreads();
        *reinterpret_cast<u32x4 *>(B.seen + 4 * tid) = u32x4{0, 0, 0, 0};
        if (tid == 0) next_block = blocks;
        __syncthreads();
        // the lists' blocks in the window, an id counting where the running maximum rises
        for (uint32_t i = wave; i < tokens; i += 4) {
            const int32_t *src = P.ids + ((t.q0 + static_cast<uint64_t>(i)) * P.lists + list) * nids;
            const int64_t room = min(static_cast<int64_t>(block_of(t.pos + static_cast<int32_t>(i))) - P.last, static_cast<int64_t>(blocks) - 1);
            int32_t most = -1;
            for (uint32_t k0 = 0; k0 < nids; k0 += 64) {
                const int32_t id = k0 + lane < nids ? src[k0 + lane] : -1;
                int32_t x = id;
#pragma unroll
                for (uint32_t d = 1; d < 64; d <<= 1) {
                    const int32_t y = __shfl_up(x, d);
                    if (lane >= d) x = max(x, y);
                }
                x = max(x, most);
                const int32_t up = __shfl_up(x, 1), before = lane ? up : most;
                most = of_lane(x, 63);
                if (id > before && id <= room && static_cast<uint32_t>(id) >= P.first) {
                    if (static_cast<uint32_t>(id) >= w0 && static_cast<uint32_t>(id) < w1) atomicOr(&B.seen[id - w0], 1u << i);
                    else if (static_cast<uint32_t>(id) >= w1) atomicMin(&next_block, static_cast<uint32_t>(id));
                }
            }
        }
        __syncthreads();
        // those that some token sees, in order; four a thread
        const u32x4 listed = *reinterpret_cast<const u32x4 *>(B.seen + 4 * tid);
        uint32_t mask[4], count = 0;
        int32_t page[4];
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
            const uint32_t b = w0 + 4 * tid + u;
            mask[u] = listed[u];
            if (b < P.first) mask[u] = ~0u;
            // among the last blocks of the tokens before position (b + last) * page_size
            mask[u] |= ~tokens_from(t.pos, (static_cast<int64_t>(b) + P.last) * page_size);
            mask[u] &= tokens_from(t.pos, static_cast<int64_t>(b) * page_size) & everyone;
            if (b >= w1) mask[u] = 0;
            page[u] = mask[u] ? table[b] : -1;
        }
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
            if (static_cast<uint32_t>(page[u]) >= P.cache.pages) mask[u] = 0;
            count += mask[u] != 0;
        }
        const uint32_t upto = sum_upto(count);
        if (lane == 63) found[wave] = upto;
        __syncthreads();
        uint32_t at = upto - count, entries = 0;
#pragma unroll
        for (uint32_t w = 0; w < 4; ++w) {
            if (w < wave) at += found[w];
            entries += found[w];
        }
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u)
            if (mask[u]) {
                B.entry_page[at] = page[u], B.entry_block[at] = static_cast<int32_t>(w0 + 4 * tid + u), B.entry_seen[at] = mask[u];
                ++at;
            }
        entries = uniform(entries);
        // where the next window begins
        uint32_t next = min(next_block, max(dense, w1));
        if (w1 < P.first) next = w1;
        w0 = uniform(max(next, w1));
        __syncthreads();

        const int32_t total = static_cast<int32_t>(entries * page_size);
        u32x4 kr[STEPS], vr[STEPS];
        uint32_t sees;  // the tokens that see this lane's token of the tile
        // (a lane loads its token's keys, as the product wants them, and of the values 16 bytes
        // beside its neighbours')
        const char *ks;
        const auto find = [&](int32_t i) {
            const int32_t n = i * 32 + static_cast<int32_t>(col), in = min(n, total - 1);
            const uint32_t e = P.cache.page_size.div(in);
            int64_t off = in - static_cast<int32_t>(e * page_size);
            const int64_t p = B.entry_page[e];
            sees = n < total ? B.entry_seen[e] & tokens_from(t.pos, static_cast<int64_t>(B.entry_block[e]) * page_size + off) : 0u;
            off = sees ? off : 0;  // (whatever lies where no row sees it stays unread: the block's first token is seen)
            ks = kbase + p * P.cache.k_page + off * P.cache.k_token;
            if (half == 0) value_at[wave][i / 4 % 2][col] = p * P.cache.v_page + off * P.cache.v_token;
            team_sync<1>();  // (other lanes read it)
        };
        const auto load_k = [&] {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) kr[s] = *reinterpret_cast<const u32x4 *>(ks + 32 * s);
        };
        const auto load_v = [&](int32_t i) {
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const uint32_t at = s * 64 + lane;
                vr[s] = *reinterpret_cast<const u32x4 *>(vbase + value_at[wave][i / 4 % 2][at / CHUNKS] + at % CHUNKS * 16);
            }
        };
        if (static_cast<int32_t>(wave) * 32 < total) {
            find(static_cast<int32_t>(wave));
            load_k();
            load_v(static_cast<int32_t>(wave));
        }
        for (int32_t i = static_cast<int32_t>(wave); i * 32 < total; i += 4) {
            const uint32_t sees_now = sees;
            const bool more = (i + 4) * 32 < total;
            if (more) find(i + 4);
            // scores: register k is that of token 8 (k / 4) + 4 half + k % 4
            f32x16 s = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < STEPS; ++k) s = T::mfma32(__builtin_bit_cast(vec, kr[k]), qv[k], s);
            if (more) load_k();
            uint32_t odd = 0;  // tokens whose values are not all finite
            if (careful) {
#pragma unroll
                for (int k = 0; k < STEPS; ++k) {
                    if (any_special<T>(vr[k])) odd |= 1u << (k * 64 + lane) / CHUNKS;
                    vr[k] = finite_part<T>(vr[k]);
                }
                odd = last_lane(wave_scan(odd, 0, [](uint32_t a, uint32_t b) { return a | b; }));
            }
#pragma unroll
            for (int k = 0; k < STEPS; ++k) {
                const uint32_t at = k * 64 + lane;
                *reinterpret_cast<u32x4 *>(vmine + at / CHUNKS * VROW + at % CHUNKS * 16) = vr[k];
            }
            if (more) load_v(i + 4);
            // the tile's tokens that this lane's row sees: those that the same tokens see, a block's as a rule,
            // together, or token by token where a tile has no more of those than blocks (1,024 tokens over 16
            // pages of 64, dim 128: 32 tokens a tile 111 us against 186 token by token, 8 148 against 148)
            uint32_t row_sees = 0, all = ~0u;
            if (by_block) {
                for (uint32_t left = ~0u; left;) {
                    const uint32_t seen_by = static_cast<uint32_t>(of_lane(static_cast<int32_t>(sees_now), __ffs(left) - 1));
                    const uint32_t those = static_cast<uint32_t>(__ballot(sees_now == seen_by));
                    left &= ~those;
                    if (seen_by != everyone) all = 0;
                    row_sees |= those & static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int32_t>(seen_by), token, 1));
                }
            } else {
                for (uint32_t x = 0; x < tokens; ++x) {
                    const uint32_t those = static_cast<uint32_t>(__ballot((sees_now >> x) & 1u));
                    all &= those;
                    row_sees = token == x ? those : row_sees;
                }
            }
            if (all != ~0u) {
                const uint32_t bits = row_sees >> (4 * half);
#pragma unroll
                for (int k = 0; k < 16; ++k) s[k] = keep_if(bits, k / 4 * 8 + k % 4, s[k]);
            }
            float top = -INFINITY;
#pragma unroll
            for (int k = 0; k < 16; ++k) top = fmaxf(top, s[k]);
            top = fmaxf(m, max_other32(top) * P.scale2);
            const float base = top == -INFINITY ? 0.0f : top;
            if (__any(top > m)) {
                const float shrink = __builtin_amdgcn_exp2f(m - base);
                l *= shrink;
#pragma unroll
                for (int k = 0; k < DB; ++k) o[k] *= shrink;
                m = top;
            }
            const float zero = UP - base;
            float sum = 0.0f;
            u32x4 pk[2], pr[2];  // the weights of 16 tokens each, in two parts
#pragma unroll
            for (int k = 0; k < 16; k += 2) {
                const float p0 = __builtin_amdgcn_exp2f(fmaf(s[k], P.scale2, zero)), p1 = __builtin_amdgcn_exp2f(fmaf(s[k + 1], P.scale2, zero));
                sum += p0 + p1;
                pk[k / 8][k % 8 / 2] = T::pack(p0, p1);
                pr[k / 8][k % 8 / 2] = rest_of<T>(p0, p1, pk[k / 8][k % 8 / 2]);
            }
            l += sum;
            team_sync<1>();  // (the values that other lanes have written)
            const char *const vt = vmine + (4 * half + lane % 16 / 4) * VROW + (lane / 16 % 2) * 32 + (lane % 4) * 8;
#pragma unroll
            for (int n = 0; n < 2 * DB; ++n) {
                const char *at = vt + 16 * (n / DB) * VROW + 64 * (n % DB);
                const s16x8 a = __builtin_shufflevector(read_transposed(at), read_transposed(at + 8 * VROW), 0, 1, 2, 3, 4, 5, 6, 7);
                o[n % DB] = T::mfma32(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, pk[n / DB]), o[n % DB]);
                o[n % DB] = T::mfma32(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, pr[n / DB]), o[n % DB]);
            }
            for (; odd; odd &= odd - 1) {
                const int at = __ffs(odd) - 1;
                const char *src = vbase + value_at[wave][i / 4 % 2][at] + half * 8;
                const bool visible = (row_sees >> at) & 1u;
#pragma unroll
                for (int k = 0; k < DB; ++k)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {  // dimensions 32 k + 8 g + 4 half and on
                        const uint2 v = *reinterpret_cast<const uint2 *>(src + 64 * k + 16 * g);
                        o[k][4 * g] += visible ? special_part<T>(v.x & 0xFFFF) : 0.0f;
                        o[k][4 * g + 1] += visible ? special_part<T>(v.x >> 16) : 0.0f;
                        o[k][4 * g + 2] += visible ? special_part<T>(v.y & 0xFFFF) : 0.0f;
                        o[k][4 * g + 3] += visible ? special_part<T>(v.y >> 16) : 0.0f;
                    }
            }
        }
    }

    if (!careful) {
        // 0 * inf is NaN: a value that is not finite leaves no output of its channel finite, of rows that see
        // it or not.  Then all again with such values taken out of the products and added to the rows that see them
        float zero = 0.0f;
#pragma unroll
        for (int k = 0; k < DB; ++k)
#pragma unroll
            for (int i = 0; i < 16; ++i) zero = fmaf(o[k][i], 0.0f, zero);
        const bool odd = __any(zero != zero);
        __syncthreads();
        if (lane == 0) found[wave] = odd;
        __syncthreads();
        if (uniform(found[0] | found[1] | found[2] | found[3])) {
            careful = true;
            goto again;
        }
    }

    // the four waves' softmaxes into one
    l = add_other32(l);
    if (half == 0) wave_m[wave][col] = m;
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, wave_m[i][col]);
    const float mine = __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.0f : top)) * DOWN;
    if (half == 0) wave_l[wave][col] = l * mine;
    float *const all_o = reinterpret_cast<float *>(lds);
#pragma unroll
    for (int k = 0; k < DB; ++k)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4 *>(all_o + (wave * kChunkRows + col) * OROW + 32 * k + 8 * g + 4 * half) =
                f32x4{o[k][4 * g], o[k][4 * g + 1], o[k][4 * g + 2], o[k][4 * g + 3]} * mine;
    __syncthreads();
    if (wave == 0 && half == 0 && real && P.lse) {
        const float sum = wave_l[0][col] + wave_l[1][col] + wave_l[2][col] + wave_l[3][col];
        P.lse[(t.q0 + static_cast<int64_t>(token)) * P.heads + head] = (top + __builtin_amdgcn_logf(sum)) * kLn2;
    }
#pragma unroll
    for (uint32_t e = 0; e < kChunkRows * D / 4; e += 256) {
        const uint32_t at = e + tid, orow = at / (D / 4), quad = at % (D / 4);
        const uint32_t otoken = P.per.div(orow), ohead = orow - otoken * P.per.d;
        if (orow < rows && ohead < heads) {
            f32x4 a = {0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i) a += *reinterpret_cast<const f32x4 *>(all_o + (i * kChunkRows + orow) * OROW + 4 * quad);
            const float sum = wave_l[0][orow] + wave_l[1][orow] + wave_l[2][orow] + wave_l[3][orow];
            a *= sum == 0.0f ? 0.0f : 1.0f / sum;
            char *dst = P.out + (t.q0 + static_cast<int64_t>(otoken)) * P.out_token +
                        (static_cast<int64_t>(list) * P.group + head0 + ohead) * P.out_head;
            *reinterpret_cast<uint2 *>(dst + 8 * quad) = uint2{T::pack(a[0], a[1]), T::pack(a[2], a[3])};
        }
    }
}

// ---------------------------------------------------------------- host side

struct BlocksPlan {
    bool chunk;  // which kernel
    uint32_t tiles, lds;
    uint64_t ml, workspace;
};

int prepare(const fg_kv_cache *c, const fg_attention *a, BlocksParams *out, BlocksPlan *plan) {
    BlocksParams &P = *out;
    if (int rc = check_cache(c, &P.cache)) return rc;
    if (!a) return fail(FG_EINVAL, "attention arguments are NULL");
    if (a->heads < 1 || a->heads > 1024 || a->heads % c->heads_kv) return fail(FG_EINVAL, "heads must be a multiple of heads_kv, at most 1024");
    if (a->lists < 1 || a->heads % a->lists || a->lists % c->heads_kv) return fail(FG_EINVAL, "lists must be a multiple of heads_kv that divides heads");
    if (!(a->scale > 0.0f) || !std::isfinite(a->scale)) return fail(FG_EINVAL, "scale must be positive and finite");
    if (a->nids > kMostBlocks) return fail(FG_EINVAL, "blocks of a list must be at most 4,096");
    if (a->tokens > kMostTokens) return fail(FG_EINVAL, "tokens must be at most 4,194,304");
    if (static_cast<uint64_t>(a->tokens) * a->heads > 0x7FFFFFFFull) return fail(FG_EINVAL, "tokens * heads must be below 2^31");
    if (a->table_width > 0x7FFFFFFFu || a->table_row < 0) return fail(FG_EINVAL, "table_width or table_row out of range");
    if (static_cast<uint64_t>(a->table_width) * c->page_size > 0x3FFFFFFFull) return fail(FG_EINVAL, "table_width * page_size must be below 2^30");
    if (a->sinks > 0x7FFFFFFFu) return fail(FG_EINVAL, "first blocks (sinks) must be below 2^31");
    if (a->window < 1) return fail(FG_EINVAL, "last blocks (window) must be >= 1");
    if (a->requests > 65536) return fail(FG_EINVAL, "requests must be at most 65,536");
    if (a->requests && a->tokens &&
        (!a->q || !a->out || !a->kv_lens || !a->q_starts || (a->nids && !a->ids) || (a->table_width && !a->table)))
        return fail(FG_EINVAL, "NULL device buffer");
    if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) % 16 ||
        (a->q_token | a->q_head | a->out_token | a->out_head) % 8)
        return fail(FG_EINVAL, "q and out must be 16-byte aligned, strides multiples of 8 elements");
    if ((a->tokens > 1 && !a->out_token) || (a->heads > 1 && !a->out_head)) return fail(FG_EINVAL, "rows of out share memory (a stride of 0)");
    P.q = static_cast<const char *>(a->q);
    P.out = static_cast<char *>(a->out);
    P.lse = a->lse;
    P.q_token = 2 * a->q_token, P.q_head = 2 * a->q_head, P.out_token = 2 * a->out_token, P.out_head = 2 * a->out_head;
    P.table = a->table;
    P.q_starts = a->q_starts;
    P.kv_lens = a->kv_lens;
    P.ids = reinterpret_cast<const int32_t *>(a->ids);
    P.table_row = a->table_row;
    P.table_width = a->table_width;
    P.requests = a->requests;
    P.tokens = a->tokens;
    P.heads = a->heads;
    P.lists = a->lists;
    P.list_heads = a->lists / c->heads_kv;
    P.nids = a->nids;
    P.first = a->sinks;
    P.last = static_cast<uint32_t>(a->window);
    P.group = a->heads / a->lists;
    P.scale2 = a->scale * 1.44269504088896341f;

    // Tiles of 32 rows once they fill half the device, whole; before that those of 16 are split among
    // workgroups.  24 of 250 pages of 32 (32 heads over 8, dim 128): 8 requests of 8 new tokens 42.5 us
    // against 41.1, of 16 43.2 against 59.9, of 64 67 against 117; 32 requests of 2 46.6 against 51.1; one
    // of 64 37.9 against 26.6.  Over many blocks windows cost more than lists in order: 256 tokens, 64 of
    // 500 blocks 30 against 42, of 2,000 41 against 48, of 7,500 81 against 52.  (At dim 256 the chunk
    // kernel's rows do not fit the registers.)
    const auto tile_tokens = [&](uint32_t rows) { return rows / std::min(P.group, rows); };
    const uint64_t chunk_tiles = std::max<uint64_t>(a->tokens / tile_tokens(kChunkRows), a->requests) * P.lists * ((P.group + kChunkRows - 1) / kChunkRows);
    plan->chunk = c->dim <= 128 && a->tokens >= 2 * static_cast<uint64_t>(a->requests) && chunk_tiles >= 128 && a->table_width <= 4 * kWindow;
    // A tile: the rows of as many tokens as it holds; for the former kernel with their lists in LDS.
    const uint32_t most_rows = plan->chunk ? kChunkRows : kTileRows, per = std::min(P.group, most_rows);
    uint32_t tokens = tile_tokens(most_rows);
    if (!plan->chunk && P.nids) tokens = std::min(tokens, std::max(1u, kMostBlocks / P.nids));
    P.per = fast_div(per);
    P.head_parts = (P.group + most_rows - 1) / most_rows;
    P.tile = fast_div(tokens);
    P.lanes = P.lists * P.head_parts;
    plan->tiles = a->tokens / tokens + (tokens > 1 ? a->requests : 0);
    plan->lds = plan->chunk ? 0 : tokens * P.nids * 12;
    const uint64_t items = static_cast<uint64_t>(plan->tiles) * P.lanes;
    if (items > kMostItems) return fail(FG_EINVAL, "more than 2^23 tiles of rows: attend to fewer tokens a call");
    const uint64_t at_a_time = std::min<uint64_t>(tokens, (a->tokens + a->requests - 1) / std::max(1u, a->requests));  // of a tile, in the mean
    const uint64_t blocks = std::min<uint64_t>(a->table_width, static_cast<uint64_t>(P.first) + P.last + at_a_time * P.nids);
    const uint64_t most = blocks * c->page_size;
    // Parts of a tile until every CU has one: 48 single tokens over 51 pages of 32, 480 tiles, 72.8 us
    // whole, 76.9 in two parts; 4 drafts of 1 to 5, 32 tiles, 14.2 us in eight.
    P.parts = 1;
    while (!plan->chunk && P.parts < kMostParts && items * P.parts < 256 && most > 2 * P.parts * kSplitTokens) P.parts *= 2;
    const uint64_t slots = items * P.parts * kTileRows;
    plan->ml = slots * c->dim * 4;
    plan->workspace = P.parts > 1 ? slots * (c->dim * 4 + 8) : 0;
    return FG_OK;
}

template <class T, int D>
int launch(const BlocksParams &P, const BlocksPlan &plan, hipStream_t st) {
    if constexpr (D <= 128) {
        if (plan.chunk) {
            hipLaunchKernelGGL((fg_blocks_chunk_kernel<T, D>), dim3(plan.tiles * P.lanes), dim3(256), 0, st, P);
            FG_HIP(hipGetLastError(), "attention launch");
            return FG_OK;
        }
    }
    FG_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(fg_blocks_kernel<T, D>), hipFuncAttributeMaxDynamicSharedMemorySize, kMostBlocks * 12), "attention LDS");
    hipLaunchKernelGGL((fg_blocks_kernel<T, D>), dim3(plan.tiles * P.parts * P.lanes), dim3(256), plan.lds, st, P);
    if (P.parts > 1) hipLaunchKernelGGL((fg_blocks_join_kernel<T, D>), dim3(plan.tiles * P.lanes), dim3(256), 0, st, P);
    FG_HIP(hipGetLastError(), "attention launch");
    return FG_OK;
}

template <class T>
int launch(const BlocksParams &P, const BlocksPlan &plan, uint32_t dim, hipStream_t st) {
    switch (dim) {
    case 64: return launch<T, 64>(P, plan, st);
    case 96: return launch<T, 96>(P, plan, st);
    case 128: return launch<T, 128>(P, plan, st);
    default: return launch<T, 256>(P, plan, st);
    }
}

}  // namespace
}  // namespace fgk

using namespace fgk;

extern "C" {

int64_t fg_attend_blocks_workspace_bytes(const fg_kv_cache *cache, const fg_attention *a) {
    return guarded<int64_t>([&]() -> int64_t {
        BlocksParams P{};
        BlocksPlan plan;
        if (int rc = prepare(cache, a, &P, &plan)) return rc;
        return static_cast<int64_t>(a->requests && a->tokens ? plan.workspace : 0);
    });
}

int fg_attend_blocks(const fg_kv_cache *cache, const fg_attention *a, void *workspace, uint64_t workspace_bytes, void *stream) {
    return guarded<int>([&]() -> int {
        BlocksParams P{};
        BlocksPlan plan;
        if (int rc = prepare(cache, a, &P, &plan)) return rc;
        if (a->requests == 0 || a->tokens == 0) return FG_OK;
        if (plan.workspace && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < plan.workspace))
            return fail(FG_EINVAL, "workspace must be 16-byte aligned and hold " + std::to_string(plan.workspace) + " bytes");
        P.part = static_cast<float *>(workspace);
        P.part_ml = reinterpret_cast<float2 *>(static_cast<char *>(workspace) + plan.ml);
        hipStream_t st = reinterpret_cast<hipStream_t>(stream);
        return cache->dtype == FG_BF16 ? launch<BF16>(P, plan, cache->dim, st) : launch<F16>(P, plan, cache->dim, st);
    });
}

}  // extern "C"
