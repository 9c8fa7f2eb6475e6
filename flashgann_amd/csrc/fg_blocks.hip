// fg_blocks.hip -- which pages of a cache a query should read: bounds of a page's keys in
// 8 bits, and the pages that promise a query the most.
//
// For a page, u and l its keys' largest and smallest value of each channel, a query q gives
// a key of it at most  sum_d max(q_d, 0) u_d + min(q_d, 0) l_d,  and the sum of that over
// the query heads of a list is the same with q+ = sum_h max(q_h, 0), q- = sum_h min(q_h, 0):
// one product of 2 dim terms a list, however many heads share it.  u and l are kept as 8-bit
// codes with a power-of-two scale, rounded outwards, so they stay bounds; q+ and q- are
// coded the same way for the product.  Integers below 2^24 times a power of two are exact
// in 32 bits: scores, and so the pages, do not depend on how the work is split.
#include "fg_blocks.hpp"
#include "fg_pick.hpp"

namespace fgk {
namespace {

typedef __attribute__((ext_vector_type(4))) int i32x4;

// 2^s as the bits of a float: the least power of two of which 127 reach `most` (not
// negative, finite), not below 2^-126.  127 = 1.984375 * 2^6.
__device__ __forceinline__ uint32_t scale_bits(float most) {
    const uint32_t e = (__float_as_uint(most) + 0x01FFFFu) >> 23;
    return max(static_cast<int32_t>(e) - 6, 1) << 23;
}
__device__ __forceinline__ float inverse(uint32_t scale_bits) { return __uint_as_float((254u << 23) - scale_bits); }

__device__ __forceinline__ uint32_t pack4(const int (&c)[4]) {
    return (c[0] & 0xFF) | (c[1] & 0xFF) << 8 | (c[2] & 0xFF) << 16 | static_cast<uint32_t>(c[3]) << 24;
}

// ---------------------------------------------------------------- bounds

constexpr uint32_t kBoundsThreads = 256, kBoundsTokens = 256;

struct BoundsParams {
    const char *k;
    int64_t k_page, k_token, k_head;  // bytes
    const int64_t *slots;
    int8_t *bounds;
    float *scales;
    uint32_t tokens, limit, heads;
    FastDiv page_size;
};

// A workgroup looks through 256 slots for those that end a page; each wave then takes a page
// of its head at a time, D / 8 lanes a row.  Eight loads a lane are under way.  Bound by the keys'
// bytes: 30,000 tokens (8 heads, dim 128, pages of 64) 15.8 us, 3.9 TB/s;
// of 64 single tokens by the latency of slots, then keys, 4.6 us.
template <class T, int D>
__global__ __launch_bounds__(kBoundsThreads) void fg_cache_bounds_kernel(BoundsParams P) {
    constexpr uint32_t LANES = D <= 64 ? 8 : D <= 128 ? 16 : 32, ROWS = 64 / LANES;  // (dim 96: 12 of 16 lanes work)
    __shared__ uint32_t full[kBoundsTokens], count;
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = tid / 64, head = blockIdx.y;
    if (tid == 0) count = 0;
    __syncthreads();
    const uint32_t t = blockIdx.x * kBoundsTokens + tid;
    if (t < P.tokens) {
        const int64_t slot = P.slots[t];
        if (slot >= 0 && slot < static_cast<int64_t>(P.limit)) {
            const uint32_t page = P.page_size.div(static_cast<uint32_t>(slot));
            if (static_cast<uint32_t>(slot) - page * P.page_size.d == P.page_size.d - 1) full[atomicAdd(&count, 1u)] = page;
        }
    }
    __syncthreads();
    const uint32_t piece = lane % LANES, sub = lane / LANES;
    const bool works = piece * 8 < D;
    for (uint32_t i = wave; i < count; i += kBoundsThreads / 64) {
        const int64_t page = full[i];
        const char *src = P.k + page * P.k_page + head * P.k_head + piece * 16;
        float hi[8], lo[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) hi[c] = -INFINITY, lo[c] = INFINITY;
        bool special = false;
        if (works) {
            // (a row past the last is the last once more)
            for (uint32_t row0 = 0; row0 < P.page_size.d; row0 += 8 * ROWS) {
                u32x4 w[8];
#pragma unroll
                for (uint32_t u = 0; u < 8; ++u) w[u] = *reinterpret_cast<const u32x4 *>(src + min(row0 + u * ROWS + sub, P.page_size.d - 1) * P.k_token);
#pragma unroll
                for (uint32_t u = 0; u < 8; ++u) {
                    special |= any_special<T>(w[u]);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const float a = as_float<T>(w[u][c] & 0xFFFF), b = as_float<T>(w[u][c] >> 16);
                        hi[2 * c] = fmaxf(hi[2 * c], a), lo[2 * c] = fminf(lo[2 * c], a);
                        hi[2 * c + 1] = fmaxf(hi[2 * c + 1], b), lo[2 * c + 1] = fminf(lo[2 * c + 1], b);
                    }
                }
            }
        }
        float most = 0.0f;
#pragma unroll
        for (int c = 0; c < 8; ++c) {
#pragma unroll
            for (uint32_t d = LANES; d < 64; d <<= 1) {
                hi[c] = fmaxf(hi[c], __shfl_xor(hi[c], d));
                lo[c] = fminf(lo[c], __shfl_xor(lo[c], d));
            }
            if (works) most = fmaxf(most, fmaxf(fabsf(hi[c]), fabsf(lo[c])));
        }
#pragma unroll
        for (uint32_t d = 1; d < LANES; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
        const bool finite = !__any(special);
        const uint32_t scale = finite ? scale_bits(most) : 0x7F800000u;
        const int64_t at = page * P.heads + head;
        if (lane == 0) P.scales[at] = __uint_as_float(scale);
        if (sub < 2 && works) {  // (two rows at least in a wave: one writes the upper bounds, one the lower)
            const float inv = finite ? inverse(scale) : 0.0f;
            int c[2][4];
#pragma unroll
            for (int i8 = 0; i8 < 8; ++i8) {
                // (floor(x) is -ceil(-x)) at least one code away from 0 where the key is not 0: the
                // product with one that lies 2^149 times below the scale is 0 before it is rounded
                const float out = sub ? -lo[i8] : hi[i8], x = fmaxf(ceilf(out * inv), out > 0.0f ? 1.0f : -127.0f);
                c[i8 / 4][i8 % 4] = finite ? static_cast<int>(sub ? -x : x) : 0;
            }
            *reinterpret_cast<uint2 *>(P.bounds + (at * 2 + sub) * D + piece * 8) = uint2{pack4(c[0]), pack4(c[1])};
        }
    }
}

// ---------------------------------------------------------------- selection

constexpr uint32_t kSelectThreads = 512, kSelectWaves = kSelectThreads / 64, kSelectRows = 16;
constexpr uint32_t kSelectLds = 128 * 1024;  // bytes of keys that a workgroup holds

struct SelectParams {
    const char *q;
    int64_t q_token, q_head;  // bytes
    const int8_t *bounds;
    const float *scales;
    const int32_t *table, *q_starts, *kv_lens;
    int64_t table_row;
    int32_t *ids;
    uint32_t *keys;     // where LDS does not hold them, or they are made and picked from by different kernels
    uint32_t table_width, requests, tokens, heads_kv, lists, list_heads, pages;
    uint32_t group;     // query heads of a list
    uint32_t count, first, last;
    FastDiv rows;       // query rows of a tile
    uint32_t stride;    // keys of a row
    uint32_t parts;     // workgroups that share a tile's blocks
    uint32_t tiles;
    FastDiv page_size;
};

// One past the last block that the row at `pos` selects from.
__device__ __forceinline__ int32_t end_of(const SelectParams &P, int32_t pos) {
    if (pos < 0) return 0;
    const int64_t end = static_cast<int64_t>(P.page_size.div(pos)) - P.last + 1;
    return static_cast<int32_t>(min(max(end, static_cast<int64_t>(0)), static_cast<int64_t>(P.table_width)));
}

// The codes of a tile's queries, 2 D bytes a row, into LDS: a wave the rows wave, wave + 8.
template <class T, int D>
__device__ __forceinline__ void code_queries(const SelectParams &P, const Tile &t, uint32_t list, char *codes, uint32_t row_bytes) {
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    constexpr uint32_t PAIRS = D / 2, N = (PAIRS + 63) / 64, R = kSelectRows / kSelectWaves;  // two channels a lane at a time
    float up[R][N][2] = {}, down[R][N][2] = {};
    const char *src[R];  // (past the tile's rows the last one again: nobody asks for its scores)
#pragma unroll
    for (uint32_t r = 0; r < R; ++r)
        src[r] = P.q + (t.q0 + static_cast<int64_t>(min(wave + r * kSelectWaves, static_cast<uint32_t>(t.rows) - 1))) * P.q_token +
                 static_cast<int64_t>(list) * P.group * P.q_head;
#pragma unroll 4
    for (uint32_t h = 0; h < P.group; ++h) {
#pragma unroll
        for (uint32_t r = 0; r < R; ++r)
#pragma unroll
            for (uint32_t n = 0; n < N; ++n) {
                const uint32_t pair = n * 64 + lane;
                if (PAIRS % 64 == 0 || pair < PAIRS) {
                    const uint32_t w = *reinterpret_cast<const uint32_t *>(src[r] + h * P.q_head + pair * 4);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float x = as_float<T>(c ? w >> 16 : w & 0xFFFF);
                        // (not fmaxf: a NaN has to stay one)
                        up[r][n][c] += x < 0.0f ? 0.0f : x;
                        down[r][n][c] += x > 0.0f ? 0.0f : x;
                    }
                }
            }
    }
#pragma unroll
    for (uint32_t r = 0; r < R; ++r) {
        char *const to = codes + (wave + r * kSelectWaves) * row_bytes;
        uint32_t most = 0;  // magnitudes as integers: infinities and NaN past all others
#pragma unroll
        for (uint32_t n = 0; n < N; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) most = max(most, max(__float_as_uint(up[r][n][c]) & 0x7FFFFFFFu, __float_as_uint(down[r][n][c]) & 0x7FFFFFFFu));
        most = wave_max(most);
        const bool finite = most < 0x7F800000u;
        const float inv = finite ? inverse(scale_bits(__uint_as_float(most))) : 0.0f;
#pragma unroll
        for (uint32_t n = 0; n < N; ++n) {
            const uint32_t pair = n * 64 + lane;
            if (PAIRS % 64 == 0 || pair < PAIRS) {
                const auto code = [&](float x) { return finite ? static_cast<int>(rintf(x * inv)) & 0xFF : 0; };
                *reinterpret_cast<uint16_t *>(to + 2 * pair) = static_cast<uint16_t>(code(up[r][n][0]) | code(up[r][n][1]) << 8);
                *reinterpret_cast<uint16_t *>(to + D + 2 * pair) = static_cast<uint16_t>(code(down[r][n][0]) | code(down[r][n][1]) << 8);
            }
        }
    }
}

// The `count` largest keys of a run by their places, ascending, -1 behind them.
template <uint32_t WAVES, class Run>
__device__ __forceinline__ void pick(const Run &run, uint32_t count, uint32_t first, int32_t *ids, Picking<WAVES> &S) {
    const uint32_t lane = threadIdx.x % 64, wave = team_wave<WAVES>();
    const Border B = border_of<WAVES>(run, count, S);
    uint32_t at = 0, equal = 0;  // ids written, and keys equal to the border, before this wave's run
    if constexpr (WAVES > 1) {
        uint32_t above = 0, same = 0;
        run.each([&](uint32_t x, uint32_t) { above += x > B.border, same += x == B.border; });
        above = wave_sum(above), same = wave_sum(same);
        if (lane == 0) S.count[0][wave] = above, S.count[1][wave] = same;
        __syncthreads();
        for (uint32_t w = 0; w < wave; ++w) {
            at += S.count[0][w] + min(S.count[1][w], B.ties - min(B.ties, equal));
            equal += S.count[1][w];
        }
    }
    if (B.valid)
        run.each([&](uint32_t x, uint32_t i) {
            const bool take = taken(B, x, equal);
            const uint64_t all = __ballot(take);
            if (take) ids[at + __popcll(all & ((1ull << lane) - 1))] = static_cast<int32_t>(first + i);
            at += __popcll(all);
        });
    for (uint32_t i = min(B.valid, count) + (WAVES > 1 ? threadIdx.x : lane); i < count; i += 64 * WAVES) ids[i] = -1;
}

// pick() for few, by a wave.  Bits of what each lane has at most give a bound that
// `count` lanes reach and a quarter more at most (none more past 20), or one that cannot be raised; the
// keys that reach it are few (16 of 1,000: 21 in the mean) and each is ranked, one a lane, by those
// above it.  False, with nothing done, where that does not serve.  Stopping at a quarter more spares turns
// for few keys (8 of 500 for 8,192 rows 19.7 us against 19.95 with none more) and makes too many candidates
// for many: 28 of 500 21.7 us, 22.9 with a quarter more there too, 32 of 1,000 33.4 against 43.6.
template <class Run>
__device__ __forceinline__ bool pick_few(const Run &run, uint32_t count, uint32_t first, int32_t *ids, u32x2 *some) {
    const uint32_t lane = threadIdx.x % 64;
    uint32_t top = 0;
    run.each([&](uint32_t x, uint32_t) { top = max(top, x); });
    if (static_cast<uint32_t>(__popcll(__ballot(top != 0))) < count) return false;
    const uint32_t most = wave_max(top), least = wave_min(top ? top : 0xFFFFFFFFu);
    uint32_t bound = least;
    if (most != least) {
        uint32_t mask = 0x80000000u >> __clz(most ^ least);
        bound = most & ~(2 * mask - 1);
        for (; mask; mask >>= 1) {
            const uint32_t reach = __popcll(__ballot(top >= (bound | mask)));
            if (reach < count) continue;
            bound |= mask;
            if (reach <= max(count, min(count + count / 4, 20u))) break;
        }
        bound = max(bound, least);
    }
    uint32_t have = 0;
    run.each([&](uint32_t x, uint32_t i) {
        const uint64_t reach = __ballot(x >= bound);
        const uint32_t at = have + __popcll(reach & ((1ull << lane) - 1));
        if (x >= bound && at < 64) some[at] = u32x2{x, i};
        have += __popcll(reach);
    });
    if (have > 64) return false;
    team_sync<1>();
    const u32x2 mine = some[lane];
    const uint32_t x = lane < have ? mine[0] : 0u;
    uint32_t above = 0;
    for (uint32_t i0 = 0; i0 < have; i0 += 8) {
#pragma unroll
        for (uint32_t u = 0; u < 8; ++u) above += static_cast<uint32_t>(of_lane(static_cast<int32_t>(x), i0 + u)) > x;
    }
    uint64_t chosen = __ballot(x != 0 && above < count);
    if (static_cast<uint32_t>(__popcll(chosen)) > count) {  // equal keys at the border: the first ones
        const uint32_t border = wave_min(chosen >> lane & 1 ? x : 0xFFFFFFFFu);
        uint64_t equal = __ballot(x == border);
        for (uint32_t more = __popcll(chosen) - count; more; --more) {
            const uint64_t last = 1ull << (63 - __clzll(equal));
            chosen &= ~last, equal &= ~last;
        }
    }
    if (chosen >> lane & 1) ids[__popcll(chosen & ((1ull << lane) - 1))] = static_cast<int32_t>(first + mine[1]);
    team_sync<1>();
    return true;
}

// Keys in registers where they fit.
template <uint32_t WAVES>
__device__ __forceinline__ void pick_from(const uint32_t *keys, uint32_t n, uint32_t count, uint32_t first, int32_t *ids, Picking<WAVES> &S) {
    if constexpr (WAVES == 1) {
        u32x2 *const some = reinterpret_cast<u32x2 *>(S.bins[0]);
        if (n && count <= 32) {
            if (n <= 64 * 8 ? pick_few(held_run<1, 8>(keys, n), count, first, ids, some)
                            : n <= 64 * 16 ? pick_few(held_run<1, 16>(keys, n), count, first, ids, some)
                                           : pick_few(stored_run<1>(keys, n), count, first, ids, some))
                return;
        }
    } else {
        const uint32_t per = run_size<WAVES>(n);
        if (n && per <= 64 * 2) return pick<WAVES>(held_run<WAVES, 2>(keys, n), count, first, ids, S);
        if (n && per <= 64 * 16) return pick<WAVES>(held_run<WAVES, 16>(keys, n), count, first, ids, S);
    }
    pick<WAVES>(stored_run<WAVES>(keys, n), count, first, ids, S);
}

enum { kFused, kScratch, kScore, kPick };  // keys in LDS; in a scratch of the workgroup; made only; picked from only

// A workgroup takes a tile of rows of one list: queries coded once, then each wave groups of
// 16 blocks through the matrix unit, rows against blocks.  Workgroups of neighbouring numbers
// take a tile's lists, so that an XCD, to which every eighth goes, sees few heads' bounds.
//
// Bound by the latency of a short workgroup.  32 single tokens over 4,000 to 24,000 (8 lists, dim 128,
// pages of 16) 25 us: the longest has 1,500 blocks, 13.5 us in the loop after 6.5 us of queries and
// first loads, 3.2 us to pick; their bounds at memory's rate would take 11 us.  A chunk of 4,096 tokens over
// 64,097 (pages of 64) 99 us: a workgroup 21 us, two a CU, in four rounds, its waves waiting for
// half of it.  Two groups of blocks under way a wave: four slow the split form by half.
template <class T, int D, int MODE, bool TEAM>
__global__ __launch_bounds__(kSelectThreads, D > 128 && !TEAM ? 2 : 4) void fg_select_kernel(SelectParams P) {
    constexpr int STEPS = 2 * D / 64, U = D <= 128 ? 2 : 1;  // groups of blocks under way at a time
    constexpr uint32_t QROW = 2 * D + 16;  // bytes of a row's codes in LDS
    constexpr uint32_t WAVES = TEAM ? kSelectWaves : 1;
    extern __shared__ uint32_t held[];
    __shared__ __attribute__((aligned(16))) char codes[kSelectRows * QROW];
    __shared__ Picking<WAVES> picking[TEAM ? 1 : kSelectWaves];
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = uniform(tid / 64), col = lane % 16, quarter = lane / 16;
    const uint32_t part = MODE == kScore ? blockIdx.y : 0, items = P.tiles * P.lists;
    for (uint32_t item = blockIdx.x; item < items; item += gridDim.x) {
        const uint32_t tile = item / P.lists, list = item - tile * P.lists;
        const Tile t = tile_of(P.q_starts, P.kv_lens, P.requests, P.tokens, P.rows, tile);
        if (t.rows == 0) continue;
        const int32_t first = static_cast<int32_t>(min(P.first, P.table_width)), end = end_of(P, t.pos + t.rows - 1);
        const uint32_t n = static_cast<uint32_t>(max(end - first, 0));
        uint32_t *const stored = P.keys + (MODE == kScratch ? blockIdx.x : static_cast<uint64_t>(t.q0) * P.lists + list) * static_cast<uint64_t>(P.stride);
        const uint32_t row_step = MODE == kScore ? P.lists * P.stride : P.stride;  // (of keys in memory: few enough where a tile has more than one row)
        if constexpr (MODE != kPick) {
            const uint32_t kv_head = list / P.list_heads;
            const int32_t *row = P.table + t.request * P.table_row + first;
            const uint32_t groups = (n + 15) / 16, step = kSelectWaves * (MODE == kScore ? P.parts : 1);
            const auto page_of = [&](uint32_t g) {  // (past the last block nothing is stored)
                return n ? row[min(g * 16 + col, n - 1)] : 0;
            };
            i32x4 b[U][STEPS];
            float scale[U];
            const auto load = [&](const int32_t (&page)[U]) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const bool real = static_cast<uint32_t>(page[u]) < P.pages;
                    const int64_t at = static_cast<int64_t>(real ? page[u] : 0) * P.heads_kv + kv_head;
                    const int8_t *src = P.bounds + at * (2 * D) + 16 * quarter;
#pragma unroll
                    for (int s = 0; s < STEPS; ++s) b[u][s] = *reinterpret_cast<const i32x4 *>(src + 64 * s);
                    const float of_page = P.scales[at];
                    scale[u] = real ? of_page : NAN;
                }
            };
            uint32_t g = wave + kSelectWaves * part;
            int32_t page[U];
#pragma unroll
            for (int u = 0; u < U; ++u) page[u] = page_of(g + u * step);
            load(page);
#pragma unroll
            for (int u = 0; u < U; ++u) page[u] = page_of(g + (U + u) * step);
            code_queries<T, D>(P, t, list, codes, QROW);
            lds_barrier();  // (the bounds stay on their way)
            i32x4 qv[STEPS];
#pragma unroll
            for (int s = 0; s < STEPS; ++s) qv[s] = *reinterpret_cast<const i32x4 *>(codes + col * QROW + 64 * s + 16 * quarter);
            int32_t ends[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) ends[i] = end_of(P, t.pos + static_cast<int32_t>(4 * quarter) + i) - first;
            const uint32_t rows = static_cast<uint32_t>(t.rows);
            const int32_t all = end_of(P, t.pos) - first;  // blocks that every row selects from
            uint32_t *const to = (MODE == kFused ? held : stored) + 4 * quarter * row_step;
            for (; g < groups; g += U * step) {
                i32x4 s4[U];
                float times[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    s4[u] = i32x4{0, 0, 0, 0};
                    times[u] = scale[u];
#pragma unroll
                    for (int s = 0; s < STEPS; ++s) s4[u] = __builtin_amdgcn_mfma_i32_16x16x64_i8(qv[s], b[u][s], s4[u], 0, 0, 0);
                }
                if (g + U * step < groups) {
                    load(page);
#pragma unroll
                    for (int u = 0; u < U; ++u) page[u] = page_of(g + (2 * U + u) * step);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const uint32_t i16 = (g + u * step) * 16 + col;
                    if (g + u * step >= groups) break;
                    uint32_t key[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) key[i] = key_of(static_cast<float>(s4[u][i]) * times[u]);
                    if (__any(!(times[u] < INFINITY))) {  // a page that is not finite, or none
#pragma unroll
                        for (int i = 0; i < 4; ++i) key[i] = times[u] != times[u] ? 0u : times[u] == INFINITY ? key_of(INFINITY) : key[i];
                    }
                    if (static_cast<int32_t>((g + u * step) * 16 + 16) > all) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) key[i] = static_cast<int32_t>(i16) < ends[i] ? key[i] : 0u;
                    }
                    if (i16 < n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (4 * quarter + i < rows) to[i * row_step + i16] = key[i];
                    }
                }
            }
            __syncthreads();
        }
        if constexpr (MODE != kScore) {
            for (uint32_t r = TEAM ? 0 : wave; r < static_cast<uint32_t>(t.rows); r += TEAM ? 1 : kSelectWaves) {
                int32_t *out = P.ids + ((t.q0 + static_cast<uint64_t>(r)) * P.lists + list) * P.count;
                if constexpr (MODE == kFused) pick_from<WAVES>(held + r * P.stride, n, P.count, first, out, picking[TEAM ? 0 : wave]);
                else pick_from<WAVES>(stored, n, P.count, first, out, picking[0]);
            }
            __syncthreads();
        }
    }
}

template <class T, int D>
int launch_select(const SelectParams &P, int mode, uint32_t grid, uint32_t lds, hipStream_t st) {
    const auto go = [&](auto kernel, const SelectParams &P, uint32_t grid, uint32_t parts, uint32_t bytes) -> int {
        if (bytes > 32 * 1024) FG_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kSelectLds), "selection LDS");
        hipLaunchKernelGGL(kernel, dim3(grid, parts), dim3(kSelectThreads), bytes, st, P);
        return FG_OK;
    };
    int rc = FG_OK;
    if (mode == kFused) rc = P.rows.d == 1 ? go(fg_select_kernel<T, D, kFused, true>, P, grid, 1, lds) : go(fg_select_kernel<T, D, kFused, false>, P, grid, 1, lds);
    else if (mode == kScratch) rc = go(fg_select_kernel<T, D, kScratch, true>, P, grid, 1, 0);
    else {
        rc = go(fg_select_kernel<T, D, kScore, true>, P, grid, P.parts, 0);
        SelectParams each = P;  // rows are picked from one by one
        each.rows = fast_div(1);
        each.tiles = P.tokens;
        if (rc == FG_OK) rc = go(fg_select_kernel<T, D, kPick, true>, each, static_cast<uint32_t>(std::min<uint64_t>(static_cast<uint64_t>(P.tokens) * P.lists, 1u << 20)), 1, 0);
    }
    if (rc != FG_OK) return rc;
    FG_HIP(hipGetLastError(), "selection launch");
    return FG_OK;
}

// How a call is run.
struct SelectPlan {
    int mode;
    uint32_t grid, lds;
    uint64_t workspace;
};

int prepare_select(const fg_kv_cache *c, const fg_attention *a, SelectParams *out, SelectPlan *plan) {
    SelectParams &P = *out;
    if (int rc = check_cache_shape(c)) return rc;
    if (!a) return fail(FG_EINVAL, "selection arguments are NULL");
    if (a->heads < 1 || a->heads > 1024 || a->heads % c->heads_kv) return fail(FG_EINVAL, "heads must be a multiple of heads_kv, at most 1024");
    if (a->lists < 1 || a->heads % a->lists || a->lists % c->heads_kv) return fail(FG_EINVAL, "lists must be a multiple of heads_kv that divides heads");
    if (a->nids < 1 || a->nids > kMostBlocks) return fail(FG_EINVAL, "blocks of a list must be in [1, 4096]");
    if (a->tokens > kMostTokens) return fail(FG_EINVAL, "tokens must be at most 4,194,304");
    if (static_cast<uint64_t>(a->tokens) * a->heads > 0x7FFFFFFFull) return fail(FG_EINVAL, "tokens * heads must be below 2^31");
    if (static_cast<uint64_t>(a->tokens) * a->lists * a->nids > 0x7FFFFFFFull) return fail(FG_EINVAL, "tokens * lists * blocks of a list must be below 2^31");
    if (a->table_width > 0x7FFFFFFFu || a->table_row < 0) return fail(FG_EINVAL, "table_width or table_row out of range");
    if (static_cast<uint64_t>(a->table_width) * c->page_size > 0x3FFFFFFFull) return fail(FG_EINVAL, "table_width * page_size must be below 2^30");
    if (a->sinks > 0x7FFFFFFFu) return fail(FG_EINVAL, "first blocks (sinks) must be below 2^31");
    if (a->window < 1) return fail(FG_EINVAL, "last blocks (window) must be >= 1");
    if (a->requests > 65536) return fail(FG_EINVAL, "requests must be at most 65,536");
    if (a->requests && a->tokens && (!a->q || !a->kv_lens || !a->q_starts || (a->table_width && !a->table))) return fail(FG_EINVAL, "NULL device buffer");
    if (reinterpret_cast<uintptr_t>(a->q) % 16 || (a->q_token | a->q_head) % 8) return fail(FG_EINVAL, "q must be 16-byte aligned, strides multiples of 8 elements");
    P.q = static_cast<const char *>(a->q);
    P.q_token = 2 * a->q_token, P.q_head = 2 * a->q_head;
    P.table = a->table;
    P.q_starts = a->q_starts;
    P.kv_lens = a->kv_lens;
    P.table_row = a->table_row;
    P.table_width = a->table_width;
    P.requests = a->requests;
    P.tokens = a->tokens;
    P.heads_kv = c->heads_kv;
    P.lists = a->lists;
    P.list_heads = a->lists / c->heads_kv;
    P.pages = c->pages;
    P.group = a->heads / a->lists;
    P.count = a->nids;
    P.first = a->sinks;
    P.last = static_cast<uint32_t>(a->window);
    P.page_size = fast_div(c->page_size);

    // Keys of a tile's rows are held in LDS: 16 rows where they fit, fewer over longer tables.  Up to two
    // rows a CU, or where most tiles would hold one or two, a workgroup takes a row: 4 requests of 8
    // new tokens over 1,000 blocks (8 lists) 17.4 us against 22.5, 32 of 1 22.0 against 32.8, of 2 27.3
    // against 33.1, of 3 37.9 against 33.0.
    const uint32_t most = std::max(1u, a->table_width - std::min(a->table_width, P.first));
    P.stride = most | 1;  // (odd: the rows of a tile lie in different banks)
    const bool one = a->tokens <= 2 * static_cast<uint64_t>(a->requests) || static_cast<uint64_t>(a->tokens) * a->lists <= 512;
    uint32_t rows = kSelectRows;
    while (rows > 1 && (static_cast<uint64_t>(rows) * P.stride * 4 > kSelectLds || one)) rows /= 2;
    P.rows = fast_div(rows);
    // (a row alone is a tile of its own number, and leaves none empty)
    P.tiles = a->tokens / rows + (rows > 1 ? a->requests : 0);
    const uint64_t items = static_cast<uint64_t>(P.tiles) * a->lists;
    if (items > 0x7FFFFFFFull) return fail(FG_EINVAL, "tokens * lists must be below 2^31");
    P.parts = 1;
    plan->grid = static_cast<uint32_t>(std::min<uint64_t>(items, 1u << 20));
    plan->lds = static_cast<uint32_t>(std::min<uint64_t>(static_cast<uint64_t>(rows) * P.stride * 4, 0xFFFFFFFFu));
    plan->workspace = 0;
    plan->mode = kFused;
    if (plan->lds > kSelectLds) {
        plan->mode = kScratch;
        plan->grid = static_cast<uint32_t>(std::min<uint64_t>(items, 512));
        plan->workspace = static_cast<uint64_t>(plan->grid) * P.stride * 4;
    }
    // Rows by themselves that are few, over many blocks: several workgroups make a row's keys, and one picks
    // from them (8 rows over 500 blocks 11.7 us against 12.2, over 1,500 12.5 against 21.9, over 8,125 17.6
    // against 81; 96 over 500 14.8 against 13.2, over 1,500 20.4 against 24.5; 128 over 3,750 38.5 against
    // 51.7; 256 over 1,500 31.8 against 30.3).  So with tiles, of 16 rows then, that are few (56 over 500 blocks
    // 16.9 us against 14.1, over 1,000 19.0 against 19.0, over 2,000 26.6 against 36.7; 208 over 2,000 57.6 against
    // 37.5), and over long tables, while the keys take 1 GiB at most.  In LDS a tile has 8 rows then (4 past 4,096
    // blocks): bounds are read twice as often, and past 2,160 blocks at dim 128, 2,030 at 256, two workgroups no
    // longer fit a CU; smaller bounds are still read faster than keys.  Keys in memory against LDS, us, 8 lists: 1,600
    // rows dim 64 3,199 blocks 198, 194, 3,699 210, 217; dim 96 2,699 209, 209, 3,199 224, 238; dim 128 2,149 201, 144,
    // 2,199 204, 211; dim 256 1,999 227, 189, 2,049 230, 288.  400 rows dim 64 3,624 66, 63, 4,224 74, 98; dim 96 2,624
    // 65, 59, 3,624 72, 77; dim 128 2,124 63, 48, 2,224 64, 62, 2,624 68, 70; dim 256 1,974 69, 49, 2,074 73, 86.
    const uint64_t keys = static_cast<uint64_t>(a->tokens) * a->lists * P.stride * 4;
    const uint64_t whole = one ? items : (static_cast<uint64_t>(a->tokens) / kSelectRows + a->requests) * a->lists;
    const bool few = most >= 1024 && whole <= (one ? 160 : 64);
    const uint32_t held_well = c->dim <= 64 ? 3400 : c->dim <= 96 ? 2800 : c->dim <= 128 ? 2160 : 2030;  // blocks
    if (keys <= (1ull << 30) && (few || (!one && P.stride > held_well))) {
        plan->mode = kScore;
        if (!one) {
            P.rows = fast_div(kSelectRows);
            P.tiles = a->tokens / kSelectRows + a->requests;
        }
        plan->grid = static_cast<uint32_t>(std::min<uint64_t>(whole, 1u << 20));
        P.parts = std::min<uint32_t>((most + 16 * kSelectWaves - 1) / (16 * kSelectWaves), static_cast<uint32_t>(std::max<uint64_t>(1, (one ? 512 : 1024) / std::max<uint64_t>(1, whole))));
        plan->workspace = keys;
    }
    return FG_OK;
}

template <class T>
int launch_select(const SelectParams &P, const SelectPlan &plan, uint32_t dim, hipStream_t st) {
    switch (dim) {
    case 64: return launch_select<T, 64>(P, plan.mode, plan.grid, plan.lds, st);
    case 96: return launch_select<T, 96>(P, plan.mode, plan.grid, plan.lds, st);
    case 128: return launch_select<T, 128>(P, plan.mode, plan.grid, plan.lds, st);
    default: return launch_select<T, 256>(P, plan.mode, plan.grid, plan.lds, st);
    }
}

template <class T>
void launch_bounds(const BoundsParams &P, uint32_t dim, dim3 grid, hipStream_t st) {
    switch (dim) {
    case 64: hipLaunchKernelGGL((fg_cache_bounds_kernel<T, 64>), grid, dim3(kBoundsThreads), 0, st, P); break;
    case 96: hipLaunchKernelGGL((fg_cache_bounds_kernel<T, 96>), grid, dim3(kBoundsThreads), 0, st, P); break;
    case 128: hipLaunchKernelGGL((fg_cache_bounds_kernel<T, 128>), grid, dim3(kBoundsThreads), 0, st, P); break;
    default: hipLaunchKernelGGL((fg_cache_bounds_kernel<T, 256>), grid, dim3(kBoundsThreads), 0, st, P); break;
    }
}

}  // namespace
}  // namespace fgk

using namespace fgk;

extern "C" {

int fg_cache_bounds(const fg_kv_cache *cache, const int64_t *d_slots, uint32_t tokens, int8_t *d_bounds, float *d_scales,
                    void *stream) {
    return guarded<int>([&]() -> int {
        CacheView view;
        if (int rc = check_cache(cache, &view, false)) return rc;
        if (tokens > 0x7FFFFFFFu) return fail(FG_EINVAL, "tokens must be below 2^31");
        if (tokens == 0) return FG_OK;
        if (!d_slots || !d_bounds || !d_scales) return fail(FG_EINVAL, "NULL device buffer");
        if (reinterpret_cast<uintptr_t>(d_bounds) % 16) return fail(FG_EINVAL, "bounds must be 16-byte aligned");
        const BoundsParams P{view.k, view.k_page, view.k_token, view.k_head, d_slots, d_bounds, d_scales, tokens,
                             cache->pages * cache->page_size, cache->heads_kv, view.page_size};
        const dim3 grid((tokens + kBoundsTokens - 1) / kBoundsTokens, cache->heads_kv);
        hipStream_t st = reinterpret_cast<hipStream_t>(stream);
        if (cache->dtype == FG_BF16) launch_bounds<BF16>(P, cache->dim, grid, st);
        else launch_bounds<F16>(P, cache->dim, grid, st);
        FG_HIP(hipGetLastError(), "bounds launch");
        return FG_OK;
    });
}

int64_t fg_select_blocks_workspace_bytes(const fg_kv_cache *cache, const fg_attention *a) {
    return guarded<int64_t>([&]() -> int64_t {
        SelectParams P{};
        SelectPlan plan;
        if (int rc = prepare_select(cache, a, &P, &plan)) return rc;
        return static_cast<int64_t>(a->requests && a->tokens ? plan.workspace : 0);
    });
}

int fg_select_blocks(const fg_kv_cache *cache, const fg_attention *a, const int8_t *d_bounds, const float *d_scales,
                     int32_t *d_ids, void *workspace, uint64_t workspace_bytes, void *stream) {
    return guarded<int>([&]() -> int {
        SelectParams P{};
        SelectPlan plan;
        if (int rc = prepare_select(cache, a, &P, &plan)) return rc;
        if (a->requests == 0 || a->tokens == 0) return FG_OK;
        if (!d_bounds || !d_scales || !d_ids) return fail(FG_EINVAL, "NULL device buffer");
        if (reinterpret_cast<uintptr_t>(d_bounds) % 16) return fail(FG_EINVAL, "bounds must be 16-byte aligned");
        if (plan.workspace && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < plan.workspace))
            return fail(FG_EINVAL, "workspace must be 16-byte aligned and hold " + std::to_string(plan.workspace) + " bytes");
        P.bounds = d_bounds;
        P.scales = d_scales;
        P.ids = d_ids;
        P.keys = static_cast<uint32_t *>(workspace);
        hipStream_t st = reinterpret_cast<hipStream_t>(stream);
        return cache->dtype == FG_BF16 ? launch_select<BF16>(P, plan, cache->dim, st) : launch_select<F16>(P, plan, cache->dim, st);
    });
}

}  // extern "C"
