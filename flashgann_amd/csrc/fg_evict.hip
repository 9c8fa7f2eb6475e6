// fg_evict.hip -- a paged cache held to a budget: the attention weight that each token has
// drawn, and which tokens stay.
//
// Weights: for token j the sum over rows of exp(scale q . k_j - lse), the column sums of the
// matrix that attention takes row by row.  With lse known there is no maximum to follow.
// Eviction: of n tokens the heaviest H stay, those below place H where they are; each hole
// there takes a token from above, so only rows that have to move are read and written.
#include "fg_blocks.hpp"
#include "fg_pick.hpp"

namespace fgk {
namespace {

// ---------------------------------------------------------------- weights

constexpr uint32_t kWeighTokens = 256, kWeighRows = 64;  // tokens of a workgroup; rows in LDS at a time

struct WeighParams {
    CacheView cache;
    const char *q;
    int64_t q_token, q_head;  // bytes
    const float *lse;
    const int32_t *table, *q_starts, *kv_lens, *known;
    int64_t table_row;
    float *weights;
    uint32_t table_width, requests, tokens, heads, heads_kv;
    uint32_t spread;  // workgroups side by side over a request's tokens
    FastDiv group;
    float scale2;  // scale * log2(e)
};

// Each of the four waves holds the keys of 64 tokens in registers and goes through the rows,
// which all share from LDS, 16 at a time on the matrix unit: a lane's column is a token, so
// its sum stays in one register till the end.
//
// Single tokens are bound by the keys' bytes: 32 over 500 to 8,000 (8 heads, dim 128) 66 us, 4.3 TB/s.
// The last 300 to 500 rows of two prompts take 131 us, at issue: vector 55%, matrix 32%, and 1,008
// workgroups on 768 places.  128 tokens a workgroup 71.9 us instead of 66, 16 rows a step 67, four
// workgroups a CU spill (92 us).
template <class T, int D>
__global__ __launch_bounds__(256, D <= 128 ? 3 : 2) void fg_weigh_kernel(WeighParams P) {
    using vec = typename T::vec;
    constexpr int STEPS = D / 32;
    constexpr uint32_t QROW = 2 * D + 16;  // bytes of a row in LDS
    constexpr int PER = kWeighRows * (D / 8) / 256;
    // rows of two steps: those being weighed and the next ones
    __shared__ __attribute__((aligned(16))) char rows_of[2][kWeighRows * QROW];
    __shared__ __attribute__((aligned(16))) float lse2[2][kWeighRows];
    __shared__ __attribute__((aligned(16))) int32_t row_pos[2][kWeighRows];  // INT_MIN: the row counts nowhere
    __shared__ uint32_t all_count[2];                                        // whether all of a step's rows count
    static_assert(kWeighRows == 64);
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = uniform(tid / 64), col = lane % 16, quarter = lane / 16;
    const uint64_t items = static_cast<uint64_t>(P.requests) * P.heads_kv * P.spread;
    for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const uint32_t x = item % P.spread, rh = static_cast<uint32_t>(item / P.spread), r = rh / P.heads_kv, h = rh - r * P.heads_kv;
        const int32_t cap = static_cast<int32_t>(P.tokens);
        const int32_t q0 = clampi(P.q_starts[r], 0, cap), fresh = clampi(P.q_starts[r + 1], q0, cap) - q0;
        const int32_t kv = max(P.kv_lens[r], 0), known = P.known[r], pos0 = kv - fresh;
        const int32_t limit = static_cast<int32_t>(min(static_cast<uint64_t>(kv), static_cast<uint64_t>(P.table_width) * P.cache.page_size.d));
        const int32_t nrows = fresh * static_cast<int32_t>(P.group.d);
        const char *const kbase = P.cache.k + h * P.cache.k_head + quarter * 16;
        for (int32_t j0 = static_cast<int32_t>(x * kWeighTokens); j0 < limit; j0 += static_cast<int32_t>(P.spread * kWeighTokens)) {
            // this lane's token of the wave's 64
            const int32_t jw = j0 + static_cast<int32_t>(wave * 64), j = jw + static_cast<int32_t>(lane);
            int2 at = {-1, 0};
            if (j < limit) {
                const uint32_t b = P.cache.page_size.div(j);
                const int32_t page = P.table[r * P.table_row + b];
                at = {static_cast<uint32_t>(page) < P.cache.pages ? page : -1, static_cast<int32_t>(j - b * P.cache.page_size.d)};
            }
            vec kf[4][STEPS];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int64_t page = max(__shfl(at.x, 16 * c + static_cast<int>(col)), 0);
                const char *src = kbase + page * P.cache.k_page + __shfl(at.y, 16 * c + static_cast<int>(col)) * P.cache.k_token;
#pragma unroll
                for (int s = 0; s < STEPS; ++s) kf[c][s] = *reinterpret_cast<const vec *>(src + 64 * s);
            }
            float sum[4] = {0, 0, 0, 0};
            // rows before position j0 see none of these tokens
            const int32_t begin = max(j0 - pos0, 0) < fresh ? max(j0 - pos0, 0) * static_cast<int32_t>(P.group.d) : nrows;
            u32x4 q_next[PER];
            float z_next = 0.0f;
            const auto load = [&](int32_t base) {
#pragma unroll
                for (int c = 0; c < PER; ++c) {
                    const uint32_t e = c * 256 + tid;
                    const int32_t row = min(base + static_cast<int32_t>(e / (D / 8)), nrows - 1), token = P.group.div(row);
                    q_next[c] = *reinterpret_cast<const u32x4 *>(P.q + (q0 + static_cast<int64_t>(token)) * P.q_token +
                                                                 (static_cast<int64_t>(h) * P.group.d + (row - token * static_cast<int32_t>(P.group.d))) * P.q_head + e % (D / 8) * 16);
                }
                if (tid < kWeighRows) {
                    const int32_t row = min(base + static_cast<int32_t>(tid), nrows - 1), token = P.group.div(row);
                    z_next = P.lse[(q0 + static_cast<int64_t>(token)) * P.heads + h * P.group.d + (row - token * static_cast<int32_t>(P.group.d))];
                }
            };
            const auto store = [&](int32_t base, uint32_t buf) {  // (rows past the last are repeated and count nowhere)
#pragma unroll
                for (int c = 0; c < PER; ++c) {
                    const uint32_t e = c * 256 + tid;
                    *reinterpret_cast<u32x4 *>(rows_of[buf] + e / (D / 8) * QROW + e % (D / 8) * 16) = q_next[c];
                }
                if (tid < kWeighRows) {
                    const int32_t row = base + static_cast<int32_t>(tid);
                    const bool counts = row < nrows && z_next != -INFINITY;
                    lse2[buf][tid] = counts ? z_next * 1.44269504088896341f : 0.0f;
                    row_pos[buf][tid] = counts ? pos0 + static_cast<int32_t>(P.group.div(row)) : INT32_MIN;
                    const bool all = __all(counts);
                    if (tid == 0) all_count[buf] = all;
                }
            };
            __syncthreads();
            if (begin < nrows) {
                load(begin);
                store(begin, 0);
            }
            wait_loads();  // of the keys: not known to have landed, they would be waited for in the loop, the next rows with them
            if (begin + static_cast<int32_t>(kWeighRows) < nrows) load(begin + kWeighRows);
            uint32_t buf = 0;
            for (int32_t base = begin; base < nrows; base += kWeighRows, buf ^= 1) {
                lds_barrier();
                if (base + static_cast<int32_t>(kWeighRows) < nrows) store(base + kWeighRows, buf ^ 1);
                if (base + 2 * static_cast<int32_t>(kWeighRows) < nrows) load(base + 2 * kWeighRows);
                const auto weigh = [&](int32_t i0, auto masked) {
                    vec qf[STEPS];
#pragma unroll
                    for (int s = 0; s < STEPS; ++s) qf[s] = *reinterpret_cast<const vec *>(rows_of[buf] + (i0 + col) * QROW + 64 * s + 16 * quarter);
                    const f32x4 z = *reinterpret_cast<const f32x4 *>(lse2[buf] + i0 + 4 * quarter);
                    const s32x4 pos = masked ? *reinterpret_cast<const s32x4 *>(row_pos[buf] + i0 + 4 * quarter) : s32x4{0, 0, 0, 0};
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        f32x4 s = {0, 0, 0, 0};
#pragma unroll
                        for (int k = 0; k < STEPS; ++k) s = T::mfma16(qf[k], kf[c][k], s);
                        float p[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], P.scale2, -z[i]));
                        if (masked) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) p[i] = pos[i] >= jw + 16 * c + static_cast<int32_t>(col) ? p[i] : 0.0f;
                        }
                        sum[c] += (p[0] + p[1]) + (p[2] + p[3]);
                    }
                };
                // (rows are in order of position)
                if (uniform(all_count[buf]) && pos0 + static_cast<int32_t>(P.group.div(base)) >= jw + 63) {
#pragma unroll
                    for (int32_t i0 = 0; i0 < static_cast<int32_t>(kWeighRows); i0 += 16) weigh(i0, std::false_type{});
                } else {
                    const int32_t here = min(nrows - base, static_cast<int32_t>(kWeighRows));
                    for (int32_t i0 = 0; i0 < here; i0 += 16)
                        if (pos0 + static_cast<int32_t>(P.group.div(base + min(i0 + 15, here - 1))) >= jw) weigh(i0, std::true_type{});
                }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) sum[c] = add_other32(add_other16(sum[c]));
            const float mine = quarter < 2 ? (quarter == 0 ? sum[0] : sum[1]) : (quarter == 2 ? sum[2] : sum[3]);
            if (at.x >= 0) {
                float *to = P.weights + (static_cast<int64_t>(at.x) * P.heads_kv + h) * P.cache.page_size.d + at.y;
                if (j >= known) *to = mine;
                else unsafeAtomicAdd(to, mine);  // (requests that share the page add too)
            }
        }
    }
}

// ---------------------------------------------------------------- eviction

constexpr uint32_t kChooseThreads = 1024, kChooseWaves = kChooseThreads / 64;
constexpr uint32_t kFewKeys = 8 * kChooseThreads, kChooseKeys = 32 * kChooseThreads;  // weights that a workgroup holds in registers
constexpr uint32_t kChooseWorkgroups = 512; // at most, where it does not
constexpr uint32_t kEvictRequests = 4096;
constexpr uint32_t kMoveThreads = 256, kMoveRows = 64;  // rows of a workgroup that fills holes
constexpr uint32_t kShiftPieces = 4;                    // 16-byte pieces of a row that a workgroup of the last tokens' move takes
constexpr uint32_t kFewMoves = 512;                     // that the workgroup which chose them makes itself

struct EvictParams {
    CacheView cache;
    float *weights;
    const int32_t *table, *kv_lens;
    int64_t table_row;
    int32_t *new_lens, *freed, *released;
    int32_t *from, *to;  // tokens, `most` for each request and head: places above H, and below
    uint32_t *counts;    // how many
    uint32_t *keys;      // where registers do not hold them: `room` for each workgroup
    uint32_t table_width, requests, heads_kv, budget, window, sinks;
    uint32_t room;       // tokens that the table names
    uint32_t most;       // tokens that may move into holes: min(budget, room - budget)
    uint32_t choosers;   // workgroups that choose; the others list the pages that go
    uint32_t pieces;     // 16-byte pieces of a row of keys
    uint32_t at_once;    // whether those that choose move too
};

__device__ __forceinline__ int32_t slot_of(const EvictParams &P, uint32_t r, uint32_t j) {
    const uint32_t b = P.cache.page_size.div(j);
    const int32_t page = P.table[r * P.table_row + b];
    return static_cast<uint32_t>(page) < P.cache.pages ? static_cast<int32_t>(page * P.cache.page_size.d + (j - b * P.cache.page_size.d)) : -1;
}
__device__ __forceinline__ uint32_t length_of(const EvictParams &P, uint32_t r) { return min(static_cast<uint32_t>(max(P.kv_lens[r], 0)), P.room); }
__device__ __forceinline__ uint32_t pages_of(const EvictParams &P, uint32_t n) {
    const uint32_t whole = P.cache.page_size.div(n);
    return whole + (whole * P.cache.page_size.d != n ? 1 : 0);
}

// The new lengths, and the pages that go one after another: every workgroup sums the lengths itself.
__device__ __forceinline__ void list_freed(const EvictParams &P, uint32_t w, uint32_t workgroups, uint32_t *first, uint32_t *sums) {
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = tid / 64, run = (P.requests + kChooseThreads - 1) / kChooseThreads;
    uint32_t mine = 0;
    for (uint32_t i = 0; i < run; ++i) {
        const uint32_t r = tid * run + i;
        if (r >= P.requests) break;
        const uint32_t n = length_of(P, r), left = min(n, P.budget);
        first[r] = mine;
        mine += pages_of(P, n) - pages_of(P, left);
        if (w == 0) P.new_lens[r] = static_cast<int32_t>(left);
    }
    uint32_t upto = mine;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    uint32_t before = upto - mine, all = 0;
    for (uint32_t i = 0; i < kChooseWaves; ++i) {
        if (i < wave) before += sums[i];
        all += sums[i];
    }
    for (uint32_t i = 0; i < run && tid * run + i < P.requests; ++i) first[tid * run + i] += before;
    __syncthreads();
    if (w == 0 && tid == 0) P.released[0] = static_cast<int32_t>(all);
    const uint32_t entries = P.requests * P.table_width;
    for (uint32_t f = w * kChooseThreads + tid; f < entries; f += workgroups * kChooseThreads) {
        int32_t page = -1;
        if (f < all) {
            uint32_t r = 0;  // the last request whose pages begin at or before f
            for (uint32_t step = 1u << (31 - __clz(P.requests)); step; step >>= 1)
                if (r + step < P.requests && first[r + step] <= f) r += step;
            page = P.table[r * P.table_row + pages_of(P, min(length_of(P, r), P.budget)) + (f - first[r])];
        }
        P.freed[f] = page;
    }
}

// One thread's part of moving rows of a request and head: 16 bytes of each, of the keys, then the
// values, and with the first of them the weight.
struct Mover {
    char *base;
    int64_t page_step, token_step;
    float *weights;  // of the head, page 0; nullptr: another thread moves them
    uint32_t weight_step;
    FastDiv page_size;
    __device__ __forceinline__ Mover(const EvictParams &P, uint32_t h, uint32_t piece) : page_size(P.cache.page_size) {
        const bool value = piece >= P.pieces;
        base = const_cast<char *>(value ? P.cache.v + h * P.cache.v_head : P.cache.k + h * P.cache.k_head) + (value ? piece - P.pieces : piece) * 16;
        page_step = value ? P.cache.v_page : P.cache.k_page, token_step = value ? P.cache.v_token : P.cache.k_token;
        weights = piece == 0 ? P.weights + static_cast<int64_t>(h) * page_size.d : nullptr;
        weight_step = P.heads_kv * page_size.d;
    }
    // U rows, source(u) to target(u), slots below 0 skipped; between loads and stores `between`
    template <uint32_t U, class S, class D, class B>
    __device__ __forceinline__ void move(S source, D target, B between) const {
        int32_t from[U], to[U];
        u32x4 x[U];
        float w[U];
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) from[u] = source(u), to[u] = target(u);
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            const uint32_t slot = max(from[u], 0), page = page_size.div(slot), at = slot - page * page_size.d;
            x[u] = *reinterpret_cast<const u32x4 *>(base + page * page_step + at * token_step);
            w[u] = weights ? weights[static_cast<int64_t>(page) * weight_step + at] : 0.0f;
        }
        between();
#pragma unroll
        for (uint32_t u = 0; u < U; ++u) {
            if (from[u] < 0 || to[u] < 0) continue;
            const uint32_t page = page_size.div(to[u]), at = to[u] - page * page_size.d;
            *reinterpret_cast<u32x4 *>(base + page * page_step + at * token_step) = x[u];
            if (weights) weights[static_cast<int64_t>(page) * weight_step + at] = w[u];
        }
    }
    // The last `window` of n tokens to places before `budget`, in steps of U * rows of them, this
    // thread's the row-th of each `rows`.  They may go to places that others of them leave, but never to
    // one that a later step reads, so a step loads all of its rows before it writes any.
    template <uint32_t U>
    __device__ __forceinline__ void shift(const EvictParams &P, uint32_t r, uint32_t n, uint32_t row, uint32_t rows, bool works) const {
        for (uint32_t i0 = 0; i0 < P.window; i0 += rows * U)
            move<U>([&](uint32_t u) { const uint32_t i = i0 + u * rows + row; return works && i < P.window ? slot_of(P, r, n - P.window + i) : -1; },
                    [&](uint32_t u) { const uint32_t i = i0 + u * rows + row; return works && i < P.window ? slot_of(P, r, P.budget - P.window + i) : -1; },
                    [] {
                        wait_loads();
                        __syncthreads();
                    });
    }
};

// The weights of U tokens j, j + step .. as keys, 0 from token `end` (1 or more) on: their pages
// first, then the weights.
template <uint32_t U, class F>
__device__ __forceinline__ void load_keys(const EvictParams &P, uint32_t r, uint32_t h, uint32_t j, uint32_t end, uint32_t step, F put) {
    int32_t page[U];
    float x[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) page[u] = P.table[r * P.table_row + P.cache.page_size.div(min(j + u * step, end - 1))];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        const uint32_t at = min(j + u * step, end - 1), off = at - P.cache.page_size.div(at) * P.cache.page_size.d;
        const int64_t real = static_cast<uint32_t>(page[u]) < P.cache.pages ? page[u] : 0;
        x[u] = P.weights[(real * P.heads_kv + h) * P.cache.page_size.d + off];
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
        const bool real = static_cast<uint32_t>(page[u]) < P.cache.pages;
        const uint32_t key = !real ? 1u : x[u] != x[u] ? key_of(INFINITY) : key_of(x[u] + 0.0f);  // (-0 as 0)
        put(u, j + u * step < end ? key : 0u);
    }
}

// A workgroup for a request and head: weights as ordered integers, the border of the heaviest,
// then which tokens move where.  K: a wave holds its run of up to 64 K weights in registers; 0: in
// a scratch.  Bound by latency: 48 requests of 8 heads, 1 to 64 over 4,096 tokens, 21 us (weights 1,
// border 4.4, places 1, moves the rest; two workgroups a CU); 4 of 20,000 to 32,000 33 us (weights
// 3.5, border 12, places 7) in 32 workgroups.
template <uint32_t K>
__global__ __launch_bounds__(kChooseThreads, K == 8 ? 8 : 4) void fg_evict_choose_kernel(EvictParams P) {
    extern __shared__ uint32_t dynamic[];
    __shared__ Picking<kChooseWaves> S;
    __shared__ int32_t few_to[K == 8 ? kFewMoves : 1], few_from[K == 8 ? kFewMoves : 1];
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = uniform(tid / 64);
    if (blockIdx.x >= P.choosers) {
        list_freed(P, blockIdx.x - P.choosers, gridDim.x - P.choosers, dynamic, S.valid);
        return;
    }
    for (uint32_t rh = blockIdx.x; rh < P.requests * P.heads_kv; rh += P.choosers) {
        const uint32_t r = rh / P.heads_kv, h = rh - r * P.heads_kv, n = length_of(P, r);
        if (n <= P.budget) {
            if (tid == 0) P.counts[rh] = 0;
            continue;
        }
        // tokens sinks .. end - 1 are chosen from: `low` of them, so that they end before place `keep`
        const uint32_t end = n - P.window, keep = P.budget - P.window, low = keep - P.sinks, span = end - P.sinks;
        const uint32_t per = run_size<kChooseWaves>(span), begin = min(wave * per, span), stop = min(begin + per, span);
        const auto choose = [&](const auto &run) {
            Border B{0xFFFFFFFFu, 0, 0};
            if (low) B = border_of<kChooseWaves>(run, low, S);
            // what each wave's run holds: keys above the border and equal to it, below place `keep` and from there on
            uint32_t above[2] = {0, 0}, same[2] = {0, 0};
            run.each([&](uint32_t x, uint32_t i) {
                const uint32_t late = i >= low, a = x > B.border, s = x == B.border;
                above[0] += a & ~late, above[1] += a & late, same[0] += s & ~late, same[1] += s & late;
            });
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint32_t a = wave_sum(above[c]), s = wave_sum(same[c]);
                if (lane == 0) S.count[c][wave] = a, S.count[2 + c][wave] = s;
            }
            __syncthreads();
            // a lane a wave: equal keys before it are the first to be taken
            const uint32_t w = lane % kChooseWaves, s0 = S.count[2][w], s1 = S.count[3][w];
            const uint32_t seen = sum_upto(s0 + s1) - (s0 + s1);  // (of the first lanes; the others' say nothing)
            const uint32_t gone = min(w * per + per, low) - min(w * per, low) - S.count[0][w] - (min(seen + s0, B.ties) - min(seen, B.ties));
            const uint32_t late = S.count[1][w] + min(seen + s0 + s1, B.ties) - min(seen + s0, B.ties);
            const uint32_t gones = sum_upto(gone), lates = sum_upto(late);
            const uint32_t holes = of_lane(static_cast<int32_t>(gones), kChooseWaves - 1);
            uint32_t equal = of_lane(static_cast<int32_t>(seen), wave), at_hole = of_lane(static_cast<int32_t>(gones - gone), wave),
                     at_late = of_lane(static_cast<int32_t>(lates - late), wave);
            const bool here = K == 8 && P.at_once;
            int32_t *const to = here ? few_to : P.to + static_cast<uint64_t>(rh) * P.most, *const from = here ? few_from : P.from + static_cast<uint64_t>(rh) * P.most;
            run.each([&](uint32_t x, uint32_t i) {
                const bool in = i < stop, take = taken(B, x, equal), hole = in && i < low && !take, rises = in && i >= low && take;
                const uint64_t hs = __ballot(hole), rs = __ballot(rises), before = (1ull << lane) - 1;
                if (hole) to[at_hole + __popcll(hs & before)] = static_cast<int32_t>(P.sinks + i);
                if (rises) from[at_late + __popcll(rs & before)] = static_cast<int32_t>(P.sinks + i);
                at_hole += __popcll(hs), at_late += __popcll(rs);
            });
            if (here) {
                const uint32_t pieces = 2 * P.pieces, rows = kChooseThreads / pieces, row = tid / pieces;
                const Mover mover(P, h, tid - row * pieces);
                __syncthreads();
                for (uint32_t i0 = 0; i0 < holes; i0 += rows)
                    mover.move<1>([&](uint32_t u) { const uint32_t i = i0 + u * rows + row; return row < rows && i < holes ? slot_of(P, r, few_from[i]) : -1; },
                                  [&](uint32_t u) { const uint32_t i = i0 + u * rows + row; return row < rows && i < holes ? slot_of(P, r, few_to[i]) : -1; }, [] {});
                __syncthreads();
                mover.shift<1>(P, r, n, row, rows, row < rows);
            } else if (tid == 0) {
                P.counts[rh] = holes;
            }
        };
        if constexpr (K > 0) {
            Held<K> run;
            run.begin = begin, run.end = stop;
            constexpr uint32_t U = K > 8 ? 8 : 4;
#pragma unroll
            for (uint32_t u0 = 0; u0 < K; u0 += U)
                if (u0 == 0 || begin + u0 * 64 < stop) load_keys<U>(P, r, h, P.sinks + begin + u0 * 64 + lane, P.sinks + max(stop, 1u), 64, [&](uint32_t u, uint32_t key) { run.key[u0 + u] = key; });
            choose(run);
        } else {
            uint32_t *const keys = P.keys + static_cast<uint64_t>(blockIdx.x) * P.room;
            for (uint32_t i0 = begin; i0 < stop; i0 += 8 * 64)
                load_keys<8>(P, r, h, P.sinks + i0 + lane, P.sinks + stop, 64, [&](uint32_t u, uint32_t key) {
                    if (i0 + u * 64 + lane < stop) keys[i0 + u * 64 + lane] = key;
                });
            // (a wave reads its own run alone: what it has written itself)
            choose(Stored<const uint32_t *>{keys, begin, stop});
        }
        __syncthreads();
    }
}

// The chosen tokens into the holes below; no other move touches a place of theirs, so any
// workgroup takes any of them.  Bound by their bytes: 4 requests of 20,000 to 32,000 to 4,096 22 us, 5 TB/s.
__global__ __launch_bounds__(kMoveThreads) void fg_evict_fill_kernel(EvictParams P) {
    const uint32_t h = blockIdx.y, r = blockIdx.z, rh = r * P.heads_kv + h, tid = threadIdx.x;
    if (length_of(P, r) <= P.budget) return;
    const uint32_t count = P.counts[rh], pieces = 2 * P.pieces, rows = kMoveThreads / pieces, row = tid / pieces;
    const Mover mover(P, h, tid - row * pieces);
    const int32_t *const from = P.from + static_cast<uint64_t>(rh) * P.most, *const to = P.to + static_cast<uint64_t>(rh) * P.most;
    for (uint32_t i0 = blockIdx.x * kMoveRows; i0 < count; i0 += gridDim.x * kMoveRows) {
        const uint32_t end = min(i0 + kMoveRows, count);
        for (uint32_t i1 = i0; i1 < end; i1 += rows * 4)
            mover.move<4>([&](uint32_t u) { const uint32_t i = i1 + u * rows + row; return row < rows && i < end ? slot_of(P, r, from[i]) : -1; },
                          [&](uint32_t u) { const uint32_t i = i1 + u * rows + row; return row < rows && i < end ? slot_of(P, r, to[i]) : -1; }, [] {});
    }
}

// The last tokens behind them, once all have left their places: a workgroup 64 bytes of every row.
__global__ __launch_bounds__(kMoveThreads) void fg_evict_shift_kernel(EvictParams P) {
    const uint32_t h = blockIdx.y, r = blockIdx.z, n = length_of(P, r), piece = blockIdx.x * kShiftPieces + threadIdx.x % kShiftPieces;
    if (n <= P.budget) return;
    const bool works = piece < 2 * P.pieces;
    Mover(P, h, works ? piece : 0).shift<4>(P, r, n, threadIdx.x / kShiftPieces, kMoveThreads / kShiftPieces, works);
}

// ---------------------------------------------------------------- host side

template <class T>
void launch_weigh(const WeighParams &P, uint32_t dim, uint32_t grid, hipStream_t st) {
    switch (dim) {
    case 64: hipLaunchKernelGGL((fg_weigh_kernel<T, 64>), dim3(grid), dim3(256), 0, st, P); break;
    case 96: hipLaunchKernelGGL((fg_weigh_kernel<T, 96>), dim3(grid), dim3(256), 0, st, P); break;
    case 128: hipLaunchKernelGGL((fg_weigh_kernel<T, 128>), dim3(grid), dim3(256), 0, st, P); break;
    default: hipLaunchKernelGGL((fg_weigh_kernel<T, 256>), dim3(grid), dim3(256), 0, st, P); break;
    }
}

int weigh(const fg_kv_cache *c, const fg_attention *a, float *weights, const int32_t *known, void *stream) {
    WeighParams P{};
    if (int rc = check_cache(c, &P.cache, false)) return rc;
    if (!a) return fail(FG_EINVAL, "attention arguments are NULL");
    if (a->heads < 1 || a->heads > 1024 || a->heads % c->heads_kv) return fail(FG_EINVAL, "heads must be a multiple of heads_kv, at most 1024");
    if (!(a->scale > 0.0f) || !std::isfinite(a->scale)) return fail(FG_EINVAL, "scale must be positive and finite");
    if (static_cast<uint64_t>(a->tokens) * a->heads > 0x7FFFFFFFull) return fail(FG_EINVAL, "tokens * heads must be below 2^31");
    if (a->table_width > 0x7FFFFFFFu || a->table_row < 0) return fail(FG_EINVAL, "table_width or table_row out of range");
    if (static_cast<uint64_t>(a->table_width) * c->page_size > 0x3FFFFFFFull) return fail(FG_EINVAL, "table_width * page_size must be below 2^30");
    if (a->tokens > kMostTokens) return fail(FG_EINVAL, "tokens must be at most 4,194,304");
    if (a->requests > 65536) return fail(FG_EINVAL, "requests must be at most 65,536");
    if (a->requests == 0) return FG_OK;
    if (!a->kv_lens || !a->q_starts || !known || !weights || (a->tokens && (!a->q || !a->lse)) || (a->table_width && !a->table))
        return fail(FG_EINVAL, "NULL device buffer");
    if (reinterpret_cast<uintptr_t>(a->q) % 16 || (a->q_token | a->q_head) % 8) return fail(FG_EINVAL, "q must be 16-byte aligned, strides multiples of 8 elements");
    P.q = static_cast<const char *>(a->q);
    P.q_token = 2 * a->q_token, P.q_head = 2 * a->q_head;
    P.lse = a->lse;
    P.table = a->table;
    P.q_starts = a->q_starts;
    P.kv_lens = a->kv_lens;
    P.known = known;
    P.table_row = a->table_row;
    P.weights = weights;
    P.table_width = a->table_width;
    P.requests = a->requests;
    P.tokens = a->tokens;
    P.heads = a->heads;
    P.heads_kv = c->heads_kv;
    P.group = fast_div(a->heads / c->heads_kv);
    P.scale2 = a->scale * 1.44269504088896341f;
    const uint64_t pairs = static_cast<uint64_t>(a->requests) * c->heads_kv;
    const uint64_t tiles = (static_cast<uint64_t>(a->table_width) * c->page_size + kWeighTokens - 1) / kWeighTokens;
    if (tiles == 0) return FG_OK;
    // a workgroup a tile, up to 16,384 of them
    P.spread = static_cast<uint32_t>(std::min<uint64_t>(tiles, std::max<uint64_t>(1, 16384 / pairs)));
    const uint32_t grid = static_cast<uint32_t>(std::min<uint64_t>(pairs * P.spread, 65536));
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (c->dtype == FG_BF16) launch_weigh<BF16>(P, c->dim, grid, st);
    else launch_weigh<F16>(P, c->dim, grid, st);
    FG_HIP(hipGetLastError(), "weigh launch");
    return FG_OK;
}

struct EvictPlan {
    bool held;
    uint64_t from, counts, keys, workspace;
};

int plan_evict(const fg_kv_cache *c, uint32_t table_width, uint32_t requests, uint32_t budget, EvictParams *out, EvictPlan *plan) {
    EvictParams &P = *out;
    if (int rc = check_cache_shape(c)) return rc;
    if (requests < 1 || requests > kEvictRequests) return fail(FG_EINVAL, "requests must be in [1, 4096]");
    if (budget < 1 || budget > 0x7FFFFFFFu) return fail(FG_EINVAL, "budget must be in [1, 2^31)");
    if (static_cast<uint64_t>(table_width) * c->page_size > 0x3FFFFFFFull) return fail(FG_EINVAL, "table_width * page_size must be below 2^30");
    if (table_width > 0x7FFFFFFFu / requests) return fail(FG_EINVAL, "requests * table_width must be below 2^31");
    P.table_width = table_width;
    P.requests = requests;
    P.heads_kv = c->heads_kv;
    P.budget = budget;
    P.room = table_width * c->page_size;
    P.most = std::min(budget, P.room - std::min(P.room, budget));
    const uint64_t pairs = static_cast<uint64_t>(requests) * c->heads_kv, slots = pairs * P.most;
    plan->held = P.room <= kChooseKeys;
    P.choosers = static_cast<uint32_t>(std::min<uint64_t>(pairs, plan->held ? 65536 : kChooseWorkgroups));
    plan->from = slots * 4;
    plan->counts = slots * 8;
    plan->keys = plan->counts + (pairs * 4 + 15) / 16 * 16;
    plan->workspace = plan->keys + (plan->held ? 0 : static_cast<uint64_t>(P.choosers) * P.room * 4);
    return FG_OK;
}

}  // namespace
}  // namespace fgk

using namespace fgk;

extern "C" {

int fg_cache_weigh(const fg_kv_cache *cache, const fg_attention *a, float *d_weights, const int32_t *d_known, void *stream) {
    return guarded<int>([&] { return weigh(cache, a, d_weights, d_known, stream); });
}

int64_t fg_cache_evict_workspace_bytes(const fg_kv_cache *cache, uint32_t table_width, uint32_t requests, uint32_t budget) {
    return guarded<int64_t>([&]() -> int64_t {
        EvictParams P{};
        EvictPlan plan;
        if (int rc = plan_evict(cache, table_width, requests, budget, &P, &plan)) return rc;
        return static_cast<int64_t>(plan.workspace);
    });
}

int fg_cache_evict(const fg_kv_cache *cache, float *d_weights, const int32_t *d_table, int64_t table_row, uint32_t table_width,
                   const int32_t *d_kv_lens, uint32_t requests, uint32_t budget, uint32_t window, uint32_t sinks,
                   int32_t *d_new_lens, int32_t *d_freed, int32_t *d_released, void *workspace, uint64_t workspace_bytes,
                   void *stream) {
    return guarded<int>([&]() -> int {
        EvictParams P{};
        EvictPlan plan;
        if (int rc = plan_evict(cache, table_width, requests, budget, &P, &plan)) return rc;
        if (int rc = check_cache(cache, &P.cache)) return rc;
        // places that share memory (a head repeated by a stride of 0, say) would be moved by several workgroups
        const bool shared = (cache->pages > 1 && (!cache->k_page || !cache->v_page)) || (cache->page_size > 1 && (!cache->k_token || !cache->v_token)) ||
                            (cache->heads_kv > 1 && (!cache->k_head || !cache->v_head));
        if (shared) return fail(FG_EINVAL, "a cache whose places share memory (a stride of 0) cannot be evicted from");
        if (static_cast<uint64_t>(window) + sinks > budget) return fail(FG_EINVAL, "window + sinks must be at most budget");
        if (table_row < 0) return fail(FG_EINVAL, "table_row out of range");
        if (!d_weights || !d_kv_lens || !d_new_lens || !d_released || (table_width && (!d_table || !d_freed))) return fail(FG_EINVAL, "NULL device buffer");
        if (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < plan.workspace)
            return fail(FG_EINVAL, "workspace must be 16-byte aligned and hold " + std::to_string(plan.workspace) + " bytes");
        // rows of one memory would be moved twice, and lengths written while others read them
        if (cache->k == cache->v) return fail(FG_EINVAL, "k and v must not be the same memory");
        if (d_new_lens < d_kv_lens + requests && d_kv_lens < d_new_lens + requests) return fail(FG_EINVAL, "new lengths must not overlap kv_lens");
        char *base = static_cast<char *>(workspace);
        P.weights = d_weights;
        P.table = d_table;
        P.kv_lens = d_kv_lens;
        P.table_row = table_row;
        P.new_lens = d_new_lens;
        P.freed = d_freed;
        P.released = d_released;
        P.to = reinterpret_cast<int32_t *>(base);
        P.from = reinterpret_cast<int32_t *>(base + plan.from);
        P.counts = reinterpret_cast<uint32_t *>(base + plan.counts);
        P.keys = reinterpret_cast<uint32_t *>(base + plan.keys);
        P.window = window;
        P.sinks = sinks;
        hipStream_t st = reinterpret_cast<hipStream_t>(stream);
        const uint64_t entries = static_cast<uint64_t>(requests) * table_width;
        const uint32_t listers = static_cast<uint32_t>(std::min<uint64_t>(64, 1 + entries / (4 * kChooseThreads)));
        P.pieces = cache->dim / 8;
        // Few can move: in the kernel that chooses (48 requests of 8 heads back to 4,096 tokens, 1 over, a window of 16
        // 21 us against 31; 500 over 65 against 80, with a window of 400 104 against 128).
        P.at_once = P.room <= kFewKeys && P.room <= budget + kFewMoves && window <= kFewMoves;
        const auto choose = P.room <= kFewKeys ? fg_evict_choose_kernel<8> : plan.held ? fg_evict_choose_kernel<32> : fg_evict_choose_kernel<0>;
        hipLaunchKernelGGL(choose, dim3(P.choosers + listers), dim3(kChooseThreads), requests * 4, st, P);
        if (P.room > budget && !P.at_once) {
            const uint32_t moves = std::min(budget - window, P.room - budget);
            const uint32_t wide = std::max<uint32_t>(1, std::min<uint64_t>((moves + kMoveRows - 1) / kMoveRows, 8192 / (static_cast<uint64_t>(requests) * cache->heads_kv)));
            if (moves) hipLaunchKernelGGL(fg_evict_fill_kernel, dim3(wide, cache->heads_kv, requests), dim3(kMoveThreads), 0, st, P);
            if (window) hipLaunchKernelGGL(fg_evict_shift_kernel, dim3((2 * P.pieces + kShiftPieces - 1) / kShiftPieces, cache->heads_kv, requests), dim3(kMoveThreads), 0, st, P);
        }
        FG_HIP(hipGetLastError(), "eviction launch");
        return FG_OK;
    });
}

}  // extern "C"
