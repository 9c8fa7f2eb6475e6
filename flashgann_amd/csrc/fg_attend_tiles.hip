// fg_attend_tiles.hip -- attention over the paged cache for blocks of many query
// rows (chunks of prompts): bound by the matrix unit and the softmax beside it.
//
// A wave holds 32 query rows, one in each lane's column; the workgroup's waves (eight;
// four at dim 256, where a wave takes all registers of its SIMD) share tiles of 64
// tokens (32 at dim 256) in LDS, two of keys and two of values, the next ones on their
// way through registers.  Per tile a wave does 2 x D/16 products of 32 keys x 16
// dimensions for the scores and 4 x D/32 of 32 dimensions x 16 keys for the output;
// a wave of 16 rows would read LDS twice as often for the same products, which alone
// would take as long as they do.
//
// The matrix unit and the softmax take about as long (at dim 128 and a tile 1,024 and
// 960 cycles a wave), and one wave issues a vector instruction every eight cycles at
// best.  So a wave works out the weights of one tile between its products for the
// scores of the next.
//
// A chunk of 8,192 tokens after 8,192 (32 heads over 8, dim 128): 1,600 to 1,740 us by
// the card, 950 to 1,030 TFLOP/s, where a library product of 8,192^3 reaches 1,226; the
// matrix unit is busy 47% of the cycles and vector instructions issue in 46%, at 1.96
// GHz.  A chunk of 4,096 after 4,096 (the same heads): dim 128 909 TFLOP/s, 96 755 (matrix
// unit 37%, vector issue 48%), 64 621 (the softmax is twice as much for the same
// products), 256 725 (29% and 28%: neither is near its limit, and a SIMD has one wave).
#include "fg_attend.hpp"

namespace fgk {
namespace {

constexpr uint32_t kRing = 16;         // tiles whose places are known at a time
constexpr uint32_t kTilesUnit = 256;   // tokens between cuts

// The barrier that publishes LDS and nothing else: loads in flight from global
// memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <class T, int D, int NW, uint32_t kTile>
__global__ __launch_bounds__(64 * NW, NW / 4) __attribute__((amdgpu_waves_per_eu(NW / 4, NW / 4))) void fg_tiles_kernel(AttendParams P) {
    using vec = typename T::vec;
    constexpr uint32_t THREADS = 64 * NW, ROWS = 32 * NW;
    constexpr int STEPS = D / 16, DB = D / 32, CHUNKS = D / 8;   // 16-byte pieces of a row
    constexpr int BLOCKS = kTile / 32, SCORES = 16 * BLOCKS;     // of 32 tokens; a lane's
    // The maximum that weights are relative to follows when a row's grows past it by more
    // than 2^8, so they go up to there; what their exponents are raised by for the product, out
    // of the sums at the end.
    constexpr int LAG = 8;
    constexpr float UP = T::kTopWeight > LAG ? T::kTopWeight - LAG : 0, DOWN = 1.0f / (1 << static_cast<int>(UP));
    constexpr uint64_t ALL = kTile == 64 ? ~0ull : (1ull << kTile) - 1;
    constexpr uint32_t PER = (kTile * CHUNKS + THREADS - 1) / THREADS;
    // LDS rows are longer than the data: eight rows' 16-byte pieces of K, and eight
    // rows' 64-byte pieces of V, then meet every bank equally often
    constexpr uint32_t KROW = 2 * D + 16, VROW = 2 * D + (D == 96 ? 128 : 64);
    __shared__ __attribute__((aligned(16))) char kbuf[2][kTile * KROW];
    __shared__ __attribute__((aligned(16))) char vbuf[2][kTile * VROW];
    // of tile i at i % kRing: where its tokens lie (bytes from the head's first key and
    // value), which of them there are, and in a tile that not every row sees which
    // hold an infinite or NaN value: 0 * inf is NaN, so those are taken out of the
    // product and added to the rows that see them
    __shared__ longlong2 place[kRing][kTile];
    __shared__ uint64_t held[kRing];
    __shared__ unsigned long long special[kRing];

    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = uniform(tid / 64), col = lane % 32, half = lane / 32;
    const uint32_t W = gridDim.x;
    // neighbours in weight, which read the same keys, on one die of eight (the
    // grid is a multiple of 8)
    const uint32_t w = blockIdx.x % 8 * (W / 8) + blockIdx.x / 8;
    const Start start = find_start<false, ROWS>(P, w);
    if (P.join && tid == 0) P.joins[w].pieces = 0;
    const uint64_t x1 = min((w + 1) * start.share, start.all);
    uint64_t before = start.before;
    uint32_t r = start.request;
    uint64_t x = w * start.share;
    if (x >= x1) return;
    Request rq = start.first;

    while (x < x1) {
        const uint64_t all = rq.weight_of(rq.blocks) * P.lists;
        if (x >= before + all) {
            before += all;
            rq = uniform_request<false, ROWS>(P, ++r);
            continue;
        }
        Span sp;
        const Piece pc = piece_of<false, ROWS>(P, rq, before, x, x1, &sp);
        if (pc.none) {
            x = x1;
            continue;
        }
        const int32_t t_lo = static_cast<int32_t>(pc.t_lo), t_hi = static_cast<int32_t>(pc.t_hi);
        const int32_t tiles = (t_hi - t_lo + static_cast<int32_t>(kTile) - 1) / static_cast<int32_t>(kTile);

        // this lane's row, and the positions that this wave's rows span
        const int32_t row_first = static_cast<int32_t>(pc.block * ROWS + wave * 32);
        const int32_t row = row_first + static_cast<int32_t>(col);
        const int32_t token = P.group.div(row);
        const int32_t pos = sp.pos0 + token;
        const bool idle = row_first >= rq.rows;  // a wave without rows
        const int32_t pos_lo = uniform(sp.pos0 + static_cast<int32_t>(P.group.div(row_first)));
        const int32_t pos_hi = uniform(sp.pos0 + static_cast<int32_t>(P.group.div(min(row_first + 31, max(rq.rows - 1, row_first)))));
        const int32_t block_lo = uniform(sp.pos0 + static_cast<int32_t>(P.group.div(pc.block * ROWS)));
        vec qv[STEPS];
        {
            const int64_t head = static_cast<int64_t>(pc.list) * P.group.d + (row - token * static_cast<int32_t>(P.group.d));
            const int64_t qrow = rq.q0 + static_cast<int64_t>(token);
            const char *src = P.q + qrow * P.q_token + head * P.q_head + half * 16;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                u32x4 v = {0, 0, 0, 0};
                if (row < rq.rows) v = *reinterpret_cast<const u32x4 *>(src + 32 * s);
                qv[s] = __builtin_bit_cast(vec, v);
            }
        }
        const char *const kbase = P.cache.k + pc.list * P.cache.k_head;
        const char *const vbase = P.cache.v + pc.list * P.cache.v_head;

        // The places of NW tiles are looked up at a time, one by each wave, every NW steps
        // (one wave at every step would hold up the others every time): the table is
        // read eight steps ahead or more, the places are written one step later, so nothing
        // waits for it.
        int32_t page = -1;
        uint32_t offset = 0;
        const auto look = [&](int32_t i) {
            const int32_t t = t_lo + i * static_cast<int32_t>(kTile) + renewed(static_cast<int32_t>(lane));
            page = -1;
            if (t < t_hi && lane < kTile) {
                const int32_t j = position_of(sp, t);
                const uint32_t b = P.cache.page_size.div(j);
                offset = j - b * P.cache.page_size.d;
                page = P.table[r * P.table_row + b];
            }
        };
        const auto note = [&](int32_t i) {
            const bool have = static_cast<uint32_t>(page) < P.cache.pages;
            const int64_t p = have ? page : 0, o = have ? offset : 0;
            const uint32_t at = renewed(static_cast<int32_t>(lane));
            if (at < kTile) place[i % kRing][at] = longlong2{p * P.cache.k_page + o * P.cache.k_token, p * P.cache.v_page + o * P.cache.v_token};
            const uint64_t there = __ballot(have);
            if (lane == 0) {
                held[i % kRing] = there;
                special[i % kRing] = 0;
            }
        };
        const int32_t shift = sp.from - sp.first;  // position less token number past the first ones
        const int32_t window = static_cast<int32_t>(min(P.window, 0x7FFFFFFFu));
        // whether every row of the workgroup sees all tokens of tile i, pages aside
        const auto whole_tile = [&](int32_t i, int32_t lo, int32_t hi) {
            const int32_t t0 = t_lo + i * static_cast<int32_t>(kTile), t1 = min(t0 + static_cast<int32_t>(kTile), t_hi) - 1;
            if (position_of(sp, t1) > lo) return false;
            return P.window == 0xFFFFFFFFu || t1 < sp.first || hi - position_of(sp, t0) < static_cast<int64_t>(P.window);
        };

        u32x4 kr[PER], vr[PER];
        // where this thread's pieces of a tile's keys (values) lie
        int64_t k_at[PER], v_at[PER];
        const auto find_k = [&](int32_t i) {
#pragma unroll
            for (uint32_t c = 0; c < PER; ++c) k_at[c] = place[i % kRing][min((tid + c * THREADS) / CHUNKS, kTile - 1)].x + (tid + c * THREADS) % CHUNKS * 16;
        };
        const auto find_v = [&](int32_t i) {
#pragma unroll
            for (uint32_t c = 0; c < PER; ++c) v_at[c] = place[i % kRing][min((tid + c * THREADS) / CHUNKS, kTile - 1)].y + (tid + c * THREADS) % CHUNKS * 16;
        };
        // (at dim 96 a tile is one and a half pieces a thread: the threads past its end load its
        // last row once more.  A branch there instead had the compiler wait for all loads
        // under way at every step: 24 mixed chunks 106 us against 87)
        const auto load_k = [&]() {
#pragma unroll
            for (uint32_t c = 0; c < PER; ++c)
                kr[c] = *reinterpret_cast<const u32x4 *>(kbase + k_at[c]);
        };
        const auto load_v = [&]() {
#pragma unroll
            for (uint32_t c = 0; c < PER; ++c)
                vr[c] = *reinterpret_cast<const u32x4 *>(vbase + v_at[c]);
        };
        const auto store_k = [&](int32_t i) {
#pragma unroll
            for (uint32_t c = 0; c < PER; ++c) {
                const uint32_t at = tid + c * THREADS;
                if (kTile * CHUNKS % THREADS == 0 || at < kTile * CHUNKS)
                    *reinterpret_cast<u32x4 *>(kbuf[i % 2] + at / CHUNKS * KROW + at % CHUNKS * 16) = kr[c];
            }
        };
        const int32_t block_hi = uniform(sp.pos0 + static_cast<int32_t>(P.group.div(min(pc.block * ROWS + ROWS, static_cast<uint32_t>(rq.rows)) - 1)));
        const auto store_v = [&](int32_t i, uint64_t there) {
            const bool edge = !whole_tile(i, block_lo, block_hi);
#pragma unroll
            for (uint32_t c = 0; c < PER; ++c) {
                const uint32_t at = tid + c * THREADS, trow = at / CHUNKS;
                if (kTile * CHUNKS % THREADS == 0 || at < kTile * CHUNKS) {
                    u32x4 v = vr[c];
                    // (a token without a page: whatever was read instead)
                    if (there != ALL && !((there >> trow) & 1)) v = u32x4{0, 0, 0, 0};
                    if (edge && any_special<T>(v)) {
                        atomicOr(&special[i % kRing], 1ull << trow);
                        v = finite_part<T>(v);
                    }
                    *reinterpret_cast<u32x4 *>(vbuf[i % 2] + trow * VROW + at % CHUNKS * 16) = v;
                }
            }
        };

        // m: of the scores before scaling; l: of the tiles that are done, l_tile: of this one
        // (one by one, weights below the last place of a long row's sum are lost)
        float m = -INFINITY, l = 0.0f, l_tile = 0.0f;
        f32x16 o[DB];
#pragma unroll
        for (int i = 0; i < DB; ++i) o[i] = f32x16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};

        // Scores: register i of s[b] is that of token 32 b + 8 (i / 4) + 4 half + i % 4.
        // Two tiles': one's are weighed while the other's are worked out.
        f32x16 s_even[BLOCKS], s_odd[BLOCKS];
        float top = -INFINITY;  // the largest of the next tile to be weighed
        uint64_t there = 0;     // its tokens
        uint64_t raw_there = 0; // those of the tile after, as read from LDS
        u32x4 pk[2 * BLOCKS];   // the weights of 16 tokens each
        // Two weights of 32.  In the values' type: the matrix unit takes both alike, and
        // the rounding of a weight is that of an output element.
        const auto weigh = [&](const f32x16 *s, int k, float base) {
            const float p0 = __builtin_amdgcn_exp2f(fmaf(s[k / 8][2 * (k % 8)], P.scale2, base));
            const float p1 = __builtin_amdgcn_exp2f(fmaf(s[k / 8][2 * (k % 8) + 1], P.scale2, base));
            l_tile = k ? l_tile + (p0 + p1) : p0 + p1;
            asm volatile("" : "+v"(l_tile));  // here, not when the sum is next looked at
            pk[k / 4][k % 4] = T::pack(p0, p1);
        };
        const auto read_key = [&](int32_t i, int n) {
            return __builtin_bit_cast(vec, *reinterpret_cast<const u32x4 *>(kbuf[i % 2] + (n / STEPS * 32 + col) * KROW + half * 16 + 32 * (n % STEPS)));
        };
        const uint32_t v_lane = (4 * half + lane % 16 / 4) * VROW + (lane / 16 % 2) * 32 + (lane % 4) * 8;
        const auto read_values = [&](int32_t i, int n) {
            const char *at = vbuf[i % 2] + v_lane + 16 * (n / DB) * VROW + 64 * (n % DB);
            return __builtin_bit_cast(vec, __builtin_shufflevector(read_transposed(at), read_transposed(at + 8 * VROW), 0, 1, 2, 3, 4, 5, 6, 7));
        };
        // (the compiler would read for one product at a time and gather the rest: LDS
        // reads run AHEAD products ahead, held there by the barriers for its scheduler)
        constexpr int AHEAD = 4;

        // Of two waves on a SIMD the one among its products issues first, the one among
        // those for the scores before the other: they fall out of step, one's matrix work
        // beside the other's vector work (a window of 1,000 over 12,000 tokens 115.4 us
        // against 111.7, the chunk of 8,192 1,667 against 1,650).
        // With a SIMD's 512 registers the compiler moved the output from the matrix unit's
        // half to the other and back at every step, in case the maximum grows; told where
        // it stays, only then (dim 256: a chunk of 4,000 after 4,000 651 us against 570).
        const auto settle = [&] {
            if constexpr (NW == 4) {
#pragma unroll
                for (int k = 0; k < DB; ++k) asm volatile("" : "+a"(o[k]));
            }
        };
        const auto first_in_line = [](auto level) {
            if constexpr (NW > 4) __builtin_amdgcn_s_setprio(level.value);
        };
        const auto step = [&](int32_t i, f32x16 *s, f32x16 *next) {
            lds_barrier();
            // the products' operands from LDS: K of the next tile, then V of this one
            vec ring[AHEAD];
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) ring[n] = read_key(i + 1, n);
            if (i % NW == 0) look(i + 8 + wave);
            if (i % NW == 1) note(i + 7 + wave);
            // LDS gets the next tile's values and the keys of the one after (past the last
            // tile what lies in page 0), whose places in it are read.  No branch among
            // the products below: the compiler would gather the weights behind it.
            const uint64_t there_next = uniform(raw_there);
            store_v(i + 1, there_next);
            const int32_t t0 = t_lo + i * static_cast<int32_t>(kTile);
            if (there != ALL || !whole_tile(i, pos_lo, pos_hi)) {
                // the tile's tokens that the row sees, then the lane's: four of every eight
                const uint64_t seen = there & (bits_below(sp.first - t0) & bits_below(pos + 1 - t0) |
                                               bits_below(pos + 1 - shift - t0) & ~bits_below(max(pos - window, -1) + 1 - shift - t0) & ~bits_below(sp.first - t0));
                const uint64_t mine = seen >> (4 * half);
                top = -INFINITY;
#pragma unroll
                for (int k = 0; k < SCORES; ++k) {
                    const int at = 8 * (k % 16 / 4) + k % 4;  // in its half of the tile
                    s[k / 16][k % 16] = keep_if(static_cast<uint32_t>(mine >> (k / 16 * 32)), at, s[k / 16][k % 16]);
                    top = fmaxf(top, s[k / 16][k % 16]);
                }
                top = max_other32(top);
            }
            top = fmaxf(m, top);
            // (the sums are no less exact for a maximum that lags)
            settle();
            if (__any((top - m) * P.scale2 > static_cast<float>(LAG))) {
                const float from = m == -INFINITY ? top : m;
                const float shrink = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((from - top) * P.scale2);
                l *= shrink;
#pragma unroll
                for (int k = 0; k < DB; ++k) o[k] *= shrink;
                settle();
                m = top;
            }
            const float base = m == -INFINITY ? 0.0f : fmaf(-m, P.scale2, UP);

            // the scores of the next tile (after the last one, of what LDS holds: unused), three
            // quarters of this one's weights between the products
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) next[b] = f32x16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
            constexpr int M = BLOCKS * STEPS, N = 2 * BLOCKS * DB;  // products for the scores, for the output
            static_assert(M % AHEAD == 0);
            first_in_line(std::integral_constant<int, 2>{});
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < M; ++k) {
                next[k / STEPS] = T::mfma32(ring[k % AHEAD], qv[k % STEPS], next[k / STEPS]);
                ring[k % AHEAD] = k + AHEAD < M ? read_key(i + 1, k + AHEAD) : read_values(i, k + AHEAD - M);
#pragma unroll
                for (int j = k * 6 * BLOCKS / M; j < (k + 1) * 6 * BLOCKS / M; ++j) weigh(s, j, base);
                if (k == 1) load_v();
                if (k == 2) store_k(i + 2);
                if (k == 3) find_k(i + 3);
                if (k == 7) load_k();
                __builtin_amdgcn_sched_barrier(0);
            }

            // this tile's values: product n adds 16 tokens, n / DB, to 32 dimensions; between
            // the products the last quarter's weights and the next scores' maximum
            top = -INFINITY;
            first_in_line(std::integral_constant<int, 1>{});
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                o[n % DB] = T::mfma32(ring[n % AHEAD], __builtin_bit_cast(vec, pk[n / DB]), o[n % DB]);
                if (n + AHEAD < N) ring[n % AHEAD] = read_values(i, n + AHEAD);
#pragma unroll
                for (int j = n * SCORES / N; j < (n + 1) * SCORES / N; ++j) top = fmaxf(top, next[j / 16][j % 16]);
#pragma unroll
                for (int j = 6 * BLOCKS + n * 2 * BLOCKS / (N - DB); j < min(6 * BLOCKS + (n + 1) * 2 * BLOCKS / (N - DB), 8 * BLOCKS); ++j) weigh(s, j, base);
                __builtin_amdgcn_sched_barrier(0);
            }
            first_in_line(std::integral_constant<int, 0>{});
            l += l_tile;
            find_v(i + 3);
            raw_there = held[(i + 2) % kRing];
            top = max_other32(top);
            if (there != ALL || !whole_tile(i, block_lo, block_hi))
                for (uint64_t odd = uniform(static_cast<uint64_t>(special[i % kRing])); odd; odd &= odd - 1) {
                    const int at = __ffsll(static_cast<unsigned long long>(odd)) - 1;
                    const char *src = vbase + place[i % kRing][at].y + renewed(static_cast<int32_t>(half)) * 8;
                    const bool shown = sees(P, pos, position_of(sp, t0 + at));
    #pragma unroll
                    for (int d = 0; d < DB; ++d)
    #pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint2 v = *reinterpret_cast<const uint2 *>(src + 64 * d + 16 * k);
                            o[d][4 * k] += shown ? special_part<T>(v.x & 0xFFFF) : 0.0f;
                            o[d][4 * k + 1] += shown ? special_part<T>(v.x >> 16) : 0.0f;
                            o[d][4 * k + 2] += shown ? special_part<T>(v.y & 0xFFFF) : 0.0f;
                            o[d][4 * k + 3] += shown ? special_part<T>(v.y >> 16) : 0.0f;
                        }
                    wait_loads();
                }
            there = there_next;
        };

        // (the last item's readers of LDS are past: see the barrier at the end)
        if (tiles > 0) {
#pragma unroll
            for (int32_t i = 0; i < 8; i += NW) {
                look(i + wave);
                note(i + wave);
            }
            lds_barrier();
            // the first tile's keys and values and the second one's keys, all under way at once
            find_k(0);
            load_k();
            u32x4 first[PER];
#pragma unroll
            for (uint32_t c = 0; c < PER; ++c) first[c] = kr[c];
            find_v(0);
            load_v();
            find_k(1);
            load_k();
            there = uniform(held[0]);
            find_v(1);
            find_k(2);
#pragma unroll
            for (uint32_t c = 0; c < PER; ++c)
                if (kTile * CHUNKS % THREADS == 0 || tid + c * THREADS < kTile * CHUNKS)
                    *reinterpret_cast<u32x4 *>(kbuf[0] + (tid + c * THREADS) / CHUNKS * KROW + (tid + c * THREADS) % CHUNKS * 16) = first[c];
            store_v(0, there);
            load_v();
            store_k(1);
            load_k();
            lds_barrier();
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) s_even[b] = f32x16{0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < BLOCKS * STEPS; ++k) s_even[k / STEPS] = T::mfma32(read_key(0, k), qv[k % STEPS], s_even[k / STEPS]);
#pragma unroll
            for (int k = 0; k < SCORES; ++k) top = fmaxf(top, s_even[k / 16][k % 16]);
            top = max_other32(top);
            find_v(2);
            raw_there = held[1];
            wait_loads();
        }
        // A wave without rows takes its share of the loads and leaves the matrix unit and LDS
        // to the others: 40 rows a list over 8 x 9,000 tokens (8 lists) took 67 us against 91
        // at dim 128 and 125 against 140 at dim 256; 128 rows (dim 128) 76 against 98, 256
        // rows 108 either way.
        if (idle) {
            for (int32_t i = 0; i < tiles; ++i) {
                lds_barrier();
                if (i % NW == 0) look(i + 8 + wave);
                if (i % NW == 1) note(i + 7 + wave);
                const uint64_t there_next = uniform(raw_there);
                store_v(i + 1, there_next);
                load_v();
                store_k(i + 2);
                find_k(i + 3);
                load_k();
                find_v(i + 3);
                raw_there = held[(i + 2) % kRing];
            }
        } else {
            for (int32_t i = 0; i < tiles; i += 2) {
                step(i, s_even, s_odd);
                if (i + 1 == tiles) break;
                step(i + 1, s_odd, s_even);
            }
        }
        lds_barrier();

        l = add_other32(l) * DOWN;
        const bool whole = pc.begins && pc.ends;
        top = m == -INFINITY ? m : m * P.scale2;
        const int32_t again = renewed(static_cast<int32_t>(tid));
        const int32_t out_row = row_first + again % 32, out_half = again / 32 % 2;
        if (out_row < rq.rows) {
            const int32_t t = P.group.div(out_row);
            const int64_t head = static_cast<int64_t>(pc.list) * P.group.d + (out_row - t * static_cast<int32_t>(P.group.d));
            const int64_t qrow = rq.q0 + static_cast<int64_t>(t);
            if (whole) {
                const float inv = l == 0.0f ? 0.0f : DOWN / l;
                char *dst = P.out + qrow * P.out_token + head * P.out_head + out_half * 8;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        *reinterpret_cast<uint2 *>(dst + 64 * d + 16 * k) =
                            uint2{T::pack(o[d][4 * k] * inv, o[d][4 * k + 1] * inv), T::pack(o[d][4 * k + 2] * inv, o[d][4 * k + 3] * inv)};
                if (P.lse && out_half == 0) P.lse[qrow * P.heads + head] = (top + __builtin_amdgcn_logf(l)) * kLn2;
            } else {
                const uint32_t slot = 2 * w + (pc.begins ? 1 : 0);
                const uint64_t at = static_cast<uint64_t>(slot) * ROWS + (out_row - static_cast<int32_t>(pc.block * ROWS));
                float *dst = P.part + at * D + out_half * 4;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        *reinterpret_cast<f32x4 *>(dst + 32 * d + 8 * k) = f32x4{o[d][4 * k], o[d][4 * k + 1], o[d][4 * k + 2], o[d][4 * k + 3]} * DOWN;
                if (out_half == 0) P.part_ml[at] = float2{top, l};
            }
        }
        if (P.join && tid == 0 && pc.begins && !pc.ends) {
            P.joins[w] = Join{workgroup_at(pc.end - 1, start.share) - w + 1, pc.block * ROWS, static_cast<uint32_t>(rq.rows), static_cast<uint32_t>(rq.q0), pc.list};
        }
        x = min(pc.end, x1);
    }
}

constexpr int waves_of(int dim) { return dim > 128 ? 4 : 8; }

template <class T, int D>
int launch(AttendParams &P, hipStream_t st) {
    constexpr int NW = waves_of(D);
    hipLaunchKernelGGL((fg_tiles_kernel<T, D, NW, (D > 128 ? 32 : 64)>), dim3(P.workgroups), dim3(64 * NW), 0, st, P);
    if (P.join) hipLaunchKernelGGL((fg_join_kernel<T, D, 32 * NW>), dim3(kJoinWorkgroups<32 * NW>), dim3(256), 0, st, P);
    FG_HIP(hipGetLastError(), "attention launch");
    return FG_OK;
}

template <class T>
int launch(AttendParams &P, uint32_t dim, hipStream_t st) {
    switch (dim) {
    case 64: return launch<T, 64>(P, st);
    case 96: return launch<T, 96>(P, st);
    case 128: return launch<T, 128>(P, st);
    default: return launch<T, 256>(P, st);
    }
}

}  // namespace

void plan_tiles(AttendParams &P, uint32_t dim, uint64_t seen) {
    P.rows = 32 * waves_of(dim);
    if (P.window != 0xFFFFFFFFu) seen += P.rows / P.group.d;  // a block's rows span so many tokens more
    // (cutting up to 512 tokens gains less than the join kernel takes)
    const uint32_t unit = seen <= 512 ? 512 : kTilesUnit;
    P.unit = fast_div(unit);
    P.workgroups = 256;
    P.join = seen > unit;
}

int launch_tiles(AttendParams &P, int dtype, uint32_t dim, hipStream_t stream) {
    return dtype == FG_BF16 ? launch<BF16>(P, dim, stream) : launch<F16>(P, dim, stream);
}

}  // namespace fgk
