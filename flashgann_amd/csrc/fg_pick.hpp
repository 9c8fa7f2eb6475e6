// fg_pick.hpp -- the largest keys of a row, exactly, where ties go to the lower place.
#ifndef FG_PICK_HPP
#define FG_PICK_HPP

#include "fg_attend.hpp"

namespace fgk {

// Floats as unsigned integers in the same order, none of them 0; not for NaN.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}

// Sums and extremes over a wave by moves between lanes that need no LDS: within rows of 16
// lanes by 1, 2, 4 and 8, then from a row's last lane to the next row, then to the upper two.
template <int CONTROL, int ROWS = 0xF>
__device__ __forceinline__ uint32_t moved(uint32_t old, uint32_t x) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(old), static_cast<int>(x), CONTROL, ROWS, 0xF, false));
}
template <class F>
__device__ __forceinline__ uint32_t wave_scan(uint32_t x, uint32_t none, F f) {  // over the lanes up to this one
    x = f(x, moved<0x111>(none, x));
    x = f(x, moved<0x112>(none, x));
    x = f(x, moved<0x114>(none, x));
    x = f(x, moved<0x118>(none, x));
    x = f(x, moved<0x142, 0xA>(none, x));
    return f(x, moved<0x143, 0xC>(none, x));
}
__device__ __forceinline__ uint32_t last_lane(uint32_t x) { return static_cast<uint32_t>(of_lane(static_cast<int32_t>(x), 63)); }
__device__ __forceinline__ uint32_t sum_upto(uint32_t x) {
    return wave_scan(x, 0, [](uint32_t a, uint32_t b) { return a + b; });
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t x) { return last_lane(sum_upto(x)); }
__device__ __forceinline__ uint32_t wave_min(uint32_t x) {
    return last_lane(wave_scan(x, 0xFFFFFFFFu, [](uint32_t a, uint32_t b) { return min(a, b); }));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    return last_lane(wave_scan(x, 0, [](uint32_t a, uint32_t b) { return max(a, b); }));
}

// The team's waves each hold a run of its keys, 64 at a time.
template <uint32_t WAVES>
__device__ __forceinline__ uint32_t run_size(uint32_t n) { return (n + 64 * WAVES - 1) / (64 * WAVES) * 64; }

// A wave's run in registers, up to 64 * K keys; 0 past its end.  Four are gone through at a time:
// a branch around each costs more.
template <uint32_t K>
struct Held {
    uint32_t key[K], begin, end;
    template <class F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll
        for (uint32_t u = 0; u < K; ++u) {
            if (u % 4 == 0 && u && begin + u * 64 >= end) break;
            f(key[u], begin + u * 64 + threadIdx.x % 64);
        }
    }
};
// In memory.
template <class Keys>
struct Stored {
    Keys keys;
    uint32_t begin, end;
    template <class F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll 4
        for (uint32_t i0 = begin; i0 < end; i0 += 64) {
            const uint32_t i = i0 + threadIdx.x % 64;
            f(i < end ? static_cast<uint32_t>(keys[i]) : 0u, i);
        }
    }
};
template <uint32_t WAVES>
__device__ __forceinline__ uint32_t team_wave() {
    if constexpr (WAVES > 1) return uniform(threadIdx.x / 64);
    else return 0;
}
template <uint32_t WAVES, class Keys>
__device__ __forceinline__ Stored<Keys> stored_run(Keys keys, uint32_t n) {
    const uint32_t per = run_size<WAVES>(n), begin = min(team_wave<WAVES>() * per, n);
    return {keys, begin, min(begin + per, n)};
}
template <uint32_t WAVES, uint32_t K, class Keys>
__device__ __forceinline__ Held<K> held_run(Keys keys, uint32_t n) {  // 1 <= n, run_size(n) <= 64 * K
    const uint32_t per = run_size<WAVES>(n), begin = min(team_wave<WAVES>() * per, n), end = min(begin + per, n);
    Held<K> h;
    h.begin = begin, h.end = end;
#pragma unroll
    for (uint32_t u = 0; u < K; ++u) h.key[u] = keys[min(begin + u * 64 + threadIdx.x % 64, n - 1)];
#pragma unroll
    for (uint32_t u = 0; u < K; ++u) h.key[u] = begin + u * 64 + threadIdx.x % 64 < end ? h.key[u] : 0u;
    return h;
}

// What a team of WAVES waves (1, or all of a workgroup) shares while it picks.  Where many add
// to a part's count, it is in several words, a lane's by its number: lanes that add to one
// word wait for each other.
constexpr uint32_t kParts = 256;
template <uint32_t WAVES>
struct Picking {
    static constexpr uint32_t kCopies = WAVES > 1 ? 4 : 1, kSets = WAVES > 1 ? 2 : 1;
    __attribute__((aligned(16))) uint32_t bins[kSets][kParts * kCopies];
    uint32_t least[2][WAVES], most[2][WAVES], valid[WAVES];
    uint32_t count[4][WAVES];
};

template <uint32_t WAVES>
__device__ __forceinline__ void team_sync() {
    if constexpr (WAVES > 1) __syncthreads();
    else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// Taken are the keys above `border` and the first `ties` of those equal to it.
struct Border {
    uint32_t border, ties, valid;  // valid: keys that are not 0
};

// The border of the `count` (1 or more) largest keys; 0 is no key.  The range between the least
// and the largest is divided into 256, and the part in which the last key to be taken lies
// again, until the keys from a part's lower end on are just those wanted or one value is left:
// four times at most (32 bits), twice for scores and weights in earnest.
template <uint32_t WAVES, class Run>
__device__ __forceinline__ Border border_of(const Run &run, uint32_t count, Picking<WAVES> &S) {
    constexpr uint32_t COPIES = Picking<WAVES>::kCopies, SETS = Picking<WAVES>::kSets, WORDS = kParts / 64 * COPIES;
    const uint32_t lane = threadIdx.x % 64, wave = team_wave<WAVES>();
    const auto clear = [&](uint32_t set) {
        if constexpr (WAVES > 1) {
            for (uint32_t w = threadIdx.x; w < kParts * COPIES; w += 64 * WAVES) S.bins[set][w] = 0;
        } else {
            *reinterpret_cast<u32x4 *>(S.bins[set] + lane * WORDS) = u32x4{0, 0, 0, 0};
            static_assert(WAVES > 1 || WORDS == 4);
        }
    };
    uint32_t least = 0xFFFFFFFFu, most = 0, valid = 0;
    run.each([&](uint32_t x, uint32_t) {
        valid += x != 0;
        most = max(most, x);
        least = min(least, x ? x : 0xFFFFFFFFu);
    });
    least = wave_min(least), most = wave_max(most), valid = wave_sum(valid);
    clear(0);
    const auto share_range = [&](uint32_t turn) {
        if constexpr (WAVES > 1) {
            if (lane == 0) S.least[turn][wave] = least, S.most[turn][wave] = most;
        }
        team_sync<WAVES>();
        if constexpr (WAVES > 1) {
            least = wave_min(S.least[turn][lane % WAVES]), most = wave_max(S.most[turn][lane % WAVES]);
        }
    };
    if constexpr (WAVES > 1) {
        if (lane == 0) S.valid[wave] = valid;
    }
    share_range(0);
    if constexpr (WAVES > 1) valid = wave_sum(lane < WAVES ? S.valid[lane % WAVES] : 0u);
    Border B{least, 0xFFFFFFFFu, valid};
    uint32_t hi = most, need = count;
    if (B.valid <= count) return B;
    for (uint32_t round = 0;; ++round) {
        const uint32_t lo = B.border, range = hi - lo;
        if (range == 0) {
            B.ties = need;
            break;
        }
        const uint32_t bits = 32 - __clz(range), shift = bits > 8 ? bits - 8 : 0;
        uint32_t *bins = S.bins[round % SETS];
        least = 0xFFFFFFFFu, most = 0;
        run.each([&](uint32_t x, uint32_t) {
            if (x >= lo && x <= hi) {
                atomicAdd(&bins[((x - lo) >> shift) * COPIES + lane % COPIES], 1u);
                least = min(least, x), most = max(most, x);
            }
        });
        least = wave_min(least), most = wave_max(most);
        if constexpr (SETS > 1) clear((round + 1) % SETS);
        share_range((round + 1) % 2);
        uint32_t mine[4] = {0, 0, 0, 0};  // a lane's four parts
#pragma unroll
        for (uint32_t w = 0; w < WORDS; w += 4) {
            const u32x4 some = *reinterpret_cast<const u32x4 *>(bins + lane * WORDS + w);
            if constexpr (COPIES == 4) mine[w / 4] = (some[0] + some[1]) + (some[2] + some[3]);
            else mine[0] = some[0], mine[1] = some[1], mine[2] = some[2], mine[3] = some[3];
        }
        const uint32_t sum = (mine[0] + mine[1]) + (mine[2] + mine[3]), upto = sum_upto(sum), above = last_lane(upto) - upto;
        // the lane whose parts hold the last key to be taken, and the part
        const uint32_t owner = __ffsll(static_cast<unsigned long long>(__ballot(above < need && above + sum >= need))) - 1;
        uint32_t part = 3, inside = mine[3], over = above;
#pragma unroll
        for (int p = 2; p >= 0; --p)
            if (part == p + 1u && over + inside < need) over += inside, part = p, inside = mine[p];
        part = 4 * owner + static_cast<uint32_t>(of_lane(static_cast<int32_t>(part), owner));
        need -= static_cast<uint32_t>(of_lane(static_cast<int32_t>(over), owner));
        inside = static_cast<uint32_t>(of_lane(static_cast<int32_t>(inside), owner));
        B.border = lo + (part << shift);
        hi = B.border + min(hi - B.border, (1u << shift) - 1);  // (the part's end may lie past 2^32)
        if (inside == need) break;  // all of the part: everything from its lower end on
        // where the keys lie closer than the parts are wide
        B.border = max(B.border, least), hi = min(hi, most);
        team_sync<WAVES>();  // (the bins are read before they are cleared again)
        if constexpr (SETS == 1) {
            clear(0);
            team_sync<WAVES>();
        }
    }
    return B;
}

// Whether lane's key x is taken; `equal` counts those equal to the border up to here.
__device__ __forceinline__ bool taken(const Border &B, uint32_t x, uint32_t &equal) {
    const bool same = x == B.border && x != 0;
    const uint64_t equals = __ballot(same);
    const bool take = x > B.border || (same && equal + __popcll(equals & ((1ull << threadIdx.x % 64) - 1)) < B.ties);
    equal += __popcll(equals);
    return take;
}

}  // namespace fgk

#endif
