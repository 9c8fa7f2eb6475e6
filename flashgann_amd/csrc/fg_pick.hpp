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

__device__ __forceinline__ uint32_t wave_sum(uint32_t v) {
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

// What a team of WAVES waves (1, or all of a workgroup) shares while it picks.
template <uint32_t WAVES>
struct Picking {
    uint32_t bins[2][64];
    uint32_t least[WAVES], most[WAVES], valid[WAVES];
    uint32_t count[2][WAVES];
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

// A wave's keys: a run of them.
struct Run {
    uint32_t begin, end;
};
template <uint32_t WAVES>
__device__ __forceinline__ Run run_of(uint32_t n) {
    const uint32_t wave = WAVES > 1 ? uniform(threadIdx.x / 64) : 0;
    const uint32_t per = (n + 64 * WAVES - 1) / (64 * WAVES) * 64, begin = min(wave * per, n);
    return {begin, min(begin + per, n)};
}

// The border of the `count` (1 or more) largest of n keys; 0 is no key.  The range between the
// least and the largest is divided into 64, and the part in which the last key to be taken lies
// again, until the keys from a part's lower end on are just those wanted or one value is left: six
// times at most (32 bits), two or three for scores in earnest.
template <uint32_t WAVES, class Keys>
__device__ __forceinline__ Border border_of(Keys keys, uint32_t n, uint32_t count, Picking<WAVES> &S) {
    const uint32_t lane = threadIdx.x % 64, wave = WAVES > 1 ? uniform(threadIdx.x / 64) : 0;
    const Run run = run_of<WAVES>(n);
    uint32_t least = 0xFFFFFFFFu, most = 0, valid = 0;
#pragma unroll 4
    for (uint32_t i = run.begin + lane; i < run.end; i += 64) {
        const uint32_t x = keys[i];
        valid += x != 0;
        most = max(most, x);
        least = min(least, x ? x : 0xFFFFFFFFu);
    }
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        least = min(least, static_cast<uint32_t>(__shfl_xor(least, d)));
        most = max(most, static_cast<uint32_t>(__shfl_xor(most, d)));
    }
    valid = wave_sum(valid);
    if (wave == 0) S.bins[0][lane] = 0;
    if constexpr (WAVES > 1) {
        if (lane == 0) S.least[wave] = least, S.most[wave] = most, S.valid[wave] = valid;
        __syncthreads();
        valid = 0;
#pragma unroll
        for (uint32_t w = 0; w < WAVES; ++w) least = min(least, S.least[w]), most = max(most, S.most[w]), valid += S.valid[w];
    } else {
        team_sync<WAVES>();
    }
    Border B{uniform(least), 0xFFFFFFFFu, uniform(valid)};
    uint32_t hi = uniform(most), need = count;
    if (B.valid <= count) return B;
    for (uint32_t round = 0;; ++round) {
        const uint32_t lo = B.border, range = hi - lo;
        if (range == 0) {
            B.ties = need;
            break;
        }
        const uint32_t bits = 32 - __clz(range), shift = bits > 6 ? bits - 6 : 0;
        uint32_t *bins = S.bins[round % 2];
#pragma unroll 4
        for (uint32_t i = run.begin + lane; i < run.end; i += 64) {
            const uint32_t x = keys[i];
            if (x >= lo && x <= hi) atomicAdd(&bins[(x - lo) >> shift], 1u);
        }
        if (wave == 0) S.bins[(round + 1) % 2][lane] = 0;
        team_sync<WAVES>();
        const uint32_t mine = bins[lane];
        uint32_t upto = mine;  // keys of this part and those above it
#pragma unroll
        for (uint32_t d = 1; d < 64; d <<= 1) {
            const uint32_t o = __shfl_down(upto, d);
            if (lane + d < 64) upto += o;
        }
        const uint32_t part = 63 - __clzll(__ballot(upto >= need));
        const uint32_t inside = of_lane(static_cast<int32_t>(mine), part);
        need -= of_lane(static_cast<int32_t>(upto), part) - inside;
        B.border = lo + (part << shift);
        hi = B.border + min(hi - B.border, (1u << shift) - 1);  // (the part's end may lie past 2^32)
        team_sync<WAVES>();  // (the bins are read before they are cleared again)
        if (inside == need) break;  // all of the part: everything from its lower end on
    }
    return B;
}

// Whether lane's key x is taken; `equal` counts those equal to the border up to here.
__device__ __forceinline__ bool taken(const Border &B, uint32_t x, uint32_t &equal) {
    const uint32_t lane = threadIdx.x % 64;
    const bool same = x == B.border && x != 0;
    const uint64_t equals = __ballot(same);
    const bool take = x > B.border || (same && equal + __popcll(equals & ((1ull << lane) - 1)) < B.ties);
    equal += __popcll(equals);
    return take;
}

}  // namespace fgk

#endif
