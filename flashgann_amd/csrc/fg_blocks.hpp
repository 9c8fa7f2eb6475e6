// fg_blocks.hpp -- what the kernels over selected pages share.
#ifndef FG_BLOCKS_HPP
#define FG_BLOCKS_HPP

#include "fg_attend.hpp"

namespace fgk {

constexpr uint32_t kMostBlocks = 4096;     // of a list: what attention over them holds in LDS
constexpr uint32_t kMostTokens = 1u << 22; // of a call
constexpr uint32_t kMostItems = 1u << 23;  // tiles and lists of a call, a grid's workgroups

// A value's 16 bits as a float.
template <class T>
__device__ __forceinline__ float as_float(uint32_t bits16);
template <>
__device__ __forceinline__ float as_float<BF16>(uint32_t x) { return __uint_as_float(x << 16); }
template <>
__device__ __forceinline__ float as_float<F16>(uint32_t x) {
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(x)));
}

// The barrier that publishes LDS and nothing else: loads in flight from global memory stay
// in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Rows of q in tiles: those of request r are tiles q_starts[r] / rows + r and on, which leaves
// room for the ragged last one of each, so a call has tokens / rows + requests at most.  A tile
// of one row is that row.
struct Tile {
    int32_t request, q0, rows, pos;  // first row of q; rows (0: no such tile); position of the first
};
__device__ __forceinline__ Tile tile_of(const int32_t *q_starts, const int32_t *kv_lens, uint32_t requests, uint32_t tokens,
                                        const FastDiv &rows, uint32_t tile) {
    const uint32_t lane = threadIdx.x % 64;
    const int32_t T = static_cast<int32_t>(tokens);
    uint32_t lo = 0;  // the last request whose tiles begin at or before `tile`, by 64 guesses at a time
    for (uint32_t len = requests; len > 1;) {
        const uint32_t stride = (len + 63) / 64, guess = lane * stride;
        const bool before = guess < len && rows.div(clampi(q_starts[lo + min(guess, len - 1)], 0, T)) + (rows.d > 1 ? lo + guess : 0) <= tile;
        const uint32_t n = max(static_cast<uint32_t>(__popcll(__ballot(before))), 1u) - 1;
        lo += n * stride;
        len = min(stride, len - n * stride);
    }
    lo = uniform(lo);
    const int32_t q0 = clampi(q_starts[lo], 0, T), n = clampi(q_starts[lo + 1], q0, T) - q0;
    const int64_t row0 = (static_cast<int64_t>(tile) - static_cast<int64_t>(rows.div(q0) + (rows.d > 1 ? lo : 0))) * rows.d;
    Tile t{static_cast<int32_t>(lo), 0, 0, 0};
    if (row0 >= 0 && row0 < n) {
        t.q0 = q0 + static_cast<int32_t>(row0);
        t.rows = min(static_cast<int32_t>(rows.d), n - static_cast<int32_t>(row0));
        t.pos = max(kv_lens[lo], 0) - n + static_cast<int32_t>(row0);
    }
    t.q0 = uniform(t.q0), t.rows = uniform(t.rows), t.pos = uniform(t.pos);
    return t;
}

}  // namespace fgk

#endif
