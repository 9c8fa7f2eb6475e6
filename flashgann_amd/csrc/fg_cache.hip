// fg_cache.hip -- a paged key/value cache: block tables and slot maps from
// request lengths, and new keys and values into their slots.
//
// Both are bound by their launch at the sizes of a decode step, and by the
// bytes they write at those of a long prompt.
#include "fg_cache.hpp"

namespace fgk {
namespace {

constexpr uint32_t kPlanThreads = 256;
constexpr uint32_t kPlanTokens = 1024;   // tokens of a workgroup
constexpr uint32_t kMaxRequests = 4096;  // three LDS words each, 48 KB
constexpr uint32_t kMaxLength = 0x7FFFFFFFu;  // tokens of a request: what int32 and FastDiv hold

struct PlanParams {
    const int32_t *lens, *fresh;
    int32_t *table;
    const int32_t *free_list;
    int32_t *q_starts, *kv_lens;
    int64_t *slots;
    int32_t *positions, *used;
    int64_t table_row;
    uint32_t requests, table_width, nfree, max_tokens;
    FastDiv page_size;
};

__device__ __forceinline__ uint32_t wave_scan(uint32_t v, uint32_t lane) {
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const uint32_t o = __shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// Pages of the first n tokens that the table has room for.
__device__ __forceinline__ uint32_t pages_of(const PlanParams &P, uint32_t n) {
    const uint32_t whole = P.page_size.div(n);
    return min(whole + (whole * P.page_size.d != n ? 1u : 0u), P.table_width);
}

// For each of N x: the largest r < requests with first[r] <= x; first is not
// decreasing.  The searches run side by side, an LDS read of each at a time.
template <uint32_t N>
__device__ __forceinline__ void owners(const uint32_t *first, uint32_t requests, const uint32_t (&x)[N], uint32_t (&r)[N]) {
#pragma unroll
    for (uint32_t k = 0; k < N; ++k) r[k] = 0;
    for (uint32_t step = 1u << (31 - __clz(requests)); step; step >>= 1) {
#pragma unroll
        for (uint32_t k = 0; k < N; ++k) {
            const uint32_t next = r[k] + step;
            if (next < requests && first[next] <= x[k]) r[k] = next;
        }
    }
}

// Every workgroup sums all the lengths itself (a few hundred requests are a
// microsecond), so one launch does and no workgroup waits for another: a
// token's page is either one that the request held, read from the table, or one of
// the free list at an index that the sums give.  Bound by latency: lengths, a scan, a
// search, the page (700 requests, 105,000 new tokens, 1.3 MB written: 8.8 us; 9.6 with a
// scan for every 256 requests and one search at a time).
__global__ __launch_bounds__(kPlanThreads) void fg_cache_plan_kernel(PlanParams P) {
    extern __shared__ uint32_t sums[];
    __shared__ uint32_t part[2][kPlanThreads / 64];
    uint32_t *start = sums, *base = sums + P.requests, *held = sums + 2 * P.requests;
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = tid / 64, B = P.requests;
    const uint32_t run = (B + kPlanThreads - 1) / kPlanThreads;  // consecutive requests of a thread
    uint32_t m = 0, e = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < run; ++i) {
        const uint32_t r = tid * run + i;
        if (r < B) {
            const uint32_t n = max(P.lens[r], 0), fresh = max(P.fresh[r], 0), pages = pages_of(P, n);
            start[r] = m, base[r] = e, held[r] = n;
            m += fresh;
            e += pages_of(P, min(n + fresh, kMaxLength)) - pages;
        }
    }
    const uint32_t ms = wave_scan(m, lane), es = wave_scan(e, lane);
    if (lane == 63) part[0][wave] = ms, part[1][wave] = es;
    __syncthreads();
    uint32_t mb = ms - m, eb = es - e, tokens = 0, pages = 0;
#pragma unroll
    for (uint32_t w = 0; w < kPlanThreads / 64; ++w) {
        if (w < wave) mb += part[0][w], eb += part[1][w];
        tokens += part[0][w], pages += part[1][w];
    }
    for (uint32_t i = 0; i < run; ++i) {
        const uint32_t r = tid * run + i;
        if (r < B) start[r] += mb, base[r] += eb;
    }
    __syncthreads();
    const uint32_t threads = gridDim.x * kPlanThreads, first = blockIdx.x * kPlanThreads + tid;
    for (uint32_t r = first; r < B; r += threads) {
        P.q_starts[r] = start[r];
        P.kv_lens[r] = min(held[r] + max(P.fresh[r], 0), kMaxLength);
    }
    if (first == 0) P.q_starts[B] = tokens, P.used[0] = pages;
    for (uint32_t p = first; p < pages; p += threads) {
        const uint32_t x[1] = {p};
        uint32_t r[1];
        owners(base, B, x, r);
        const uint32_t b = pages_of(P, held[r[0]]) + p - base[r[0]];
        if (b < P.table_width) P.table[r[0] * P.table_row + b] = p < P.nfree ? P.free_list[p] : -1;
    }
    constexpr uint32_t N = kPlanTokens / kPlanThreads;
    uint32_t x[N], r[N];
#pragma unroll
    for (uint32_t k = 0; k < N; ++k) x[k] = blockIdx.x * kPlanTokens + k * kPlanThreads + tid;
    owners(start, B, x, r);
#pragma unroll
    for (uint32_t k = 0; k < N; ++k) {
        if (x[k] >= P.max_tokens) break;
        int64_t slot = -1;
        uint32_t pos = 0;
        if (x[k] < tokens) {
            const uint32_t n = held[r[k]];
            pos = min(n + x[k] - start[r[k]], kMaxLength);  // (the last of them: past the end)
            const uint32_t b = P.page_size.div(pos), own = pages_of(P, n);
            if (b < P.table_width && pos < kMaxLength) {
                const uint32_t p = base[r[k]] + b - own;
                const int32_t page = b < own ? P.table[r[k] * P.table_row + b] : p < P.nfree ? P.free_list[p] : -1;
                if (page >= 0) slot = static_cast<int64_t>(page) * P.page_size.d + (pos - b * P.page_size.d);
            }
        }
        P.slots[x[k]] = slot;
        P.positions[x[k]] = pos;
    }
}

constexpr uint32_t kAppendThreads = 256;

struct AppendParams {
    CacheView cache;
    const char *k, *v;
    int64_t k_token, k_head, v_token, v_head;  // bytes
    const int64_t *slots;
    uint32_t tokens, per_block, limit;  // limit: pages * page_size
    FastDiv chunks, head_chunks;        // 16-byte pieces of a token, of a head
};

// A 16-byte piece of keys and of values a thread, neighbours in a token's row: bound by
// the bytes.  30,000 tokens of 8 x 128 (240 MB read and written) 36.6 us, 44 where
// neither is in a cache: 6.6 and 5.4 TB/s, a copy 4.7; 64 tokens 2.4 us, a launch.
__global__ __launch_bounds__(kAppendThreads) void fg_cache_append_kernel(AppendParams P) {
    const uint32_t t0 = blockIdx.x * P.per_block;
    const uint32_t n = min(P.per_block, P.tokens - t0) * P.chunks.d;
    for (uint32_t c = threadIdx.x; c < n; c += kAppendThreads) {
        const uint32_t dt = P.chunks.div(c), in = c - dt * P.chunks.d, h = P.head_chunks.div(in);
        const int64_t t = t0 + dt, off = (in - h * P.head_chunks.d) * 16u, slot = P.slots[t];
        if (slot < 0 || slot >= static_cast<int64_t>(P.limit)) continue;
        const int64_t page = P.cache.page_size.div(static_cast<uint32_t>(slot)), at = slot - page * P.cache.page_size.d;
        const uint4 k = *reinterpret_cast<const uint4 *>(P.k + t * P.k_token + h * P.k_head + off);
        const uint4 v = *reinterpret_cast<const uint4 *>(P.v + t * P.v_token + h * P.v_head + off);
        *reinterpret_cast<uint4 *>(const_cast<char *>(P.cache.k) + page * P.cache.k_page + at * P.cache.k_token +
                                   h * P.cache.k_head + off) = k;
        *reinterpret_cast<uint4 *>(const_cast<char *>(P.cache.v) + page * P.cache.v_page + at * P.cache.v_token +
                                   h * P.cache.v_head + off) = v;
    }
}

}  // namespace

int check_cache(const fg_kv_cache *c, CacheView *view) {
    if (!c) return fail(FG_EINVAL, "cache is NULL");
    if (c->dtype != FG_BF16 && c->dtype != FG_F16) return fail(FG_EINVAL, "cache dtype must be FG_BF16 or FG_F16");
    if (c->dim != 64 && c->dim != 96 && c->dim != 128 && c->dim != 256) return fail(FG_EINVAL, "dim must be 64, 96, 128 or 256");
    if (c->heads_kv < 1 || c->heads_kv > 1024) return fail(FG_EINVAL, "heads_kv must be in [1, 1024]");
    if (c->page_size < 1 || c->pages < 1 || static_cast<uint64_t>(c->pages) * c->page_size > 0x7FFFFFFFull)
        return fail(FG_EINVAL, "the cache must hold 1 to 2^31 - 1 tokens");
    if (!c->k || !c->v) return fail(FG_EINVAL, "NULL cache buffer");
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) % 16)
        return fail(FG_EINVAL, "cache buffers must be 16-byte aligned");
    if ((c->k_page | c->k_token | c->k_head | c->v_page | c->v_token | c->v_head) % 8)
        return fail(FG_EINVAL, "cache strides must be multiples of 8 elements");
    *view = {static_cast<const char *>(c->k), static_cast<const char *>(c->v),
             2 * c->k_page, 2 * c->k_token, 2 * c->k_head, 2 * c->v_page, 2 * c->v_token, 2 * c->v_head,
             c->pages, fast_div(c->page_size)};
    return FG_OK;
}

}  // namespace fgk

using namespace fgk;

extern "C" {

int fg_cache_plan(const int32_t *d_lens, const int32_t *d_new, uint32_t requests, int32_t *d_table, int64_t table_row,
                  uint32_t table_width, const int32_t *d_free, uint32_t nfree, uint32_t page_size,
                  uint32_t max_tokens, int32_t *d_q_starts, int32_t *d_kv_lens, int64_t *d_slots,
                  int32_t *d_positions, int32_t *d_used, void *stream) {
    return guarded<int>([&]() -> int {
        if (requests < 1 || requests > kMaxRequests) return fail(FG_EINVAL, "requests must be in [1, 4096]");
        if (page_size < 1 || page_size > 0x7FFFFFFFu) return fail(FG_EINVAL, "page_size must be in [1, 2^31)");
        if (max_tokens > 0x7FFFFFFFu) return fail(FG_EINVAL, "max_tokens must be below 2^31");
        if (table_width > 0x7FFFFFFFu / requests) return fail(FG_EINVAL, "requests * table_width must be below 2^31");
        if (!d_lens || !d_new || !d_q_starts || !d_kv_lens || !d_used || (table_width && !d_table) ||
            (nfree && !d_free) || (max_tokens && (!d_slots || !d_positions)))
            return fail(FG_EINVAL, "NULL device buffer");
        const PlanParams P{d_lens, d_new, d_table, d_free, d_q_starts, d_kv_lens, d_slots, d_positions, d_used,
                           table_row, requests, table_width, nfree, max_tokens, fast_div(page_size)};
        const uint32_t grid = max_tokens ? (max_tokens + kPlanTokens - 1) / kPlanTokens : 1;
        hipLaunchKernelGGL(fg_cache_plan_kernel, dim3(grid), dim3(kPlanThreads), requests * 12,
                           reinterpret_cast<hipStream_t>(stream), P);
        FG_HIP(hipGetLastError(), "cache plan launch");
        return FG_OK;
    });
}

int fg_cache_append(const fg_kv_cache *cache, const void *k, const void *v, int64_t k_token, int64_t k_head,
                    int64_t v_token, int64_t v_head, const int64_t *d_slots, uint32_t tokens, void *stream) {
    return guarded<int>([&]() -> int {
        AppendParams P;
        if (int rc = check_cache(cache, &P.cache)) return rc;
        if (tokens > 0x7FFFFFFFu) return fail(FG_EINVAL, "tokens must be below 2^31");
        if (tokens == 0) return FG_OK;
        if (!k || !v || !d_slots) return fail(FG_EINVAL, "NULL device buffer");
        if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 ||
            (k_token | k_head | v_token | v_head) % 8)
            return fail(FG_EINVAL, "keys and values must be 16-byte aligned, strides multiples of 8 elements");
        P.k = static_cast<const char *>(k);
        P.v = static_cast<const char *>(v);
        P.k_token = 2 * k_token, P.k_head = 2 * k_head, P.v_token = 2 * v_token, P.v_head = 2 * v_head;
        P.slots = d_slots;
        P.tokens = tokens;
        P.limit = cache->pages * cache->page_size;
        P.head_chunks = fast_div(cache->dim / 8);
        P.chunks = fast_div(cache->heads_kv * (cache->dim / 8));
        // one piece a thread, whole tokens a workgroup
        P.per_block = P.chunks.d >= kAppendThreads ? 1 : kAppendThreads / P.chunks.d;
        const uint32_t grid = (tokens + P.per_block - 1) / P.per_block;
        hipLaunchKernelGGL(fg_cache_append_kernel, dim3(grid), dim3(kAppendThreads), 0,
                           reinterpret_cast<hipStream_t>(stream), P);
        FG_HIP(hipGetLastError(), "cache append launch");
        return FG_OK;
    });
}

}  // extern "C"
