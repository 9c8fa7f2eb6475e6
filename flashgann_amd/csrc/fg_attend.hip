// fg_attend.hip -- attention over a paged key/value cache.
//
// For a row with query q, scores s_j = scale2 * (q . k_j) of the visible tokens
// (scale2 = scale * log2 e, so that weights are powers of two), maximum m:
//   out = sum 2^(s_j - m) v_j / l,  l = sum 2^(s_j - m),  lse = ln 2 (m + log2 l)
// in one pass over the tokens: a new maximum m' multiplies what is summed so far
// by 2^(m - m').  Weights and so sums may carry a common power of two (kTopWeight), taken
// out, exactly, with the sums.  Products run on the matrix unit, transposed: S' = K Q', then
// O' = V' P', so that a query row is a lane's column in both.  Its weights leave
// the first product in the lanes where the second wants them, once the second's
// contraction takes the tokens in the order that the first leaves them, and V is
// read from LDS in that order by the transposing read.
#include "fg_attend.hpp"

namespace fgk {
namespace {

// ---------------------------------------------------------------- few rows
//
// Blocks of 16 query rows; each of the four waves takes every fourth tile of 32
// tokens and keeps a softmax of its own, joined through LDS at the end.  Bound by the
// cache's bytes, a tile being 32 x D keys and values against 16 rows: 64 single tokens
// over 500 to 16,000 (32 heads over 8, dim 128; 2.4 GB) 450 to 480 us, 5.0 to 5.3 TB/s
// where a copy reaches 4.7.  Two workgroups a CU: with four the same took 469 instead of
// 476, but one token over 131,070 41.8 instead of 36.2 (twice the parts), and registers
// for three waves a SIMD 516.  Short calls are bound by latency: lengths, table, keys,
// output one after another, 8 us for 4 tokens over 200 to 1,500, and 4 us of the join.
constexpr uint32_t kRowsUnit = 128;    // tokens a unit: one tile of each wave
constexpr uint32_t kPlaces = 1024;     // token places resolved at a time

template <class T, int D, bool FOUND>
__global__ __launch_bounds__(256, D > 128 ? 1 : 2) void fg_rows_kernel(AttendParams P) {
    using vec = typename T::vec;
    constexpr int STEPS = D / 32, DB = D / 16;
    constexpr uint32_t VROW = 2 * D + 32;  // bytes of a row of V in LDS: 16 rows' 32-byte pieces meet each bank twice
    constexpr uint32_t OROW = D + 4;       // floats of a row of O in LDS
    constexpr float UP = T::kTopWeight, DOWN = 1.0f / (1 << T::kTopWeight);  // what is added to a weight's exponent, what takes it out
    static_assert(kRows * OROW * 4 <= 32 * VROW);
    __shared__ __attribute__((aligned(16))) char vbuf[4][32 * VROW];
    __shared__ int2 place[kPlaces];
    __shared__ float wave_m[4][kRows], wave_l[4][kRows];

    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = uniform(tid / 64), col = lane % 16, quarter = lane / 16;
    const uint32_t w = blockIdx.x;
    const Start start = find_start<FOUND, kRows>(P, w);
    if (P.join && tid == 0) P.joins[w].pieces = 0;
    const uint64_t x1 = min((w + 1) * start.share, start.all);
    uint64_t before = start.before;
    uint32_t r = start.request;
    char *const vmine = vbuf[wave];

    Request rq = start.first;
    for (uint64_t x = w * start.share; x < x1;) {
        const uint64_t all = rq.weight_of(rq.blocks) * P.lists;
        if (x >= before + all) {
            before += all;
            rq = uniform_request<FOUND, kRows>(P, ++r);
            continue;
        }
        Span sp;
        const Piece pc = piece_of<FOUND, kRows>(P, rq, before, x, x1, &sp);
        if (pc.none) {
            x = x1;
            continue;
        }
        const uint32_t list = pc.list, block = pc.block;
        const int32_t t_lo = static_cast<int32_t>(pc.t_lo), t_hi = static_cast<int32_t>(pc.t_hi);
        const int32_t row0 = static_cast<int32_t>(block * kRows);

        // this lane's row: its query, and where its token stands
        const int32_t row = row0 + static_cast<int32_t>(col);
        const int32_t token = P.group.div(row);
        const int32_t pos = sp.pos0 + token;
        const bool ragged = !FOUND && P.group.div(row0) != P.group.div(min(row0 + static_cast<int32_t>(kRows), rq.rows) - 1);
        vec qv[STEPS];
        {
            const int64_t head = static_cast<int64_t>(list) * P.group.d + (row - token * static_cast<int32_t>(P.group.d));
            const char *src = P.q + (rq.q0 + static_cast<int64_t>(token)) * P.q_token + head * P.q_head + quarter * 16;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                u32x4 v = {0, 0, 0, 0};
                if (row < rq.rows) v = *reinterpret_cast<const u32x4 *>(src + 64 * s);
                qv[s] = __builtin_bit_cast(vec, v);
            }
        }
        const uint32_t kv_head = list / P.list_heads;
        const char *const kbase = P.cache.k + kv_head * P.cache.k_head + quarter * 16;
        const char *const vbase = P.cache.v + kv_head * P.cache.v_head + quarter * 16;

        float m = -INFINITY, l = 0.0f;
        f32x4 o[DB];
#pragma unroll
        for (int i = 0; i < DB; ++i) o[i] = f32x4{0, 0, 0, 0};

        for (int32_t c0 = t_lo; c0 < t_hi; c0 += kPlaces) {
            const int32_t n = min(t_hi - c0, static_cast<int32_t>(kPlaces));
            __syncthreads();
            for (int32_t i = tid; i < ((n + 31) & ~31); i += 256) {
                const int32_t t = c0 + i;
                int2 at = {-1, 0};
                if (t < min(t_hi, sp.dense)) {
                    at = place_of(P, r, position_of(sp, t));
                } else if (FOUND && t < t_hi) {
                    const int32_t k = t - sp.dense;
                    const uint32_t *ids = P.ids + (static_cast<uint64_t>(r) * P.lists + list) * P.nids;
                    const uint32_t id = ids[k];
                    const bool repeat = k > 0 && ids[k - 1] == id;
                    // (a window of the whole context or more leaves from = first: no id counts)
                    if (!repeat && id < static_cast<uint32_t>(min(sp.from, rq.limit)) && id >= static_cast<uint32_t>(sp.first))
                        at = place_of(P, r, static_cast<int32_t>(id));
                }
                place[i] = at;
            }
            __syncthreads();

            u32x4 kr[2][STEPS], vr[2][STEPS];
            bool held[2];
            const auto load = [&](int32_t tile) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int2 at = place[tile * 32 + 16 * b + col];
                    held[b] = at.x >= 0;
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
            for (int32_t tile = wave; tile * 32 < n; tile += 4) {
                // scores: register i of s[b] is token 16 b + 4 quarter + i
                f32x4 s[2];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    s[b] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < STEPS; ++k) s[b] = T::mfma16(__builtin_bit_cast(vec, kr[b][k]), qv[k], s[b]);
                }
                const uint32_t held0 = static_cast<uint32_t>(__ballot(held[0])) & 0xFFFFu;
                const uint32_t held1 = static_cast<uint32_t>(__ballot(held[1])) & 0xFFFFu;
                uint32_t odd = 0;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    bool special = false;
#pragma unroll
                    for (int k = 0; k < STEPS; ++k) {
                        // (a token without a page: whatever was read instead)
                        u32x4 v = held[b] ? vr[b][k] : u32x4{0, 0, 0, 0};
                        if (ragged && any_special<T>(v)) {
                            // 0 * inf is NaN: where not every row sees a token, infinities and NaNs
                            // are taken out of the product and added to the rows that see them
                            special = true;
                            v = finite_part<T>(v);
                        }
                        *reinterpret_cast<u32x4 *>(vmine + (16 * b + col) * VROW + 64 * k + 16 * quarter) = v;
                    }
                    if (ragged) {
                        uint64_t any = __ballot(special);
                        any |= any >> 32;
                        odd |= static_cast<uint32_t>((any | any >> 16) & 0xFFFF) << (16 * b);
                    }
                }
                if ((tile + 4) * 32 < n) load(tile + 4);

                float p[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) p[i] = s[i / 4][i % 4] * P.scale2;
                uint32_t see = ((held0 >> (4 * quarter)) & 15u) | (((held1 >> (4 * quarter)) & 15u) << 4);
                if (ragged) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int32_t j = position_of(sp, c0 + tile * 32 + 16 * (i / 4) + 4 * static_cast<int32_t>(quarter) + i % 4);
                        see &= ~(static_cast<uint32_t>(!sees(P, pos, j)) << i);
                    }
                }
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    p[i] = (see >> i) & 1u ? p[i] : -INFINITY;
                    top = fmaxf(top, p[i]);
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
                // (a tile's first: one by one, those below the last place of a long row's sum are lost)
                l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                // weights in the values' type: the matrix unit takes both alike, and
                // the rounding of a weight is that of an output element
                u32x4 pk = {T::pack(p[0], p[1]), T::pack(p[2], p[3]), T::pack(p[4], p[5]), T::pack(p[6], p[7])};
                const vec pv = __builtin_bit_cast(vec, pk);
                const char *vt = vmine + (4 * quarter + col / 4) * VROW + (col % 4) * 8;
#pragma unroll
                for (int i = 0; i < DB; ++i) {
                    const s16x4 a0 = read_transposed(vt + 32 * i), a1 = read_transposed(vt + 16 * VROW + 32 * i);
                    const s16x8 a = __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7);
                    o[i] = T::mfma16(__builtin_bit_cast(vec, a), pv, o[i]);
                }
                for (; odd; odd &= odd - 1) {
                    const int32_t at = tile * 32 + __ffs(odd) - 1;
                    const int2 where = place[at];
                    const char *src = vbase + where.x * P.cache.v_page + where.y * P.cache.v_token - quarter * 8;
                    const bool shown = sees(P, pos, position_of(sp, c0 + at));
#pragma unroll
                    for (int i = 0; i < DB; ++i) {
                        const uint2 v = *reinterpret_cast<const uint2 *>(src + 32 * i);
                        o[i][0] += shown ? special_part<T>(v.x & 0xFFFF) : 0.0f;
                        o[i][1] += shown ? special_part<T>(v.x >> 16) : 0.0f;
                        o[i][2] += shown ? special_part<T>(v.y & 0xFFFF) : 0.0f;
                        o[i][3] += shown ? special_part<T>(v.y >> 16) : 0.0f;
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
        const bool whole = pc.begins && pc.ends;
        const uint32_t slot = (2 * w + (pc.begins ? 1 : 0)) * kRows;
        l = wave_l[0][col] + wave_l[1][col] + wave_l[2][col] + wave_l[3][col];
        if (wave == 0 && quarter == 0 && row < rq.rows) {
            if (!whole)
                P.part_ml[slot + col] = float2{top, l};
            else if (P.lse)
                P.lse[(rq.q0 + static_cast<int64_t>(token)) * P.heads + list * P.group.d + (row - token * static_cast<int32_t>(P.group.d))] =
                    (top + __builtin_amdgcn_logf(l)) * kLn2;
        }
#pragma unroll
        for (uint32_t e = 0; e < kRows * D / 4; e += 256) {
            const uint32_t at = e + tid, orow = at / (D / 4), quad = at % (D / 4);
            const int32_t out_row = row0 + static_cast<int32_t>(orow);
            if ((kRows * D / 4 % 256 == 0 || at < kRows * D / 4) && out_row < rq.rows) {
                f32x4 a = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < 4; ++i) a += *reinterpret_cast<const f32x4 *>(reinterpret_cast<float *>(vbuf[i]) + orow * OROW + 4 * quad);
                if (whole) {
                    const float sum = wave_l[0][orow] + wave_l[1][orow] + wave_l[2][orow] + wave_l[3][orow];
                    a *= sum == 0.0f ? 0.0f : 1.0f / sum;
                    const int32_t t = P.group.div(out_row);
                    char *dst = P.out + (rq.q0 + static_cast<int64_t>(t)) * P.out_token +
                                static_cast<int64_t>(list * P.group.d + (out_row - t * P.group.d)) * P.out_head;
                    *reinterpret_cast<uint2 *>(dst + 8 * quad) = uint2{T::pack(a[0], a[1]), T::pack(a[2], a[3])};
                } else {
                    *reinterpret_cast<f32x4 *>(P.part + static_cast<uint64_t>(slot + orow) * D + 4 * quad) = a;
                }
            }
        }
        if (P.join && tid == 0 && pc.begins && !pc.ends)
            P.joins[w] = Join{workgroup_at(pc.end - 1, start.share) - w + 1, static_cast<uint32_t>(row0), static_cast<uint32_t>(rq.rows),
                              static_cast<uint32_t>(rq.q0), list};
        __syncthreads();
        x = min(pc.end, x1);
    }
}

// ---------------------------------------------------------------- host side

template <class T, int D, bool FOUND>
int launch(AttendParams &P, hipStream_t st) {
    hipLaunchKernelGGL((fg_rows_kernel<T, D, FOUND>), dim3(P.workgroups), dim3(256), 0, st, P);
    if (P.join) hipLaunchKernelGGL((fg_join_kernel<T, D, kRows>), dim3(kJoinWorkgroups<kRows>), dim3(256), 0, st, P);
    FG_HIP(hipGetLastError(), "attention launch");
    return FG_OK;
}

template <class T, bool FOUND>
int launch(AttendParams &P, uint32_t dim, hipStream_t st) {
    switch (dim) {
    case 64: return launch<T, 64, FOUND>(P, st);
    case 96: return launch<T, 96, FOUND>(P, st);
    case 128: return launch<T, 128, FOUND>(P, st);
    default: return launch<T, 256, FOUND>(P, st);
    }
}

// Checks the arguments and fills all of P but the workspace's addresses.
template <bool FOUND>
int prepare(const fg_kv_cache *c, const fg_attention *a, AttendParams *out) {
    AttendParams &P = *out;
    if (int rc = check_cache(c, &P.cache)) return rc;
    if (!a) return fail(FG_EINVAL, "attention arguments are NULL");
    if (a->heads < 1 || a->heads > 1024 || a->heads % c->heads_kv)
        return fail(FG_EINVAL, "heads must be a multiple of heads_kv, at most 1024");
    if (!(a->scale > 0.0f) || !std::isfinite(a->scale)) return fail(FG_EINVAL, "scale must be positive and finite");
    if (static_cast<uint64_t>(a->tokens) * a->heads > 0x7FFFFFFFull)
        return fail(FG_EINVAL, "tokens * heads must be below 2^31");
    if (a->table_width > 0x7FFFFFFFu || a->table_row < 0) return fail(FG_EINVAL, "table_width or table_row out of range");
    if (static_cast<uint64_t>(a->table_width) * c->page_size > 0x3FFFFFFFull)
        return fail(FG_EINVAL, "table_width * page_size must be below 2^30");
    if (a->sinks > 0x7FFFFFFFu) return fail(FG_EINVAL, "sinks must be below 2^31");
    if (FOUND) {
        if (a->window < 0) return fail(FG_EINVAL, "window must be >= 0");
        if (a->lists < 1 || a->heads % a->lists || a->lists % c->heads_kv)
            return fail(FG_EINVAL, "lists must be a multiple of heads_kv that divides heads");
        if (a->nids > 0x1FFFFFFFu) return fail(FG_EINVAL, "ids of a list must be below 2^29");
        if (a->requests != a->tokens) return fail(FG_EINVAL, "one query row a request");
    } else {
        if (a->window != -1 && a->window < 1) return fail(FG_EINVAL, "window must be >= 1, or -1 for none");
        if (a->lists) return fail(FG_EINVAL, "lists are for retrieved tokens");
    }
    if (a->requests > 65536) return fail(FG_EINVAL, "requests must be at most 65,536");
    if (a->requests && a->tokens &&
        (!a->q || !a->out || !a->kv_lens || (!FOUND && !a->q_starts) || (FOUND && a->nids && !a->ids) ||
         (a->table_width && !a->table)))
        return fail(FG_EINVAL, "NULL device buffer");
    if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) % 16 ||
        (a->q_token | a->q_head | a->out_token | a->out_head) % 8)
        return fail(FG_EINVAL, "q and out must be 16-byte aligned, strides multiples of 8 elements");
    P.q = static_cast<const char *>(a->q);
    P.out = static_cast<char *>(a->out);
    P.lse = a->lse;
    P.q_token = 2 * a->q_token, P.q_head = 2 * a->q_head, P.out_token = 2 * a->out_token, P.out_head = 2 * a->out_head;
    P.table = a->table;
    P.table_row = a->table_row;
    P.q_starts = a->q_starts;
    P.kv_lens = a->kv_lens;
    P.ids = a->ids;
    P.table_width = a->table_width;
    P.requests = a->requests;
    P.tokens = a->tokens;
    P.heads = a->heads;
    P.lists = FOUND ? a->lists : c->heads_kv;
    P.list_heads = P.lists / c->heads_kv;
    P.nids = FOUND ? a->nids : 0;
    P.window = static_cast<uint32_t>(a->window);
    P.sinks = a->window == -1 ? 0 : a->sinks;
    P.group = fast_div(a->heads / P.lists);
    P.scale2 = a->scale * 1.44269504088896341f;

    // What the host knows of the sizes: the table's room bounds a request's tokens.
    uint64_t seen = static_cast<uint64_t>(a->table_width) * c->page_size;
    if (a->window != -1)
        seen = std::min(seen, static_cast<uint64_t>(a->sinks) + static_cast<uint32_t>(a->window) + (kRows - 1) / P.group.d + 1);
    seen += P.nids;
    // Rows of a list: past one block the few-rows kernel reads the keys again for each,
    // the tile kernel once.  At dim 128, 8 key/value heads: 20 rows over 8 x 9,000 tokens
    // 118 us against 85; 40 rows 171 against 88.  Over short contexts the second reading
    // is from the caches and an item is cheaper: 32 rows over 64 x 100 tokens 19.8 us
    // against 22.5, 40 rows 26.5 against 23.2.
    P.tiles = !FOUND && static_cast<uint64_t>(a->max_q) * P.group.d > (seen <= 512 ? 2 * kRows : kRows);
    if (P.tiles) {
        plan_tiles(P, c->dim, seen);
        return FG_OK;
    }
    const uint64_t blocks = (static_cast<uint64_t>(a->tokens) * P.group.d + kRows - 1) / kRows + a->requests;
    const uint64_t items = std::min<uint64_t>(blocks * P.lists, 1u << 20);
    // Cutting an item of up to 512 tokens (four tiles a wave) gains less than the
    // join kernel takes: one token over 168 tokens a list, 32 lists, took 19.4 us cut
    // and 11.7 whole.  784 tokens a list, 256 lists: 28.7 cut, 31.2 whole.
    const uint32_t unit = seen <= 512 ? 512 : kRowsUnit;
    const uint64_t pieces = items * std::max<uint64_t>(1, std::min<uint64_t>((seen + unit - 1) / unit, kWorkgroups));
    P.rows = kRows;
    P.unit = fast_div(unit);
    P.join = seen > unit;
    P.workgroups = 8;
    while (P.workgroups < pieces && P.workgroups < kWorkgroups) P.workgroups *= 2;
    return FG_OK;
}

// Two parts a workgroup, their maxima and sums, and a join record each.
struct Workspace {
    uint64_t ml, joins, total;
};
Workspace workspace_of(const AttendParams &P, uint32_t dim) {
    if (!P.join) return {0, 0, 0};
    const uint64_t rows = 2ull * P.workgroups * P.rows;
    return {rows * dim * 4, rows * (dim * 4 + 8), rows * (dim * 4 + 8) + P.workgroups * sizeof(Join)};
}

template <bool FOUND>
int attend(const fg_kv_cache *c, const fg_attention *a, void *workspace, uint64_t workspace_bytes, void *stream) {
    AttendParams P{};
    if (int rc = prepare<FOUND>(c, a, &P)) return rc;
    if (a->requests == 0 || a->tokens == 0) return FG_OK;
    const Workspace ws = workspace_of(P, c->dim);
    if (ws.total && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < ws.total))
        return fail(FG_EINVAL, "workspace must be 16-byte aligned and hold " + std::to_string(ws.total) + " bytes");
    char *base = static_cast<char *>(workspace);
    P.part = reinterpret_cast<float *>(base);
    P.part_ml = reinterpret_cast<float2 *>(base + ws.ml);
    P.joins = reinterpret_cast<Join *>(base + ws.joins);
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (P.tiles) return launch_tiles(P, c->dtype, c->dim, st);
    return c->dtype == FG_BF16 ? launch<BF16, FOUND>(P, c->dim, st) : launch<F16, FOUND>(P, c->dim, st);
}

}  // namespace
}  // namespace fgk

extern "C" {

int64_t fg_attend_workspace_bytes(const fg_kv_cache *cache, const fg_attention *a) {
    return fgk::guarded<int64_t>([&]() -> int64_t {
        fgk::AttendParams P{};
        const int rc = a && a->lists ? fgk::prepare<true>(cache, a, &P) : fgk::prepare<false>(cache, a, &P);
        return rc ? rc : static_cast<int64_t>(a->requests && a->tokens ? fgk::workspace_of(P, cache->dim).total : 0);
    });
}

int fg_attend(const fg_kv_cache *cache, const fg_attention *a, void *workspace, uint64_t workspace_bytes, void *stream) {
    return fgk::guarded<int>([&] { return fgk::attend<false>(cache, a, workspace, workspace_bytes, stream); });
}

int fg_attend_retrieved(const fg_kv_cache *cache, const fg_attention *a, void *workspace, uint64_t workspace_bytes,
                        void *stream) {
    return fgk::guarded<int>([&] { return fgk::attend<true>(cache, a, workspace, workspace_bytes, stream); });
}

}  // extern "C"
