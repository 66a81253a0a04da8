// The attention's kernels (what they compute: hnsw_attend.hip), for one row type in each file that includes this.
#pragma once
#include "hnsw_attend.h"

namespace hnsw_amd {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWaves = 4;                 // wavefronts of a workgroup of attend_tile_kernel and attend_join_kernel
constexpr uint32_t kScanTokens = 4096;    // of one table of block entries in LDS (all tokens), and
constexpr uint32_t kListTokens = 1024;    // of one table of token entries (listed tokens)
// What meets the values' codes is a token's weight: its probability times its block's value scale, as a 16-bit float in units of 2^-11 of a
// reference that each row has for itself, the largest weight it has seen.  (A row's own: next to tokens that it does not see, or that weigh
// nothing in it, blocks of any scale leave it its precision.)  The reference is only moved when a weight is more than this above it, in base
// 2: moving it costs as much as a third of a tile (the outputs are multiplied by the change), and over random scores some row of 16 sees a new
// maximum in every second tile.  Weights are then below 2^15.9, and 16-bit floats go to 65504.
constexpr float kLead = 4.9f;
constexpr float kPScale = 2048.0f, kPScaleLog = 11.0f;
__device__ __forceinline__ float max_over_groups(float x)       // over the four lanes that share lane & 15
{
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_over_groups(float x)
{
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <class T> constexpr int kQTerms = sizeof(T) == 4 ? 2 : 1;                  // 16-bit floats that a query element is split into
template <class T> constexpr int kPTerms = std::is_same_v<T, bf16> ? 1 : 2;         // and a weight

// A value scale in base 2: -inf for 0, and finite where a scale is none (tokens that a row does not see weigh 2^-inf whatever it is).
__device__ __forceinline__ float log2_of_scale(float s) { return fminf(__builtin_amdgcn_logf(s), 128.0f); }
// log2 of a sum that is in units of 2^top (the whole parts are added first: they can be large, of opposite sign)
__device__ __forceinline__ float log2_of_sum(float top, float l)
{
    return (top + (float)__builtin_amdgcn_frexp_expf(l)) + __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(l));
}
// A value scale's inverse in units of 2^11, by which a weight gives its probability back, so that one exponential gives both: the sum of the
// probabilities is kept in units of the weights' reference, which is within 2^40 of the largest probability as long as scales are
// within 2^40 of 1.  For others (blocks of zeros among them) this is 0: from the first such block on a wavefront sums probabilities apart, in
// units of their own maximum.  (Three prompts of 900 rows over 4000 tokens: 258 us, 322 where the first block is one of zeros; single
// tokens of 64 requests 125 and 125; with a second exponential for all, before there was the inverse, 285 instead of 270.)
__device__ __forceinline__ float inverse_of_scale(float s) { return s >= 0x1p-40f && s <= 0x1p40f ? __builtin_amdgcn_rcpf(s) * (1.0f / kPScale) : 0.0f; }
// A reference that exponents are taken relative to.  Whole where weights have two terms, so that differences to scales that are powers of
// two are exact; the largest weight itself where they have one, so that this one, which can be nearly all of them, is a power of two.
template <class T> __device__ __forceinline__ float reference(float x) { return kPTerms<T> == 1 ? x : floorf(x); }

__device__ __forceinline__ f16x2 as_f16x2(uint32_t w) { return __builtin_bit_cast(f16x2, w); }

// Two signed bytes, each in the low half of a 16-bit lane of w (the high halves are 0), as 16-bit floats: with its sign bit turned a
// byte is code + 128, and 0x6400 | b is the 16-bit float 1024 + b, so 1152 less is the code, exactly.
__device__ __forceinline__ f16x2 bytes_to_f16(uint32_t w)
{
    return as_f16x2(w ^ 0x64806480u) - f16x2{(_Float16)1152.0f, (_Float16)1152.0f};
}

// Eight consecutive codes of a row as 16-bit floats (exact for both kinds of codes).  Signed bytes come out in the order
// 0 2 1 3 4 6 5 7, which the queries are laid out to match.
template <int CODES> __device__ __forceinline__ f16x8 decode8(uint32_t w0, uint32_t w1)
{
    union { f16x8 v; f16x2 h[4]; } u;
    if constexpr (CODES == HNSW_AMD_CODES_I8) {
        u.h[0] = bytes_to_f16(w0 & 0x00ff00ffu);
        u.h[1] = bytes_to_f16((w0 >> 8) & 0x00ff00ffu);
        u.h[2] = bytes_to_f16(w1 & 0x00ff00ffu);
        u.h[3] = bytes_to_f16((w1 >> 8) & 0x00ff00ffu);
    } else {
        u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, false);
        u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, 1.0f, true);
        u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, false);
        u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, 1.0f, true);
    }
    return u.v;
}
constexpr int kOrderI8[8] = {0, 2, 1, 3, 4, 6, 5, 7};

// Byte b of eight rows' words (one word of each of two times four rows), as 16-bit floats: a column of the values.
template <int CODES> __device__ __forceinline__ void decode_columns(const uint32_t (&w)[8], f16x8 (&out)[4])
{
    union U { f16x8 v; f16x2 h[4]; };
    U u[4];
    if constexpr (CODES == HNSW_AMD_CODES_I8) {
#pragma unroll
        for (int b = 0; b < 4; b++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                u[b].h[j] = bytes_to_f16(__builtin_amdgcn_perm(w[2 * j + 1], w[2 * j], 0x0c000c00u | ((4u + b) << 16) | (uint32_t)b));
    } else {
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t* x = &w[4 * half];
            const uint32_t a0 = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), a1 = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);
            const uint32_t c0 = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u), c1 = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
            const uint32_t t[4] = {__builtin_amdgcn_perm(c0, a0, 0x05040100u), __builtin_amdgcn_perm(c0, a0, 0x07060302u),
                                   __builtin_amdgcn_perm(c1, a1, 0x05040100u), __builtin_amdgcn_perm(c1, a1, 0x07060302u)};
#pragma unroll
            for (int b = 0; b < 4; b++) {
                u[b].h[2 * half] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(t[b], 1.0f, false);
                u[b].h[2 * half + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(t[b], 1.0f, true);
            }
        }
    }
#pragma unroll
    for (int b = 0; b < 4; b++) out[b] = u[b].v;
}

// Where a request's rows lie among the query rows, kept within n_rows whatever cu_q holds.
struct Span { uint32_t first, count; };
__device__ __forceinline__ Span rows_of(const AttendArgs& a, uint32_t b)
{
    if (!a.cu_q) return {b, 1};
    const int64_t lo = min(max((int64_t)a.cu_q[b], (int64_t)0), (int64_t)a.n_rows), hi = min(max((int64_t)a.cu_q[b + 1], lo), (int64_t)a.n_rows);
    return {(uint32_t)lo, (uint32_t)(hi - lo)};
}
__device__ __forceinline__ uint32_t length_of(const AttendArgs& a, int32_t len)
{
    const int64_t cap = (int64_t)a.width * a.block_tokens;
    return (uint32_t)min(max((int64_t)len, (int64_t)0), cap);
}
// r / group of a row and head (both below 2^24: a product with the reciprocal is off by one at most)
__device__ __forceinline__ uint32_t of_group(const AttendArgs& a, uint32_t r)
{
    const uint32_t q = (uint32_t)((float)r * a.group_inverse);
    const int32_t rest = (int32_t)(r - q * a.group);
    return rest < 0 ? q - 1 : rest >= (int32_t)a.group ? q + 1 : q;
}
// tokens that row i of a request's n rows sees
__device__ __forceinline__ uint32_t seen_by(const AttendArgs& a, uint32_t len, uint32_t n, uint32_t i)
{
    if (!a.causal) return len;
    const int64_t s = (int64_t)len - n + i + 1;
    return (uint32_t)min(max(s, (int64_t)0), (int64_t)len);
}

// Unit u of the rows cut into tiles of `tile` (row, head) pairs, request after request: its request, that request's rows, and the tile
// within it; false when there are fewer units.
__device__ __forceinline__ bool unit_of(const AttendArgs& a, uint32_t u, uint32_t group, uint32_t tile, uint32_t lane, uint32_t& request, Span& rows, uint32_t& part)
{
    if (!a.cu_q) {
        const uint32_t per = (group + tile - 1) / tile;
        request = u / per;
        part = u - request * per;
        rows = {request, 1};
        return request < a.n_requests;
    }
    uint32_t before = 0;
    for (uint32_t b0 = 0; b0 < a.n_requests; b0 += 64) {
        Span s{0, 0};
        if (b0 + lane < a.n_requests) s = rows_of(a, b0 + lane);
        const uint32_t n = (uint32_t)(((uint64_t)s.count * group + tile - 1) / tile), upto = wave_inclusive_sum(n);
        const unsigned long long m = __ballot(before + upto > u);
        if (m) {
            const int at = __builtin_ctzll(m);
            request = b0 + at;
            rows = {(uint32_t)__builtin_amdgcn_readlane(s.first, at), (uint32_t)__builtin_amdgcn_readlane(s.count, at)};
            part = u - before - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(n, at));
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// A query row as it lies in memory, eight elements from column col(s) on for step s (zeros behind dim, or where there is no row): the
// loads.
template <class T, int KS> struct RawQuery { Eight<T> x[KS]; };
template <class T, int KS, class Col>
__device__ __forceinline__ void load_query(const AttendArgs& a, bool there, uint32_t row, uint32_t head, uint32_t vec, Col&& col, RawQuery<T, KS>& raw)
{
    const T* x = (const T*)a.q + (int64_t)row * a.q_row_stride + (int64_t)head * a.q_head_stride;
#pragma unroll
    for (int s = 0; s < KS; s++) {
        const uint32_t c = col(s);
        raw.x[s] = Eight<T>{};
        if (there && c < a.dim) {
            if (vec) load8<T, true>(x + c, raw.x[s]);
            else load8<T, false>(x + c, raw.x[s]);
        }
    }
}
// Its operands, and what the products with codes are multiplied by to be scores in base 2.  The row is scaled by the power of two that
// puts its largest element into [2^14, 2^15).  The four lanes that share a row call this together.
template <class T, int CODES, int KS, int QT>
__device__ __forceinline__ float query_operands(const AttendArgs& a, const RawQuery<T, KS>& raw, f16x8 (&q)[KS][QT])
{
    const float sign = a.scale < 0.0f ? -1.0f : 1.0f;           // (goes into the queries, so that factors are not negative)
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
        for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(raw.x[s][j]));
    top = max_over_groups(top);
    const int e = top > 0.0f && top < __builtin_inff() ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float y = ldexpf(raw.x[s][CODES == HNSW_AMD_CODES_I8 ? kOrderI8[j] : j] * sign, e);
            const _Float16 hi = (_Float16)y;
            q[s][0][j] = hi;
            if constexpr (QT == 2) q[s][1][j] = (_Float16)(y - (float)hi);
        }
    return ldexpf(fabsf(a.scale) * kLog2e, -e);
}

// Wavefronts of a SIMD that the registers must leave room for: what hides the latency of the loads.
constexpr int rows_depth(int dp, int mt, int nw) { return dp <= 128 && mt == 1 && (dp == 64 || nw != 4) ? 2 : 1; }
constexpr int rows_waves(int dp, int mt, int nw) { return dp == 64 ? (mt == 1 ? 4 : 3) : dp == 128 && mt == 1 && rows_depth(dp, mt, nw) == 1 ? 3 : 2; }

// The arguments in scalar registers, asked for together: left to themselves they are loaded where they are used first, and every line
// of them is another wait in a chain that bounds short calls.
__device__ __forceinline__ void arguments_now(const AttendArgs& a, const Partials& parts)
{
    asm volatile("" ::"s"(a.k_codes), "s"(a.v_codes), "s"(a.k_scale), "s"(a.v_scale), "s"(a.n_blocks), "s"(a.n_heads), "s"(a.dim), "s"(a.q), "s"(a.table), "s"(a.lens),
                 "s"(a.width), "s"(a.scale), "s"(a.out), "s"(parts.chunk));
}

// Attention of few query rows over many tokens: for single tokens the codes are read once and that is the time.
//
// The workgroup takes one key head of one request (or one list), up to 16 * MT rows of queries and one chunk of the tokens; its
// NW wavefronts take tiles of 32 tokens in turn, each with a softmax of its own, and join at the end.  Scores are computed
// transposed, S^T = K Q^T, with v_mfma_f32_16x16x32_f16: the lane that then holds scores of query (lane & 15) is the one that needs
// their probabilities as the operand of O^T = V^T P^T, so that nothing is exchanged between lanes, and the softmax's maximum and
// sum are scalars of a lane.  Codes go from memory to registers as the matrix instructions want them, without LDS:
//   keys    lane (m, g): row m of 16, 16-byte pieces g, g + 4, ... (the order of the dims is free as long as the queries have it too)
//   values  lane (m, g): the same DP / 16 bytes of rows 4g .. 4g + 3 of both halves of the tile; a byte of eight rows is an operand
// and the next tile is under way while one is computed.  Codes become 16-bit floats, which hold both kinds exactly.
// Queries are scaled by a power of two to just under 2^15 and rounded to 16-bit floats (nothing is lost of bf16 and f16 but what
// lies 2^-29 under the row's largest element); 32-bit queries are split into two terms.  A block's key scale multiplies the
// scores, its value scale goes into the weights by way of their exponents.  Weights as 16-bit floats in units of 2^-11 reach down to
// 2^-35 of the row's largest: 2^-11 of each is rounded away for bf16 rows (whose outputs keep 2^-8), and a second term takes that up for
// the others.  Sums, maxima and outputs are in 32 bits.
// A workgroup's start is a chain of loads that wait for one another (length, table, codes; for lists: ids, table, codes): the first
// tile's codes are asked for as soon as the table is there, and queries and scales are made ready meanwhile.
// Measured (memory bounds the long ones, that chain the short ones; reading alone reaches 6.3 TB/s here, and this kernel 5.8 over 4.3 GB):
// 64 requests of 1 to 8192 tokens, 8 heads of 128 dims, 540 MB: 113 us and 5 of joining; 2 requests of 150000 and more, 678 MB: 126 us and 5.5;
// one request of 777 tokens, 8 heads of 64 dims: 9.6 us; lists of 100 tokens, 64 requests of 32 lists, 56 MB of single rows: 18 us, 3.1 TB/s.
template <class T, int CODES, int DP, int MT, int NW, bool FOUND>
__global__ __launch_bounds__(64 * NW, rows_waves(DP, MT, NW)) void attend_rows_kernel(AttendArgs a, Partials parts, uint32_t heads, uint32_t q_vec)
{
    constexpr int KS = DP / 32, KW = DP / 64, VW = DP / 64, VB = DP / 16, QT = kQTerms<T>, PT = kPTerms<T>, DEPTH = rows_depth(DP, MT, NW);
    constexpr uint32_t kThreads = 64 * NW, kTable = FOUND ? (NW == 1 ? 256 : kListTokens) : (NW == 1 ? 1024 : kScanTokens);      // items of a table
    constexpr uint32_t kEntries = FOUND ? kTable + kTile : kTable / 16 + 1, kMine = FOUND ? kTable / kThreads : 1;   // (one a thread of all tokens: 16 to a block at least)
    static_assert(FOUND || kTable / 16 <= kThreads);
    constexpr int kOutLd = DP + 4, kJoin = NW == 1 ? 1 : NW / 2;
    __shared__ uint32_t ent_row[kEntries];                      // first row of a block's (a token's) codes, in rows of dim bytes; ~0: of no block
    // its key scale (-1: of no block; the sign says so, a scale of -0 is made 0), its value scale in base 2, and that one's inverse
    __shared__ __align__(16) float ent_k[FOUND ? kEntries : 1], ent_v[FOUND ? kEntries : 1], ent_z[FOUND ? kEntries : 1];
    __shared__ __align__(16) float4 ent[FOUND ? 1 : kEntries];
    __shared__ __align__(16) float join[kJoin][16 * MT][kOutLd];
    __shared__ float join_m[NW][16 * MT], join_v[NW][16 * MT], join_l[NW][16 * MT];
    __shared__ uint32_t red_n[NW];

    arguments_now(a, parts);
    const uint32_t tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t head = blockIdx.x % heads, unit = blockIdx.x / heads, split = blockIdx.y;
    const uint32_t dim = a.dim, bs = a.block_tokens, bs_log = 31 - __builtin_clz(bs);
    const uint32_t group = a.group;                             // rows of a token: query heads that share this key head, or list
    const uint32_t kv = FOUND ? head / a.lists : head;

    // which rows: `first` + r / group is the query row of row r, head * group + r % group its head
    uint32_t b, first, count, r0;
    if constexpr (FOUND) {
        const uint32_t per = (group + 16 * MT - 1) / (16 * MT);
        first = unit / per;
        r0 = (unit - first * per) * 16 * MT;
        if (first >= a.n_rows) return;
        b = __builtin_amdgcn_readfirstlane(a.cu_q ? request_of(a.cu_q, a.n_requests, first) : first);
        if (b >= a.n_requests) return;
        count = 1;
    } else {
        uint32_t part;
        Span s;
        if (!unit_of(a, unit, group, 16 * MT, lane, b, s, part)) return;
        first = s.first;
        count = s.count;
        r0 = part * 16 * MT;
    }
    const uint32_t n_r = count * group;                         // (fits: n_rows * q_heads < 2^24)
    if (r0 >= n_r) return;

    // the length, the first table's block numbers (or ids) and the queries, asked for together (loads come back in order, and the queries
    // are needed last)
    const int32_t len_raw = a.lens[b];
    const uint32_t begin = split * parts.chunk;
    uint32_t early[kMine];
#pragma unroll
    for (uint32_t e = 0; e < kMine; e++) {
        early[e] = ~0u;
        if constexpr (FOUND) {
            const uint32_t i = begin + e * kThreads + tid;
            if (i < a.n_ids) early[e] = (uint32_t)a.ids[((size_t)first * heads + head) * a.n_ids + i];
        } else {
            const uint32_t i = (begin >> bs_log) + tid;
            if (tid < kEntries && i < a.width) early[e] = (uint32_t)a.table[(size_t)b * a.width + i];
        }
    }
    // the rows of this lane's columns: their queries, and what they see
    RawQuery<T, KS> raw[MT];
    uint32_t seen[MT], least, most;
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const uint32_t r = r0 + 16 * mt + m;
        const bool there = r < n_r;
        const uint32_t i = there ? of_group(a, r) : 0, h = head * group + (there ? r - i * group : 0);
        load_query<T, KS>(a, there, first + i, h, q_vec, [&](int s) { return 64 * (s / 2) + 16 * g + 8 * (s % 2); }, raw[mt]);
    }
    const uint32_t len = __builtin_amdgcn_readfirstlane(length_of(a, len_raw));
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const uint32_t r = r0 + 16 * mt + m;
        if constexpr (FOUND) {
            const Span s = rows_of(a, b);
            seen[mt] = seen_by(a, len, s.count, first - s.first);
        } else {
            seen[mt] = r < n_r ? seen_by(a, len, count, of_group(a, r)) : 0;
        }
    }
    // (rows follow one another in what they see)
    if constexpr (FOUND) {
        least = most = seen[0];
    } else {
        least = seen_by(a, len, count, of_group(a, r0));
        most = seen_by(a, len, count, of_group(a, min(r0 + 16 * MT, n_r) - 1));
    }

    const uint32_t all = FOUND ? a.n_ids : most;                // items: tokens, or list entries
    if (!FOUND && split > 0 && begin >= all) return;            // (a row that sees no token of a chunk does not ask for its part)
    const uint32_t end = split + 1 < parts.n_splits ? min(begin + parts.chunk, all) : all;

    f16x8 q[MT][KS][QT];
    float factor[MT];                                           // of the products: scores in base 2
    f32x4 o[MT][VB];
    // references of the weights, and of the sums of probabilities, which are the weights' up to the first unusual scale
    float top_v[MT], top[MT], sum[MT];
    bool far = false;                                           // there has been one
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        top[mt] = top_v[mt] = -__builtin_inff();
        sum[mt] = 0.0f;
#pragma unroll
        for (int i = 0; i < VB; i++) o[mt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    u32x4 tk[DEPTH][2][KW];                                     // tiles' codes, keys and values
    uint32_t tv[DEPTH][8][VW];
    uint32_t c0 = begin, c1 = 0, n = 0, e0 = 0, safe = 0;       // the table: items c0 .. c1, n of them; its first block; a row of codes of a live token
    uint32_t bh[kMine], at[kMine];                              // (block, head) of this thread's entries, ~0: of none, and their places

    // Entries c0 .. c1 but for the scales; false where there is nothing in them.
    auto open_table = [&]() {
        c1 = min(end - c0, kTable) + c0;
        n = c1 - c0;
        if constexpr (FOUND) {
            // listed tokens that the row sees and that exist, moved together (in order): entries, then 32 or less that weigh nothing
            const int32_t* ids = a.ids + ((size_t)first * heads + head) * a.n_ids;
            uint32_t id[kMine], kept = 0;
#pragma unroll
            for (uint32_t e = 0; e < kMine; e++) id[e] = e * kThreads + tid >= n ? ~0u : c0 == begin ? early[e] : (uint32_t)ids[c0 + e * kThreads + tid];
#pragma unroll
            for (uint32_t e = 0; e < kMine; e++) {
                const uint32_t blk = id[e] < seen[0] ? (uint32_t)a.table[(size_t)b * a.width + (id[e] >> bs_log)] : ~0u;
                bh[e] = blk < a.n_blocks ? blk * a.n_heads + kv : ~0u;
            }
#pragma unroll
            for (uint32_t e = 0; e < kMine; e++) {
                if (e * kThreads >= n) break;
                const unsigned long long mine = __ballot(bh[e] != ~0u);
                if (e) __syncthreads();
                if (lane == 0) red_n[wave] = (uint32_t)__popcll(mine);
                __syncthreads();
                at[e] = kept + (uint32_t)__popcll(mine & ((1ull << lane) - 1));
                for (uint32_t w = 0; w < NW; w++) {
                    if (w < wave) at[e] += red_n[w];
                    kept += red_n[w];
                }
                if (bh[e] != ~0u) ent_row[at[e]] = (bh[e] << bs_log) + (id[e] & (bs - 1));
            }
            n = __builtin_amdgcn_readfirstlane(kept);
            if (n == 0) return false;
            __syncthreads();
            if (tid < kTile) { ent_row[n + tid] = ent_row[n - 1]; ent_k[n + tid] = 0.0f; ent_v[n + tid] = -__builtin_inff(); ent_z[n + tid] = 1.0f; }
            __syncthreads();
            return true;
        } else {
            e0 = c0 >> bs_log;
            const bool mine = tid <= ((c1 - 1) >> bs_log) - e0;
            const uint32_t blk = !mine ? ~0u : c0 == begin ? early[0] : (uint32_t)a.table[(size_t)b * a.width + e0 + tid];
            bh[0] = blk < a.n_blocks ? blk * a.n_heads + kv : ~0u;
            if (mine) ent_row[tid] = bh[0] == ~0u ? ~0u : bh[0] << bs_log;
            const unsigned long long fine = __ballot(bh[0] != ~0u);
            const uint32_t live = fine ? (__builtin_amdgcn_readlane(bh[0], __builtin_ctzll(fine)) << bs_log) + 1 : 0;    // (all lanes take part)
            if (lane == 0) red_n[wave] = live;
            __syncthreads();
            safe = 0;
#pragma unroll
            for (int w = 0; w < NW; w++) safe = safe ? safe : red_n[w];
            safe = __builtin_amdgcn_readfirstlane(safe);
            return safe-- != 0;
        }
    };
    // Where tile j's codes are: of all tokens, the two runs of 16 lie in a block each (tokens behind the last one are the last one).
    struct Where { uint64_t at[2]; uint32_t limit[2]; };
    auto locate = [&](uint32_t j) {
        Where w{};
        if constexpr (!FOUND) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t start = min(c0 + 32 * j + 16 * h, c1 - 1);
                const uint32_t base = __builtin_amdgcn_readfirstlane(ent_row[(start >> bs_log) - e0]);
                // (no block: one live token over and over; stale codes can be NaN, which a weight of 0 would not remove)
                w.at[h] = (uint64_t)(base == ~0u ? safe : base + (start & (bs - 1))) * dim;
                w.limit[h] = base == ~0u ? 0u : min(c1 - 1 - start, 15u);
            }
        }
        return w;
    };
    auto fetch_keys = [&](auto buf, uint32_t j, const Where& w) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint8_t* p = a.k_codes;
            uint32_t off = 0;
            if constexpr (FOUND) {
                p += (uint64_t)ent_row[32 * j + 16 * h + m] * dim;
            } else {
                p += w.at[h];
                off = (w.limit[h] == 15 ? m : min(m, w.limit[h])) * dim;
            }
#pragma unroll
            for (int i = 0; i < KW; i++) {
                const uint32_t c = 64 * i + 16 * g;
                tk[buf.value][h][i] = *reinterpret_cast<const u32x4*>(p + off + (c < dim ? c : 0));
            }
        }
    };
    auto fetch_values = [&](auto buf, uint32_t j, const Where& w) {
        const uint32_t c = VB * m;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const uint8_t* p = a.v_codes;
                uint32_t off = 0;
                if constexpr (FOUND) {
                    p += (uint64_t)ent_row[32 * j + 16 * h + 4 * g + r] * dim;
                } else if (w.limit[h] == 15) {
                    p += w.at[h] + (uint64_t)r * dim;
                    off = 4 * g * dim;
                } else {
                    p += w.at[h];
                    off = min(4 * g + r, w.limit[h]) * dim;
                }
                if constexpr (VW == 2) {
                    const u32x2 x = *reinterpret_cast<const u32x2*>(p + off + (c < dim ? c : 0));
                    tv[buf.value][4 * h + r][0] = x[0]; tv[buf.value][4 * h + r][1] = x[1];
                } else if constexpr (VW == 4) {
                    const u32x4 x = *reinterpret_cast<const u32x4*>(p + off + (c < dim ? c : 0));
#pragma unroll
                    for (int i = 0; i < 4; i++) tv[buf.value][4 * h + r][i] = x[i];
                } else {                                        // (a lane's bytes can end with the row in their middle)
#pragma unroll
                    for (int i = 0; i < VW; i++) tv[buf.value][4 * h + r][i] = *reinterpret_cast<const uint32_t*>(p + off + (c + 4 * i < dim ? c + 4 * i : 0));
                }
            }
    };

    auto first_tiles = [&]() {
        auto one = [&](auto buf) {
            const uint32_t j = wave + buf.value * NW;
            if (32 * j < n) {
                const Where w = locate(j);
                fetch_keys(buf, j, w);
                fetch_values(buf, j, w);
            }
        };
        one(std::integral_constant<int, 0>{});
        if constexpr (DEPTH == 2) one(std::integral_constant<int, 1>{});
    };
    bool some = begin < end && open_table();                    // (the same in all threads)
    if (some) first_tiles();
#pragma unroll
    for (int mt = 0; mt < MT; mt++) factor[mt] = query_operands<T, CODES, KS, QT>(a, raw[mt], q[mt]);
    while (c0 < end) {
        if (some) {
            // the entries' scales
#pragma unroll
            for (uint32_t e = 0; e < kMine; e++) {
                if constexpr (FOUND) {
                    if (bh[e] != ~0u) {
                        const float sv = a.v_scale[bh[e]];
                        ent_k[at[e]] = a.k_scale[bh[e]];
                        ent_v[at[e]] = log2_of_scale(sv);
                        ent_z[at[e]] = inverse_of_scale(sv);
                    }
                } else if (tid <= ((c1 - 1) >> bs_log) - e0) {
                    const float sv = bh[0] != ~0u ? a.v_scale[bh[0]] : 1.0f;
                    ent[tid] = make_float4(bh[0] != ~0u ? a.k_scale[bh[0]] + 0.0f : -1.0f, log2_of_scale(sv), inverse_of_scale(sv), 0.0f);
                }
            }
            __syncthreads();

            auto take = [&](auto buf, uint32_t j) {
                const uint32_t i0 = 32 * j, ahead = j + DEPTH * NW;
                const bool more = 32 * ahead < n;
                f32x4 s[MT][2];
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int ks = 0; ks < KS; ks++) {
                        const f16x8 k = decode8<CODES>(tk[buf.value][h][ks / 2][2 * (ks % 2)], tk[buf.value][h][ks / 2][2 * (ks % 2) + 1]);
#pragma unroll
                        for (int mt = 0; mt < MT; mt++)
#pragma unroll
                            for (int qt = 0; qt < QT; qt++)
                                s[mt][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[mt][ks][qt], ks + qt ? s[mt][h] : f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
                    }
                // the keys' registers are free: a later tile's keys are under way while this one's weights meet its values
                Where next{};
                if (more) {
                    next = locate(ahead);
                    fetch_keys(buf, ahead, next);
                }
                float fk[2][4], lv[2][4], inverse[2][4];        // the scales of this lane's tokens 4g + r of both halves
                bool gone[2] = {false, false}, ragged, odd = false;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if constexpr (FOUND) {
                        const float4 x = *reinterpret_cast<const float4*>(&ent_k[i0 + 16 * h + 4 * g]), y = *reinterpret_cast<const float4*>(&ent_v[i0 + 16 * h + 4 * g]),
                                     z = *reinterpret_cast<const float4*>(&ent_z[i0 + 16 * h + 4 * g]);
                        fk[h][0] = x.x; fk[h][1] = x.y; fk[h][2] = x.z; fk[h][3] = x.w;
                        lv[h][0] = y.x; lv[h][1] = y.y; lv[h][2] = y.z; lv[h][3] = y.w;
                        inverse[h][0] = z.x; inverse[h][1] = z.y; inverse[h][2] = z.z; inverse[h][3] = z.w;
                        odd |= __ballot(fminf(fminf(z.x, z.y), fminf(z.z, z.w)) == 0.0f) != 0;
                    } else {
                        const uint32_t e = (min(c0 + i0 + 16 * h, c1 - 1) >> bs_log) - e0;
                        const float4 x = ent[e];
#pragma unroll
                        for (int r = 0; r < 4; r++) { fk[h][r] = x.x; lv[h][r] = x.y; inverse[h][r] = x.z; }
                        gone[h] = __builtin_amdgcn_readfirstlane(__float_as_uint(x.x)) >> 31;
                        odd |= __builtin_amdgcn_readfirstlane(__float_as_uint(x.z)) == 0;
                    }
                }
                const bool was_far = far;
                far = far || odd;
                if constexpr (FOUND) ragged = i0 + 32 > n;
                else ragged = c0 + i0 + 32 > least || c0 + i0 + 32 > c1 || gone[0] || gone[1];
                f16x8 p[MT][PT];
#pragma unroll
                for (int mt = 0; mt < MT; mt++) {
                    float x[2][4], local = -__builtin_inff();
#pragma unroll
                    for (int h = 0; h < 2; h++)
#pragma unroll
                        for (int r = 0; r < 4; r++) x[h][r] = s[mt][h][r] * (fk[h][r] * factor[mt]);
                    if (ragged) {
                        const int left = (int)((FOUND ? n : min(seen[mt], c1) - c0) - i0 - 4 * g);
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int r = 0; r < 4; r++) x[h][r] = 16 * h + r < left && !gone[h] ? x[h][r] : -__builtin_inff();
                    }
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if constexpr (FOUND) {
#pragma unroll
                            for (int r = 0; r < 4; r++) local = fmaxf(local, x[h][r] + lv[h][r]);
                        } else {
                            local = fmaxf(local, fmaxf(fmaxf(x[h][0], x[h][1]), fmaxf(x[h][2], x[h][3])) + lv[h][0]);
                        }
                    }
                    if (far || __ballot(local > top_v[mt] + kLead)) {          // rare after the first tile, but for unusual scales
                        const float before = top_v[mt], now = fmaxf(before, reference<T>(max_over_groups(local)));
                        const float shrink = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(before - now);
                        top_v[mt] = now;
#pragma unroll
                        for (int i = 0; i < VB; i++) o[mt][i] *= shrink;
                        if (!far) {
                            sum[mt] *= shrink;
                        } else {                                // the sum by itself
                            if (!was_far) top[mt] = before;
#pragma unroll
                            for (int i = 0; i < 8; i++) inverse[i / 4][i % 4] = 0.0f;
                            float most_x = -__builtin_inff();
#pragma unroll
                            for (int i = 0; i < 8; i++) most_x = fmaxf(most_x, x[i / 4][i % 4]);
                            const float now_x = fmaxf(top[mt], reference<T>(max_over_groups(most_x))), ref = now_x == -__builtin_inff() ? 0.0f : now_x;
                            sum[mt] *= __builtin_amdgcn_exp2f(top[mt] - ref);
                            top[mt] = now_x;
#pragma unroll
                            for (int i = 0; i < 8; i++) sum[mt] += __builtin_amdgcn_exp2f(x[i / 4][i % 4] - ref);
                        }
                    }
                    // (the factor of 2^11 in the exponent costs bits of it, which 32-bit rows keep)
                    constexpr bool kApart = sizeof(T) == 4;
                    const float ref = (top_v[mt] == -__builtin_inff() ? 0.0f : top_v[mt]) - (kApart ? 0.0f : kPScaleLog);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float part_sum = 0.0f;
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const float w = __builtin_amdgcn_exp2f(x[h][r] + (lv[h][r] - ref)) * (kApart ? kPScale : 1.0f);
                            part_sum = FOUND ? __builtin_fmaf(w, inverse[h][r], part_sum) : part_sum + w;
                            const _Float16 hi = (_Float16)w;
                            p[mt][0][4 * h + r] = hi;
                            if constexpr (PT == 2) p[mt][1][4 * h + r] = (_Float16)(w - (float)hi);
                        }
                        sum[mt] = FOUND ? sum[mt] + part_sum : __builtin_fmaf(part_sum, inverse[h][0], sum[mt]);
                    }
                }
#pragma unroll
                for (int i = 0; i < VW; i++) {
                    uint32_t w[8];
                    f16x8 v[4];
#pragma unroll
                    for (int r = 0; r < 8; r++) w[r] = tv[buf.value][r][i];
                    decode_columns<CODES>(w, v);
#pragma unroll
                    for (int c = 0; c < 4; c++)
#pragma unroll
                        for (int mt = 0; mt < MT; mt++)
#pragma unroll
                            for (int pt = 0; pt < PT; pt++) o[mt][4 * i + c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[c], p[mt][pt], o[mt][4 * i + c], 0, 0, 0);
                }
                if (more) fetch_values(buf, ahead, next);
            };
            for (uint32_t j = wave; 32 * j < n; j += DEPTH * NW) {
                take(std::integral_constant<int, 0>{}, j);
                if constexpr (DEPTH == 2) {
                    if (32 * (j + NW) >= n) break;
                    take(std::integral_constant<int, 1>{}, j + NW);
                }
            }
        }
        c0 += kTable;
        if (c0 >= end) break;
        __syncthreads();                                        // the table's last readers are done
        some = open_table();
        if (some) first_tiles();
    }

    // the wavefronts' softmaxes become one
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        if (!far) top[mt] = top_v[mt];
        sum[mt] = sum_over_groups(sum[mt]);
        if (g == 0) { join_m[wave][16 * mt + m] = top[mt]; join_v[wave][16 * mt + m] = top_v[mt]; join_l[wave][16 * mt + m] = sum[mt]; }
    }
    __syncthreads();
    auto top_of = [&](const float (&tops)[NW][16 * MT], uint32_t r) {
        float x = tops[0][r];
#pragma unroll
        for (int w = 1; w < NW; w++) x = fmaxf(x, tops[w][r]);
        return x;
    };
    auto ref_of = [&](const float (&tops)[NW][16 * MT], uint32_t r) { const float x = top_of(tops, r); return x == -__builtin_inff() ? 0.0f : x; };
    auto put = [&](bool add) {
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const float f = __builtin_amdgcn_exp2f(top_v[mt] - ref_of(join_v, 16 * mt + m));
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int i = 0; i < VB; i += 4) {
                    float4* to = reinterpret_cast<float4*>(&join[wave % kJoin][16 * mt + m][(4 * g + r) * VB + i]);
                    float4 x = make_float4(o[mt][i][r] * f, o[mt][i + 1][r] * f, o[mt][i + 2][r] * f, o[mt][i + 3][r] * f);
                    if (add) { const float4 y = *to; x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w); }
                    *to = x;
                }
        }
    };
    if (wave >= kJoin || NW == 1) put(false);
    __syncthreads();
    if constexpr (NW > 1) {
        if (wave < kJoin) put(true);
        __syncthreads();
    }
    auto joined = [&](uint32_t r, uint32_t d) {
        float x = join[0][r][d];
#pragma unroll
        for (int w = 1; w < kJoin; w++) x += join[w][r][d];
        return x;
    };
    for (uint32_t r = wave; r < 16 * MT && r0 + r < n_r; r += NW) {
        const uint32_t i = of_group(a, r0 + r);
        const size_t to = (size_t)(first + i) * a.q_heads + head * group + (r0 + r - i * group);
        const float ref = ref_of(join_m, r), ref_v = top_of(join_v, r);          // (the latter -inf: all scales are 0, and the outputs)
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) l += join_l[w][r] * __builtin_amdgcn_exp2f(join_m[w][r] - ref);
        const float inv = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(ref_v - ref - kPScaleLog) / l;
        if (parts.n_splits == 1) {
            for (uint32_t d = lane; d < dim; d += 64) ((T*)a.out)[to * dim + d] = from_float<T>(joined(r, d) * inv);
            if (lane == 0 && a.lse) a.lse[to] = l == 0.0f ? -__builtin_inff() : log2_of_sum(ref, l) * 0.6931471805599453f;
        } else {
            const size_t at = to * parts.n_splits + split;
            for (uint32_t d = lane; d < dim; d += 64) parts.out[at * dim + d] = joined(r, d) * inv;
            if (lane == 0) parts.lse[at] = l == 0.0f ? -__builtin_inff() : log2_of_sum(ref, l);
        }
    }
}

// Attention of many query rows: prompts.  The codes of 64 tokens become 16-bit floats once for all 64 * MT rows of the workgroup: in
// LDS, keys [token][dim] (rows of an odd number of 16-byte pieces, so that operands are read without bank conflicts), values
// [dim][token] (the eight tokens of a matrix operand next to each other, the pieces of a row in an order that differs by row to
// the same end), while the next tile's codes are on their way to registers: each wavefront moves the keys of 16 tokens and a quarter
// of the values' octets, so that the blocks they lie in are scalars.
// HALVES = 2: twice the wavefronts, which take the tiles in turn and join at the end: half the steps of one after the other where
// workgroups are too few to hide them.  (Up to 64 dims, where two such workgroups fit a compute unit: 163 rows each of eight requests over
// 1000 tokens, 16 heads: 34.3 us, 37.4 without.  At 128 dims only one fits: with more than 256 workgroups the rounds cost more than the steps, 300 rows
// each of four requests over 700 tokens 43.8 -> 51.3; with fewer they would win, 35 -> 30, which no rule here takes.)
// Each wavefront has 16 * MT rows and their softmax to itself.  The arithmetic is that of attend_rows_kernel.
// What bounds it: per tile and wavefront 371 vector instructions (by the counters, starts included; 32 of them are exponentials; 1870 cycles of issue)
// and 64 matrix instructions (1020 cycles), of which the registers leave room for two wavefronts a SIMD to overlap.  Three prompts of 900 rows
// over 4000 tokens, 32 query heads of 128 dims, 156 GFLOP: 275 us, 566 TFLOP/s, the vector units busy 43 % of it and the matrix units 23 %: neither is
// the limit, but that the two overlap little, and that 688 workgroups on 512 places leave some compute units three to do and others two.
template <class T, int CODES, int DP, int MT, int NBUF, int HALVES>
__global__ __launch_bounds__(256 * HALVES, HALVES == 2 ? 4 : 2) void attend_tile_kernel(AttendArgs a, Partials parts, uint32_t q_vec)
{
    constexpr int KS = DP / 32, DT = DP / 16, QT = kQTerms<T>, PT = kPTerms<T>;
    constexpr int kTokens = 64, kKeyLd = DP + 8;                 // 16-bit elements
    constexpr int KL = DP / 64, VL = (DP + 127) / 128;          // 16-byte pieces of keys, and words x 8 tokens of values, that a thread moves
    constexpr uint32_t kEntries = kScanTokens / 16 + 1;
    static_assert(kScanTokens / 16 <= 256 && (HALVES == 1 || NBUF == 2));
    constexpr int kAll = kWaves * HALVES;                       // wavefronts
    __shared__ uint32_t ent_row[kEntries], some[kAll];        // first row of a block's codes, in rows of dim bytes; ~0: of no block
    __shared__ __align__(16) float4 ent[kEntries];              // key scale (-1: there is no block), value scale in base 2, its inverse
    __shared__ __align__(16) _Float16 keys[NBUF * HALVES][kTokens * kKeyLd];
    __shared__ __align__(16) _Float16 vals[NBUF * HALVES][DP * kTokens];
    auto val_at = [](uint32_t d, uint32_t oct) { return d * kTokens + 8 * (oct ^ ((d >> 1) & 7)); };

    arguments_now(a, parts);
    const uint32_t tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
    const uint32_t of_all = __builtin_amdgcn_readfirstlane(tid >> 6), wave = of_all % kWaves, half = of_all / kWaves;
    const uint32_t kv = blockIdx.x % a.n_heads, split = blockIdx.y;
    const uint32_t unit = gridDim.x / a.n_heads - 1 - blockIdx.x / a.n_heads;   // the last rows of a prompt see the most: first
    const uint32_t dim = a.dim, bs = a.block_tokens, bs_log = 31 - __builtin_clz(bs);
    const uint32_t group = a.group;
    constexpr uint32_t kRows = kWaves * 16 * MT;
    uint32_t b, part;
    Span rows;
    if (!unit_of(a, unit, group, kRows, lane, b, rows, part)) return;
    const uint32_t n_r = rows.count * group, r0 = part * kRows + wave * 16 * MT;
    // the length, the first table's block numbers and the queries, asked for together (loads come back in order, and the queries are
    // needed last)
    const int32_t len_raw = a.lens[b];
    const uint32_t begin = split * parts.chunk, e_begin = begin >> bs_log;
    const uint32_t early = tid < kEntries && e_begin + tid < a.width ? (uint32_t)a.table[(size_t)b * a.width + e_begin + tid] : ~0u;
    RawQuery<T, KS> raw[MT];
    uint32_t seen[MT];
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const uint32_t r = r0 + 16 * mt + m;
        const bool there = r < n_r;
        const uint32_t i = there ? of_group(a, r) : 0, h = kv * group + (there ? r - i * group : 0);
        seen[mt] = i;
        load_query<T, KS>(a, there, rows.first + i, h, q_vec, [&](int s) { return 32 * s + 8 * g; }, raw[mt]);
    }
    const uint32_t len = __builtin_amdgcn_readfirstlane(length_of(a, len_raw));
#pragma unroll
    for (int mt = 0; mt < MT; mt++) seen[mt] = r0 + 16 * mt + m < n_r ? seen_by(a, len, rows.count, seen[mt]) : 0;
    // (rows follow one another in what they see; a wavefront without rows sees nothing)
    const uint32_t least = r0 < n_r ? seen_by(a, len, rows.count, of_group(a, r0)) : 0;
    const uint32_t most = r0 < n_r ? seen_by(a, len, rows.count, of_group(a, min(r0 + 16 * MT, n_r) - 1)) : 0;
    // what the workgroup's last row sees
    const uint32_t last_r = min((part + 1) * kRows, n_r) - 1;
    const uint32_t all = seen_by(a, len, rows.count, of_group(a, last_r));
    if (split > 0 && begin >= all) return;
    const uint32_t end = split + 1 < parts.n_splits ? min(begin + parts.chunk, all) : all;

    f16x8 q[MT][KS][QT];
    float factor[MT];
    f32x4 o[MT][DT];
    float top_v[MT], top[MT], sum[MT];                          // (as in attend_rows_kernel)
    bool far = false;
#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        top[mt] = top_v[mt] = -__builtin_inff();
        sum[mt] = 0.0f;
#pragma unroll
        for (int i = 0; i < DT; i++) o[mt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // the table: tokens c0 .. c1, its first block, a row of codes of a live token, (block, head) of this thread's entry (~0: of none)
    uint32_t c0 = begin, c1 = 0, e0 = 0, safe = 0, bh = ~0u;
    u32x4 kr[KL];
    uint32_t vr[VL][8];
    const uint32_t k_row = lane >> 2, oct = 2 * wave + (lane >> 5), v_row = 4 * (oct & 3), v_word = lane & 31;
    uint32_t k_off[KL], v_off[VL];                              // of a whole tile's codes
#pragma unroll
    for (int i = 0; i < KL; i++) k_off[i] = k_row * dim + (64 * i + 16 * (lane & 3) < dim ? 64 * i + 16 * (lane & 3) : 0);
#pragma unroll
    for (int i = 0; i < VL; i++) v_off[i] = v_row * dim + (4 * (v_word + 32 * i) < dim ? 4 * (v_word + 32 * i) : 0);
    // The next tile's codes: this wavefront's keys are 16 tokens of one block, its values the octets of two runs of 16 tokens.  (Tokens
    // behind the last one are the last one; those of no block are one live token over and over: stale codes can be NaN, which a weight
    // of 0 would not remove.)
    auto fetch = [&](uint32_t t0) {
        const uint32_t last = c1 - 1, kt = min(t0 + 16 * wave, last), vt0 = min(t0 + 32 * (wave >> 1), last), vt1 = min(t0 + 32 * (wave >> 1) + 16, last);
        uint32_t ek = ent_row[(kt >> bs_log) - e0], ev0 = ent_row[(vt0 >> bs_log) - e0], ev1 = ent_row[(vt1 >> bs_log) - e0];
        ek = __builtin_amdgcn_readfirstlane(ek);
        ev0 = __builtin_amdgcn_readfirstlane(ev0);
        ev1 = __builtin_amdgcn_readfirstlane(ev1);
        auto codes_at = [&](const uint8_t* codes, uint32_t base, uint32_t pos) {
            return codes + (uint64_t)(base == ~0u ? safe : base + (pos & (bs - 1))) * dim;
        };
        const uint8_t *kb = codes_at(a.k_codes, ek, kt), *vb0 = codes_at(a.v_codes, ev0, vt0), *vb1 = codes_at(a.v_codes, ev1, vt1);
        if (t0 + kTokens <= c1 && ek != ~0u && ev0 != ~0u && ev1 != ~0u) {
#pragma unroll
            for (int i = 0; i < KL; i++) kr[i] = *reinterpret_cast<const u32x4*>(kb + k_off[i]);
#pragma unroll
            for (int i = 0; i < VL; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    vr[i][r] = *reinterpret_cast<const uint32_t*>(vb0 + (size_t)r * dim + v_off[i]);
                    vr[i][4 + r] = *reinterpret_cast<const uint32_t*>(vb1 + (size_t)r * dim + v_off[i]);
                }
        } else {
            const uint32_t k_back = k_row - min(k_row, ek == ~0u ? 0u : last - kt);                 // rows that are not there
            const uint32_t v_left0 = ev0 == ~0u ? 0u : last - vt0, v_left1 = ev1 == ~0u ? 0u : last - vt1;
#pragma unroll
            for (int i = 0; i < KL; i++) kr[i] = *reinterpret_cast<const u32x4*>(kb + (k_off[i] - k_back * dim));
#pragma unroll
            for (int i = 0; i < VL; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const uint32_t row = v_row + r;
                    vr[i][r] = *reinterpret_cast<const uint32_t*>(vb0 + (v_off[i] - v_row * dim + min(row, v_left0) * dim));
                    vr[i][4 + r] = *reinterpret_cast<const uint32_t*>(vb1 + (v_off[i] - v_row * dim + min(row, v_left1) * dim));
                }
        }
    };
    // the codes in registers become 16-bit floats in LDS, piece by piece: eight of a row of keys, or eight of a column of values
    constexpr int kPieces = 2 * KL + 4 * VL;
    auto store_piece = [&](int buf, int j) {
        if (j < 2 * KL) {
            const int i = j / 2, half = j % 2;
            *reinterpret_cast<f16x8*>(&keys[buf][(16 * wave + k_row) * kKeyLd + 64 * i + 16 * (lane & 3) + 8 * half]) = decode8<CODES>(kr[i][2 * half], kr[i][2 * half + 1]);
        } else {
            const int i = (j - 2 * KL) / 4, col = (j - 2 * KL) % 4;
            const uint32_t c = 4 * (v_word + 32 * i);
            f16x8 v[4];
            decode_columns<CODES>(vr[i], v);
            if (DP % 128 == 0 || c < DP) *reinterpret_cast<f16x8*>(&vals[buf][val_at(c + col, oct)]) = v[col];
        }
    };
    auto store = [&](int buf) {
#pragma unroll
        for (int j = 0; j < kPieces; j++) store_piece(buf, j);
    };
    auto compute = [&](uint32_t t0, int buf, int other) {
        if (t0 >= most || (HALVES == 2 && t0 >= c1)) {                                   // none of this wavefront's rows sees the tile
            if constexpr (NBUF == 2) store(other);
            return;
        }
        float4 x[4];
#pragma unroll
        for (int t = 0; t < 4; t++) x[t] = ent[(min(t0 + 16 * t, c1 - 1) >> bs_log) - e0];
        f32x4 s[MT][4];
#pragma unroll
        for (int ks = 0; ks < KS; ks++)
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const f16x8 k = *reinterpret_cast<const f16x8*>(&keys[buf][(16 * t + m) * kKeyLd + 32 * ks + 8 * g]);
#pragma unroll
                for (int mt = 0; mt < MT; mt++)
#pragma unroll
                    for (int qt = 0; qt < QT; qt++)
                        s[mt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[mt][ks][qt], ks + qt ? s[mt][t] : f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            }
        bool gone[4], any_gone = false, odd = false;
#pragma unroll
        for (int t = 0; t < 4; t++) {
            gone[t] = __builtin_amdgcn_readfirstlane(__float_as_uint(x[t].x)) >> 31;
            any_gone |= gone[t];
            odd |= __builtin_amdgcn_readfirstlane(__float_as_uint(x[t].z)) == 0;
        }
        const bool was_far = far;
        far = far || odd;
        const bool ragged = t0 + kTokens > least || t0 + kTokens > c1 || any_gone;
        float f[MT][4], ref[MT];
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            float local = -__builtin_inff();
            if (ragged) {
                const int left = (int)(min(seen[mt], c1) - t0 - 4 * g);         // (both are below 2^31)
#pragma unroll
                for (int t = 0; t < 4; t++)
#pragma unroll
                    for (int r = 0; r < 4; r++) s[mt][t][r] = 16 * t + r < left && !gone[t] ? s[mt][t][r] : -__builtin_inff();
            }
#pragma unroll
            for (int t = 0; t < 4; t++) {
                f[mt][t] = fmaxf(x[t].x * factor[mt], 0x1p-126f);               // (not 0, which masked scores would make NaN)
                const float most_s = fmaxf(fmaxf(s[mt][t][0], s[mt][t][1]), fmaxf(s[mt][t][2], s[mt][t][3]));
                local = fmaxf(local, __builtin_fmaf(f[mt][t], most_s, x[t].y));
            }
            if (far || __ballot(local > top_v[mt] + kLead)) {
                const float before = top_v[mt], now = fmaxf(before, reference<T>(max_over_groups(local)));
                const float shrink = now == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(before - now);
                top_v[mt] = now;
#pragma unroll
                for (int i = 0; i < DT; i++) o[mt][i] *= shrink;
                if (!far) {
                    sum[mt] *= shrink;
                } else {                                        // the sum by itself
                    if (!was_far) top[mt] = before;
#pragma unroll
                    for (int t = 0; t < 4; t++) x[t].z = 0.0f;
                    float most_x = -__builtin_inff();
#pragma unroll
                    for (int t = 0; t < 4; t++) most_x = fmaxf(most_x, f[mt][t] * fmaxf(fmaxf(s[mt][t][0], s[mt][t][1]), fmaxf(s[mt][t][2], s[mt][t][3])));
                    const float now_x = fmaxf(top[mt], reference<T>(max_over_groups(most_x))), by = now_x == -__builtin_inff() ? 0.0f : now_x;
                    sum[mt] *= __builtin_amdgcn_exp2f(top[mt] - by);
                    top[mt] = now_x;
#pragma unroll
                    for (int t = 0; t < 4; t++)
#pragma unroll
                        for (int r = 0; r < 4; r++) sum[mt] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][t][r], f[mt][t], -by));
                }
            }
            ref[mt] = (top_v[mt] == -__builtin_inff() ? 0.0f : top_v[mt]) - kPScaleLog;
        }
        // the two halves of the tile: weights of one while the other's meet the values, and the next tile's codes become
        // 16-bit floats meanwhile (their loads were issued before the scores)
        f16x8 p[2][MT][PT];
        auto weigh = [&](int mt, int t) {
            const float by = x[t].y - ref[mt];
            float part_sum = 0.0f;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][t][r], f[mt][t], by));
                part_sum += w;
                const _Float16 hi = (_Float16)w;
                p[t / 2][mt][0][4 * (t % 2) + r] = hi;
                if constexpr (PT == 2) p[t / 2][mt][1][4 * (t % 2) + r] = (_Float16)(w - (float)hi);
            }
            sum[mt] = __builtin_fmaf(part_sum, x[t].z, sum[mt]);
        };
        // the values' operands are read from LDS kAhead products ahead
        constexpr int kAhead = 2;
        f16x8 v[kAhead];
        auto read_values = [&](int j) { v[j % kAhead] = *reinterpret_cast<const f16x8*>(&vals[buf][val_at(16 * (j % DT) + m, 4 * (j / DT) + g)]); };
        auto meet = [&](int j) {
            const f16x8 now = v[j % kAhead];
            if (j + kAhead < 2 * DT) read_values(j + kAhead);
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int pt = 0; pt < PT; pt++) o[mt][j % DT] = __builtin_amdgcn_mfma_f32_16x16x32_f16(now, p[j / DT][mt][pt], o[mt][j % DT], 0, 0, 0);
        };
#pragma unroll
        for (int j = 0; j < kAhead; j++) read_values(j);
#pragma unroll
        for (int j = 0; j < 2 * MT; j++) weigh(j / 2, j % 2);
#pragma unroll
        for (int i = 0; i < DT; i++) {
            meet(i);
#pragma unroll
            for (int j = i * 2 * MT / DT; j < (i + 1) * 2 * MT / DT; j++) weigh(j / 2, 2 + j % 2);
        }
#pragma unroll
        for (int i = 0; i < DT; i++) {
            meet(DT + i);
            if constexpr (NBUF == 2) {
#pragma unroll
                for (int j = i * kPieces / DT; j < (i + 1) * kPieces / DT; j++) store_piece(other, j);
            }
        }
    };

    auto open_table = [&]() {                                   // false where no block of it exists
        c1 = min(end - c0, kScanTokens) + c0;
        e0 = c0 >> bs_log;
        const bool mine = tid <= ((c1 - 1) >> bs_log) - e0;
        const uint32_t blk = !mine ? ~0u : c0 == begin ? early : (uint32_t)a.table[(size_t)b * a.width + e0 + tid];
        bh = blk < a.n_blocks ? blk * a.n_heads + kv : ~0u;
        if (mine) ent_row[tid] = bh == ~0u ? ~0u : bh << bs_log;
        const unsigned long long fine = __ballot(bh != ~0u);
        const uint32_t live = fine ? (__builtin_amdgcn_readlane(bh, __builtin_ctzll(fine)) << bs_log) + 1 : 0;        // (all lanes take part)
        if (lane == 0) some[of_all] = live;
        __syncthreads();
        safe = 0;
#pragma unroll
        for (int w = 0; w < kAll; w++) safe = safe ? safe : some[w];
        safe = __builtin_amdgcn_readfirstlane(safe);
        return safe-- != 0;
    };
    bool has = begin < end && open_table();                     // (the same in all threads)
    // (with two halves of the wavefronts these take tiles in turn)
    auto first_tile = [&]() { if (HALVES == 1 || c0 + half * kTokens < c1) fetch(c0 + half * kTokens); };
    if (has) first_tile();
#pragma unroll
    for (int mt = 0; mt < MT; mt++) factor[mt] = query_operands<T, CODES, KS, QT>(a, raw[mt], q[mt]);
    while (c0 < end) {
        if (has) {
            // the entries' scales
            const float sk = bh != ~0u ? a.k_scale[bh] + 0.0f : -1.0f, sv = bh != ~0u ? a.v_scale[bh] : 1.0f;
            if (tid <= ((c1 - 1) >> bs_log) - e0) ent[tid] = make_float4(sk, log2_of_scale(sv), inverse_of_scale(sv), 0.0f);
            const int own = NBUF * half;                        // this half's buffers
            store(own);
            __syncthreads();
            int buf = 0;
            for (uint32_t first = c0; first < c1; first += HALVES * kTokens) {
                const uint32_t t0 = first + half * kTokens, next = t0 + HALVES * kTokens;
                if (next < c1) fetch(next);
                compute(t0, own + buf, own + (buf ^ 1));
                if constexpr (NBUF == 1) {                      // the only buffer is about to be overwritten
                    __syncthreads();
                    store(0);
                } else {
                    buf ^= 1;
                }
                __syncthreads();
            }
        }
        c0 += kScanTokens;
        if (c0 >= end) break;
        __syncthreads();                                        // the table's last readers are done
        has = open_table();
        if (has) first_tile();
    }

#pragma unroll
    for (int mt = 0; mt < MT; mt++)
        if (!far) top[mt] = top_v[mt];
    if constexpr (HALVES == 2) {
        // the second half's softmaxes go to the first through the tiles' memory, lane by lane
        constexpr int kPer = 4 * DT + 3, kLd = MT * kPer;
        static_assert(sizeof(keys) >= 256 * kLd * 4);
        float* mine = reinterpret_cast<float*>(&keys[0][0]) + wave * 64 + lane;
        __syncthreads();
        if (half == 1) {
#pragma unroll
            for (int mt = 0; mt < MT; mt++) {
                float* to = mine + 256 * (mt * kPer);
                to[0] = top[mt];
                to[256] = sum[mt];
                to[512] = top_v[mt];
#pragma unroll
                for (int i = 0; i < DT; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) to[256 * (3 + 4 * i + r)] = o[mt][i][r];
            }
        }
        __syncthreads();
        if (half == 1) return;
#pragma unroll
        for (int mt = 0; mt < MT; mt++) {
            const float* from = mine + 256 * (mt * kPer);
            auto both = [](float& mine_, float there, float& x, float& y) {
                const float now = fmaxf(mine_, there), ref = now == -__builtin_inff() ? 0.0f : now;
                x = __builtin_amdgcn_exp2f(mine_ - ref);
                y = __builtin_amdgcn_exp2f(there - ref);
                mine_ = now;
            };
            float x, y;
            both(top[mt], from[0], x, y);
            sum[mt] = sum[mt] * x + from[256] * y;
            both(top_v[mt], from[512], x, y);
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) o[mt][i][r] = o[mt][i][r] * x + from[256 * (3 + 4 * i + r)] * y;
        }
    }

#pragma unroll
    for (int mt = 0; mt < MT; mt++) {
        const float l = sum_over_groups(sum[mt]);
        const uint32_t r = r0 + 16 * mt + m;
        if (r >= n_r) continue;
        const uint32_t i = of_group(a, r);
        const size_t to = (size_t)(rows.first + i) * a.q_heads + kv * group + (r - i * group);
        const float unit = top_v[mt] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(top_v[mt] - top[mt] - kPScaleLog);
        const float inv = l == 0.0f ? 0.0f : unit / l, lse = l == 0.0f ? -__builtin_inff() : log2_of_sum(top[mt], l);
        if (parts.n_splits == 1) {
            T* out = (T*)a.out + to * dim + 4 * g;
#pragma unroll
            for (int t = 0; t < DT; t++)
                if (16 * t < (int)dim) store4<T>(out + 16 * t, o[mt][t][0] * inv, o[mt][t][1] * inv, o[mt][t][2] * inv, o[mt][t][3] * inv);
            if (g == 0 && a.lse) a.lse[to] = lse * 0.6931471805599453f;
        } else {
            const size_t at = to * parts.n_splits + split;
            float* out = parts.out + at * dim + 4 * g;
#pragma unroll
            for (int t = 0; t < DT; t++)
                if (16 * t < (int)dim) store4<float>(out + 16 * t, o[mt][t][0] * inv, o[mt][t][1] * inv, o[mt][t][2] * inv, o[mt][t][3] * inv);
            if (g == 0) parts.lse[at] = lse;
        }
    }
}

// Chunks that a row's softmax has parts of.
__device__ __forceinline__ uint32_t chunks_of(const AttendArgs& a, const Partials& parts, uint32_t b, uint32_t row)
{
    if (a.found) return parts.n_splits;
    const Span s = rows_of(a, b);
    const uint32_t sees = seen_by(a, length_of(a, a.lens[b]), s.count, row - s.first);
    return min(parts.n_splits, (uint32_t)(((uint64_t)sees + parts.chunk - 1) / parts.chunk));
}

// The chunks' outputs of a row and head become one: weights 2^(lse - largest).  One workgroup each: dim / 4 lanes take a chunk, so that
// 256 / (dim / 4) chunks are read at a time.  What bounds this is the chain of loads that wait for one another, so the first 8 chunks of
// every lane are asked for before it is known how many there are (the workspace holds all of them; what was not written is not used).
// (2 rows of 64 heads of 128 dims in 49 chunks: 5.1 us, 6.0 with the loads one after the other.)
template <class T>
__global__ __launch_bounds__(256) void attend_join_kernel(AttendArgs a, Partials parts)
{
    constexpr uint32_t kFirst = 8;
    __shared__ float red[kWaves], weight[256];
    __shared__ __align__(16) float4 out_s[256];
    const uint32_t tid = threadIdx.x, lane = tid & 63, to = blockIdx.x, row = to / a.q_heads;
    const float* lse = parts.lse + (size_t)to * parts.n_splits;
    const float* x = parts.out + (size_t)to * parts.n_splits * a.dim;
    const uint32_t lanes = a.dim / 4, per = 256 / lanes, mine = tid / lanes, d = (tid - mine * lanes) * 4;
    const float first_lse = tid < parts.n_splits ? lse[tid] : 0.0f;
    float4 first[kFirst];
#pragma unroll
    for (uint32_t j = 0; j < kFirst; j++) {
        const uint32_t i = mine + j * per;
        first[j] = mine < per && i < parts.n_splits && i < 256 ? *reinterpret_cast<const float4*>(x + (size_t)i * a.dim + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const uint32_t b = a.cu_q ? request_of(a.cu_q, a.n_requests, row) : row;
    if (b >= a.n_requests) return;
    const uint32_t n = chunks_of(a, parts, b, row);
    float top = tid < n ? first_lse : -__builtin_inff();
    for (uint32_t i = tid + 256; i < n; i += 256) top = fmaxf(top, lse[i]);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
    if (lane == 0) red[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float ref = top == -__builtin_inff() ? 0.0f : top;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.0f;
    auto add = [&](float f, const float4& y) { o.x += f * y.x; o.y += f * y.y; o.z += f * y.z; o.w += f * y.w; };
    for (uint32_t i0 = 0; i0 < n; i0 += 256) {
        const float w = i0 + tid < n ? __builtin_amdgcn_exp2f((i0 ? lse[i0 + tid] : first_lse) - ref) : 0.0f;
        l += w;
        __syncthreads();
        weight[tid] = w;
        __syncthreads();
        const uint32_t here = min(n - i0, 256u);
        if (mine < per) {
            uint32_t i = mine;
            if (i0 == 0)
#pragma unroll
                for (uint32_t j = 0; j < kFirst; j++, i += per)
                    if (i < here) add(weight[i], first[j]);
#pragma unroll 4
            for (; i < here; i += per) add(weight[i], *reinterpret_cast<const float4*>(x + (size_t)(i0 + i) * a.dim + d));
        }
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) l += __shfl_xor(l, off);
    __syncthreads();
    if (lane == 0) red[tid >> 6] = l;
    out_s[tid] = o;
    __syncthreads();
    l = red[0] + red[1] + red[2] + red[3];
    if (mine == 0) {
        for (uint32_t i = 1; i < per; i++) {
            const float4 y = out_s[tid + i * lanes];
            o.x += y.x; o.y += y.y; o.z += y.z; o.w += y.w;
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        store4<T>((T*)a.out + (size_t)to * a.dim + d, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    }
    if (tid == 0 && a.lse) a.lse[to] = l == 0.0f ? -__builtin_inff() : (ref + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

// The same for few chunks: dim / 4 lanes take a row and head, and all of its chunks (2048 rows of 128 dims in 2 chunks: 4.8 us; 204 of 96 dims in 8: 3.9, 4.7 one after the other).
constexpr uint32_t kFewChunks = 8;
template <class T>
__global__ __launch_bounds__(256) void attend_join_few_kernel(AttendArgs a, Partials parts)
{
    const uint32_t lanes = a.dim / 4, per = 256 / lanes, mine = threadIdx.x / lanes, d = (threadIdx.x - mine * lanes) * 4;
    const uint64_t to = (uint64_t)blockIdx.x * per + mine;
    if (mine >= per || to >= (uint64_t)a.n_rows * a.q_heads) return;
    const float* lse = parts.lse + to * parts.n_splits;
    const float* x = parts.out + to * parts.n_splits * a.dim + d;
    float4 y[kFewChunks];
    float ls[kFewChunks];
#pragma unroll
    for (uint32_t i = 0; i < kFewChunks; i++) {
        ls[i] = i < parts.n_splits ? lse[i] : 0.0f;
        y[i] = i < parts.n_splits ? *reinterpret_cast<const float4*>(x + (size_t)i * a.dim) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const uint32_t row = (uint32_t)(to / a.q_heads);
    const uint32_t b = a.cu_q ? request_of(a.cu_q, a.n_requests, row) : row;
    if (b >= a.n_requests) return;
    const uint32_t n = chunks_of(a, parts, b, row);
    float top = -__builtin_inff(), l = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kFewChunks; i++) top = i < n ? fmaxf(top, ls[i]) : top;
    const float ref = top == -__builtin_inff() ? 0.0f : top;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (uint32_t i = 0; i < kFewChunks; i++)
        if (i < n) {
            const float f = __builtin_amdgcn_exp2f(ls[i] - ref);
            l += f;
            o.x += f * y[i].x; o.y += f * y[i].y; o.z += f * y[i].z; o.w += f * y[i].w;
        }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    store4<T>((T*)a.out + to * a.dim + d, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    if (d == 0 && a.lse) a.lse[to] = l == 0.0f ? -__builtin_inff() : (ref + __builtin_amdgcn_logf(l)) * 0.6931471805599453f;
}

}  // namespace

template <class T> void launch_attend(const AttendArgs& a, const Cut& cut, uint32_t codes_, float* workspace, hipStream_t stream)
{
    const char* who = a.found ? "cache_attend_found" : "cache_attend";
    const Partials parts{workspace, workspace + (uint64_t)a.n_rows * a.q_heads * cut.n_splits * a.dim, cut.n_splits, cut.chunk};
    const int64_t step = 16 / (int64_t)sizeof(T);
    const uint32_t q_vec = (reinterpret_cast<uintptr_t>(a.q) & 15u) == 0 && a.q_row_stride % step == 0 && a.q_head_stride % step == 0;
    const dim3 grid(cut.units * cut.heads, cut.n_splits);
    auto rows = [&](auto codes, auto dp, auto mt, auto nw) {
        if (a.found) hipLaunchKernelGGL((attend_rows_kernel<T, codes.value, dp.value, mt.value, nw.value, true>), grid, dim3(64 * nw.value), 0, stream, a, parts, cut.heads, q_vec);
        else hipLaunchKernelGGL((attend_rows_kernel<T, codes.value, dp.value, mt.value, nw.value, false>), grid, dim3(64 * nw.value), 0, stream, a, parts, cut.heads, q_vec);
    };
    auto by_size = [&](auto codes, auto dp) {
        if (cut.tiles) {
            auto tiles = [&](auto mt) {
                constexpr int kHalves = mt.value == 1 && dp.value == 64 ? 2 : 1;
                hipLaunchKernelGGL((attend_tile_kernel<T, codes.value, dp.value, mt.value, dp.value <= 128 ? 2 : 1, kHalves>), grid, dim3(256 * kHalves), 0, stream, a, parts, q_vec);
            };
            if (dp.value <= 128 && cut.mt == 2) tiles(std::integral_constant<int, dp.value <= 128 ? 2 : 1>{});
            else tiles(std::integral_constant<int, 1>{});
        } else if (dp.value <= 128 && cut.mt == 2) {
            if constexpr (dp.value <= 128) rows(codes, dp, std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
        } else if (cut.waves == 1) {
            rows(codes, dp, std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
        } else if (cut.waves == 8) {
            rows(codes, dp, std::integral_constant<int, 1>{}, std::integral_constant<int, 8>{});
        } else {
            rows(codes, dp, std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
        }
    };
    auto by_dim = [&](auto codes) {
        if (a.dim <= 64) by_size(codes, std::integral_constant<int, 64>{});
        else if (a.dim <= 128) by_size(codes, std::integral_constant<int, 128>{});
        else if (a.dim <= 192) by_size(codes, std::integral_constant<int, 192>{});
        else by_size(codes, std::integral_constant<int, 256>{});
    };
    if (codes_ == HNSW_AMD_CODES_I8) by_dim(std::integral_constant<int, HNSW_AMD_CODES_I8>{});
    else by_dim(std::integral_constant<int, HNSW_AMD_CODES_E4M3>{});
    check_launch(who);
    if (cut.n_splits > 1) {
        // few chunks: many rows to a workgroup (20480 rows of 64 dims in 2 chunks: 5.6 us, 38 with a workgroup each)
        if (cut.n_splits <= kFewChunks) {
            const uint32_t per = 256 / (a.dim / 4);
            hipLaunchKernelGGL((attend_join_few_kernel<T>), dim3((a.n_rows * a.q_heads + per - 1) / per), dim3(256), 0, stream, a, parts);
        } else {
            hipLaunchKernelGGL((attend_join_kernel<T>), dim3(a.n_rows * a.q_heads), dim3(256), 0, stream, a, parts);
        }
        check_launch(who);
    }
}

}  // namespace hnsw_amd
