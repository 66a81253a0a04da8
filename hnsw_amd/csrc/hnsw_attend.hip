// Attention over the token cache (hnsw_cache.hip), over all tokens of a request or over those that a search listed.
//
//   out_i = sum_t p_it v_t / sum_t p_it,   p_it = exp(scale * q_i . k_t),   lse_i = log sum_t p_it
//
// A row that sees no token gives zeros and lse = -inf.  The reference indexes vectors and has no counterpart of this.
#include <algorithm>

#include "hnsw_attend.h"

namespace hnsw_amd {

static void check_attend(const hnsw_amd_token_cache* c, const AttendArgs& a, const char* who)
{
    check_cache(c, who);
    const std::string w(who);
    if (a.q_heads < 1 || a.q_heads % c->n_heads) throw std::invalid_argument(w + ": the query heads must be a multiple of the cache's heads");
    if (a.n_requests < 1) throw std::invalid_argument(w + ": no requests");
    if (a.width < 1 || (uint64_t)a.width * c->block_tokens > 0x7fffffffull) throw std::invalid_argument(w + ": the table's width in tokens must be 1..2^31 - 1");
    if (!a.cu_q && a.n_rows != a.n_requests) throw std::invalid_argument(w + ": without cu_q there is one query row for each request");
    if (a.n_rows > 0x7fffffffu || (uint64_t)a.n_rows * a.q_heads >= 1ull << 24) throw std::invalid_argument(w + ": too many rows and heads for one call");
    if (a.found && (a.id_heads < 1 || a.id_heads % c->n_heads || a.q_heads % a.id_heads))
        throw std::invalid_argument(w + ": the lists' heads must be a multiple of the cache's heads and divide the query heads");
    if (reinterpret_cast<uintptr_t>(a.out) & 15u) throw std::invalid_argument(w + ": the output must be aligned to 16 bytes");
    if (!(a.scale == a.scale) || a.scale - a.scale != 0.0f) throw std::invalid_argument(w + ": scale must be finite");
}

// How a call's work is cut.  `items`: tokens of the longest request, or list entries.
static Cut cut_work(uint32_t dim, uint32_t n_rows, uint32_t q_heads, uint32_t n_requests, uint32_t heads, uint32_t items, bool by_request, bool ragged)
{
    Cut c{};
    c.heads = heads;
    const uint32_t group = q_heads / heads;
    const double rows = (double)group * (by_request ? (double)n_rows / n_requests : 1.0);      // that share the tokens
    // Many rows: 128 (beyond 128 dims 64) a workgroup, through LDS.  Few: 16, or 32, in registers; the codes are decoded once for both
    // halves (beyond 128 dims two halves' outputs do not fit the registers).  Sixteen requests of 2000 tokens, 8 heads of 128 dims: with 64
    // rows of queries to a key head 38 us in registers and 63 through LDS, with 96 55 and 61, with 256 81 and 78, with 512 152 and 100;
    // eight of 1000 tokens, 16 heads of 64 dims and 16-bit float rows: 64 rows 21.9 and 22.7, 100 33 and 24.
    c.tiles = by_request && ragged && rows > 96.0;
    c.mt = rows > 16.0 && dim <= 128 ? 2 : 1;
    c.waves = 4;
    auto units_of = [&](uint64_t tile) {
        return by_request && ragged ? n_requests + (uint64_t)n_rows * group / tile : (uint64_t)(by_request ? n_requests : n_rows) * ((group + tile - 1) / tile);
    };
    uint64_t chunk = 0;
    if (c.tiles) {
        // 128 rows in chunks (512 tokens at least) until there are two workgroups for every compute unit, or 64 rows and one: half the rows
        // cost 0.6 of a tile of tokens' time, a workgroup's start three tiles' and joining chunks six.  What these say was measured
        // on 25 shapes; the choice is the faster one, or within 3 %, in all of them.  (1000 rows over 1000 tokens of 8 heads of 128
        // dims: 48 us with 128 rows, 36 with 64; 512 over 8000: 109 and 203.)
        double least = 0.0;
        auto consider = [&](uint32_t mt, uint64_t want, double tile_time) {
            const uint64_t have = units_of(64 * mt) * heads, splits = (want + have - 1) / have;
            const uint64_t each = std::max<uint64_t>((((uint64_t)items + splits - 1) / splits + 63) / 64 * 64, 512), n = ((uint64_t)items + each - 1) / each;
            const double time = std::max(1.0, (double)(have * n) / 512) * (3.0 + (double)std::min<uint64_t>(each, items) / 64) * tile_time + (n > 1 ? 6.0 : 0.0);
            if (least > 0.0 && time >= least) return;
            least = time;
            c.mt = mt;
            chunk = each;
        };
        if (dim <= 128) {
            consider(2, 512, 1.0);
            consider(1, 256, 0.6);
        } else {
            consider(1, 512, 1.0);
        }
    }
    const uint64_t units = units_of(c.tiles ? 64 * c.mt : 16 * c.mt), have = units * heads;
    c.units = (uint32_t)std::min<uint64_t>(units, 1u << 24);             // (as many are refused)
    if (c.tiles) {
        // (cut above)
    } else if (c.mt == 1 && have >= 1024 && items <= 256) {
        // short requests (lists) in number: a wavefront for each, nothing to join.  (Lists of 32, 100, 200 and 256 entries in 2048 workgroups: 8.4,
        // 18.5, 27.7 and 31.8 us, in chunks 18.5, 23.9, 31.5 and 34.7; in 1024: 6.4, 11.3, 18.0 and 19.4, in chunks 11.2, 13.9, 19.0 and
        // 20.4; in 768: 6.2, 10.2, 15.5 and 16.7, in chunks 7.8, 10.1, 14.3 and 15.4.)
        c.waves = 1;
        chunk = 256;
    } else if (c.mt == 1 && have < 512 && items <= 1024) {
        // few short ones: one chunk, as a second launch to join more of them mostly costs more than it saves (300 and 1000 tokens of 128 dims,
        // 504 workgroups: 11.8 and 25.4 us, in chunks 19.0 and 29.5; 256: 9.0 and 16.6, in chunks 12.1 and 18.5; 64: 8.6 and 12.5, in chunks 9.2
        // and 10.9; and it would still win at 504 of 2000 tokens, 42.3 and 48.9, but not at 64 of 2000, 21.2 and 12.9).  Eight wavefronts for
        // it where it is not so short that they cost more in starting (64 dims, 256 workgroups: 100 tokens 6.6 us, with four 6.2; 160: 6.9 and
        // 7.0; 500: 8.7 and 9.2; 1000: 11.4 and 13.2; at 128 dims four are 0.3 to 0.6 us faster up to 500 tokens and 0.4 slower at 1000)
        // and all fit the chip at once, beyond 64 dims one such workgroup to a compute unit (320 of 1000 tokens of 128 dims: 26.6, with
        // four 19.3)
        c.waves = items > 128 && have <= (dim <= 64 ? 512 : 256) ? 8 : 4;
        chunk = 1024;
    } else {
        // one round of three workgroups a compute unit, but no chunk of more than 4096: a long request among short ones is not left to
        // a few workgroups (64 requests of 1 to 8192 tokens, 8 heads: 117 us, 121 with 8192; 17 of 100 to 3000, 4 heads: 15.4 us, 18.5 with half
        // as many workgroups and 16.6 with twice)
        chunk = std::min<uint64_t>(have * items / 768, 4096);
        chunk = std::max<uint64_t>((chunk + 127) / 128 * 128, 128);
    }
    chunk = std::max<uint64_t>(chunk, ((uint64_t)items / 32768 + 127) / 128 * 128);      // (the chunks are a grid's second extent, below 2^16)
    c.chunk = (uint32_t)std::min<uint64_t>(chunk, 0x80000000ull);
    c.n_splits = std::max<uint32_t>(1, (uint32_t)(((uint64_t)items + c.chunk - 1) / c.chunk));
    return c;
}

static uint64_t workspace_of(const Cut& c, uint32_t n_rows, uint32_t q_heads, uint32_t dim)
{
    return c.n_splits == 1 ? 0 : (uint64_t)n_rows * q_heads * c.n_splits * (dim + 1) * 4;
}

static uint32_t items_of(uint32_t width, uint32_t block_tokens, uint32_t max_len)
{
    const uint64_t cap = (uint64_t)width * block_tokens;
    return (uint32_t)(max_len && max_len < cap ? max_len : (cap < 0x7fffffffull ? cap : 0x7fffffffull));
}

uint64_t attend_workspace(const hnsw_amd_token_cache* c, uint32_t n_rows, uint32_t q_heads, uint32_t n_requests, uint32_t width, uint32_t max_len)
{
    if (!c->n_heads || !n_requests || !q_heads || q_heads % c->n_heads) return 0;      // (the call itself says what is wrong)
    return workspace_of(cut_work(c->dim, n_rows, q_heads, n_requests, c->n_heads, items_of(width, c->block_tokens, max_len), true, n_rows != n_requests), n_rows, q_heads, c->dim);
}

uint64_t attend_found_workspace(const hnsw_amd_token_cache* c, uint32_t n_rows, uint32_t q_heads, uint32_t id_heads, uint32_t n_ids)
{
    if (!id_heads || !q_heads || q_heads % id_heads) return 0;
    return workspace_of(cut_work(c->dim, n_rows, q_heads, n_rows, id_heads, n_ids, false, false), n_rows, q_heads, c->dim);
}

void cache_attend(const hnsw_amd_token_cache* c, const void* q, uint32_t n_rows, uint32_t q_heads, int64_t q_row_stride, int64_t q_head_stride,
                  uint32_t row_type, const int32_t* table, uint32_t width, const int32_t* lens, uint32_t n_requests, const int32_t* cu_q,
                  bool found, const int32_t* ids, uint32_t n_ids, uint32_t id_heads, int causal, float scale, uint32_t max_len, void* out, float* lse,
                  void* workspace, uint64_t workspace_bytes, int device, void* stream)
{
    const char* who = found ? "cache_attend_found" : "cache_attend";
    if (!c) throw std::invalid_argument(std::string(who) + ": NULL argument");
    AttendArgs a{(const uint8_t*)c->k_codes, (const uint8_t*)c->v_codes, c->k_scale, c->v_scale, c->n_blocks, c->n_heads, c->block_tokens, c->dim,
                 q, q_row_stride, q_head_stride, n_rows, q_heads, table, lens, cu_q, ids, width, n_requests, n_ids, id_heads, causal, found ? 1 : 0, scale, out, lse, 0, 1, 0.0f};
    check_attend(c, a, who);
    a.group = q_heads / (found ? id_heads : c->n_heads);
    a.lists = found ? id_heads / c->n_heads : 1;
    a.group_inverse = 1.0f / (float)a.group;
    check_row_type(row_type, who);
    if (n_rows == 0) return;
    const Cut cut = found ? cut_work(c->dim, n_rows, q_heads, n_rows, id_heads, n_ids, false, false)
                          : cut_work(c->dim, n_rows, q_heads, n_requests, c->n_heads, items_of(width, c->block_tokens, max_len), true, n_rows != n_requests);
    const uint64_t need = workspace_of(cut, n_rows, q_heads, c->dim);
    if (need > workspace_bytes || (need && !workspace)) throw std::invalid_argument(std::string(who) + ": the workspace is too small");
    if (reinterpret_cast<uintptr_t>(workspace) & 15u) throw std::invalid_argument(std::string(who) + ": the workspace must be aligned to 16 bytes");
    if ((uint64_t)cut.units * cut.heads >= 1ull << 24) throw std::invalid_argument(std::string(who) + ": too much work for one call");
    const OnDevice on(device);
    if (row_type == HNSW_AMD_TYPE_F32) launch_attend<float>(a, cut, c->codes, (float*)workspace, (hipStream_t)stream);
    else if (row_type == HNSW_AMD_TYPE_F16) launch_attend<_Float16>(a, cut, c->codes, (float*)workspace, (hipStream_t)stream);
    else launch_attend<bf16>(a, cut, c->codes, (float*)workspace, (hipStream_t)stream);
}

}  // namespace hnsw_amd
