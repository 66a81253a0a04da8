// Attention over the token cache (hnsw_cache.hip), over all tokens of a request or over those that a search listed.
//
//   out_i = sum_t p_it v_t / sum_t p_it,   p_it = exp(scale * q_i . k_t),   lse_i = log sum_t p_it
//
// A row that sees no token gives zeros and lse = -inf.  The reference indexes vectors and has no counterpart of this.
#include "hnsw_cache.h"

namespace hnsw_amd {

struct AttendArgs {
    const uint8_t *k_codes, *v_codes;
    const float *k_scale, *v_scale;
    uint32_t n_blocks, n_heads, block_tokens, dim;
    const void* q;
    int64_t q_row_stride, q_head_stride;
    uint32_t n_rows, q_heads;
    const int32_t *table, *lens, *cu_q, *ids;
    uint32_t width, n_requests, n_ids, id_heads;
    int32_t causal, found;      // found: over the listed tokens `ids`
    float scale;
    void* out;
    float* lse;
};

namespace {

// The simplest form: one workgroup per query row and head, 256 tokens at a time.
template <class T, int CODES>
__global__ __launch_bounds__(256) void attend_simple_kernel(AttendArgs a)
{
    __shared__ float q_s[256], p_s[256], red[4];
    __shared__ uint64_t at_s[256];
    __shared__ float sv_s[256];
    const uint32_t tid = threadIdx.x, lane = tid & 63, head = blockIdx.x % a.q_heads, row = blockIdx.x / a.q_heads;
    const uint32_t b = a.cu_q ? request_of(a.cu_q, a.n_requests, row) : row;
    if (b >= a.n_requests) return;
    const uint32_t kv = head / (a.q_heads / a.n_heads);
    const int64_t cap = (int64_t)a.width * a.block_tokens;
    int64_t len = a.lens[b];
    if (len < 0) len = 0;
    if (len > cap) len = cap;
    int64_t seen = len;
    if (a.cu_q && a.causal) seen = len - (a.cu_q[b + 1] - a.cu_q[b]) + (int64_t)(row - a.cu_q[b]) + 1;
    if (seen > len) seen = len;
    const int64_t items = a.found ? (int64_t)a.n_ids : seen;
    const int32_t* ids = a.found ? a.ids + ((size_t)row * a.id_heads + head / (a.q_heads / a.id_heads)) * a.n_ids : nullptr;
    if (tid < a.dim) q_s[tid] = to_float(((const T*)a.q)[(int64_t)row * a.q_row_stride + (int64_t)head * a.q_head_stride + tid]);
    float m = -__builtin_inff(), l = 0.0f, o = 0.0f;
    for (int64_t t0 = 0; t0 < items; t0 += 256) {
        __syncthreads();
        float s = -__builtin_inff();
        uint64_t at = ~0ull;
        float sv = 0.0f;
        if (t0 + tid < items) {
            const int64_t t = a.found ? (int64_t)(uint32_t)ids[t0 + tid] : t0 + tid;
            const int32_t blk = t < seen ? a.table[(size_t)b * a.width + t / a.block_tokens] : -1;
            if ((uint32_t)blk < a.n_blocks) {
                const uint64_t bh = (uint64_t)blk * a.n_heads + kv;
                at = (bh * a.block_tokens + t % a.block_tokens) * a.dim;
                float dot = 0.0f;
                for (uint32_t i = 0; i < a.dim / 4; i++) {
                    float x[4];
                    decode4<CODES>(*reinterpret_cast<const uint32_t*>(a.k_codes + at + 4 * i), x);
#pragma unroll
                    for (int j = 0; j < 4; j++) dot = __builtin_fmaf(x[j], q_s[4 * i + j], dot);
                }
                s = dot * a.k_scale[bh] * a.scale;
                sv = a.v_scale[bh];
            }
        }
        float top = s;
#pragma unroll
        for (int o2 = 32; o2 >= 1; o2 >>= 1) top = fmaxf(top, __shfl_xor(top, o2));
        if (lane == 0) red[tid >> 6] = top;
        __syncthreads();
        const float mn = fmaxf(m, fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]))), ref = mn == -__builtin_inff() ? 0.0f : mn;
        const float p = expf(s - ref), shrink = expf(m - ref);
        p_s[tid] = p; at_s[tid] = at; sv_s[tid] = sv;
        float sum = p;
#pragma unroll
        for (int o2 = 32; o2 >= 1; o2 >>= 1) sum += __shfl_xor(sum, o2);
        __syncthreads();
        if (lane == 0) red[tid >> 6] = sum;
        __syncthreads();
        l = l * shrink + (red[0] + red[1] + red[2] + red[3]);
        m = mn;
        o *= shrink;
        if (tid < a.dim)
            for (int j = 0; j < 256; j++)
                if (at_s[j] != ~0ull) {
                    float x[4];
                    decode4<CODES>(*reinterpret_cast<const uint32_t*>(a.v_codes + at_s[j] + (tid & ~3u)), x);
                    o += p_s[j] * sv_s[j] * x[tid & 3];
                }
    }
    const size_t to = (size_t)row * a.q_heads + head;
    if (tid < a.dim) ((T*)a.out)[to * a.dim + tid] = from_float<T>(l > 0.0f ? o / l : (l == 0.0f ? 0.0f : l));
    if (tid == 0 && a.lse) a.lse[to] = l == 0.0f ? -__builtin_inff() : m + logf(l);
}

}  // namespace

static void check_attend(const hnsw_amd_token_cache* c, const AttendArgs& a, const char* who)
{
    check_cache(c, who);
    const std::string w(who);
    if (a.q_heads < 1 || a.q_heads % c->n_heads) throw std::invalid_argument(w + ": the query heads must be a multiple of the cache's heads");
    if (a.n_requests < 1) throw std::invalid_argument(w + ": no requests");
    if (a.width < 1 || (uint64_t)a.width * c->block_tokens > 0x7fffffffull) throw std::invalid_argument(w + ": the table's width in tokens must be 1..2^31 - 1");
    if (!a.cu_q && a.n_rows != a.n_requests) throw std::invalid_argument(w + ": without cu_q there is one query row for each request");
    if (a.n_rows > 0x7fffffffu || (uint64_t)a.n_rows * a.q_heads > 0x7fffffffull) throw std::invalid_argument(w + ": too many rows and heads for one call");
    if (a.found && (a.id_heads < 1 || a.id_heads % c->n_heads || a.q_heads % a.id_heads))
        throw std::invalid_argument(w + ": the lists' heads must be a multiple of the cache's heads and divide the query heads");
    if (!(a.scale == a.scale) || a.scale - a.scale != 0.0f) throw std::invalid_argument(w + ": scale must be finite");
}

uint64_t attend_workspace(const hnsw_amd_token_cache*, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) { return 0; }
uint64_t attend_found_workspace(const hnsw_amd_token_cache*, uint32_t, uint32_t, uint32_t, uint32_t) { return 0; }

void cache_attend(const hnsw_amd_token_cache* c, const void* q, uint32_t n_rows, uint32_t q_heads, int64_t q_row_stride, int64_t q_head_stride,
                  uint32_t row_type, const int32_t* table, uint32_t width, const int32_t* lens, uint32_t n_requests, const int32_t* cu_q,
                  bool found, const int32_t* ids, uint32_t n_ids, uint32_t id_heads, int causal, float scale, uint32_t max_len, void* out, float* lse,
                  void* workspace, uint64_t workspace_bytes, int device, void* stream)
{
    const char* who = found ? "cache_attend_found" : "cache_attend";
    if (!c) throw std::invalid_argument(std::string(who) + ": NULL argument");
    AttendArgs a{(const uint8_t*)c->k_codes, (const uint8_t*)c->v_codes, c->k_scale, c->v_scale, c->n_blocks, c->n_heads, c->block_tokens, c->dim,
                 q, q_row_stride, q_head_stride, n_rows, q_heads, table, lens, cu_q, ids, width, n_requests, n_ids, id_heads, causal, found ? 1 : 0, scale, out, lse};
    check_attend(c, a, who);
    check_row_type(row_type, who);
    (void)max_len; (void)workspace; (void)workspace_bytes;
    if (n_rows == 0) return;
    const OnDevice on(device);
    by_types(row_type, c->codes, [&](auto t, auto codes) {
        hipLaunchKernelGGL((attend_simple_kernel<decltype(t), codes.value>), dim3(n_rows * q_heads), dim3(256), 0, (hipStream_t)stream, a);
    });
    check_launch(who);
}

}  // namespace hnsw_amd
