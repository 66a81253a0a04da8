// The token cache: keys and values of a language model's tokens, held in 8 bits with one scale for each block of tokens and
// head, in blocks that requests take from a common stock.  This file grows requests (block tables, slot maps), writes rows
// into their slots and reads them back; hnsw_attend.hip reads the cache with attention.
//
//   codes [n_blocks][n_heads][block_tokens][dim] bytes, scale [n_blocks][n_heads] f32, value = code * scale
//
// A token's row of one head is contiguous, so that a token found by a search is one 128-byte line (at 128 dims), and the rows
// of a block and head are contiguous, so that a scan streams.
// The reference indexes vectors and has no counterpart of this.
#include <algorithm>

#include "hnsw_cache.h"

namespace hnsw_amd {

namespace {

constexpr uint32_t kMaxRequests = 8192;      // of one planning call: its prefix sums live in LDS (4 words each)

struct PlanArgs {
    const int32_t *lens, *grow;
    int32_t* table;
    int32_t* ring;
    const int64_t* state;
    int64_t* slots;
    int32_t *cu_new, *lens_out, *status;
    int64_t* state_out;
    uint32_t n_requests, width, n_blocks, block_tokens, n_slots, per;      // per: slots in a row that a thread maps
    uint32_t taker, giver, counter;     // the first threads that enter taken blocks, give blocks back and write lengths
};

// last b in [0, n) with pre[b] <= i (pre ascending, pre[0] = 0)
__device__ __forceinline__ uint32_t last_not_after(const uint32_t* pre, uint32_t n, uint32_t i)
{
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (pre[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
}

// One launch: every workgroup recomputes the prefix sums over the requests (a few KB out of the L2, cheaper than a second
// launch that would wait for them) and then takes its share of the slots, table entries and returned blocks.  Nothing that a
// workgroup reads is written by another: lengths and ring state go to buffers of their own, the table is written only beyond
// what the requests held, and the ring only behind its tail, where no free block lies.
// What bounds it is the chain of loads that wait for one another: lengths, table or ring, slots.  (64 requests, a token each: 4.0 us;
// 1000 requests, 318000 tokens, 2.8 MB: 8.2 us.)
__global__ void plan_kernel(PlanArgs a)
{
    extern __shared__ uint32_t lds[];
    const uint32_t n = a.n_requests, bs = a.block_tokens, bs_log = 31 - __builtin_clz(bs), tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
    uint32_t* len_s = lds;            // tokens held
    uint32_t* cu_s = len_s + n;       // new tokens before this request
    uint32_t* need_s = cu_s + n;      // blocks taken before this request
    uint32_t* back_s = need_s + n;    // blocks given back before this request
    __shared__ uint32_t wsum[3][16];
    __shared__ unsigned long long total_grow, total_back;
    __shared__ uint32_t trouble;
    if (tid == 0) { total_grow = 0; total_back = 0; trouble = 0; }
    const int64_t head = a.state[0], tail = a.state[1], avail = tail - head;
    __syncthreads();

    const uint32_t per = (n + blockDim.x - 1) / blockDim.x, lo = min(tid * per, n), hi = min(lo + per, n);
    uint32_t g_sum = 0, need_sum = 0, back_sum = 0, bad = 0;
    unsigned long long g_all = 0, back_all = 0;
    auto counts = [&](uint32_t b, uint32_t& len, uint32_t& g, uint32_t& need, uint32_t& back) {
        const int32_t l = a.lens[b], r = a.grow[b];
        if (l < 0 || r < -1) bad |= HNSW_AMD_PLAN_BAD_LENGTH;
        len = (uint32_t)max(l, 0);
        g = (uint32_t)max(r, 0);
        const uint32_t have = (len + bs - 1) >> bs_log;                                  // (lengths are below 2^31)
        const uint32_t want = (uint32_t)(((unsigned long long)len + g + bs - 1) >> bs_log);
        if (want > a.width) bad |= HNSW_AMD_PLAN_TABLE_FULL;
        need = want - have;
        back = r == -1 ? have : 0;
    };
    for (uint32_t b = lo; b < hi; b++) {
        uint32_t len, g, need, back;
        counts(b, len, g, need, back);
        len_s[b] = len; cu_s[b] = g_sum; need_s[b] = need_sum; back_s[b] = back_sum;
        g_sum += g; need_sum += need; back_sum += back; g_all += g; back_all += back;
    }
    const uint32_t gi = wave_inclusive_sum(g_sum), ni = wave_inclusive_sum(need_sum), bi = wave_inclusive_sum(back_sum);
    // (the totals in two parts, so that 32 bits hold their sums: a thread has 16 requests at most, below 2^35)
    auto total = [](unsigned long long x) { return ((unsigned long long)wave_inclusive_sum((uint32_t)(x >> 16)) << 16) + wave_inclusive_sum((uint32_t)x & 0xffffu); };
    const unsigned long long g_total = total(g_all), back_total = total(back_all);
    if (lane == 63) {
        wsum[0][wave] = gi; wsum[1][wave] = ni; wsum[2][wave] = bi;
        atomicAdd(&total_grow, g_total);
        atomicAdd(&total_back, back_total);
    }
    if (bad) atomicOr(&trouble, bad);
    __syncthreads();
    uint32_t g0 = gi - g_sum, n0 = ni - need_sum, b0 = bi - back_sum, given = 0, taken = 0, grown = 0;
    for (uint32_t w = 0; w < waves; w++) {
        if (w < wave) { g0 += wsum[0][w]; n0 += wsum[1][w]; b0 += wsum[2][w]; }
        grown += wsum[0][w]; taken += wsum[1][w]; given += wsum[2][w];
    }
    for (uint32_t b = lo; b < hi; b++) { cu_s[b] += g0; need_s[b] += n0; back_s[b] += b0; }
    uint32_t status = trouble;
    if (head < 0 || avail < 0 || avail > (int64_t)a.n_blocks) status |= HNSW_AMD_PLAN_BAD_LENGTH;
    if (total_grow > a.n_slots) status |= HNSW_AMD_PLAN_SLOTS_FULL;
    // (the 32-bit sums can only have wrapped where one of the 64-bit totals is refused)
    if (!status && (int64_t)taken > avail) status |= HNSW_AMD_PLAN_NO_BLOCKS;
    if (!status && (int64_t)total_back > (int64_t)a.n_blocks - avail) status |= HNSW_AMD_PLAN_BAD_LENGTH;
    if (status) { grown = 0; taken = 0; given = 0; }                                // all or nothing
    auto wrap = [&](int64_t x) { return x >> 32 ? (uint32_t)((uint64_t)x % a.n_blocks) : (uint32_t)x % a.n_blocks; };      // (64-bit division is long)
    const uint32_t head_at = status ? 0u : wrap(head), tail_at = status ? 0u : wrap(tail);
    __syncthreads();

    auto ring_at = [&](uint32_t from, uint32_t i) { const unsigned long long p = (unsigned long long)from + i; return (uint32_t)(p >= a.n_blocks ? p - a.n_blocks : p); };
    const uint32_t stride = gridDim.x * blockDim.x, me = blockIdx.x * blockDim.x + tid;
    // slots in a row: one search for the request, one block looked up for most of them
    for (uint32_t t0 = a.per * me; t0 < a.n_slots; t0 += a.per * stride) {
        uint32_t b = t0 < grown ? last_not_after(cu_s, n, t0) : n, block = ~0u, of = ~0u;        // (block `block` of request `of` is number blk)
        int32_t blk = -1;
        for (uint32_t t = t0; t < t0 + a.per && t < a.n_slots; t++) {
            int64_t slot = -1;
            if (t < grown) {
                while (b + 1 < n && cu_s[b + 1] <= t) b++;
                const uint32_t pos = len_s[b] + (t - cu_s[b]), j = pos >> bs_log, have = (len_s[b] + bs - 1) >> bs_log;
                if (j != block || b != of) {
                    blk = j < have ? a.table[(size_t)b * a.width + j] : a.ring[ring_at(head_at, need_s[b] + j - have)];
                    block = j;
                    of = b;
                }
                if ((uint32_t)blk < a.n_blocks) slot = ((int64_t)blk << bs_log) + (pos & (bs - 1));
            }
            a.slots[t] = slot;
        }
    }
    // (the other work begins in other wavefronts than the slots: each is a chain of loads that wait for one another)
    auto from = [&](uint32_t first) { return me >= first ? me - first : me + stride - first; };
    for (uint32_t i = from(a.taker); i < taken; i += stride) {
        const uint32_t b = last_not_after(need_s, n, i), have = (len_s[b] + bs - 1) >> bs_log;
        a.table[(size_t)b * a.width + have + (i - need_s[b])] = a.ring[ring_at(head_at, i)];
    }
    for (uint32_t i = from(a.giver); i < given; i += stride) {
        const uint32_t b = last_not_after(back_s, n, i);
        a.ring[ring_at(tail_at, i)] = a.table[(size_t)b * a.width + (i - back_s[b])];
    }
    for (uint32_t b = from(a.counter); b < n; b += stride) {
        const int32_t r = a.grow[b];
        a.lens_out[b] = status ? a.lens[b] : (r < 0 ? 0 : (int32_t)(len_s[b] + (uint32_t)r));
        a.cu_new[b] = status ? 0 : (int32_t)cu_s[b];
    }
    if (me == 0) {
        a.cu_new[n] = (int32_t)grown;
        a.state_out[0] = head + taken;
        a.state_out[1] = tail + given;
        a.status[0] = (int32_t)status;
    }
}

struct AppendArgs {
    uint8_t* codes[2];
    float* scale[2];
    const void* rows[2];
    int64_t row_stride[2], head_stride[2];
    const int64_t* slots;
    uint32_t n_rows, n_blocks, n_heads, block_tokens, dim, span;
};

// The least e with peak <= max * 2^e, in [-100, 121] (121: the largest f32 over 127; below 2^-100 values count as zero).
__device__ __forceinline__ int scale_exponent(float peak, float most)
{
    int e = (int)((__float_as_uint(peak) >> 23) & 255u) - 127 - (most > 200.0f ? 9 : 7);      // peak < 2^(x + 1) and most > 2^(x of most): e or e - 1, e - 2
    e = max(min(e, 121), -100);
    while (e < 121 && peak > ldexpf(most, e)) e++;
    return e;
}

// Four wavefronts take a.span rows of one head's keys or values, run by run (a run: rows whose slots follow one another in one block).  First the
// rows' largest value, which gives the block's scale; where that raises the scale of a block that held earlier tokens, their codes move to it;
// then the rows' codes.  What a wavefront has looked at first stays in its registers between the two.  Short runs (single tokens of many
// requests) are latency: a wavefront takes each by itself.  Long runs (prompts) are memory: all four wavefronts take each, and so they do
// with runs of one block that slots which are left out keep apart, one after the other.
// A power of two as scale makes x / scale exact, so a code is ONE rounding of x, and moving codes to a larger scale one more.
// (64 rows of 8 heads of 128 dims: 4.4 us.  Three prompts, 21500 rows, 132 MB: 41 us, 3.2 TB/s: slots, rows, largest value and codes follow
// one another in a workgroup, and seven workgroups a compute unit hide most of that; five, with the rows kept as 32-bit values: 45 us.)
template <class T, int CODES, bool VEC>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a)
{
    constexpr int kKeep = 4;                                    // passes over the rows whose values are kept
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t part = blockIdx.x % 2, head = blockIdx.x / 2 % a.n_heads;
    const uint64_t t0 = (uint64_t)(blockIdx.x / 2 / a.n_heads) * a.span;
    __shared__ float peaks[4];
    const uint32_t bs = a.block_tokens, bs_log = 31 - __builtin_clz(bs), dim = a.dim, lanes_per_row = dim / 8, rows_per_wave = 64 / lanes_per_row;
    const uint32_t wave_row = lane / lanes_per_row, my_col = (lane - wave_row * lanes_per_row) * 8;
    const bool active = wave_row < rows_per_wave;
    const int64_t n_slots = (int64_t)a.n_blocks << bs_log;
    const T* rows = (const T*)a.rows[part];
    const int64_t row_stride = a.row_stride[part], col = a.head_stride[part] * head + my_col;
    auto load = [&](uint32_t row, Eight<T>& x) { load8<T, VEC>(rows + (int64_t)row * row_stride + col, x); };

    const uint32_t end = (uint32_t)(t0 + a.span < a.n_rows ? t0 + a.span : a.n_rows);
    for (uint32_t base = (uint32_t)t0; base < end; base += 62) {
        // lanes 1 .. 62 have the slots of rows base .. base + 61, the others those before and behind
        const int64_t at = (int64_t)base - 1 + lane;
        const int64_t slot_l = at >= 0 && at < (int64_t)a.n_rows ? a.slots[at] : -1;
        const bool valid = slot_l >= 0 && slot_l < n_slots;
        const int64_t prev_l = __shfl_up(slot_l, 1);
        const bool after = valid && lane > 0 && (uint64_t)(slot_l ^ prev_l) < bs && prev_l < slot_l;     // the row before is of the same block, and of
        const unsigned long long follow = __ballot(after && prev_l == slot_l - 1);                           // the same run, or slots between the two
        const unsigned long long behind = __ballot(after) & ~follow;                                         // are left out
        unsigned long long firsts = __ballot(valid && !after) & ~(1ull << 63) & ~1ull;
        if (end - base < 62) firsts &= (2ull << (end - base)) - 1;

        // The run of n rows from row0 and `slot` on, by wavefront `sub` of `of`.
        auto take = [&](uint32_t row0, int64_t slot, uint32_t n, uint32_t sub, auto of) {
            constexpr uint32_t kOf = of.value;
            const uint32_t my_row = sub * rows_per_wave + wave_row, step = rows_per_wave * kOf;
            const uint32_t block = (uint32_t)(slot >> bs_log), off = (uint32_t)(slot & (bs - 1));
            float* scale = a.scale[part] + (size_t)block * a.n_heads + head;
            uint8_t* codes = a.codes[part] + ((size_t)block * a.n_heads + head) * bs * dim;
            const float before = *scale;
            Eight<T> kept[kKeep];
            float peak = 0.0f;
            auto look = [&](const Eight<T>& x) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float y = fabsf(x[j]);
                    peak = y < __builtin_inff() ? fmaxf(peak, y) : peak;            // (NaN and infinities do not set the scale)
                }
            };
            if (active) {
#pragma unroll
                for (int i = 0; i < kKeep; i++)
                    if (my_row + i * step < n) load(row0 + my_row + i * step, kept[i]);
#pragma unroll
                for (int i = 0; i < kKeep; i++)
                    if (my_row + i * step < n) look(kept[i]);
                for (uint32_t r = my_row + kKeep * step; r < n; r += step) {
                    Eight<T> x;
                    load(row0 + r, x);
                    look(x);
                }
            }
            peak = wave_max_not_negative(peak);
            if constexpr (kOf > 1) {
                if (lane == 0) peaks[sub] = peak;
                __syncthreads();
                peak = fmaxf(fmaxf(peaks[0], peaks[1]), fmaxf(peaks[2], peaks[3]));
            }
            int e = scale_exponent(peak, kCodeMax<CODES>);
            const bool held = off > 0 && before > 0.0f && before < __builtin_inff();        // the block holds earlier tokens
            if (held) {
                int eb = (int)((__float_as_uint(before) >> 23) & 255u) - 127;
                if (eb < -100) eb = -100;
                else if (__float_as_uint(before) & 0x7fffffu) eb++;                 // (a scale from elsewhere: the next power of two)
                e = max(e, min(eb, 121));
            }
            const float now = ldexpf(1.0f, e);
            if (held && now != before) {
                const float ratio = before / now;
                for (uint32_t i = sub * 64 + lane; i < bs * dim / 4; i += 64 * kOf) {
                    const uint32_t o = i * 4 / dim;
                    if (o >= off && o < off + n) continue;                          // about to be written
                    float x[4];
                    uint32_t* w = reinterpret_cast<uint32_t*>(codes) + i;
                    decode4<CODES>(*w, x);
#pragma unroll
                    for (int j = 0; j < 4; j++) x[j] *= ratio;
                    *w = encode4<CODES>(x);
                }
            }
            const float inv = ldexpf(1.0f, -e);
            auto write = [&](uint32_t r, const Eight<T>& x) {
                float lo[4], hi[4];
#pragma unroll
                for (int j = 0; j < 4; j++) { lo[j] = x[j] * inv; hi[j] = x[j + 4] * inv; }
                *reinterpret_cast<u32x2*>(codes + (size_t)(off + r) * dim + my_col) = u32x2{encode4<CODES>(lo), encode4<CODES>(hi)};
            };
            if (active) {
#pragma unroll
                for (int i = 0; i < kKeep; i++)
                    if (my_row + i * step < n) write(my_row + i * step, kept[i]);
                for (uint32_t r = my_row + kKeep * step; r < n; r += step) {
                    Eight<T> x;
                    load(row0 + r, x);
                    write(r, x);
                }
            }
            if constexpr (kOf > 1) __syncthreads();             // (all have read the old scale and the peaks)
            if (lane == 0 && sub == 0) *scale = now;
        };
        // the run's length, of which n rows are known
        auto extend = [&](uint32_t row0, int64_t slot, uint32_t n) {
            const uint32_t off = (uint32_t)(slot & (bs - 1));
            for (;;) {
                const uint32_t i = n + lane;
                const bool more = off + i < bs && (uint64_t)row0 + i < a.n_rows && a.slots[row0 + i] == slot + i;
                const unsigned long long more_l = __ballot(more);
                if (more_l != ~0ull) return n + (uint32_t)__builtin_ctzll(~more_l);
                n += 64;
            }
        };
        auto whole = [](int64_t x, int l) { return ((int64_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)x, l); };
        // (the same runs in the same order in all four wavefronts, so that all of them meet at the barriers)
        uint32_t turn = 0;
        while (firsts) {
            const int l = __builtin_ctzll(firsts);
            firsts &= firsts - 1;
            uint32_t row0 = base + l - 1, n = 1 + (uint32_t)__builtin_ctzll(~(follow >> (l + 1)));
            int64_t slot = whole(slot_l, l);
            if (l + n == 64) n = extend(row0, slot, n);         // the run goes on behind what the wavefront has in view
            // the slot of the next row of this block, -1: there is none
            auto next = [&]() -> int64_t {
                if ((uint32_t)(slot & (bs - 1)) + n >= bs || (uint64_t)row0 + n >= a.n_rows) return -1;
                const int64_t x = whole(a.slots[row0 + n], 0);
                return x >= slot + n && (x >> bs_log) == (slot >> bs_log) ? x : -1;
            };
            const bool gap = __builtin_expect(l + n < 64, 1) ? (behind >> (l + n)) & 1 : next() >= 0;
            if (gap || n > 2 * rows_per_wave) {
                for (;;) {
                    take(row0, slot, n, wave, std::integral_constant<int, 4>{});
                    if (__builtin_expect(!gap, 1)) break;
                    const int64_t x = next();
                    if (x < 0) break;
                    row0 += n;
                    slot = x;
                    n = extend(row0, slot, 1);
                    __syncthreads();                            // (scale and codes of the rows before)
                }
            } else if (turn++ % 4 == wave) {
                take(row0, slot, n, 0u, std::integral_constant<int, 1>{});
            }
        }
    }
}

struct ReadArgs {
    const uint8_t* codes[2];
    const float* scale[2];
    void* out[2];
    const int64_t* slots;
    uint32_t n_rows, n_blocks, n_heads, block_tokens, dim;
};

// Eight values a lane; blockIdx.y: keys or values.  Bound by memory (21500 rows in 32 bits, 220 MB: 42 us, 5.3 TB/s).
template <class T, int CODES>
__global__ __launch_bounds__(256) void read_kernel(ReadArgs a)
{
    const uint32_t part = blockIdx.y, groups = a.dim / 8;
    T* out = (T*)a.out[part];
    if (!out) return;
    const uint32_t i = blockIdx.x * 256 + threadIdx.x, row = i / groups, col = (i - row * groups) * 8, t = row / a.n_heads, head = row - t * a.n_heads;   // (below 2^32)
    if (t >= a.n_rows) return;
    const int64_t slot = a.slots[t];
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const uint32_t bs_log = 31 - __builtin_clz(a.block_tokens);
    if (slot >= 0 && slot < (int64_t)a.n_blocks << bs_log) {
        const uint64_t at = (uint64_t)(slot >> bs_log) * a.n_heads + head;
        const float s = a.scale[part][at];
        const u32x2 w = *reinterpret_cast<const u32x2*>(a.codes[part] + ((at << bs_log) + (uint64_t)(slot & (a.block_tokens - 1))) * a.dim + col);
        float lo[4], hi[4];
        decode4<CODES>(w[0], lo);
        decode4<CODES>(w[1], hi);
#pragma unroll
        for (int j = 0; j < 4; j++) { x[j] = lo[j] * s; x[j + 4] = hi[j] * s; }
    }
    T* to = out + (uint64_t)row * a.dim + col;
    store4<T>(to, x[0], x[1], x[2], x[3]);
    store4<T>(to + 4, x[4], x[5], x[6], x[7]);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

void check_cache(const hnsw_amd_token_cache* c, const char* who)
{
    const std::string w(who);
    if (!c || !c->k_codes || !c->v_codes || !c->k_scale || !c->v_scale) throw std::invalid_argument(w + ": NULL argument");
    if (c->codes != HNSW_AMD_CODES_I8 && c->codes != HNSW_AMD_CODES_E4M3) throw std::invalid_argument(w + ": codes must be HNSW_AMD_CODES_I8 or _E4M3");
    if (c->block_tokens < 16 || c->block_tokens > 256 || (c->block_tokens & (c->block_tokens - 1))) throw std::invalid_argument(w + ": block_tokens must be 16, 32, 64, 128 or 256");
    if (c->dim < 16 || c->dim > 256 || c->dim % 16) throw std::invalid_argument(w + ": dim must be a multiple of 16 up to 256");
    if (c->n_heads < 1 || c->n_blocks < 1) throw std::invalid_argument(w + ": a cache has at least one block and one head");
    if (c->n_blocks > 0x7fffffffu || (unsigned __int128)c->n_blocks * c->n_heads * c->block_tokens > 0xffffffffull)
        throw std::invalid_argument(w + ": at most 2^32 - 1 rows (blocks x heads x block_tokens)");
    if (!aligned16(c->k_codes) || !aligned16(c->v_codes)) throw std::invalid_argument(w + ": codes must be aligned to 16 bytes");
}

void cache_plan(const int32_t* lens, const int32_t* grow, uint32_t n_requests, int32_t* table, uint32_t width, int32_t* ring, uint32_t n_blocks,
                const int64_t* state, uint32_t block_tokens, uint32_t n_slots, int64_t* slots, int32_t* cu_new, int32_t* lens_out,
                int64_t* state_out, int32_t* status, int device, void* stream)
{
    if (n_requests < 1 || n_requests > kMaxRequests) throw std::invalid_argument("cache_plan: 1..8192 requests a call");
    if (block_tokens < 16 || block_tokens > 256 || (block_tokens & (block_tokens - 1))) throw std::invalid_argument("cache_plan: block_tokens must be 16, 32, 64, 128 or 256");
    if (width < 1 || (uint64_t)width * block_tokens > 0x7fffffffull) throw std::invalid_argument("cache_plan: the table's width in tokens must be 1..2^31 - 1");
    if (n_blocks < 1 || n_blocks > 0x7fffffffu) throw std::invalid_argument("cache_plan: n_blocks must be 1..2^31 - 1");
    if (n_slots > 0x7fffffffu) throw std::invalid_argument("cache_plan: n_slots must be below 2^31");
    // every workgroup reads the inputs, while others write
    const uint64_t n = n_requests;
    const struct { const void* at; uint64_t bytes; } in[] = {{lens, 4 * n}, {grow, 4 * n}, {state, 16}},
                                                     out[] = {{slots, 8ull * n_slots}, {cu_new, 4 * (n + 1)}, {lens_out, 4 * n}, {state_out, 16}, {status, 4}};
    for (const auto& i : in)
        for (const auto& o : out)
            if ((uintptr_t)i.at < (uintptr_t)o.at + o.bytes && (uintptr_t)o.at < (uintptr_t)i.at + i.bytes)
                throw std::invalid_argument("cache_plan: the results need buffers of their own");
    const OnDevice on(device);
    // A slot a thread, or four in a row where there are more than a few workgroups of them; 512 workgroups at most.  (64 requests, one slot
    // each: 6.0 us, 7.5 with four.  1000 requests, 318000 slots: 10.7 us, 11.9 with one; 14.3 with workgroups of 1024 whose first threads do
    // all the other work.  All of these with prefix sums that took 2 us more than they do now.)
    const uint32_t per = n_slots > 4096 ? 4 : 1;
    auto whole = [](uint64_t x) { return (x + 63) / 64 * 64; };
    const uint64_t mappers = whole((n_slots + per - 1) / per), takers = whole(n_slots / block_tokens + n_requests), others = whole(n_requests);
    const uint64_t items = mappers + takers + 2 * others;
    const uint32_t threads = items <= 256 ? 256 : 512, groups = (uint32_t)std::min<uint64_t>((items + threads - 1) / threads, 512), stride = groups * threads;
    const PlanArgs a{lens, grow, table, ring, state, slots, cu_new, lens_out, status, state_out, n_requests, width, n_blocks, block_tokens, n_slots, per,
                     (uint32_t)(mappers % stride), (uint32_t)((mappers + takers) % stride), (uint32_t)((mappers + takers + others) % stride)};
    const size_t lds = (size_t)n_requests * 16;
    if (lds > 48 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(plan_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) throw std::runtime_error(std::string("HIP: cache_plan: ") + hipGetErrorString(e));
    }
    hipLaunchKernelGGL(plan_kernel, dim3(groups), dim3(threads), lds, (hipStream_t)stream, a);
    check_launch("cache_plan");
}

void cache_append(const hnsw_amd_token_cache* c, const void* k, const void* v, uint32_t n_rows, uint32_t row_type, int64_t k_row_stride,
                  int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride, const int64_t* slots, int device, void* stream)
{
    check_cache(c, "cache_append");
    check_row_type(row_type, "cache_append");
    if (n_rows == 0) return;
    if (n_rows > 0x7fffffffu) throw std::invalid_argument("cache_append: at most 2^31 - 1 rows");
    const OnDevice on(device);
    AppendArgs a{{(uint8_t*)c->k_codes, (uint8_t*)c->v_codes}, {c->k_scale, c->v_scale}, {k, v}, {k_row_stride, v_row_stride}, {k_head_stride, v_head_stride},
                 slots, n_rows, c->n_blocks, c->n_heads, c->block_tokens, c->dim, 1};
    // A workgroup looks at four rows, so that single tokens run side by side; at more where that would be more than 1024 workgroups, up to 64
    // (a prompt, of whose runs each is one workgroup's).  Measured with reading the blocks back behind it, 8 heads of 128 dims: 64 single
    // rows 8.8 us with 4, 12.3 with 16; 600 rows of three prompts 11.9 with 4, 10.2 with 8; 4000 single rows 194 with 4, 186 with 32; 21500
    // rows of three prompts 118 with 16, 80 with 64 (72 since the rows are kept in 16 bits).
    const uint64_t share = (uint64_t)n_rows * c->n_heads * 2 / 1024;
    a.span = share < 8 ? 4 : share < 16 ? 8 : share < 32 ? 16 : share < 64 ? 32 : 64;
    const uint64_t groups = (uint64_t)((n_rows + a.span - 1) / a.span) * c->n_heads * 2;
    if (groups >= 1ull << 24) throw std::invalid_argument("cache_append: too many rows and heads for one call");
    by_types(row_type, c->codes, [&](auto t, auto codes) {
        using T = decltype(t);
        const int64_t step = 16 / (int64_t)sizeof(T);
        const bool vec = aligned16(k) && aligned16(v) && k_row_stride % step == 0 && k_head_stride % step == 0 && v_row_stride % step == 0 && v_head_stride % step == 0;
        auto go = [&](auto v) { hipLaunchKernelGGL((append_kernel<T, codes.value, v.value>), dim3((uint32_t)groups), dim3(256), 0, (hipStream_t)stream, a); };
        if (vec) go(std::true_type{});
        else go(std::false_type{});
    });
    check_launch("cache_append");
}

void cache_read(const hnsw_amd_token_cache* c, const int64_t* slots, uint32_t n_rows, uint32_t row_type, void* k, void* v, int device, void* stream)
{
    check_cache(c, "cache_read");
    check_row_type(row_type, "cache_read");
    if (n_rows == 0 || (!k && !v)) return;
    if (!aligned16(k) || !aligned16(v)) throw std::invalid_argument("cache_read: outputs must be aligned to 16 bytes");
    const uint64_t groups = ((uint64_t)n_rows * c->n_heads * (c->dim / 8) + 255) / 256;
    if (groups >= 1ull << 24) throw std::invalid_argument("cache_read: too many rows for one call");
    const OnDevice on(device);
    const ReadArgs a{{(const uint8_t*)c->k_codes, (const uint8_t*)c->v_codes}, {c->k_scale, c->v_scale}, {k, v}, slots, n_rows, c->n_blocks, c->n_heads, c->block_tokens, c->dim};
    by_types(row_type, c->codes, [&](auto t, auto codes) {
        hipLaunchKernelGGL((read_kernel<decltype(t), codes.value>), dim3((uint32_t)groups, 2), dim3(256), 0, (hipStream_t)stream, a);
    });
    check_launch("cache_read");
}

}  // namespace hnsw_amd
