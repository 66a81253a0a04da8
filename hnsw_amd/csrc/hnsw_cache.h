// Shared pieces of the token cache's kernels (hnsw_cache.hip: planning, writing and reading; hnsw_attend.hip: attention).
#pragma once
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <cstdint>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "../../include/hnsw_amd.h"

namespace hnsw_amd {

// Makes `device` current for the scope of a call and puts the caller's device back.
class OnDevice {
public:
    explicit OnDevice(int device)
    {
        hipError_t e = hipGetDevice(&before_);
        if (e == hipSuccess && before_ != device) { e = hipSetDevice(device); moved_ = e == hipSuccess; }
        if (e != hipSuccess) throw std::runtime_error(std::string("HIP: selecting the device: ") + hipGetErrorString(e));
    }
    ~OnDevice() { if (moved_) (void)hipSetDevice(before_); }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;

private:
    int before_ = 0;
    bool moved_ = false;
};

inline void check_launch(const char* what)
{
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) throw std::runtime_error(std::string("HIP: ") + what + " launch: " + hipGetErrorString(e));
}

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

struct bf16 { uint16_t bits; };

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(_Float16 x) { return (float)x; }
__device__ __forceinline__ float to_float(bf16 x) { return __uint_as_float((uint32_t)x.bits << 16); }
template <class T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float<float>(float x) { return x; }
template <> __device__ __forceinline__ _Float16 from_float<_Float16>(float x) { return (_Float16)x; }
template <> __device__ __forceinline__ bf16 from_float<bf16>(float x) { return bf16{__builtin_bit_cast(uint16_t, (__bf16)x)}; }

// Two values as two 16-bit ones in a word (rounded to nearest, ties to even).
template <class T> __device__ __forceinline__ uint32_t pack2(float x, float y)
{
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    if constexpr (std::is_same_v<T, bf16>) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, bf16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{x, y}, f16x2));
}
// Four consecutive outputs (the address is a multiple of 8 bytes).
template <class T> __device__ __forceinline__ void store4(T* to, float a, float b, float c, float d)
{
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(to) = make_float4(a, b, c, d);
    else *reinterpret_cast<u32x2*>(to) = u32x2{pack2<T>(a, b), pack2<T>(c, d)};
}

// Eight elements of a row as they lie in memory (half the registers of their values where they have 16 bits);
// VEC: the address is a multiple of 16 bytes.
template <class T> struct Eight {
    uint32_t w[2 * sizeof(T)];
    __device__ __forceinline__ float operator[](int j) const
    {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
        else return to_float(__builtin_bit_cast(T, (uint16_t)(w[j >> 1] >> (16 * (j & 1)))));
    }
};
template <class T, bool VEC> __device__ __forceinline__ void load8(const T* p, Eight<T>& x)
{
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) {
            const u32x4 w = reinterpret_cast<const u32x4*>(p)[i];
#pragma unroll
            for (int j = 0; j < 4; j++) x.w[4 * i + j] = w[j];
        }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 8; j++) x.w[j] = __float_as_uint(p[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) x.w[j] = (uint32_t)__builtin_bit_cast(uint16_t, p[2 * j]) | (uint32_t)__builtin_bit_cast(uint16_t, p[2 * j + 1]) << 16;
    }
}

// Values of the four codes in a word.
template <int CODES> __device__ __forceinline__ void decode4(uint32_t w, float (&x)[4])
{
    if constexpr (CODES == HNSW_AMD_CODES_I8) {
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = (float)(int8_t)(w >> (8 * j));
    } else {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        x[0] = a[0]; x[1] = a[1]; x[2] = b[0]; x[3] = b[1];
    }
}
template <int CODES> constexpr float kCodeMax = CODES == HNSW_AMD_CODES_I8 ? 127.0f : 448.0f;

// The codes of four values that are already divided by their scale: rounded to nearest, ties to even, infinities and what
// lies outside the range at the largest code, NaN as 0 (a code of a live token is always finite).
template <int CODES> __device__ __forceinline__ uint32_t encode4(const float (&x)[4])
{
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        y[j] = fminf(fmaxf(x[j], -kCodeMax<CODES>), kCodeMax<CODES>);
        y[j] = x[j] != x[j] ? 0.0f : y[j];
    }
    if constexpr (CODES == HNSW_AMD_CODES_I8) {
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) w |= ((uint32_t)(int)rintf(y[j]) & 0xffu) << (8 * j);
        return w;
    } else {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
    }
}

// Across the 64 lanes with the data-parallel moves of the vector unit, which take a few cycles where a shuffle through LDS takes a hundred.
__device__ __forceinline__ uint32_t wave_inclusive_sum(uint32_t x)
{
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xf, 0xf, false);      // 1, 2, 4, 8 lanes up within 16
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xf, 0xf, false);
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xa, 0xf, false);      // the last lane of 16 to the next 16
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xc, 0xf, false);      // the last lane of 32 to the other 32
    return x;
}
__device__ __forceinline__ float wave_max_not_negative(float y)
{
    int x = __float_as_int(y);                                  // (floats that are not negative are ordered as integers)
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
    return __int_as_float(__builtin_amdgcn_readlane(x, 63));
}

// The request that row t belongs to: largest b with cu[b] <= t (cu ascending, cu[0] = 0); n when t is behind the last one.
__device__ __forceinline__ uint32_t request_of(const int32_t* cu, uint32_t n, uint32_t t)
{
    if ((int64_t)t >= (int64_t)cu[n]) return n;
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if ((int64_t)cu[mid] <= (int64_t)t) lo = mid; else hi = mid;
    }
    return lo;
}

void check_cache(const hnsw_amd_token_cache* c, const char* who);

inline void check_row_type(uint32_t row_type, const char* who)
{
    if (row_type > HNSW_AMD_TYPE_BF16) throw std::invalid_argument(std::string(who) + ": row type must be HNSW_AMD_TYPE_F32, _F16 or _BF16");
}

// f(T{}, integral_constant<codes>) for the types of a call (checked before).
template <class F> void by_types(uint32_t row_type, uint32_t codes, F&& f)
{
    auto both = [&](auto t) {
        if (codes == HNSW_AMD_CODES_I8) f(t, std::integral_constant<int, HNSW_AMD_CODES_I8>{});
        else f(t, std::integral_constant<int, HNSW_AMD_CODES_E4M3>{});
    };
    if (row_type == HNSW_AMD_TYPE_F32) both(float{});
    else if (row_type == HNSW_AMD_TYPE_F16) both(_Float16{});
    else both(bf16{});
}

}  // namespace hnsw_amd
