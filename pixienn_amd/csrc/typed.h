// Vectors of 32- and 16-bit floating values in memory, and their conversion from and to fp32.
#pragma once

#include "common.h"

namespace pxh {

template<int T>
constexpr int kSize = T == PXH_F32 ? 4 : T == PXH_E4M3 ? 1 : 2;

inline size_t size_of(int type) { return type == PXH_F32 ? 4 : type == PXH_E4M3 ? 1 : 2; }

// Values of one 128-bit access.
template<int T>
constexpr int kVec = 16 / kSize<T>;

__device__ __forceinline__ float bf16_up(uint32_t low) { return __uint_as_float(low << 16); }

// Two fp32 values as a pair of 16-bit ones, rounded to nearest even (one instruction for bf16).
template<int T>
__device__ __forceinline__ uint32_t pair_of(float a, float b)
{
    if constexpr (T == PXH_BF16) {
        typedef __bf16 two __attribute__((ext_vector_type(2)));
        const two t = { static_cast<__bf16>(a), static_cast<__bf16>(b) };
        return __builtin_bit_cast(uint32_t, t);
    } else {
        typedef _Float16 two __attribute__((ext_vector_type(2)));
        const two t = { static_cast<_Float16>(a), static_cast<_Float16>(b) };
        return __builtin_bit_cast(uint32_t, t);
    }
}

// The two values of a word of 16-bit ones.
template<int T>
__device__ __forceinline__ void unpair(uint32_t w, float& a, float& b)
{
    if constexpr (T == PXH_BF16) {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xffff0000u);
    } else {
        typedef _Float16 two __attribute__((ext_vector_type(2)));
        const two t = __builtin_bit_cast(two, w);
        a = static_cast<float>(t.x);
        b = static_cast<float>(t.y);
    }
}

// V values of type T as raw words.
template<int T, int V>
struct Raw {
    static constexpr int kWords = V * kSize<T> / 4;
    uint32_t w[kWords];

    __device__ __forceinline__ void get(float (&x)[V]) const
    {
        if constexpr (T == PXH_F32) {
#pragma unroll
            for (int k = 0; k < V; ++k) x[k] = __uint_as_float(w[k]);
        } else {
#pragma unroll
            for (int k = 0; k < kWords; ++k) unpair<T>(w[k], x[2 * k], x[2 * k + 1]);
        }
    }
    __device__ __forceinline__ void set(const float (&x)[V])
    {
        if constexpr (T == PXH_F32) {
#pragma unroll
            for (int k = 0; k < V; ++k) w[k] = __float_as_uint(x[k]);
        } else {
#pragma unroll
            for (int k = 0; k < kWords; ++k) w[k] = pair_of<T>(x[2 * k], x[2 * k + 1]);
        }
    }
};

// Global memory, whatever the compiler knows of a pointer: one that comes out of a table in memory would be accessed as one that
// may as well lie in LDS, and waited for as such.
template<typename W>
__device__ __forceinline__ auto global_memory(const void* p) { return (const __attribute__((address_space(1))) W*) p; }
template<typename W>
__device__ __forceinline__ auto global_memory(void* p) { return (__attribute__((address_space(1))) W*) p; }

// V values at element e of p, as one access of up to 128 bits; NT: past the caches.  The access takes any alignment: the
// hardware has 128-bit accesses at every byte, and a row of an odd number of 16-bit values begins at a multiple of 2, so
// that no row needs another form for where it begins.
template<int T, int V, bool NT = false>
__device__ __forceinline__ Raw<T, V> load_raw(const void* p, size_t e)
{
    constexpr int N = V * kSize<T>;
    static_assert(N <= 16, "one access");
    typedef uint32_t words __attribute__((ext_vector_type(N / 4), aligned(1)));
    const auto at = global_memory<words>(static_cast<const char*>(p) + e * kSize<T>);
    const words b = NT ? __builtin_nontemporal_load(at) : *at;
    return __builtin_bit_cast(Raw<T, V>, b);
}

template<int T, int V, bool NT = false>
__device__ __forceinline__ void store_raw(void* p, size_t e, const Raw<T, V>& r)
{
    constexpr int N = V * kSize<T>;
    static_assert(N <= 16, "one access");
    typedef uint32_t words __attribute__((ext_vector_type(N / 4), aligned(1)));
    const auto at = global_memory<words>(static_cast<char*>(p) + e * kSize<T>);
    const words b = __builtin_bit_cast(words, r);
    if constexpr (NT) __builtin_nontemporal_store(b, at);
    else *at = b;
}

// The same at a byte offset of the lane's own from a place that is the workgroup's: an address in scalar registers, one
// register for the offset however many vectors a lane holds.
template<int T, int V, bool NT = false>
__device__ __forceinline__ Raw<T, V> load_raw_at(const char* place, uint32_t offset)
{
    return load_raw<T, V, NT>(place + offset, 0);
}

template<int T, int V, bool NT = false>
__device__ __forceinline__ void store_raw_at(char* place, uint32_t offset, const Raw<T, V>& r)
{
    store_raw<T, V, NT>(place + offset, 0, r);
}

// One value.
template<int T>
__device__ __forceinline__ float load_one(const void* p, size_t e)
{
    if constexpr (T == PXH_F32) return global_memory<float>(p)[e];
    else {
        const uint32_t h = global_memory<uint16_t>(p)[e];
        if constexpr (T == PXH_BF16) return bf16_up(h);
        else return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(h)));
    }
}

template<int T>
__device__ __forceinline__ void store_one(void* p, size_t e, float x)
{
    if constexpr (T == PXH_F32) global_memory<float>(p)[e] = x;
    else global_memory<uint16_t>(p)[e] = static_cast<uint16_t>(pair_of<T>(x, x));
}

// x rounded to T and back.
template<int T>
__device__ __forceinline__ float rounded(float x)
{
    if constexpr (T == PXH_F32) return x;
    else {
        float a, b;
        unpair<T>(pair_of<T>(x, x), a, b);
        return a;
    }
}

// V values at element e < n of a row of n, the row's last ones, and `fill` behind them: without a branch, so that several such
// loads go out together.
template<int T, int V>
__device__ __forceinline__ Raw<T, V> load_end(const void* p, int e, int n, float fill = 0.0f)
{
    float x[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const float l = load_one<T>(p, min(e + k, n - 1));
        x[k] = e + k < n ? l : fill;
    }
    Raw<T, V> r;
    r.set(x);
    return r;
}

// V values at element e of a row of n: whole vectors in one access, the row's last ones value by value, and `fill` behind them.
template<int T, int V, bool NT = false>
__device__ __forceinline__ Raw<T, V> load_row(const void* p, int e, int n, float fill = 0.0f)
{
    if (e + V <= n) return load_raw<T, V, NT>(p, e);
    return load_end<T, V>(p, e, n, fill);
}

template<int T, int V, bool NT = false>
__device__ __forceinline__ void store_row(void* p, int e, int n, const Raw<T, V>& r)
{
    if (e + V <= n) {
        store_raw<T, V, NT>(p, e, r);
        return;
    }
    float x[V];
    r.get(x);
#pragma unroll
    for (int k = 0; k < V; ++k)
        if (e + k < n) store_one<T>(p, e + k, x[k]);
}

// The scale of e4m3 values of which the largest magnitude is `peak`: a product with 1/448, as torch has a quotient by a number, so that
// its operations give the same codes (a unit of a scale turns one code of 10^6 that are rounded stochastically, and as many at a tie).
constexpr float kE4m3Max = 448.0f;
constexpr float kLeastScale = 0x1p-126f;        // its reciprocal is finite, and zeros have zeros
constexpr float kMostScale = 0x1.fffffep+127f;  // beside an infinity the others are zeros

__device__ __forceinline__ float scale_of(float peak) { return __builtin_amdgcn_fmed3f(peak * (1.0f / kE4m3Max), kLeastScale, kMostScale); }

// x / scale from the scale's rounded reciprocal and one correction by the remainder (Markstein), which is the rounded quotient.
__device__ __forceinline__ float quotient_of(float x, float scale, float inverse)
{
    const float q = x * inverse;
    return fmaf(fmaf(-q, scale, x), inverse, q);
}

// Calls f.template operator()<T>() for a run-time type of values; false for another one.
template<typename F>
inline bool dispatch_type(int type, F&& f)
{
    switch (type) {
    case PXH_F32: f.template operator()<PXH_F32>(); return true;
    case PXH_BF16: f.template operator()<PXH_BF16>(); return true;
    case PXH_F16: f.template operator()<PXH_F16>(); return true;
    default: return false;
    }
}

// The sum over a workgroup of LANES lanes, the same in every lane; `slots` is LDS of a float per wave.
template<int LANES>
__device__ __forceinline__ float group_sum(float v, float* slots)
{
    v = wave_sum_by_rows(v);
    if constexpr (LANES > kWave) {
        const int wave = threadIdx.x / kWave;
        if ((threadIdx.x & (kWave - 1)) == 0) slots[wave] = v;
        __syncthreads();
        v = slots[0];
#pragma unroll
        for (int k = 1; k < LANES / kWave; ++k) v += slots[k];
        __syncthreads();
    }
    return v;
}

}  // namespace pxh
