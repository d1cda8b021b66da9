// Rows of values and the sums of their columns, for the norms.
#pragma once

#include "typed.h"

namespace pxh {

// Rows of one launch: a grid has fewer than 2^32 work items.
constexpr long long kLaunchRows = 1 << 21;

template<int T>
__host__ __device__ __forceinline__ const char* row_of(const void* p, long long row, long long stride)
{
    return static_cast<const char*>(p) + row * stride * kSize<T>;
}

template<int T>
__host__ __device__ __forceinline__ char* row_of(void* p, long long row, long long stride)
{
    return static_cast<char*>(p) + row * stride * kSize<T>;
}

// V weights from column e on; zeros behind the last one.
template<int T, int V>
__device__ __forceinline__ void weights_at(const void* weight, bool f32, int e, int width, float (&w)[V])
{
    if (f32 && T != PXH_F32) {
#pragma unroll
        for (int q = 0; q < V; q += 4) {
            float part[4];
            load_row<PXH_F32, 4>(weight, e + q, width).get(part);
#pragma unroll
            for (int k = 0; k < 4; ++k) w[q + k] = part[k];
        }
    } else {
        load_row<T, V>(weight, e, width).get(w);
    }
}

// Over the workers' rows of partial sums, `pitch` values apart: a workgroup of 1024 lanes takes 64 columns, and its waves share the
// workers.  The total is in the first wave's lanes; `sums` is LDS.  All lanes call it.
constexpr int kColumnLanes = 1024, kColumnWaves = kColumnLanes / kWave;

__device__ __forceinline__ float sum_of_workers(const float* partial, int workers, size_t pitch, int column, bool there,
                                                float (&sums)[kColumnWaves][kWave])
{
    constexpr int kAhead = 8;
    const int wave = threadIdx.x / kWave;
    float sum = 0.0f;
    if (there) {
        int w = wave;
        for (; w + (kAhead - 1) * kColumnWaves < workers; w += kAhead * kColumnWaves) {
            float v[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) v[k] = partial[static_cast<size_t>(w + k * kColumnWaves) * pitch + column];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) sum += v[k];
        }
        for (; w < workers; w += kColumnWaves) sum += partial[static_cast<size_t>(w) * pitch + column];
    }
    sums[wave][threadIdx.x % kWave] = sum;
    __syncthreads();
    float all = 0.0f;
    if (wave == 0) {
#pragma unroll
        for (int k = 0; k < kColumnWaves; ++k) all += sums[k][threadIdx.x];
    }
    return all;
}

// What the entry points of a norm refuse alike.
inline int check_norm_rows(const char* who, int type, int weight_type, long long rows, int width)
{
    if (type != PXH_F32 && type != PXH_BF16 && type != PXH_F16) return fail_invalid("%s: type %d is not fp32, bf16 or half", who, type);
    if (weight_type != type && weight_type != PXH_F32)
        return fail_invalid("%s: the weights are of the tensors' type or fp32 (got type %d)", who, weight_type);
    if (rows < 0 || rows > 0x7fffffffll) return fail_invalid("%s: %lld rows", who, rows);
    if (width <= 0 || width > 1 << 30) return fail_invalid("%s: rows of %d values", who, width);
    return PXH_OK;
}

}  // namespace pxh
