// Root-mean-square norm over rows, with the residual's addition in front of it and 8-bit results, and its gradients.
#include "rows.h"
#include "stream.h"

namespace pxh {
namespace {

// ---------------------------------------------------------------- forward
//   h = x + residual (rounded as it is kept);  rstd = 1 / sqrt(mean(h^2) + eps);  y = h * rstd * weight
struct NormArgs {
    const void* x;
    const void* residual;
    void* sum;
    const void* weight;
    void* y;
    float* scales;
    float* rstd;
    long long rows, x_stride, residual_stride, sum_stride, y_stride;
    int width, group;
    float eps;
};

// The largest value among the lanes that hold one group of 128 values: 16 lanes of 8 values or 32 of 4.
template<int V>
__device__ __forceinline__ float scale_group_max(float v)
{
    v = fmaxf(v, lane_in_row<0xB1>(v));
    v = fmaxf(v, lane_in_row<0x4E>(v));
    v = fmaxf(v, lane_in_row<0x141>(v));
    v = fmaxf(v, lane_in_row<0x140>(v));
    if constexpr (V == 4) v = fmaxf(v, __shfl_xor(v, 16, kWave));
    return v;
}

// Four values no larger than 448 by more than a rounding: the conversion rounds to nearest even and leaves NaN.
__device__ __forceinline__ uint32_t e4m3_of(float a, float b, float c, float d)
{
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
    return static_cast<uint32_t>(w);
}

// V 8-bit values at column e of a row of n.
template<int V>
__device__ __forceinline__ void store_e4m3(char* y, int e, int n, const float (&q)[V])
{
    uint32_t w[V / 4];
#pragma unroll
    for (int k = 0; k < V / 4; ++k) w[k] = e4m3_of(q[4 * k], q[4 * k + 1], q[4 * k + 2], q[4 * k + 3]);
    if (e + V <= n) {
        typedef uint32_t words __attribute__((ext_vector_type(V / 4), aligned(1)));
        *reinterpret_cast<words*>(y + e) = __builtin_bit_cast(words, w);
        return;
    }
#pragma unroll
    for (int k = 0; k < V; ++k)
        if (e + k < n) y[e + k] = static_cast<char>(w[k / 4] >> (8 * (k & 3)));
}

// V values of a row and what goes with them: the residual and the weights.
template<int T, bool WIDE>
struct NormVector {
    static constexpr int V = kVec<T>;
    static constexpr int W = WIDE ? PXH_F32 : T;
    static constexpr int kParts = V * kSize<W> / 16;                // accesses for the weights
    static constexpr int kPart = V / kParts;
    Raw<T, V> h, more;
    Raw<W, kPart> w[kParts];

    template<bool NT>
    __device__ __forceinline__ void load(const NormArgs& a, const char* x, const char* residual, int e)
    {
        const int n = a.width;
        if (e + V <= n) {
            h = load_raw<T, V, NT>(x, e);
            if (residual) more = load_raw<T, V, NT>(residual, e);
#pragma unroll
            for (int q = 0; q < kParts; ++q) w[q] = load_raw<W, kPart>(a.weight, e + q * kPart);
        } else if (e < n) {
            h = load_end<T, V>(x, e, n);
            if (residual) more = load_end<T, V>(residual, e, n);
#pragma unroll
            for (int q = 0; q < kParts; ++q) w[q] = load_end<W, kPart>(a.weight, e + q * kPart, n);
        }
    }

    // h with the residual, rounded as it is kept
    __device__ __forceinline__ void add()
    {
        float p[V], q[V];
        h.get(p);
        more.get(q);
#pragma unroll
        for (int k = 0; k < V; ++k) p[k] += q[k];
        h.set(p);
    }

    __device__ __forceinline__ void weights(float (&out)[V]) const
    {
#pragma unroll
        for (int q = 0; q < kParts; ++q) {
            float part[kPart];
            w[q].get(part);
#pragma unroll
            for (int k = 0; k < kPart; ++k) out[q * kPart + k] = part[k];
        }
    }
};

// A row is walked in vectors, lane by lane.  K vectors a lane stay in registers between the sum and the result; the residual and the
// weights are asked for with the row, so that there is one trip to memory.  K == 0: a row of any width, which is read again.
// Bound by its streams: 4096 x 8192 bf16 with a residual and the sum kept, to 8 bits with a scale for 128, is 236 MB in 39.7 us,
// 5.9 TB/s where a copy has 6.6; 8 x 4096 is one launch, 3.8 us (an empty one 3.5).
template<int T, bool EIGHT, bool WIDE, int LANES, int K, bool NT>
__global__ __launch_bounds__(LANES > kWave ? LANES : kBlock) void rms_norm_kernel(NormArgs a)
{
    constexpr int V = kVec<T>;
    constexpr int kRows = LANES > kWave ? 1 : kBlock / kWave;       // rows per workgroup, a wave each if several
    constexpr int kUnroll = K ? K : 1;
    __shared__ float2 slots[LANES / kWave];
    const int lane = threadIdx.x % LANES;
    const long long row = static_cast<long long>(blockIdx.x) * kRows + threadIdx.x / LANES;
    if (row >= a.rows) return;                                       // whole waves, and only where nothing is waited for
    const char* x = row_of<T>(a.x, row, a.x_stride);
    const char* residual = a.residual ? row_of<T>(a.residual, row, a.residual_stride) : nullptr;
    char* sum = a.sum ? row_of<T>(a.sum, row, a.sum_stride) : nullptr;
    const int n = a.width;
    const int steps = K ? K : (n + LANES * V - 1) / (LANES * V);
    const bool whole_row = EIGHT && a.group == 0;

    NormVector<T, WIDE> kept[kUnroll];
    if constexpr (K > 0) {
#pragma unroll
        for (int s = 0; s < K; ++s) {
            kept[s] = NormVector<T, WIDE>{};
            kept[s].template load<NT>(a, x, residual, (s * LANES + lane) * V);
        }
    }
    float squares = 0.0f, peak = 0.0f;
#pragma unroll kUnroll
    for (int s = 0; s < steps; ++s) {
        const int e = (s * LANES + lane) * V;
        if (e >= n) break;
        NormVector<T, WIDE>& v = kept[K ? s : 0];
        if constexpr (K == 0) v.template load<NT>(a, x, residual, e);
        if (residual) {
            v.add();
            if (sum) store_row<T, V, NT>(sum, e, n, v.h);
        }
        float h[V];
        v.h.get(h);
#pragma unroll
        for (int k = 0; k < V; ++k) squares = fmaf(h[k], h[k], squares);
        if (whole_row) {
            float w[V];
            v.weights(w);
#pragma unroll
            for (int k = 0; k < V; ++k) peak = fmaxf(peak, fabsf(h[k] * w[k]));
        }
    }
    squares = wave_sum_by_rows(squares);
    if (whole_row) peak = wave_max_by_rows(peak);
    if constexpr (LANES > kWave) {
        if ((lane & (kWave - 1)) == 0) slots[lane / kWave] = make_float2(squares, peak);
        __syncthreads();
        squares = 0.0f;
#pragma unroll
        for (int k = 0; k < LANES / kWave; ++k) {
            squares += slots[k].x;
            peak = fmaxf(peak, slots[k].y);
        }
    }
    const float rstd = 1.0f / sqrtf(squares / static_cast<float>(n) + a.eps);
    if (a.rstd && lane == 0) a.rstd[row] = rstd;
    float scale = 1.0f, inverse = 1.0f;
    if (whole_row) {
        scale = scale_of(peak * rstd);
        inverse = 1.0f / scale;
        if (lane == 0) a.scales[row] = scale;
    }
    const int groups = (n + 127) / 128;
#pragma unroll kUnroll
    for (int s = 0; s < steps; ++s) {
        const int e = (s * LANES + lane) * V;
        // with a scale per group all lanes of a wave go on together
        if ((s * LANES + lane / kWave * kWave) * V >= n) break;
        NormVector<T, WIDE>& v = kept[K ? s : 0];
        if constexpr (K == 0) {
            v = NormVector<T, WIDE>{};
            // x may have been overwritten by the sum, which is what is wanted
            v.template load<NT>(a, sum ? sum : x, sum ? nullptr : residual, e);
            if (residual && !sum) v.add();
        }
        float y[V], w[V];
        v.h.get(y);
        v.weights(w);
#pragma unroll
        for (int k = 0; k < V; ++k) y[k] = y[k] * rstd * w[k];
        if constexpr (EIGHT) {
            if (a.group) {
                float most = 0.0f;
#pragma unroll
                for (int k = 0; k < V; ++k) most = fmaxf(most, fabsf(y[k]));
                scale = scale_of(scale_group_max<V>(most));
                inverse = 1.0f / scale;
                if (e % 128 == 0 && e < n) a.scales[row * groups + e / 128] = scale;
            }
#pragma unroll
            for (int k = 0; k < V; ++k) y[k] = quotient_of(y[k], scale, inverse);
            if (e < n) store_e4m3<V>(static_cast<char*>(a.y) + row * a.y_stride, e, n, y);
        } else {
            Raw<T, V> r;
            r.set(y);
            if (e < n) store_row<T, V, NT>(row_of<T>(a.y, row, a.y_stride), e, n, r);
        }
    }
}

template<int T, bool EIGHT, bool WIDE, int LANES, int K, bool NT>
int launch_norm(const NormArgs& a, hipStream_t s)
{
    constexpr int kRows = LANES > kWave ? 1 : kBlock / kWave;
    for (long long done = 0; done < a.rows; done += kLaunchRows) {
        NormArgs part = a;
        part.x = row_of<T>(a.x, done, a.x_stride);
        part.residual = a.residual ? row_of<T>(a.residual, done, a.residual_stride) : nullptr;
        part.sum = a.sum ? row_of<T>(a.sum, done, a.sum_stride) : nullptr;
        part.y = static_cast<char*>(a.y) + done * a.y_stride * (EIGHT ? 1 : kSize<T>);
        part.scales = a.scales + (EIGHT ? done * (a.group ? (a.width + 127) / 128 : 1) : 0);
        part.rstd = a.rstd ? a.rstd + done : nullptr;
        part.rows = a.rows - done < kLaunchRows ? a.rows - done : kLaunchRows;
        const dim3 grid(grid_for(part.rows, kRows)), block(kRows * LANES);
        hipLaunchKernelGGL((rms_norm_kernel<T, EIGHT, WIDE, LANES, K, NT>), grid, block, 0, s, part);
        if (int rc = check_launch("pxh_rms_norm_forward")) return rc;
    }
    return PXH_OK;
}

// Lanes and vectors a lane, by the vectors of a row: few vectors while the row is short, whose time is that of one trip through the chain
// (1024 x 8192 bf16: 512 lanes of two 11.2 us, 1024 of one 12.5, 256 of four 11.5; 1111 x 1537 fp32: 256 of two 4.3, 512 of one
// 4.8; 8 x 4096 bf16 128 of four 4.5, and 3.7).  Beyond 2048 vectors 512 lanes of eight would win some and lose some (2048 x 20001
// with a residual 66.6 us in place of 72.6, 4000 x 32768 without one 104.8 in place of 101.1, 8 x 32768 6.5 in place of 5.9).
// NT, past the caches, where the tensors do not fit: 4096 x 8192 to 8 bits 44.5 -> 39.7 us, 16384 x 4096 92.3 -> 88.7; 2048 x 4096 would go
// from 11.3 to 13.5.
template<int T, bool EIGHT, bool WIDE, bool NT>
int norm_forward(const NormArgs& a, hipStream_t s)
{
    const int vectors = (a.width + kVec<T> - 1) / kVec<T>;
    if (vectors <= 64) return launch_norm<T, EIGHT, WIDE, 64, 1, NT>(a, s);
    if (vectors <= 128) return launch_norm<T, EIGHT, WIDE, 128, 1, NT>(a, s);
    if (vectors <= 256) return launch_norm<T, EIGHT, WIDE, 256, 1, NT>(a, s);
    if (vectors <= 512) return launch_norm<T, EIGHT, WIDE, 256, 2, NT>(a, s);
    if (vectors <= 1024) return launch_norm<T, EIGHT, WIDE, 512, 2, NT>(a, s);
    if (vectors <= 2048) return launch_norm<T, EIGHT, WIDE, 1024, 2, NT>(a, s);
    if (vectors <= 4096) return launch_norm<T, EIGHT, WIDE, 1024, 4, NT>(a, s);
    return launch_norm<T, EIGHT, WIDE, 1024, 0, false>(a, s);           // read twice: through the caches
}

template<int T, bool EIGHT, bool WIDE>
int norm_forward(const NormArgs& a, hipStream_t s)
{
    const size_t tensors = 1 + (a.residual != nullptr) + (a.sum != nullptr) + !EIGHT;
    const bool past = static_cast<size_t>(a.rows) * static_cast<size_t>(a.width) * kSize<T> * tensors >= kStreamingBytes;
    return past ? norm_forward<T, EIGHT, WIDE, true>(a, s) : norm_forward<T, EIGHT, WIDE, false>(a, s);
}

// ---------------------------------------------------------------- backward
struct NormBackwardArgs {
    const void* dy;
    const void* h;
    const void* weight;
    const float* rstd;
    const void* dsum;
    void* dx;
    float* partial;         // [workers][width]
    long long rows, dy_stride, h_stride, dsum_stride, dx_stride;
    int width;
    bool weight_f32;
};

// dx of every row, and the part of dw that this worker's rows give: a worker (LANES lanes) takes every workers-th row, and asks for
// the next one before it waits for the sum over this one.  At four vectors a lane there are no registers for that, nor for
// the weights, which are read again for every row.  The widest forms for 16 bits spill all the same, at two vectors 17 registers and at
// four 142, most of them for the rows' ends, value by value in every step: 4096 x 16384 bf16 with dsum is 537 MB in 100.5 us, 5.3 TB/s, and
// 2048 x 32768 takes 166.  16384 x 4096 bf16 with dsum: 537 MB in 88.7 us with the launch that adds up dw,
// 6.05 TB/s, where a kernel that only moves three streams in and one out has 6.3.
template<int T, int LANES, int K, bool NT>
__global__ __launch_bounds__(LANES > kWave ? LANES : kBlock) void rms_norm_backward_kernel(NormBackwardArgs a, int workers)
{
    constexpr int V = kVec<T>;
    constexpr int kPer = LANES > kWave ? 1 : kBlock / kWave;
    constexpr int kWaves = LANES / kWave;
    constexpr bool kAhead = K <= 2;
    __shared__ float slots[2][kWaves];
    const int lane = threadIdx.x % LANES;
    const int worker = blockIdx.x * kPer + threadIdx.x / LANES;
    if (worker >= workers) return;              // single waves, which wait for nobody
    const int n = a.width;
    float w[kAhead ? K : 1][V], dw[K][V];
#pragma unroll
    for (int s = 0; s < K; ++s) {
        const int e = (s * LANES + lane) * V;
#pragma unroll
        for (int k = 0; k < V; ++k) dw[s][k] = 0.0f;
        if (kAhead) {
#pragma unroll
            for (int k = 0; k < V; ++k) w[s][k] = 0.0f;
            if (e < n) weights_at<T, V>(a.weight, a.weight_f32, e, n, w[s]);
        }
    }
    struct Row {
        Raw<T, V> g[K], h[K], more[K];
        float rstd;
    };
    const auto ask = [&](long long row, Row& r) {
        if (row >= a.rows) return;
        const char* dy = row_of<T>(a.dy, row, a.dy_stride);
        const char* h = row_of<T>(a.h, row, a.h_stride);
        r.rstd = a.rstd[row];
#pragma unroll
        for (int s = 0; s < K; ++s) {
            const int e = (s * LANES + lane) * V;
            if (e >= n) break;
            r.g[s] = load_row<T, V, NT>(dy, e, n);
            r.h[s] = load_row<T, V, NT>(h, e, n);
            if (kAhead && a.dsum) r.more[s] = load_row<T, V, NT>(row_of<T>(a.dsum, row, a.dsum_stride), e, n);
        }
    };
    Row next;
    if (kAhead) ask(worker, next);
    int turn = 0;
    for (long long row = worker; row < a.rows; row += workers) {
        if (!kAhead) ask(row, next);
        const Row r = next;
        float dot = 0.0f;
#pragma unroll
        for (int s = 0; s < K; ++s) {
            const int e = (s * LANES + lane) * V;
            if (e >= n) break;
            float g[V], x[V], u[V];
            r.g[s].get(g);
            r.h[s].get(x);
            if (!kAhead) weights_at<T, V>(a.weight, a.weight_f32, e, n, u);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float xhat = x[k] * r.rstd;
                dw[s][k] = fmaf(g[k], xhat, dw[s][k]);
                dot = fmaf(g[k] * (kAhead ? w[kAhead ? s : 0][k] : u[k]), xhat, dot);
            }
        }
        if (kAhead) ask(row + workers, next);
        dot = wave_sum_by_rows(dot);
        if constexpr (kWaves > 1) {
            // two places in turn: no wave is more than one row ahead of another
            float* const slot = slots[turn];
            turn ^= 1;
            if ((lane & (kWave - 1)) == 0) slot[lane / kWave] = dot;
            __syncthreads();
            dot = slot[0];
#pragma unroll
            for (int k = 1; k < kWaves; ++k) dot += slot[k];
        }
        const float c = r.rstd * (dot / static_cast<float>(n));
#pragma unroll
        for (int s = 0; s < K; ++s) {
            const int e = (s * LANES + lane) * V;
            if (e >= n) break;
            float g[V], x[V], u[V], more[V] = {};
            r.g[s].get(g);
            r.h[s].get(x);
            if (!kAhead) weights_at<T, V>(a.weight, a.weight_f32, e, n, u);
            if (a.dsum) {
                if (kAhead) r.more[s].get(more);
                else load_row<T, V>(row_of<T>(a.dsum, row, a.dsum_stride), e, n).get(more);
            }
#pragma unroll
            for (int k = 0; k < V; ++k) g[k] = fmaf(r.rstd, g[k] * (kAhead ? w[kAhead ? s : 0][k] : u[k]) - x[k] * c, more[k]);
            Raw<T, V> out;
            out.set(g);
            store_row<T, V, NT>(row_of<T>(a.dx, row, a.dx_stride), e, n, out);
        }
    }
#pragma unroll
    for (int s = 0; s < K; ++s) {
        const int e = (s * LANES + lane) * V;
        Raw<PXH_F32, 4> part;
#pragma unroll
        for (int q = 0; q < V; q += 4) {
#pragma unroll
            for (int k = 0; k < 4; ++k) part.w[k] = __float_as_uint(dw[s][q + k]);
            store_row<PXH_F32, 4>(a.partial + static_cast<size_t>(worker) * n, e + q, n, part);
        }
    }
}

// Rows of any width: dx alone, the row is read twice.
template<int T>
__global__ __launch_bounds__(1024) void rms_norm_backward_wide_kernel(NormBackwardArgs a, long long first)
{
    constexpr int V = kVec<T>;
    __shared__ float slots[1024 / kWave];
    const int n = a.width;
    const long long row = first + blockIdx.x;
    const char* dy = row_of<T>(a.dy, row, a.dy_stride);
    const char* h = row_of<T>(a.h, row, a.h_stride);
    const float rstd = a.rstd[row];
    float dot = 0.0f;
    for (int e = threadIdx.x * V; e < n; e += 1024 * V) {
        float g[V], x[V], w[V];
        load_row<T, V>(dy, e, n).get(g);
        load_row<T, V>(h, e, n).get(x);
        weights_at<T, V>(a.weight, a.weight_f32, e, n, w);
#pragma unroll
        for (int k = 0; k < V; ++k) dot = fmaf(g[k] * w[k], x[k] * rstd, dot);
    }
    const float c = group_sum<1024>(dot, slots) / static_cast<float>(n);
    for (int e = threadIdx.x * V; e < n; e += 1024 * V) {
        float g[V], x[V], w[V], more[V] = {};
        load_row<T, V>(dy, e, n).get(g);
        load_row<T, V>(h, e, n).get(x);
        weights_at<T, V>(a.weight, a.weight_f32, e, n, w);
        if (a.dsum) load_row<T, V>(row_of<T>(a.dsum, row, a.dsum_stride), e, n).get(more);
#pragma unroll
        for (int k = 0; k < V; ++k) g[k] = fmaf(rstd, g[k] * w[k] - x[k] * rstd * c, more[k]);
        Raw<T, V> r;
        r.set(g);
        store_row<T, V>(row_of<T>(a.dx, row, a.dx_stride), e, n, r);
    }
}

// ... and the parts of dw, one column to a lane, before dx (which may be dy itself) is written.
template<int T>
__global__ __launch_bounds__(kBlock) void rms_norm_wide_dw_kernel(NormBackwardArgs a, int workers)
{
    const int e = blockIdx.x * kBlock + threadIdx.x;
    if (e >= a.width) return;
    float dw = 0.0f;
    for (long long row = blockIdx.y; row < a.rows; row += workers)
        dw = fmaf(load_one<T>(row_of<T>(a.dy, row, a.dy_stride), e), load_one<T>(row_of<T>(a.h, row, a.h_stride), e) * a.rstd[row], dw);
    a.partial[static_cast<size_t>(blockIdx.y) * a.width + e] = dw;
}

// dw[column] (+)= the sum of the workers' parts: 64 columns to a workgroup, whose waves share the workers.
__global__ __launch_bounds__(kColumnLanes) void rms_norm_dw_kernel(const float* partial, int workers, int width, float* dw, int accumulate)
{
    __shared__ float sums[kColumnWaves][kWave];
    const int column = blockIdx.x * kWave + threadIdx.x % kWave;
    const float all = sum_of_workers(partial, workers, width, column, column < width, sums);
    if (threadIdx.x < kWave && column < width) dw[column] = accumulate ? dw[column] + all : all;
}

// Workers that share the rows of the backward pass, each with a row of partial sums: a workgroup as wide as a row for each of 256 compute
// units (16384 x 4096 bf16: 1024 workers 108 us, 512 96, 256 89.5; 777 x 5121 half 17.1 with 512, 14.9 with 256), more of them where
// a row takes a few waves (16384 x 1024: 35 us with 512, 27 with 1024), fewer for rows of any width.
constexpr int kWideWorkers = 32;
int workers_for(long long rows, int width)
{
    const int most = width <= 2048 ? 1024 : width <= 32768 ? 256 : kWideWorkers;
    return static_cast<int>(rows < most ? rows : most);
}

template<int T, int LANES, int K>
int launch_backward(const NormBackwardArgs& a, int workers, hipStream_t s)
{
    constexpr int kPer = LANES > kWave ? 1 : kBlock / kWave;
    const dim3 grid(grid_for(workers, kPer)), block(LANES * kPer);
    // past the caches where the tensors do not fit (16384 x 4096 bf16 105 -> 97 us; 2048 x 4096 would go from 17 to 20)
    const size_t bytes = static_cast<size_t>(a.rows) * static_cast<size_t>(a.width) * kSize<T> * (a.dsum ? 4 : 3);
    if (bytes >= kStreamingBytes) hipLaunchKernelGGL((rms_norm_backward_kernel<T, LANES, K, true>), grid, block, 0, s, a, workers);
    else hipLaunchKernelGGL((rms_norm_backward_kernel<T, LANES, K, false>), grid, block, 0, s, a, workers);
    return check_launch("pxh_rms_norm_backward");
}

template<int T>
int norm_backward(const NormBackwardArgs& a, int& workers, hipStream_t s)
{
    const int vectors = (a.width + kVec<T> - 1) / kVec<T>;
    if (vectors <= 64) return launch_backward<T, 64, 1>(a, workers, s);
    if (vectors <= 128) return launch_backward<T, 128, 1>(a, workers, s);
    if (vectors <= 256) return launch_backward<T, 256, 1>(a, workers, s);
    if (vectors <= 512) return launch_backward<T, 512, 1>(a, workers, s);
    if (vectors <= 1024) return launch_backward<T, 1024, 1>(a, workers, s);
    if (vectors <= 2048) return launch_backward<T, 1024, 2>(a, workers, s);
    if (vectors <= 4096) return launch_backward<T, 1024, 4>(a, workers, s);
    if (workers > kWideWorkers) workers = kWideWorkers;
    hipLaunchKernelGGL((rms_norm_wide_dw_kernel<T>), dim3(grid_for(a.width, kBlock), workers), dim3(kBlock), 0, s, a, workers);
    if (int rc = check_launch("pxh_rms_norm_backward")) return rc;
    for (long long done = 0; done < a.rows; done += kLaunchRows) {
        const long long rows = a.rows - done < kLaunchRows ? a.rows - done : kLaunchRows;
        hipLaunchKernelGGL((rms_norm_backward_wide_kernel<T>), dim3(static_cast<unsigned>(rows)), dim3(1024), 0, s, a, done);
        if (int rc = check_launch("pxh_rms_norm_backward")) return rc;
    }
    return PXH_OK;
}

}  // namespace
}  // namespace pxh

using namespace pxh;

extern "C" {

int pxh_rms_norm_forward(const void* x, const void* residual, void* sum, const void* weight, void* y, float* scales,
                         float* rstd, int type, int weight_type, int y_type, long long rows, int width, long long x_stride,
                         long long residual_stride, long long sum_stride, long long y_stride, int group, float eps, void* stream)
{
    const char* who = "pxh_rms_norm_forward";
    if (int rc = check_norm_rows(who, type, weight_type, rows, width)) return rc;
    const bool eight = y_type == PXH_E4M3;
    if (!eight && y_type != type) return fail_invalid("%s: y is of the type of x or e4m3 (got type %d)", who, y_type);
    if (group != 0 && group != 128) return fail_invalid("%s: a scale for 128 values or, with 0, for a row (got %d)", who, group);
    if (sum && !residual) return fail_invalid("%s: a sum without a residual", who);
    if (!(eps >= 0.0f)) return fail_invalid("%s: eps %g", who, static_cast<double>(eps));
    if (rows == 0) return PXH_OK;
    if (!x || !weight || !y) return fail_invalid("%s: null pointer", who);
    if (eight && !scales) return fail_invalid("%s: 8-bit values without scales", who);
    if (x_stride < width || y_stride < width || (residual && residual_stride < width) || (sum && sum_stride < width))
        return fail_invalid("%s: rows of %d values that overlap", who, width);
    const NormArgs a{ x, residual, sum, weight, y, scales, rstd, rows, x_stride, residual_stride, sum_stride, y_stride, width, group, eps };
    int rc = PXH_OK;
    dispatch_type(type, [&]<int T>() {
        constexpr bool kMayWiden = T != PXH_F32;
        hipStream_t s = as_stream(stream);
        if (kMayWiden && weight_type == PXH_F32) rc = eight ? norm_forward<T, true, kMayWiden>(a, s) : norm_forward<T, false, kMayWiden>(a, s);
        else rc = eight ? norm_forward<T, true, false>(a, s) : norm_forward<T, false, false>(a, s);
    });
    return rc;
}

size_t pxh_rms_norm_workspace_bytes(long long rows, int width)
{
    if (rows <= 0 || width <= 0) return 0;
    // the largest that any of the shapes up to this one takes
    size_t most = 0;
    for (int w: { 2048, 32768, width }) {
        const int here = width < w ? width : w;
        const size_t floats = static_cast<size_t>(workers_for(rows, here)) * static_cast<size_t>(here);
        if (floats > most) most = floats;
    }
    return most * sizeof(float);
}

int pxh_rms_norm_backward(const void* dy, const void* h, const void* weight, const float* rstd, const void* dsum, void* dx,
                          float* dw, int type, int weight_type, long long rows, int width, long long dy_stride,
                          long long h_stride, long long dsum_stride, long long dx_stride, int accumulate, void* workspace,
                          size_t workspace_bytes, void* stream)
{
    const char* who = "pxh_rms_norm_backward";
    if (int rc = check_norm_rows(who, type, weight_type, rows, width)) return rc;
    if (!dw) return fail_invalid("%s: null pointer", who);
    hipStream_t s = as_stream(stream);
    if (rows > 0) {
        if (!dy || !h || !weight || !rstd || !dx) return fail_invalid("%s: null pointer", who);
        if (dy_stride < width || h_stride < width || dx_stride < width || (dsum && dsum_stride < width))
            return fail_invalid("%s: rows of %d values that overlap", who, width);
    }
    int workers = rows > 0 ? workers_for(rows, width) : 0;
    void* ws = nullptr;
    if (rows > 0)
        if (int rc = resolve_workspace(workspace, workspace_bytes, pxh_rms_norm_workspace_bytes(rows, width), &ws, s)) return rc;
    const NormBackwardArgs a{ dy, h, weight, rstd, dsum, dx, static_cast<float*>(ws), rows, dy_stride, h_stride, dsum_stride, dx_stride,
                              width, weight_type == PXH_F32 };
    int rc = PXH_OK;
    if (rows > 0) dispatch_type(type, [&]<int T>() { rc = norm_backward<T>(a, workers, s); });
    if (rc) return rc;
    // without rows the sum over them is zero
    if (workers == 0 && accumulate) return PXH_OK;
    hipLaunchKernelGGL(rms_norm_dw_kernel, dim3(grid_for(width, kWave)), dim3(kColumnLanes), 0, s, a.partial, workers, width, dw, accumulate);
    return check_launch(who);
}

}
