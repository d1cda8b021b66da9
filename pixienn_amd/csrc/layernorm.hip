// Layer norm over rows, with the residual's addition in front of it, and its gradients.
#include "rows.h"
#include "stream.h"

namespace pxh {
namespace {

// ---------------------------------------------------------------- forward
//   h = x + residual (rounded as it is kept);  mean = mean(h);  rstd = 1 / sqrt(mean((h - mean)^2) + eps);  y = (h - mean) * rstd * weight + bias
struct LayerNormArgs {
    const void* x;
    const void* residual;
    void* sum;
    const void* weight;
    const void* bias;
    void* y;
    float* mean;
    float* rstd;
    long long rows, x_stride, residual_stride, sum_stride, y_stride;
    int width;
    float eps;
};

// The sum over the lanes of a row, the same in each: of a wave, or, with SHARED, of the workgroup's waves, as many as it has.
constexpr int kMostWaves = 16;

template<bool SHARED>
__device__ __forceinline__ float sum_of_row(float v, float* slots)
{
    v = wave_sum_by_rows(v);
    if constexpr (SHARED) {
        const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
        if (lane == 0) slots[wave] = v;
        __syncthreads();
        v = lane < waves ? slots[lane] : 0.0f;
        v = wave_sum_by_rows(v);
    }
    return v;
}

// Where a lane's vector e of a row of n values lies: at the row's last V values where it would go beyond them.  The first `skip` of those
// are the neighbour's as well (all of them where the lane has none): they count in no sum, and are written twice alike.  No access by
// the value at the row's end, and no branch around a load.  n >= V.
struct Place {
    int at, skip;
    __device__ __forceinline__ Place(int e, int n, int v) : at(min(e, n - v)), skip(e - at) {}
};

// V weights as they lie in memory, of the tensors' type or, WIDE, of fp32.
template<int T, int V, bool WIDE>
struct Weights {
    static constexpr int W = WIDE ? PXH_F32 : T, kParts = V * kSize<W> / 16, kPart = V / kParts;
    Raw<W, kPart> r[kParts];

    __device__ __forceinline__ void load(const void* p, int e)
    {
#pragma unroll
        for (int q = 0; q < kParts; ++q) r[q] = load_raw<W, kPart>(p, e + q * kPart);
    }
    __device__ __forceinline__ void get(float (&x)[V]) const
    {
#pragma unroll
        for (int q = 0; q < kParts; ++q) {
            float part[kPart];
            r[q].get(part);
#pragma unroll
            for (int k = 0; k < kPart; ++k) x[q * kPart + k] = part[k];
        }
    }
};

// A row is walked in vectors, lane by lane, by a wave or, with SHARED, by a workgroup of as many waves as its vectors fill.  K vectors a
// lane stay in registers from the sum over the squares of what is left without the mean (not a difference of two sums, which loses what a
// large mean leaves of the digits) to the result; up to two of them with their weights, asked for with the row.  K == 0: a row of any
// width, which is read three times.
// Bound by the memory, and by a launch where there is little of it: 16384 x 4096 bf16 with residual and bias 91 us (537 MB at 5.9 TB/s), without a
// residual 50 (5.3 TB/s); 2111 x 5001 fp32 with a bias 17.1, of which the kernel is 15.7 (85 MB at 5.4 TB/s; with row ends value by value it
// was 4 more), 16 x 4096 bf16 with residual and bias 4.5.
template<int T, bool WIDE, bool SHARED, int K, bool NT>
__global__ __launch_bounds__(SHARED ? kMostWaves * kWave : kBlock) void layer_norm_kernel(LayerNormArgs a)
{
    constexpr int V = kVec<T>;
    constexpr int kRows = SHARED ? 1 : kBlock / kWave;              // rows per workgroup
    constexpr bool kAhead = K == 1 || K == 2;
    __shared__ float slots[2][SHARED ? kMostWaves : 1];
    const int lanes = SHARED ? static_cast<int>(blockDim.x) : kWave, lane = SHARED ? threadIdx.x : threadIdx.x % kWave;
    const long long row = static_cast<long long>(blockIdx.x) * kRows + (SHARED ? 0 : threadIdx.x / kWave);
    if (row >= a.rows) return;                                       // whole waves, and only where nothing is waited for
    const char* x = row_of<T>(a.x, row, a.x_stride);
    const char* residual = a.residual ? row_of<T>(a.residual, row, a.residual_stride) : nullptr;
    char* sum = a.sum ? row_of<T>(a.sum, row, a.sum_stride) : nullptr;
    char* y = row_of<T>(a.y, row, a.y_stride);
    const int n = a.width;
    float total = 0.0f, squares = 0.0f;
    if constexpr (K > 0) {
        Raw<T, V> kept[K], more[K];
        Weights<T, V, WIDE> weight[kAhead ? K : 1], bias[kAhead ? K : 1];
#pragma unroll
        for (int s = 0; s < K; ++s) {
            const Place p((s * lanes + lane) * V, n, V);
            kept[s] = load_raw<T, V, NT>(x, p.at);
            if (residual) more[s] = load_raw<T, V, NT>(residual, p.at);
            if (kAhead) {
                weight[kAhead ? s : 0].load(a.weight, p.at);
                if (a.bias) bias[kAhead ? s : 0].load(a.bias, p.at);
            }
        }
#pragma unroll
        for (int s = 0; s < K; ++s) {
            // only a row's last step can have such (looked after by the host)
            const int skip = s + 1 < K ? 0 : Place((s * lanes + lane) * V, n, V).skip;
            float h[V];
            kept[s].get(h);
            if (residual) {
                float q[V];
                more[s].get(q);
#pragma unroll
                for (int k = 0; k < V; ++k) h[k] += q[k];
                kept[s].set(h);
                kept[s].get(h);
            }
#pragma unroll
            for (int k = 0; k < V; ++k) total += k >= skip ? h[k] : 0.0f;
        }
        const float mean = sum_of_row<SHARED>(total, slots[0]) / static_cast<float>(n);
#pragma unroll
        for (int s = 0; s < K; ++s) {
            const Place p((s * lanes + lane) * V, n, V);
            const int skip = s + 1 < K ? 0 : p.skip;
            // not before every lane has read, where the sum takes the residual's place
            if (sum && skip < V) store_raw<T, V, NT>(sum, p.at, kept[s]);
            float h[V];
            kept[s].get(h);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float d = k >= skip ? h[k] - mean : 0.0f;
                squares = fmaf(d, d, squares);
            }
        }
        const float rstd = 1.0f / sqrtf(sum_of_row<SHARED>(squares, slots[1]) / static_cast<float>(n) + a.eps);
        if (lane == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
#pragma unroll
        for (int s = 0; s < K; ++s) {
            const Place p((s * lanes + lane) * V, n, V);
            if (p.skip >= V) break;
            float h[V], w[V], b[V] = {};
            kept[s].get(h);
            if constexpr (!kAhead) {
                weight[0].load(a.weight, p.at);
                if (a.bias) bias[0].load(a.bias, p.at);
            }
            weight[kAhead ? s : 0].get(w);
            if (a.bias) bias[kAhead ? s : 0].get(b);
#pragma unroll
            for (int k = 0; k < V; ++k) h[k] = fmaf((h[k] - mean) * rstd, w[k], b[k]);
            Raw<T, V> r;
            r.set(h);
            store_raw<T, V, NT>(y, p.at, r);
        }
    } else {
        const auto ask = [&](int e, float (&h)[V]) {
            // x may have been overwritten by the sum, which is what is wanted
            Raw<T, V> r = load_row<T, V>(sum ? sum : x, e, n);
            r.get(h);
            if (residual && !sum) {
                float q[V];
                load_row<T, V>(residual, e, n).get(q);
#pragma unroll
                for (int k = 0; k < V; ++k) h[k] += q[k];
                r.set(h);
                r.get(h);
            }
        };
        if (sum) {
            for (int e = lane * V; e < n; e += lanes * V) {
                float h[V], q[V];
                load_row<T, V>(x, e, n).get(h);
                load_row<T, V>(residual, e, n).get(q);
#pragma unroll
                for (int k = 0; k < V; ++k) h[k] += q[k];
                Raw<T, V> r;
                r.set(h);
                store_row<T, V>(sum, e, n, r);
            }
        }
        for (int e = lane * V; e < n; e += lanes * V) {
            float h[V];
            ask(e, h);
#pragma unroll
            for (int k = 0; k < V; ++k) total += h[k];               // zeros behind the row's last value
        }
        const float mean = sum_of_row<SHARED>(total, slots[0]) / static_cast<float>(n);
        for (int e = lane * V; e < n; e += lanes * V) {
            float h[V];
            ask(e, h);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float d = e + k < n ? h[k] - mean : 0.0f;
                squares = fmaf(d, d, squares);
            }
        }
        const float rstd = 1.0f / sqrtf(sum_of_row<SHARED>(squares, slots[1]) / static_cast<float>(n) + a.eps);
        if (lane == 0) {
            if (a.mean) a.mean[row] = mean;
            if (a.rstd) a.rstd[row] = rstd;
        }
        for (int e = lane * V; e < n; e += lanes * V) {
            float h[V], w[V], b[V] = {};
            ask(e, h);
            weights_at<T, V>(a.weight, WIDE, e, n, w);
            if (a.bias) weights_at<T, V>(a.bias, WIDE, e, n, b);
#pragma unroll
            for (int k = 0; k < V; ++k) h[k] = fmaf((h[k] - mean) * rstd, w[k], b[k]);
            Raw<T, V> r;
            r.set(h);
            store_row<T, V>(y, e, n, r);
        }
    }
}

template<int T, bool WIDE, bool SHARED, int K, bool NT>
int launch_norm(const LayerNormArgs& a, int lanes, hipStream_t s)
{
    constexpr int kRows = SHARED ? 1 : kBlock / kWave;
    for (long long done = 0; done < a.rows; done += kLaunchRows) {
        LayerNormArgs part = a;
        part.x = row_of<T>(a.x, done, a.x_stride);
        part.residual = a.residual ? row_of<T>(a.residual, done, a.residual_stride) : nullptr;
        part.sum = a.sum ? row_of<T>(a.sum, done, a.sum_stride) : nullptr;
        part.y = row_of<T>(a.y, done, a.y_stride);
        part.mean = a.mean ? a.mean + done : nullptr;
        part.rstd = a.rstd ? a.rstd + done : nullptr;
        part.rows = a.rows - done < kLaunchRows ? a.rows - done : kLaunchRows;
        const dim3 grid(grid_for(part.rows, kRows)), block(SHARED ? lanes : kBlock);
        hipLaunchKernelGGL((layer_norm_kernel<T, WIDE, SHARED, K, NT>), grid, block, 0, s, part);
        if (int rc = check_launch("pxh_layer_norm_forward")) return rc;
    }
    return PXH_OK;
}

// Waves of a row whose lanes take `each` of its vectors.
inline int lanes_for(int vectors, int each) { return ((vectors + each - 1) / each + kWave - 1) / kWave * kWave; }

// Vectors a lane by the vectors of a row, few while the row is short; as many waves as they fill, so that only the last of a lane's vectors
// can lie beyond the row.  Rows of less than one vector go the way of the widest.
template<int T, bool WIDE, bool NT>
int norm_forward(const LayerNormArgs& a, hipStream_t s)
{
    const int vectors = (a.width + kVec<T> - 1) / kVec<T>;
    if (a.width < kVec<T>) return launch_norm<T, WIDE, true, 0, false>(a, kWave, s);
    if (vectors <= 64) return launch_norm<T, WIDE, false, 1, NT>(a, kWave, s);
    if (vectors <= 256) return launch_norm<T, WIDE, true, 1, NT>(a, lanes_for(vectors, 1), s);
    if (vectors <= 1024) return launch_norm<T, WIDE, true, 2, NT>(a, lanes_for(vectors, 2), s);
    if (vectors <= 4096) return launch_norm<T, WIDE, true, 4, NT>(a, lanes_for(vectors, 4), s);
    return launch_norm<T, WIDE, true, 0, false>(a, 1024, s);        // read several times: through the caches
}

// ---------------------------------------------------------------- backward
//   g = dy * weight;  xhat = (h - mean) * rstd;  dx = rstd * (g - mean(g) - xhat * mean(g * xhat)) + dsum
//   dw (+)= sum over the rows of dy * xhat;  db (+)= sum of dy
struct LayerNormBackwardArgs {
    const void* dy;
    const void* h;
    const void* weight;
    const float* mean;
    const float* rstd;
    const void* dsum;
    void* dx;
    float* partial;         // [workers][2][width]: of dw, of db
    long long rows, dy_stride, h_stride, dsum_stride, dx_stride;
    int width;
    bool weight_f32, bias;
};

// Two sums over the lanes of a row, the same in each.  `slot` is one of two places, used in turn from row to row: no wave is more than
// one row ahead of another.
template<bool SHARED>
__device__ __forceinline__ float2 two_sums(float a, float b, float2* slot)
{
    a = wave_sum_by_rows(a);
    b = wave_sum_by_rows(b);
    if constexpr (SHARED) {
        const int lane = threadIdx.x % kWave, waves = blockDim.x / kWave;
        if (lane == 0) slot[threadIdx.x / kWave] = make_float2(a, b);
        __syncthreads();
        const float2 v = lane < waves ? slot[lane] : make_float2(0.0f, 0.0f);
        return make_float2(wave_sum_by_rows(v.x), wave_sum_by_rows(v.y));
    }
    return make_float2(a, b);
}

// dx of every row, and the part of dw and db that this worker's rows give: a worker (a wave, or a workgroup) takes every workers-th row, and
// asks for the next one before it waits for the sums over this one.  Bound by the memory: 16384 x 4096 bf16 with dsum, dw and db 90.5 us with the
// sums behind it (546 MB with the workers' sums, at 6.0 TB/s), 2048 x 16384 58 (4.6 TB/s: sixteen waves wait for one sum, and none is loaded ahead).
template<int T, bool WIDE, bool SHARED, int K, bool NT>
__global__ __launch_bounds__(SHARED ? kMostWaves * kWave : kBlock) void layer_norm_backward_kernel(LayerNormBackwardArgs a, int workers)
{
    constexpr int V = kVec<T>;
    constexpr int kPer = SHARED ? 1 : kBlock / kWave;
    constexpr bool kAhead = K == 1 || T == PXH_F32;        // two vectors of 16-bit values leave no registers for it
    __shared__ float2 slots[2][SHARED ? kMostWaves : 1];
    const int lanes = SHARED ? static_cast<int>(blockDim.x) : kWave, lane = SHARED ? threadIdx.x : threadIdx.x % kWave;
    const int worker = blockIdx.x * kPer + (SHARED ? 0 : threadIdx.x / kWave);
    if (worker >= workers) return;              // single waves, which wait for nobody
    const int n = a.width;
    float dw[K][V], db[K][V];
    float w[kAhead ? K : 1][V];
#pragma unroll
    for (int s = 0; s < K; ++s) {
#pragma unroll
        for (int k = 0; k < V; ++k) dw[s][k] = db[s][k] = 0.0f;
        if (kAhead) {
            Weights<T, V, WIDE> u;
            u.load(a.weight, Place((s * lanes + lane) * V, n, V).at);
            u.get(w[kAhead ? s : 0]);
        }
    }
    struct Row {
        Raw<T, V> g[K], h[K], more[kAhead ? K : 1];
        float mean, rstd;
    };
    const auto ask = [&](long long row, Row& r) {
        if (row >= a.rows) return;
        const char* dy = row_of<T>(a.dy, row, a.dy_stride);
        const char* h = row_of<T>(a.h, row, a.h_stride);
        r.mean = a.mean[row];
        r.rstd = a.rstd[row];
#pragma unroll
        for (int s = 0; s < K; ++s) {
            const int at = Place((s * lanes + lane) * V, n, V).at;
            r.g[s] = load_raw<T, V, NT>(dy, at);
            r.h[s] = load_raw<T, V, NT>(h, at);
            if (kAhead && a.dsum) r.more[kAhead ? s : 0] = load_raw<T, V, NT>(row_of<T>(a.dsum, row, a.dsum_stride), at);
        }
    };
    Row next;
    if (kAhead) ask(worker, next);
    int turn = 0;
    for (long long row = worker; row < a.rows; row += workers) {
        if (!kAhead) ask(row, next);
        const Row r = next;
        float plain = 0.0f, dot = 0.0f;
#pragma unroll
        for (int s = 0; s < K; ++s) {
            const Place p((s * lanes + lane) * V, n, V);
            const int skip = s + 1 < K ? 0 : p.skip;
            float g[V], x[V], u[V];
            r.g[s].get(g);
            r.h[s].get(x);
            if constexpr (!kAhead) {
                Weights<T, V, WIDE> t;
                t.load(a.weight, p.at);
                t.get(u);
            }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float own = k >= skip ? g[k] : 0.0f;
                const float xhat = (x[k] - r.mean) * r.rstd;
                dw[s][k] = fmaf(own, xhat, dw[s][k]);
                db[s][k] += own;
                const float gw = own * (kAhead ? w[kAhead ? s : 0][k] : u[k]);
                plain += gw;
                dot = fmaf(gw, xhat, dot);
            }
        }
        if (kAhead) ask(row + workers, next);
        const float2 sums = two_sums<SHARED>(plain, dot, slots[turn]);
        turn ^= 1;
        const float c0 = sums.x / static_cast<float>(n), c1 = r.rstd * (sums.y / static_cast<float>(n));
#pragma unroll
        for (int s = 0; s < K; ++s) {
            const Place p((s * lanes + lane) * V, n, V);
            float g[V], x[V], u[V], more[V] = {};
            r.g[s].get(g);
            r.h[s].get(x);
            if constexpr (!kAhead) {
                Weights<T, V, WIDE> t;
                t.load(a.weight, p.at);
                t.get(u);
            }
            if (a.dsum) {
                if (kAhead) r.more[kAhead ? s : 0].get(more);
                else load_raw<T, V>(row_of<T>(a.dsum, row, a.dsum_stride), p.at).get(more);
            }
#pragma unroll
            for (int k = 0; k < V; ++k)
                g[k] = fmaf(r.rstd, (g[k] * (kAhead ? w[kAhead ? s : 0][k] : u[k]) - c0) - (x[k] - r.mean) * c1, more[k]);
            Raw<T, V> out;
            out.set(g);
            char* const dx = row_of<T>(a.dx, row, a.dx_stride);
            if (p.skip == 0) {
                store_raw<T, V, NT>(dx, p.at, out);
            } else {
                // not the neighbour's: where dx takes the place of dsum, they may have been read behind its store
#pragma unroll
                for (int k = 0; k < V; ++k)
                    if (k >= p.skip) store_one<T>(dx, p.at + k, g[k]);
            }
        }
    }
    float* const partial = a.partial + static_cast<size_t>(worker) * 2 * n;
#pragma unroll
    for (int s = 0; s < K; ++s) {
        const Place p((s * lanes + lane) * V, n, V);
        if (p.skip == 0) {
            Raw<PXH_F32, 4> part;
#pragma unroll
            for (int q = 0; q < V; q += 4) {
#pragma unroll
                for (int k = 0; k < 4; ++k) part.w[k] = __float_as_uint(dw[s][q + k]);
                store_raw<PXH_F32, 4>(partial, p.at + q, part);
                if (a.bias) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) part.w[k] = __float_as_uint(db[s][q + k]);
                    store_raw<PXH_F32, 4>(partial + n, p.at + q, part);
                }
            }
        } else {
            // the neighbour's sums are the neighbour's
#pragma unroll
            for (int k = 0; k < V; ++k) {
                if (k < p.skip) continue;
                partial[p.at + k] = dw[s][k];
                if (a.bias) partial[n + p.at + k] = db[s][k];
            }
        }
    }
}

// Rows of any width: dx alone, the row is read twice (1024 x 32768 bf16 with dsum 58 us, 405 MB at 7.0 TB/s, some of it from the caches; with the
// sums in front of it, 29, and behind it, 5, the call takes 103 with tensors that no cache holds).
template<int T>
__global__ __launch_bounds__(1024) void layer_norm_backward_wide_kernel(LayerNormBackwardArgs a, long long first)
{
    constexpr int V = kVec<T>;
    __shared__ float2 slot[1024 / kWave];
    const int n = a.width;
    const long long row = first + blockIdx.x;
    const char* dy = row_of<T>(a.dy, row, a.dy_stride);
    const char* h = row_of<T>(a.h, row, a.h_stride);
    const float mean = a.mean[row], rstd = a.rstd[row];
    float plain = 0.0f, dot = 0.0f;
    for (int e = threadIdx.x * V; e < n; e += 1024 * V) {
        float g[V], x[V], w[V];
        load_row<T, V>(dy, e, n).get(g);
        load_row<T, V>(h, e, n).get(x);
        weights_at<T, V>(a.weight, a.weight_f32, e, n, w);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float gw = g[k] * w[k];
            plain += gw;
            dot = fmaf(gw, (x[k] - mean) * rstd, dot);
        }
    }
    const float2 sums = two_sums<true>(plain, dot, slot);
    const float c0 = sums.x / static_cast<float>(n), c1 = rstd * (sums.y / static_cast<float>(n));
    for (int e = threadIdx.x * V; e < n; e += 1024 * V) {
        float g[V], x[V], w[V], more[V] = {};
        load_row<T, V>(dy, e, n).get(g);
        load_row<T, V>(h, e, n).get(x);
        weights_at<T, V>(a.weight, a.weight_f32, e, n, w);
        if (a.dsum) load_row<T, V>(row_of<T>(a.dsum, row, a.dsum_stride), e, n).get(more);
#pragma unroll
        for (int k = 0; k < V; ++k) g[k] = fmaf(rstd, (g[k] * w[k] - c0) - (x[k] - mean) * c1, more[k]);
        Raw<T, V> r;
        r.set(g);
        store_row<T, V>(row_of<T>(a.dx, row, a.dx_stride), e, n, r);
    }
}

// ... and the parts of dw and db, one column to a lane, before dx (which may be dy itself) is written.
template<int T>
__global__ __launch_bounds__(kBlock) void layer_norm_wide_sums_kernel(LayerNormBackwardArgs a, int workers)
{
    const int e = blockIdx.x * kBlock + threadIdx.x;
    if (e >= a.width) return;
    float dw = 0.0f, db = 0.0f;
    for (long long row = blockIdx.y; row < a.rows; row += workers) {
        const float g = load_one<T>(row_of<T>(a.dy, row, a.dy_stride), e);
        dw = fmaf(g, (load_one<T>(row_of<T>(a.h, row, a.h_stride), e) - a.mean[row]) * a.rstd[row], dw);
        db += g;
    }
    float* const partial = a.partial + static_cast<size_t>(blockIdx.y) * 2 * a.width;
    partial[e] = dw;
    partial[a.width + e] = db;
}

// The sums of the workers' parts: blockIdx.y 0 for dw, 1 for db.
__global__ __launch_bounds__(kColumnLanes) void layer_norm_sums_kernel(const float* partial, int workers, int width, float* dw, float* db,
                                                                        int accumulate)
{
    __shared__ float sums[kColumnWaves][kWave];
    const int column = blockIdx.x * kWave + threadIdx.x % kWave;
    const size_t which = blockIdx.y;
    const float all = sum_of_workers(partial + which * width, workers, static_cast<size_t>(width) * 2, column, column < width, sums);
    float* const out = which ? db : dw;
    if (threadIdx.x < kWave && column < width) out[column] = accumulate ? out[column] + all : all;
}

// Workers that share the rows of the backward pass, each with two rows of partial sums.
constexpr int kWideWorkers = 32;
int workers_for(long long rows, int width)
{
    const int most = width <= 2048 ? 1024 : width <= 32768 ? 256 : kWideWorkers;
    return static_cast<int>(rows < most ? rows : most);
}

template<int T, bool WIDE, bool SHARED, int K>
int launch_backward(const LayerNormBackwardArgs& a, int workers, int lanes, hipStream_t s)
{
    constexpr int kPer = SHARED ? 1 : kBlock / kWave;
    const dim3 grid(grid_for(workers, kPer)), block(SHARED ? lanes : kBlock);
    // past the caches where the tensors do not fit
    const size_t bytes = static_cast<size_t>(a.rows) * static_cast<size_t>(a.width) * kSize<T> * (a.dsum ? 4 : 3);
    if (bytes >= kStreamingBytes) hipLaunchKernelGGL((layer_norm_backward_kernel<T, WIDE, SHARED, K, true>), grid, block, 0, s, a, workers);
    else hipLaunchKernelGGL((layer_norm_backward_kernel<T, WIDE, SHARED, K, false>), grid, block, 0, s, a, workers);
    return check_launch("pxh_layer_norm_backward");
}

template<int T, bool WIDE>
int norm_backward(const LayerNormBackwardArgs& a, int& workers, hipStream_t s)
{
    const int vectors = (a.width + kVec<T> - 1) / kVec<T>;
    if (a.width >= kVec<T>) {
        if (vectors <= 64) return launch_backward<T, WIDE, false, 1>(a, workers, 64, s);
        if (vectors <= 1024) return launch_backward<T, WIDE, true, 1>(a, workers, lanes_for(vectors, 1), s);
        if (vectors <= 2048) return launch_backward<T, WIDE, true, 2>(a, workers, lanes_for(vectors, 2), s);
    }
    if (workers > kWideWorkers) workers = kWideWorkers;
    hipLaunchKernelGGL((layer_norm_wide_sums_kernel<T>), dim3(grid_for(a.width, kBlock), workers), dim3(kBlock), 0, s, a, workers);
    if (int rc = check_launch("pxh_layer_norm_backward")) return rc;
    for (long long done = 0; done < a.rows; done += kLaunchRows) {
        const long long rows = a.rows - done < kLaunchRows ? a.rows - done : kLaunchRows;
        hipLaunchKernelGGL((layer_norm_backward_wide_kernel<T>), dim3(static_cast<unsigned>(rows)), dim3(1024), 0, s, a, done);
        if (int rc = check_launch("pxh_layer_norm_backward")) return rc;
    }
    return PXH_OK;
}

}  // namespace
}  // namespace pxh

using namespace pxh;

extern "C" {

int pxh_layer_norm_forward(const void* x, const void* residual, void* sum, const void* weight, const void* bias, void* y, float* mean,
                           float* rstd, int type, int weight_type, long long rows, int width, long long x_stride,
                           long long residual_stride, long long sum_stride, long long y_stride, float eps, void* stream)
{
    const char* who = "pxh_layer_norm_forward";
    if (int rc = check_norm_rows(who, type, weight_type, rows, width)) return rc;
    if (sum && !residual) return fail_invalid("%s: a sum without a residual", who);
    if (!(eps >= 0.0f)) return fail_invalid("%s: eps %g", who, static_cast<double>(eps));
    if (rows == 0) return PXH_OK;
    if (!x || !weight || !y) return fail_invalid("%s: null pointer", who);
    if (x_stride < width || y_stride < width || (residual && residual_stride < width) || (sum && sum_stride < width))
        return fail_invalid("%s: rows of %d values that overlap", who, width);
    const LayerNormArgs a{ x, residual, sum, weight, bias, y, mean, rstd, rows, x_stride, residual_stride, sum_stride, y_stride, width, eps };
    const size_t tensors = 2 + (residual != nullptr) + (sum != nullptr);
    const bool past = static_cast<size_t>(rows) * static_cast<size_t>(width) * size_of(type) * tensors >= kStreamingBytes;
    int rc = PXH_OK;
    dispatch_type(type, [&]<int T>() {
        constexpr bool kMayWiden = T != PXH_F32;
        hipStream_t s = as_stream(stream);
        if (kMayWiden && weight_type == PXH_F32) rc = past ? norm_forward<T, kMayWiden, true>(a, s) : norm_forward<T, kMayWiden, false>(a, s);
        else rc = past ? norm_forward<T, false, true>(a, s) : norm_forward<T, false, false>(a, s);
    });
    return rc;
}

size_t pxh_layer_norm_workspace_bytes(long long rows, int width)
{
    if (rows <= 0 || width <= 0) return 0;
    // the largest that any of the shapes up to this one takes
    size_t most = 0;
    for (int w: { 2048, 32768, width }) {
        const int here = width < w ? width : w;
        const size_t floats = static_cast<size_t>(workers_for(rows, here)) * static_cast<size_t>(here) * 2;
        if (floats > most) most = floats;
    }
    return most * sizeof(float);
}

int pxh_layer_norm_backward(const void* dy, const void* h, const void* weight, const float* mean, const float* rstd, const void* dsum,
                            void* dx, float* dw, float* db, int type, int weight_type, long long rows, int width, long long dy_stride,
                            long long h_stride, long long dsum_stride, long long dx_stride, int accumulate, void* workspace,
                            size_t workspace_bytes, void* stream)
{
    const char* who = "pxh_layer_norm_backward";
    if (int rc = check_norm_rows(who, type, weight_type, rows, width)) return rc;
    if (!dw) return fail_invalid("%s: null pointer", who);
    hipStream_t s = as_stream(stream);
    int workers = 0;
    void* ws = nullptr;
    if (rows > 0) {
        if (!dy || !h || !weight || !mean || !rstd || !dx) return fail_invalid("%s: null pointer", who);
        if (dy_stride < width || h_stride < width || dx_stride < width || (dsum && dsum_stride < width))
            return fail_invalid("%s: rows of %d values that overlap", who, width);
        workers = workers_for(rows, width);
        if (int rc = resolve_workspace(workspace, workspace_bytes, pxh_layer_norm_workspace_bytes(rows, width), &ws, s)) return rc;
    }
    const LayerNormBackwardArgs a{ dy, h, weight, mean, rstd, dsum, dx, static_cast<float*>(ws), rows, dy_stride, h_stride, dsum_stride,
                                   dx_stride, width, weight_type == PXH_F32, db != nullptr };
    int rc = PXH_OK;
    if (rows > 0) dispatch_type(type, [&]<int T>() {
        constexpr bool kMayWiden = T != PXH_F32;
        rc = kMayWiden && weight_type == PXH_F32 ? norm_backward<T, kMayWiden>(a, workers, s) : norm_backward<T, false>(a, workers, s);
    });
    if (rc) return rc;
    // without rows the sums over them are zero
    if (workers == 0 && accumulate) return PXH_OK;
    hipLaunchKernelGGL(layer_norm_sums_kernel, dim3(grid_for(width, kWave), db ? 2 : 1), dim3(kColumnLanes), 0, s, a.partial, workers, width, dw,
                       db, accumulate);
    return check_launch(who);
}

}
