// AdamW over all parameter tensors of a table, states in 32 or in 8 bits, gradients clipped by their common norm.
#include "stream.h"
#include "typed.h"

#include <cmath>
#include <cstring>
#include <exception>
#include <new>
#include <vector>

namespace pxh {
namespace {

constexpr int kStateBlock = 256;            // values with one scale: four to a lane of a wave
constexpr int kSteps = 4;                   // blocks of a wave
constexpr int kChunk = kSteps * kBlock * 4; // values of a workgroup
constexpr int kNormWorkers = 2048;

struct AdamwRecord {
    float* w;
    const void* d;
    void* m;
    void* v;
    float* m_scale;
    float* v_scale;
    void* copy;
    uint32_t n;
    uint32_t place;             // of its first value among the random numbers
    int d_type, copy_type, decay;
};

struct Chunk {
    uint32_t tensor, first;     // first: of the tensor's values
};

struct AdamwStep {
    float beta1, beta2, a1, a2;         // a: 1 - beta
    float c1, c2;                       // 1 - beta^t, and the square root of 1 - beta2^t
    float lr, lr_c1, inverse_c2, eps, shrink, d_scale;
    uint32_t seed;
};

// Two rounds of an odd factor (of the golden ratio and the square root of two) and the high bits folded into the low ones.
constexpr uint32_t kMix1 = 0x9E3779B9u, kMix2 = 0x6A09E667u;

__host__ __device__ __forceinline__ uint32_t second_round(uint32_t x)
{
    x ^= x >> 15;
    x *= kMix2;
    x ^= x >> 13;
    return x;
}

__host__ __device__ __forceinline__ uint32_t mixed(uint32_t x) { return second_round(x * kMix1); }

// Four values of a lane.
template<int D>
struct Quad {
    float w[4];
    Raw<D, 4> d;
    Raw<PXH_F32, 4> m32, v32;           // states in 32 bits
    uint32_t m8, v8;                    // ... in 8
};

template<int BITS, int D, bool NT>
__device__ __forceinline__ void load_quad(const AdamwRecord& r, uint32_t e, Quad<D>& q)
{
    load_raw<PXH_F32, 4, NT>(r.w, e).get(q.w);
    q.d = load_raw<D, 4, NT>(r.d, e);
    if constexpr (BITS == 32) {
        q.m32 = load_raw<PXH_F32, 4, NT>(r.m, e);
        q.v32 = load_raw<PXH_F32, 4, NT>(r.v, e);
    } else {
        q.m8 = load_raw<PXH_E4M3, 4, NT>(r.m, e).w[0];
        q.v8 = load_raw<PXH_E4M3, 4, NT>(r.v, e).w[0];
    }
}

// ... of which only those below n are there; zeros behind them.
template<int BITS, int D>
__device__ __forceinline__ void load_last(const AdamwRecord& r, uint32_t e, Quad<D>& q)
{
    float d[4] = {}, m[4] = {}, v[4] = {};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (e + k >= r.n) continue;
        q.w[k] = load_one<PXH_F32>(r.w, e + k);
        d[k] = load_one<D>(r.d, e + k);
        if constexpr (BITS == 32) {
            m[k] = load_one<PXH_F32>(r.m, e + k);
            v[k] = load_one<PXH_F32>(r.v, e + k);
        } else {
            q.m8 |= static_cast<uint32_t>(global_memory<uint8_t>(r.m)[e + k]) << (8 * k);
            q.v8 |= static_cast<uint32_t>(global_memory<uint8_t>(r.v)[e + k]) << (8 * k);
        }
    }
    q.d.set(d);
    q.m32.set(m);
    q.v32.set(v);
}

// What a lane writes of four values: all, or those below n.
template<int BITS, bool NT>
__device__ __forceinline__ void store_quad(const AdamwRecord& r, uint32_t e, const float (&w)[4], const float (&m)[4], const float (&v)[4],
                                           uint32_t m8, uint32_t v8)
{
    if (e + 4 <= r.n) {
        Raw<PXH_F32, 4> f;
        f.set(w);
        store_raw<PXH_F32, 4, NT>(r.w, e, f);
        if constexpr (BITS == 32) {
            f.set(m);
            store_raw<PXH_F32, 4, NT>(r.m, e, f);
            f.set(v);
            store_raw<PXH_F32, 4, NT>(r.v, e, f);
        } else {
            store_raw<PXH_E4M3, 4, NT>(r.m, e, Raw<PXH_E4M3, 4>{ { m8 } });
            store_raw<PXH_E4M3, 4, NT>(r.v, e, Raw<PXH_E4M3, 4>{ { v8 } });
        }
        if (r.copy) {
            if (r.copy_type == PXH_BF16) {
                Raw<PXH_BF16, 4> h;
                h.set(w);
                store_raw<PXH_BF16, 4, NT>(r.copy, e, h);
            } else {
                Raw<PXH_F16, 4> h;
                h.set(w);
                store_raw<PXH_F16, 4, NT>(r.copy, e, h);
            }
        }
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (e + k >= r.n) continue;
        store_one<PXH_F32>(r.w, e + k, w[k]);
        if constexpr (BITS == 32) {
            store_one<PXH_F32>(r.m, e + k, m[k]);
            store_one<PXH_F32>(r.v, e + k, v[k]);
        } else {
            global_memory<uint8_t>(r.m)[e + k] = static_cast<uint8_t>(m8 >> (8 * k));
            global_memory<uint8_t>(r.v)[e + k] = static_cast<uint8_t>(v8 >> (8 * k));
        }
        if (r.copy) {
            if (r.copy_type == PXH_BF16) store_one<PXH_BF16>(r.copy, e + k, w[k]);
            else store_one<PXH_F16>(r.copy, e + k, w[k]);
        }
    }
}

// ---------------------------------------------------------------- states in 32 bits
__device__ __forceinline__ void step_32(const AdamwStep& s, float clip, bool decay, const float (&d)[4], float (&w)[4], float (&m)[4],
                                        float (&v)[4])
{
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float g = d[k] * s.d_scale * clip;
        m[k] = fmaf(s.beta1, m[k], s.a1 * g);
        v[k] = fmaf(s.beta2, v[k], s.a2 * (g * g));
        const float step = (m[k] / s.c1) / (sqrtf(v[k]) / s.c2 + s.eps);
        const float old = w[k];
        w[k] = fmaf(s.lr, step, old);
        if (decay) w[k] = fmaf(-s.shrink, old, w[k]);
    }
}

// ---------------------------------------------------------------- states in 8 bits
// The states and their roots are formed operation by operation, each rounded to fp32, since a bit of theirs may turn what they are rounded
// to; the quotient of the step, whose last bits are lost in the weight, by the hardware's reciprocal.
__device__ __forceinline__ void step_8(const AdamwStep& s, float m_scale, float v_scale, float clip, bool decay, uint32_t m8, uint32_t v8,
                                       const float (&d)[4], float (&w)[4], float (&m)[4], float (&root)[4])
{
    const auto m01 = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(m8), false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(m8), true);
    const auto v01 = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(v8), false), v23 = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(v8), true);
    const float mc[4] = { m01[0], m01[1], m23[0], m23[1] }, vc[4] = { v01[0], v01[1], v23[0], v23[1] };
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float g = d[k] * s.d_scale * clip;
        m[k] = s.beta1 * (mc[k] * m_scale) + s.a1 * g;
        const float before = vc[k] * v_scale;
        root[k] = sqrtf(s.beta2 * (before * before) + s.a2 * (g * g));
        const float q = m[k] * __builtin_amdgcn_rcpf(fmaf(root[k], s.inverse_c2, s.eps));
        const float old = w[k];
        w[k] = fmaf(s.lr_c1, q, old);
        if (decay) w[k] = fmaf(-s.shrink, old, w[k]);
    }
}

__device__ __forceinline__ float largest(const float (&x)[4])
{
    return fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
}

__device__ __forceinline__ float max_of_halves(float a, float b)
{
    // a's two halves of the wave against each other in the lower half, b's in the upper one
    const auto t = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}

__device__ __forceinline__ float max_of_rows(float a, float b)
{
    // the same for the even and odd rows of 16
    const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}

// The maxima of eight values over the wave: lanes 8 j to 8 j + 7 have that of value j.  The lanes and the values are halved together, 18
// instructions for all eight (one by one it is 14 for each, and as many scales to be formed).
__device__ __forceinline__ float eight_maxima(const float (&x)[8])
{
    float y[4], z[2];
#pragma unroll
    for (int k = 0; k < 4; ++k) y[k] = max_of_halves(x[k], x[k + 4]);
#pragma unroll
    for (int k = 0; k < 2; ++k) z[k] = max_of_rows(y[k], y[k + 2]);
    const bool upper = threadIdx.x & 8;
    float v = fmaxf(upper ? z[1] : z[0], lane_in_row<0x128>(upper ? z[0] : z[1]));      // the lane eight further on in the row
    v = fmaxf(v, lane_in_row<0xB1>(v));
    v = fmaxf(v, lane_in_row<0x4E>(v));
    return fmaxf(v, lane_in_row<0x141>(v));
}

// The same of values that are numbers: one that is not does not take its block's scale with it.
__device__ __forceinline__ float largest_number(const float (&x)[4])
{
    float most = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) most = fmaxf(most, fabsf(x[k]) < INFINITY ? fabsf(x[k]) : 0.0f);
    return most;
}

// Four values over their block's scale as e4m3, up with the probability of what is cut off, by the upper 20 bits of the noise (the
// hardware's conversion, which is the addition of those bits below the last place, subnormals among it).  What is no number, whose weight
// is lost, has a NaN for its quotient, and is kept as the largest value: the lesser of a NaN and a number is the number.
__device__ __forceinline__ void to_e4m3(const AdamwStep& s, uint32_t place, const float (&m)[4], const float (&root)[4], float m_scale,
                                        float m_inverse, float v_scale, float v_inverse, uint32_t& m8, uint32_t& v8)
{
    // the four places differ in their last two bits only: one product for all
    const uint32_t base = ((place ^ s.seed) & ~3u) * kMix1;
    int mw = 0, vw = 0;
    const auto put = [&]<int K>() {
        const uint32_t noise = second_round(base + ((K ^ s.seed) & 3u) * kMix1);
        const float x = fmaxf(fminf(quotient_of(m[K], m_scale, m_inverse), kE4m3Max), -kE4m3Max);
        mw = __builtin_amdgcn_cvt_sr_fp8_f32(x, static_cast<int>(noise), mw, K);
        // at least the least value there is, unless it is zero
        const float v = fmaxf(fminf(quotient_of(root[K], v_scale, v_inverse), kE4m3Max), fminf(root[K] * 0x1p100f, 0x1p-9f));
        vw = __builtin_amdgcn_cvt_sr_fp8_f32(v, static_cast<int>(noise << 12), vw, K);
    };
    put.template operator()<0>();
    put.template operator()<1>();
    put.template operator()<2>();
    put.template operator()<3>();
    m8 = static_cast<uint32_t>(mw);
    v8 = static_cast<uint32_t>(vw);
}

// ---------------------------------------------------------------- the step
// A wave takes four blocks, 1024 values apart; all of their loads go out before the first is used.  Bound by its streams: 184.6 M values with
// 8-bit states, bf16 gradients and copies are 2.97 GB in 457 us, 6.5 TB/s, beside 65 for the norm's read of the gradients; 50 M
// with 32-bit ones 238 us for four streams in and three out, as a kernel that only moves those.
template<int BITS, int D, bool NT>
__device__ __forceinline__ void step_chunk(const AdamwRecord& r, const AdamwStep& s, uint32_t first, float clip)
{
    const bool decay = r.decay != 0;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const uint32_t e = first + threadIdx.x * 4;
    const uint32_t block = first / kStateBlock + wave;              // of the first step; the others four further on each
    const uint32_t blocks = (r.n + kStateBlock - 1) / kStateBlock;
    if (block >= blocks) return;                                    // a whole wave
    Quad<D> q[kSteps];
    float m_scale[kSteps], v_scale[kSteps];
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        q[k] = Quad<D>{};
        if (e + k * kBlock * 4 + 4 <= r.n) load_quad<BITS, D, NT>(r, e + k * kBlock * 4, q[k]);
        if constexpr (BITS == 8) {
            const uint32_t at = min(block + k * (kBlock / kWave), blocks - 1);
            m_scale[k] = global_memory<float>(r.m_scale)[at];
            v_scale[k] = global_memory<float>(r.v_scale)[at];
        }
    }
    if (first + kChunk > r.n) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            const uint32_t at = e + k * kBlock * 4;
            if (at < r.n && at + 4 > r.n) load_last<BITS, D>(r, at, q[k]);
        }
    }
    if constexpr (BITS == 32) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            float d[4], m[4], v[4];
            q[k].d.get(d);
            q[k].m32.get(m);
            q[k].v32.get(v);
            step_32(s, clip, decay, d, q[k].w, m, v);
            store_quad<BITS, NT>(r, e + k * kBlock * 4, q[k].w, m, v, 0, 0);
        }
    } else {
        float m[kSteps][4], root[kSteps][4], most[2 * kSteps];
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            float d[4];
            q[k].d.get(d);
            step_8(s, m_scale[k], v_scale[k], clip, decay, q[k].m8, q[k].v8, d, q[k].w, m[k], root[k]);
            most[k] = largest(m[k]);
            most[k + kSteps] = largest(root[k]);
        }
        // lanes 8 j and on: the scale of m in step j, and of the root in step j - 4
        const uint32_t lane = threadIdx.x % kWave, j = lane / 8;
        float peak = eight_maxima(most);
        if (__any(peak == INFINITY)) {
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                most[k] = largest_number(m[k]);
                most[k + kSteps] = largest_number(root[k]);
            }
            peak = eight_maxima(most);
        }
        const float scale = scale_of(peak), inverse = 1.0f / scale;
        const uint32_t of = block + (j % kSteps) * (kBlock / kWave);
        if (lane % 8 == 0 && of < blocks) global_memory<float>(j < kSteps ? r.m_scale : r.v_scale)[of] = scale;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            uint32_t m8, v8;
            to_e4m3(s, r.place + e + k * kBlock * 4, m[k], root[k], from_lane(scale, 8 * k), from_lane(inverse, 8 * k),
                    from_lane(scale, 8 * (k + kSteps)), from_lane(inverse, 8 * (k + kSteps)), m8, v8);
            store_quad<BITS, NT>(r, e + k * kBlock * 4, q[k].w, m[k], root[k], m8, v8);
        }
    }
}

template<int BITS, bool NT>
__global__ __launch_bounds__(kBlock) void adamw_kernel(const AdamwRecord* records, const Chunk* chunks, AdamwStep s, const float* factor)
{
    const Chunk c = chunks[blockIdx.x];
    const AdamwRecord r = records[c.tensor];
    const float clip = factor ? *factor : 1.0f;
    if (clip != clip) return;                   // the norm is not finite: the step is left out
    if (r.d_type == PXH_F32) step_chunk<BITS, PXH_F32, NT>(r, s, c.first, clip);
    else if (r.d_type == PXH_BF16) step_chunk<BITS, PXH_BF16, NT>(r, s, c.first, clip);
    else step_chunk<BITS, PXH_F16, NT>(r, s, c.first, clip);
}

// ---------------------------------------------------------------- the norm of all gradients
template<int D>
struct Gradients {
    Raw<D, 4> raw[kSteps];

    __device__ __forceinline__ void load(const AdamwRecord& r, uint32_t first)
    {
        const uint32_t e = first + threadIdx.x * 4;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            raw[k] = Raw<D, 4>{};
            if (e + k * kBlock * 4 + 4 <= r.n) raw[k] = load_raw<D, 4>(r.d, e + k * kBlock * 4);
        }
    }

    __device__ __forceinline__ double squares(const AdamwRecord& r, uint32_t first) const
    {
        double sum = 0.0;
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            float d[4];
            raw[k].get(d);
#pragma unroll
            for (int j = 0; j < 4; ++j) sum = fma(static_cast<double>(d[j]), static_cast<double>(d[j]), sum);
        }
        if (first + kChunk > r.n) {             // the tensor's last values, which fill no vector
            const uint32_t e = r.n / 4 * 4 + threadIdx.x;
            if (threadIdx.x < 4 && e < r.n) {
                const double d = load_one<D>(r.d, e);
                sum = fma(d, d, sum);
            }
        }
        return sum;
    }
};

// A workgroup asks for so many chunks at once, where all gradients are of one type: one after the other a chunk is three trips
// to memory for 8 KB (184.6 M values of bf16: 86 us, and 66 with four).
constexpr int kChunksAhead = 4;

template<int D>
__device__ __forceinline__ double squares_of(const AdamwRecord* records, const Chunk* chunks, uint32_t count)
{
    double sum = 0.0;
    for (uint32_t i = blockIdx.x * kChunksAhead; i < count; i += gridDim.x * kChunksAhead) {
        Gradients<D> d[kChunksAhead];
        Chunk c[kChunksAhead];
#pragma unroll
        for (int k = 0; k < kChunksAhead; ++k) c[k] = chunks[min(i + k, count - 1)];
#pragma unroll
        for (int k = 0; k < kChunksAhead; ++k) d[k].load(records[c[k].tensor], c[k].first);
#pragma unroll
        for (int k = 0; k < kChunksAhead; ++k)
            if (i + k < count) sum += d[k].squares(records[c[k].tensor], c[k].first);
    }
    return sum;
}

__device__ __forceinline__ double squares_of_any(const AdamwRecord* records, const Chunk* chunks, uint32_t count)
{
    double sum = 0.0;
    const auto take = [&]<int D>(const AdamwRecord& r, uint32_t first) {
        Gradients<D> d;
        d.load(r, first);
        sum += d.squares(r, first);
    };
    for (uint32_t i = blockIdx.x; i < count; i += gridDim.x) {
        const Chunk c = chunks[i];
        const AdamwRecord& r = records[c.tensor];
        if (r.d_type == PXH_F32) take.template operator()<PXH_F32>(r, c.first);
        else if (r.d_type == PXH_BF16) take.template operator()<PXH_BF16>(r, c.first);
        else take.template operator()<PXH_F16>(r, c.first);
    }
    return sum;
}

// Each workgroup leaves the sum over its chunks, and the last one to be done makes the norm and the clipping factor of them, in their
// order.  The sums cross from one die's cache to another's, as does the count of those that are done; that is zero again behind
// the last.  D: the type of all gradients, or -1.
template<int D>
__global__ __launch_bounds__(kBlock) void adamw_squares_kernel(const AdamwRecord* records, const Chunk* chunks, uint32_t count, double* partial,
                                                               uint32_t* done, float d_scale, float max_norm, float* factor, float* norm_out)
{
    __shared__ double slots[kBlock / kWave];
    __shared__ bool last;
    double sum;
    if constexpr (D < 0) sum = squares_of_any(records, chunks, count);
    else sum = squares_of<D>(records, chunks, count);
    sum = block_sum(sum, slots);
    if (threadIdx.x == 0) {
        __hip_atomic_store(partial + blockIdx.x, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // the sum is where every die sees it before the count says so; a release here would write back and empty the caches of
        // 2048 workgroups (65 us)
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        __builtin_amdgcn_s_waitcnt(0x0F70);      // vmcnt(0)
        last = __hip_atomic_fetch_add(done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
    }
    __syncthreads();
    if (!last) return;
    sum = 0.0;
    for (uint32_t i = threadIdx.x; i < gridDim.x; i += kBlock) sum += __hip_atomic_load(partial + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    sum = block_sum(sum, slots);
    if (threadIdx.x == 0) {
        // rounded once, to nearest: one beyond the largest number becomes an infinity, and leaves the step out as any other
        const double exact = sqrt(sum) * fabs(static_cast<double>(d_scale));
        const float norm = static_cast<float>(exact);
        float f = 1.0f;
        if (max_norm > 0.0f) {
            if (!(norm < INFINITY)) f = __builtin_nanf("");
            else if (exact > max_norm) f = static_cast<float>(max_norm / exact);
        }
        *factor = f;
        if (norm_out) *norm_out = norm;
        __hip_atomic_store(done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
}

}  // namespace
}  // namespace pxh

using namespace pxh;

extern "C" {

struct pxh_adamw_table {
    int device, count, bits;
    int d_type;                 // of all gradients, or -1
    uint32_t chunks;
    bool streaming;             // too large to stay cached from step to step
    void* memory;
    const AdamwRecord* records;
    const Chunk* chunk_list;
    double* partial;
    float* factor;
    uint32_t* done;             // workgroups of the norm that have left their sum; zero between launches
};

int pxh_adamw_table_create(int count, const pxh_adamw_tensor* tensors, int state_bits, pxh_adamw_table** table)
{
    const char* who = "pxh_adamw_table_create";
    if (!table) return fail_invalid("%s: null pointer", who);
    *table = nullptr;
    if (count < 0 || (count && !tensors)) return fail_invalid("%s: bad argument", who);
    if (count > 1 << 20) return fail_invalid("%s: %d tensors; a table holds %d at most", who, count, 1 << 20);
    if (state_bits != 8 && state_bits != 32) return fail_invalid("%s: states of 8 or 32 bits (got %d)", who, state_bits);
    try {
        std::vector<AdamwRecord> records;
        std::vector<Chunk> chunks;
        uint32_t place = 0;
        size_t bytes = 0;
        for (int i = 0; i < count; ++i) {
            const pxh_adamw_tensor& t = tensors[i];
            if (t.n == 0) continue;
            if (t.n > 0x7fffffffu) return fail_invalid("%s: tensor %d has 2^31 values or more", who, i);
            if (t.d_type != PXH_F32 && t.d_type != PXH_BF16 && t.d_type != PXH_F16)
                return fail_invalid("%s: tensor %d: gradients of type %d are not fp32, bf16 or half", who, i, t.d_type);
            if (t.copy && t.copy_type != PXH_BF16 && t.copy_type != PXH_F16)
                return fail_invalid("%s: tensor %d: a copy of type %d is not bf16 or half", who, i, t.copy_type);
            if (!t.w || !t.d || !t.m || !t.v || (state_bits == 8 && (!t.m_scale || !t.v_scale)))
                return fail_invalid("%s: null pointer for tensor %d", who, i);
            const uint32_t n = static_cast<uint32_t>(t.n);
            // before their list is made, which could be larger than memory
            if (chunks.size() + (n + kChunk - 1) / kChunk > (1u << 24) - 1) {
                set_error("%s: more values than one launch takes", who);
                return PXH_ERR_UNSUPPORTED;
            }
            const uint32_t tensor = static_cast<uint32_t>(records.size());
            records.push_back({ t.w, t.d, t.m, t.v, t.m_scale, t.v_scale, t.copy, n, place, t.d_type, t.copy_type, t.apply_decay != 0 });
            for (uint32_t at = 0; at < n; at += kChunk) chunks.push_back({ tensor, at });
            place += (n + kStateBlock - 1) / kStateBlock * kStateBlock;
            bytes += t.n * (8 + 2 * state_bits / 4 + size_of(t.d_type) + (t.copy ? 2 : 0));
        }
        auto* t = new pxh_adamw_table{};
        t->count = static_cast<int>(records.size());
        t->bits = state_bits;
        t->d_type = records.empty() ? -1 : records[0].d_type;
        for (const AdamwRecord& r: records)
            if (r.d_type != t->d_type) t->d_type = -1;
        t->chunks = static_cast<uint32_t>(chunks.size());
        t->streaming = bytes >= kStreamingBytes;
        if (hipGetDevice(&t->device) != hipSuccess) t->device = -1;
        if (t->count == 0) {
            *table = t;
            return PXH_OK;
        }
        const auto align = [](size_t b) { return (b + 255) & ~static_cast<size_t>(255); };
        const size_t record_bytes = align(records.size() * sizeof(AdamwRecord)), chunk_bytes = align(chunks.size() * sizeof(Chunk));
        const size_t head = record_bytes + chunk_bytes;
        hipError_t e = hipSuccess;
        std::vector<char> image;
        try {
            image.resize(head + 256);       // behind them the factor and the count, which has to begin at zero
        } catch (...) {
            delete t;
            throw;
        }
        std::memcpy(image.data(), records.data(), records.size() * sizeof(AdamwRecord));
        std::memcpy(image.data() + record_bytes, chunks.data(), chunks.size() * sizeof(Chunk));
        e = hipMalloc(&t->memory, image.size() + kNormWorkers * sizeof(double));
        if (e == hipSuccess) {
            e = hipMemcpy(t->memory, image.data(), image.size(), hipMemcpyHostToDevice);
            if (e != hipSuccess) (void) hipFree(t->memory);
        }
        if (e != hipSuccess) {
            set_error("%s: %s", who, hipGetErrorString(e));
            delete t;
            return static_cast<int>(e);
        }
        char* base = static_cast<char*>(t->memory);
        t->records = reinterpret_cast<const AdamwRecord*>(base);
        t->chunk_list = reinterpret_cast<const Chunk*>(base + record_bytes);
        t->factor = reinterpret_cast<float*>(base + head);
        t->done = reinterpret_cast<uint32_t*>(base + head + 128);
        t->partial = reinterpret_cast<double*>(base + image.size());
        *table = t;
        return PXH_OK;
    } catch (const std::exception&) {
        return fail_invalid("%s: out of host memory", who);
    }
}

void pxh_adamw_table_destroy(pxh_adamw_table* table)
{
    if (!table) return;
    if (table->memory) (void) hipFree(table->memory);
    delete table;
}

int pxh_adamw_table_count(const pxh_adamw_table* table) { return table ? table->count : 0; }

int pxh_adamw_update_table(const pxh_adamw_table* table, int t, float lr, double beta1, double beta2, float eps, float decay,
                           float d_scale, float max_norm, float* norm_out, unsigned seed, void* stream)
{
    const char* who = "pxh_adamw_update_table";
    if (!table) return fail_invalid("%s: null table", who);
    if (t < 1) return fail_invalid("%s: step %d", who, t);
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0)) return fail_invalid("%s: beta %g, %g", who, beta1, beta2);
    if (!(eps >= 0.0f) || !(max_norm >= 0.0f)) return fail_invalid("%s: eps %g, max_norm %g", who, static_cast<double>(eps), static_cast<double>(max_norm));
    if (table->count == 0 && !norm_out) return PXH_OK;
    int device = -1;
    if (hipGetDevice(&device) != hipSuccess || device != table->device)
        return fail_invalid("%s: the table is of device %d, the current one is %d", who, table->device, device);
    hipStream_t s = as_stream(stream);
    if (table->count == 0) return pxh_fill_f32(norm_out, 1, 0.0f, stream);
    const bool clips = max_norm > 0.0f;
    if (clips || norm_out) {
        // fewer chunks than that are a workgroup each
        const bool ahead = table->d_type >= 0 && table->chunks >= kNormWorkers;
        const uint32_t groups = ahead ? (table->chunks + kChunksAhead - 1) / kChunksAhead : table->chunks;
        const dim3 workers(groups < static_cast<uint32_t>(kNormWorkers) ? groups : kNormWorkers);
        const auto launch = [&](auto* kernel) {
            hipLaunchKernelGGL(kernel, workers, dim3(kBlock), 0, s, table->records, table->chunk_list, table->chunks, table->partial, table->done,
                               d_scale, max_norm, table->factor, norm_out);
        };
        if (!ahead || !dispatch_type(table->d_type, [&]<int D>() { launch(&adamw_squares_kernel<D>); })) launch(&adamw_squares_kernel<-1>);
        if (int rc = check_launch(who)) return rc;
    }
    AdamwStep step{};
    // constants from the arguments in 64 bits, each rounded once
    const double c1 = 1.0 - std::pow(beta1, t), c2 = std::sqrt(1.0 - std::pow(beta2, t));
    step.beta1 = static_cast<float>(beta1); step.beta2 = static_cast<float>(beta2);
    step.a1 = static_cast<float>(1.0 - beta1); step.a2 = static_cast<float>(1.0 - beta2);
    step.c1 = static_cast<float>(c1); step.c2 = static_cast<float>(c2);
    step.lr_c1 = static_cast<float>(static_cast<double>(lr) / c1); step.inverse_c2 = static_cast<float>(1.0 / c2);
    step.lr = lr; step.eps = eps; step.d_scale = d_scale;
    step.shrink = static_cast<float>(static_cast<double>(lr) * static_cast<double>(decay));
    step.seed = mixed((seed & 0x7fffffffu) + 1u);
    const float* factor = clips ? table->factor : nullptr;
    const dim3 grid(table->chunks), block(kBlock);
    if (table->bits == 8) {
        if (table->streaming) hipLaunchKernelGGL((adamw_kernel<8, true>), grid, block, 0, s, table->records, table->chunk_list, step, factor);
        else hipLaunchKernelGGL((adamw_kernel<8, false>), grid, block, 0, s, table->records, table->chunk_list, step, factor);
    } else {
        if (table->streaming) hipLaunchKernelGGL((adamw_kernel<32, true>), grid, block, 0, s, table->records, table->chunk_list, step, factor);
        else hipLaunchKernelGGL((adamw_kernel<32, false>), grid, block, 0, s, table->records, table->chunk_list, step, factor);
    }
    return check_launch(who);
}

}
