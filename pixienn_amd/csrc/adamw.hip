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
constexpr int kChunk = 16 * kStateBlock;    // values of a workgroup
constexpr int kSteps = kChunk / (kBlock * 4);
constexpr int kNormWorkers = 2048;
constexpr float kE4m3Max = 448.0f;
constexpr float kLeastScale = 0x1p-126f;

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
    float lr, eps, shrink, d_scale;
    uint32_t seed;
};

// Two rounds of an odd factor (of the golden ratio and the square root of two) and the high bits folded into the low ones.
__host__ __device__ __forceinline__ uint32_t mixed(uint32_t x)
{
    x *= 0x9E3779B9u;
    x ^= x >> 15;
    x *= 0x6A09E667u;
    x ^= x >> 13;
    return x;
}

// |x| / scale as e4m3 bits, rounded up with the probability of what is cut off: scaled by 2^-120 the value has e4m3's
// exponent, its subnormals among fp32's own, and 20 random bits are added below the last place.  A NaN stays one.
__device__ __forceinline__ uint32_t stochastic(float x, float inverse, uint32_t noise)
{
    const float small = fabsf(x) * inverse * 0x1p-120f;
    const uint32_t code = (__float_as_uint(small) + noise) >> 20;
    return x != x ? 0x7fu : code > 0x7eu ? 0x7eu : code;
}

__device__ __forceinline__ void from_e4m3(uint32_t codes, float scale, float (&x)[4])
{
    const auto low = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes), false);
    const auto high = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes), true);
    x[0] = low[0] * scale; x[1] = low[1] * scale; x[2] = high[0] * scale; x[3] = high[1] * scale;
}

// Four values of a lane.
struct Quad {
    float w[4], d[4], m[4], v[4];       // v: its root, with states in 8 bits
};

template<int BITS, int D, bool NT>
__device__ __forceinline__ void load_quad(const AdamwRecord& r, uint32_t e, Quad& q)
{
    load_raw<PXH_F32, 4, NT>(r.w, e).get(q.w);
    load_raw<D, 4, NT>(r.d, e).get(q.d);
    if constexpr (BITS == 32) {
        load_raw<PXH_F32, 4, NT>(r.m, e).get(q.m);
        load_raw<PXH_F32, 4, NT>(r.v, e).get(q.v);
    } else {
        from_e4m3(load_raw<PXH_E4M3, 4, NT>(r.m, e).w[0], r.m_scale[e / kStateBlock], q.m);
        from_e4m3(load_raw<PXH_E4M3, 4, NT>(r.v, e).w[0], r.v_scale[e / kStateBlock], q.v);
    }
}

// ... of which only those below n are there; zeros behind them.
template<int BITS, int D>
__device__ __forceinline__ void load_tail(const AdamwRecord& r, uint32_t e, Quad& q)
{
    uint32_t m = 0, v = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const bool there = e + k < r.n;
        q.w[k] = there ? r.w[e + k] : 0.0f;
        q.d[k] = there ? load_one<D>(r.d, e + k) : 0.0f;
        if constexpr (BITS == 32) {
            q.m[k] = there ? static_cast<const float*>(r.m)[e + k] : 0.0f;
            q.v[k] = there ? static_cast<const float*>(r.v)[e + k] : 0.0f;
        } else if (there) {
            m |= static_cast<uint32_t>(static_cast<const uint8_t*>(r.m)[e + k]) << (8 * k);
            v |= static_cast<uint32_t>(static_cast<const uint8_t*>(r.v)[e + k]) << (8 * k);
        }
    }
    if constexpr (BITS == 8) {
        const uint32_t block = min(e, r.n - 1) / kStateBlock;
        from_e4m3(m, r.m_scale[block], q.m);
        from_e4m3(v, r.v_scale[block], q.v);
    }
}

// One step of four values; the states as they are before they are rounded, v or its root.
template<int BITS>
__device__ __forceinline__ void step_quad(const AdamwStep& s, float factor, bool decay, Quad& q)
{
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float g = q.d[k] * factor;
        const float m = fmaf(s.beta1, q.m[k], s.a1 * g);
        const float before = BITS == 8 ? q.v[k] * q.v[k] : q.v[k];
        const float v = fmaf(s.beta2, before, s.a2 * (g * g));
        const float root = sqrtf(v);
        const float step = (m / s.c1) / (root / s.c2 + s.eps);
        const float w = q.w[k];
        q.w[k] = fmaf(s.lr, step, w);
        if (decay) q.w[k] = fmaf(-s.shrink, w, q.w[k]);
        q.m[k] = m;
        q.v[k] = BITS == 8 ? root : v;
    }
}

// The largest magnitude of a wave's values, as a scale.
__device__ __forceinline__ float block_scale(const float (&x)[4])
{
    const float most = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    return fmaxf(wave_max_by_rows(most) * (1.0f / kE4m3Max), kLeastScale);
}

struct Codes {
    uint32_t m, v;
    float m_scale, v_scale;
};

// All lanes of a wave, with the values of one block.
__device__ __forceinline__ Codes to_e4m3(const AdamwStep& s, uint32_t place, const Quad& q)
{
    Codes c{ 0, 0, block_scale(q.m), block_scale(q.v) };
    const float mi = 1.0f / c.m_scale, vi = 1.0f / c.v_scale;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t noise = mixed((place + k) ^ s.seed);
        const uint32_t m = stochastic(q.m[k], mi, noise >> 12) | (q.m[k] < 0.0f ? 0x80u : 0u);
        const uint32_t v = stochastic(q.v[k], vi, noise & 0xfffffu);
        c.m |= m << (8 * k);
        c.v |= (v == 0 && q.v[k] != 0.0f ? 1u : v) << (8 * k);
    }
    return c;
}

template<int BITS, bool NT>
__device__ __forceinline__ void store_quad(const AdamwStep& s, const AdamwRecord& r, uint32_t e, const Quad& q)
{
    Raw<PXH_F32, 4> f;
    f.set(q.w);
    store_raw<PXH_F32, 4, NT>(r.w, e, f);
    if constexpr (BITS == 32) {
        f.set(q.m);
        store_raw<PXH_F32, 4, NT>(r.m, e, f);
        f.set(q.v);
        store_raw<PXH_F32, 4, NT>(r.v, e, f);
    } else {
        const Codes c = to_e4m3(s, r.place + e, q);
        store_raw<PXH_E4M3, 4, NT>(r.m, e, Raw<PXH_E4M3, 4>{ { c.m } });
        store_raw<PXH_E4M3, 4, NT>(r.v, e, Raw<PXH_E4M3, 4>{ { c.v } });
        if (e % kStateBlock == 0) {
            r.m_scale[e / kStateBlock] = c.m_scale;
            r.v_scale[e / kStateBlock] = c.v_scale;
        }
    }
    if (r.copy) {
        if (r.copy_type == PXH_BF16) {
            Raw<PXH_BF16, 4> h;
            h.set(q.w);
            store_raw<PXH_BF16, 4>(r.copy, e, h);
        } else {
            Raw<PXH_F16, 4> h;
            h.set(q.w);
            store_raw<PXH_F16, 4>(r.copy, e, h);
        }
    }
}

template<int BITS>
__device__ __forceinline__ void store_tail(const AdamwStep& s, const AdamwRecord& r, uint32_t e, const Quad& q)
{
    Codes c{};
    if constexpr (BITS == 8) {
        c = to_e4m3(s, r.place + e, q);                 // the whole wave
        if (e % kStateBlock == 0 && e < r.n) {
            r.m_scale[e / kStateBlock] = c.m_scale;
            r.v_scale[e / kStateBlock] = c.v_scale;
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if (e + k >= r.n) break;
        r.w[e + k] = q.w[k];
        if constexpr (BITS == 32) {
            static_cast<float*>(r.m)[e + k] = q.m[k];
            static_cast<float*>(r.v)[e + k] = q.v[k];
        } else {
            static_cast<uint8_t*>(r.m)[e + k] = static_cast<uint8_t>(c.m >> (8 * k));
            static_cast<uint8_t*>(r.v)[e + k] = static_cast<uint8_t>(c.v >> (8 * k));
        }
        if (r.copy) {
            if (r.copy_type == PXH_BF16) store_one<PXH_BF16>(r.copy, e + k, q.w[k]);
            else store_one<PXH_F16>(r.copy, e + k, q.w[k]);
        }
    }
}

template<int BITS, int D, bool NT>
__device__ __forceinline__ void step_chunk(const AdamwRecord& r, const AdamwStep& s, uint32_t first, float factor)
{
    const bool decay = r.decay != 0;
    const uint32_t e = first + threadIdx.x * 4;
    if (first + kChunk <= r.n) {
        Quad q[kSteps];
#pragma unroll
        for (int k = 0; k < kSteps; ++k) load_quad<BITS, D, NT>(r, e + k * kBlock * 4, q[k]);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            step_quad<BITS>(s, factor, decay, q[k]);
            store_quad<BITS, NT>(s, r, e + k * kBlock * 4, q[k]);
        }
        return;
    }
    for (int k = 0; k < kSteps; ++k) {
        const uint32_t at = e + k * kBlock * 4;
        if (at / kStateBlock * kStateBlock >= r.n) return;      // whole waves: a wave has a block of its own
        Quad q;
        load_tail<BITS, D>(r, at, q);
        step_quad<BITS>(s, factor, decay, q);
        store_tail<BITS>(s, r, at, q);
    }
}

template<int BITS, bool NT>
__global__ __launch_bounds__(kBlock) void adamw_kernel(const AdamwRecord* records, const Chunk* chunks, AdamwStep s, const float* factor)
{
    const Chunk c = chunks[blockIdx.x];
    const AdamwRecord r = records[c.tensor];
    float f = s.d_scale;
    if (factor) {
        const float clip = *factor;
        if (clip != clip) return;               // the norm is not finite: the step is left out
        f *= clip;
    }
    if (r.d_type == PXH_F32) step_chunk<BITS, PXH_F32, NT>(r, s, c.first, f);
    else if (r.d_type == PXH_BF16) step_chunk<BITS, PXH_BF16, NT>(r, s, c.first, f);
    else step_chunk<BITS, PXH_F16, NT>(r, s, c.first, f);
}

// ---------------------------------------------------------------- the norm of all gradients
template<int D>
__device__ __forceinline__ double squares_of_chunk(const AdamwRecord& r, uint32_t first)
{
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        const uint32_t e = first + (k * kBlock + threadIdx.x) * 4;
        float d[4] = {};
        if (e + 4 <= r.n) load_raw<D, 4>(r.d, e).get(d);
        else
            for (int i = 0; i < 4; ++i)
                if (e + i < r.n) d[i] = load_one<D>(r.d, e + i);
        sum += fmaf(d[0], d[0], fmaf(d[1], d[1], fmaf(d[2], d[2], d[3] * d[3])));
    }
    return sum;
}

__global__ __launch_bounds__(kBlock) void adamw_squares_kernel(const AdamwRecord* records, const Chunk* chunks, uint32_t count, double* partial)
{
    __shared__ double slots[kBlock / kWave];
    double sum = 0.0;
    for (uint32_t i = blockIdx.x; i < count; i += gridDim.x) {
        const Chunk c = chunks[i];
        const AdamwRecord& r = records[c.tensor];
        if (r.d_type == PXH_F32) sum += squares_of_chunk<PXH_F32>(r, c.first);
        else if (r.d_type == PXH_BF16) sum += squares_of_chunk<PXH_BF16>(r, c.first);
        else sum += squares_of_chunk<PXH_F16>(r, c.first);
    }
    sum = block_sum(sum, slots);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

__global__ __launch_bounds__(kBlock) void adamw_norm_kernel(const double* partial, int count, float d_scale, float max_norm, float* factor,
                                                            float* norm_out)
{
    __shared__ double slots[kBlock / kWave];
    double sum = 0.0;
    for (int i = threadIdx.x; i < count; i += kBlock) sum += partial[i];
    sum = block_sum(sum, slots);
    if (threadIdx.x == 0) {
        const float norm = static_cast<float>(sqrt(sum) * fabs(static_cast<double>(d_scale)));
        float f = 1.0f;
        if (max_norm > 0.0f) {
            if (!(norm <= 3.4028234e38f)) f = __builtin_nanf("");
            else if (norm > max_norm) f = max_norm / norm;
        }
        *factor = f;
        if (norm_out) *norm_out = norm;
    }
}

}  // namespace
}  // namespace pxh

using namespace pxh;

extern "C" {

struct pxh_adamw_table {
    int device, count, bits;
    uint32_t chunks;
    bool streaming;             // too large to stay cached from step to step
    void* memory;
    const AdamwRecord* records;
    const Chunk* chunk_list;
    double* partial;
    float* factor;
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
            const uint32_t tensor = static_cast<uint32_t>(records.size());
            records.push_back({ t.w, t.d, t.m, t.v, t.m_scale, t.v_scale, t.copy, n, place, t.d_type, t.copy_type, t.apply_decay != 0 });
            for (uint32_t at = 0; at < n; at += kChunk) chunks.push_back({ tensor, at });
            place += (n + kStateBlock - 1) / kStateBlock * kStateBlock;
            bytes += t.n * (8 + 2 * state_bits / 4 + size_of(t.d_type) + (t.copy ? 2 : 0));
        }
        if (chunks.size() > (1u << 24) - 1) {
            set_error("%s: more values than one launch takes", who);
            return PXH_ERR_UNSUPPORTED;
        }
        auto* t = new pxh_adamw_table{};
        t->count = static_cast<int>(records.size());
        t->bits = state_bits;
        t->chunks = static_cast<uint32_t>(chunks.size());
        t->streaming = bytes >= kStreamingBytes;
        if (hipGetDevice(&t->device) != hipSuccess) t->device = -1;
        if (t->count == 0) {
            *table = t;
            return PXH_OK;
        }
        const auto align = [](size_t b) { return (b + 255) & ~static_cast<size_t>(255); };
        const size_t record_bytes = align(records.size() * sizeof(AdamwRecord)), chunk_bytes = align(chunks.size() * sizeof(Chunk));
        hipError_t e = hipSuccess;
        std::vector<char> image;
        try {
            image.resize(record_bytes + chunk_bytes);
        } catch (...) {
            delete t;
            throw;
        }
        std::memcpy(image.data(), records.data(), records.size() * sizeof(AdamwRecord));
        std::memcpy(image.data() + record_bytes, chunks.data(), chunks.size() * sizeof(Chunk));
        e = hipMalloc(&t->memory, image.size() + align(kNormWorkers * sizeof(double)) + 256);
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
        t->partial = reinterpret_cast<double*>(base + image.size());
        t->factor = reinterpret_cast<float*>(base + image.size() + align(kNormWorkers * sizeof(double)));
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

int pxh_adamw_update_table(const pxh_adamw_table* table, int t, float lr, float beta1, float beta2, float eps, float decay,
                           float d_scale, float max_norm, float* norm_out, unsigned seed, void* stream)
{
    const char* who = "pxh_adamw_update_table";
    if (!table) return fail_invalid("%s: null table", who);
    if (t < 1) return fail_invalid("%s: step %d", who, t);
    if (!(beta1 >= 0.0f && beta1 < 1.0f && beta2 >= 0.0f && beta2 < 1.0f)) return fail_invalid("%s: beta %g, %g", who, static_cast<double>(beta1), static_cast<double>(beta2));
    if (!(eps >= 0.0f) || !(max_norm >= 0.0f)) return fail_invalid("%s: eps %g, max_norm %g", who, static_cast<double>(eps), static_cast<double>(max_norm));
    if (table->count == 0 && !norm_out) return PXH_OK;
    int device = -1;
    if (hipGetDevice(&device) != hipSuccess || device != table->device)
        return fail_invalid("%s: the table is of device %d, the current one is %d", who, table->device, device);
    hipStream_t s = as_stream(stream);
    if (table->count == 0) {
        hipLaunchKernelGGL(adamw_norm_kernel, dim3(1), dim3(kBlock), 0, s, nullptr, 0, d_scale, 0.0f, norm_out, norm_out);
        return check_launch(who);
    }
    const bool clips = max_norm > 0.0f;
    if (clips || norm_out) {
        const unsigned workers = table->chunks < static_cast<uint32_t>(kNormWorkers) ? table->chunks : kNormWorkers;
        hipLaunchKernelGGL(adamw_squares_kernel, dim3(workers), dim3(kBlock), 0, s, table->records, table->chunk_list, table->chunks, table->partial);
        if (int rc = check_launch(who)) return rc;
        hipLaunchKernelGGL(adamw_norm_kernel, dim3(1), dim3(kBlock), 0, s, table->partial, static_cast<int>(workers), d_scale, max_norm,
                           table->factor, norm_out);
        if (int rc = check_launch(who)) return rc;
    }
    AdamwStep step{};
    step.beta1 = beta1; step.beta2 = beta2;
    step.a1 = static_cast<float>(1.0 - static_cast<double>(beta1)); step.a2 = static_cast<float>(1.0 - static_cast<double>(beta2));
    step.c1 = static_cast<float>(1.0 - std::pow(static_cast<double>(beta1), t));
    step.c2 = static_cast<float>(std::sqrt(1.0 - std::pow(static_cast<double>(beta2), t)));
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
