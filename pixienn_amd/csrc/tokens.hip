// Log probabilities of given tokens, entropy, the most probable alternatives, and the gradient of the logits.
#include "typed.h"

#include <cmath>

namespace pxh {
namespace {

constexpr float kLog2e = 1.44269504f;
constexpr float kLn2 = 0.693147181f;
constexpr float kFar = -200.0f;         // 2^-200 is no longer an fp32 number: what is this far below the maximum counts nothing

// Of a set of values l: their maximum, and relative to it the sum of e = 2^t and of e * t with t = (l - max) * c, c = scale * log2(e).
// A maximum of minus infinity (no value yet, or nothing but masked ones) has sums of zero.
struct Sums {
    float peak, sum, weighted;

    __device__ __forceinline__ float reference() const { return peak == -INFINITY ? 0.0f : peak; }

    // V more values
    template<int V>
    __device__ __forceinline__ void add(const float (&l)[V], float c)
    {
        float most = l[0];
#pragma unroll
        for (int k = 1; k < V; ++k) most = fmaxf(most, l[k]);
        const float next = fmaxf(peak, most);
        const float ref = next == -INFINITY ? 0.0f : next;
        const float t = (peak - ref) * c;
        const float f = __builtin_amdgcn_exp2f(t);
        weighted = f * fmaf(fmaxf(t, kFar), sum, weighted);
        sum *= f;
        peak = next;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float u = (l[k] - ref) * c;
            const float e = __builtin_amdgcn_exp2f(u);
            sum += e;
            weighted = fmaf(e, fmaxf(u, kFar), weighted);
        }
    }
};

__device__ __forceinline__ Sums nothing() { return Sums{ -INFINITY, 0.0f, 0.0f }; }

// Over a workgroup; the result in every lane.  The maximum first, then the sums relative to it: an exponential per lane.
template<int LANES>
__device__ __forceinline__ Sums group_join(Sums s, float c, Sums* slots)
{
    const float peak = wave_max_by_rows(s.peak);
    Sums w{ peak, 0.0f, 0.0f };
    {
        const float t = (s.peak - w.reference()) * c;
        const float f = __builtin_amdgcn_exp2f(t);
        w.weighted = wave_sum_by_rows(f * fmaf(fmaxf(t, kFar), s.sum, s.weighted));
        w.sum = wave_sum_by_rows(s.sum * f);
    }
    if constexpr (LANES > kWave) {
        if ((threadIdx.x & (kWave - 1)) == 0) slots[threadIdx.x / kWave] = w;
        __syncthreads();
        Sums all = nothing();
#pragma unroll
        for (int k = 0; k < LANES / kWave; ++k) all.peak = fmaxf(all.peak, slots[k].peak);
        const float ref = all.reference();
#pragma unroll
        for (int k = 0; k < LANES / kWave; ++k) {
            const Sums o = slots[k];
            const float t = (o.peak - ref) * c;
            const float f = __builtin_amdgcn_exp2f(t);
            all.weighted += f * fmaf(fmaxf(t, kFar), o.sum, o.weighted);
            all.sum += o.sum * f;
        }
        __syncthreads();
        w = all;
    }
    return w;
}

struct TokenArgs {
    const void* logits;
    const void* targets;
    const float* d_logp;
    const float* d_entropy;
    float* logp;
    float* entropy;
    float* lse;
    float* top_logp;
    int* top_ids;
    const float* lse_in;
    const float* entropy_in;
    void* dlogits;
    long long rows, stride, d_stride;
    int vocab, wide, top;
    float scale;
};

// The place of a row's token, -1 where none is given.
__device__ __forceinline__ int target_of(const TokenArgs& a, long long row)
{
    if (!a.targets) return -1;
    const long long t = a.wide ? static_cast<const long long*>(a.targets)[row] : static_cast<const int*>(a.targets)[row];
    return t >= 0 && t < a.vocab ? static_cast<int>(t) : -1;
}

struct RowResult {
    float lse, log_sum, entropy;        // log_sum: relative to the peak; minus infinity where there is nothing
};

// What a row's sums say, with the given token's place (or -1) and logit.
__device__ __forceinline__ RowResult finish_row(const TokenArgs& a, long long row, const Sums& s, int target, float given, bool writes)
{
    const bool empty = s.peak == -INFINITY;
    const float log_sum = logf(s.sum);
    RowResult r;
    r.log_sum = log_sum;
    r.lse = empty ? -INFINITY : fmaf(s.peak, a.scale, log_sum);
    r.entropy = empty ? 0.0f : log_sum - s.weighted / s.sum * kLn2;
    if (writes) {
        if (a.lse) a.lse[row] = r.lse;
        if (a.entropy) a.entropy[row] = r.entropy;
        if (a.logp) {
            a.logp[row] = target < 0 ? 0.0f : empty ? -INFINITY : (given - s.peak) * a.scale - log_sum;
        }
    }
    return r;
}

// One number that orders by value, then by the lowest index; NaN below everything.
__device__ __forceinline__ unsigned long long key_of(float z, uint32_t index)
{
    const uint32_t bits = __float_as_uint(z + 0.0f);
    const uint32_t order = z != z ? 0u : (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
    return (static_cast<unsigned long long>(order) << 32) | ~index;
}

// ---------------------------------------------------------------- forward
// A workgroup per row, one pass over it; then a pass for each alternative, over what the caches hold.
template<int T, int LANES>
__global__ __launch_bounds__(LANES) void token_logprobs_kernel(TokenArgs a)
{
    constexpr int V = kVec<T>;
    __shared__ Sums slots[LANES / kWave];
    __shared__ unsigned long long best;
    const long long row = blockIdx.x;
    const char* logits = static_cast<const char*>(a.logits) + row * a.stride * kSize<T>;
    const float c = a.scale * kLog2e;
    const int target = target_of(a, row);
    const float given = target < 0 ? 0.0f : load_one<T>(logits, target);
    Sums s = nothing();
    for (int e = threadIdx.x * V; e < a.vocab; e += LANES * V) {
        float l[V];
        load_row<T, V>(logits, e, a.vocab, -INFINITY).get(l);
        s.add(l, c);
    }
    s = group_join<LANES>(s, c, slots);
    const RowResult r = finish_row(a, row, s, target, given, threadIdx.x == 0);
    unsigned long long before = ~0ull;
    for (int j = 0; j < a.top; ++j) {
        if (threadIdx.x == 0) best = 0;
        __syncthreads();
        unsigned long long mine = 0;
        for (int e = threadIdx.x; e < a.vocab; e += LANES) {
            const unsigned long long key = key_of(load_one<T>(logits, e) * a.scale, e);
            if (key < before && key > mine) mine = key;
        }
        atomicMax(&best, mine);
        __syncthreads();
        before = best;
        __syncthreads();
        if (threadIdx.x == 0) {
            const uint32_t id = ~static_cast<uint32_t>(before);
            a.top_ids[row * a.top + j] = static_cast<int>(id);
            a.top_logp[row * a.top + j] = load_one<T>(logits, id) * a.scale - r.lse;
        }
    }
}

// ---------------------------------------------------------------- gradient
//   d_j = scale * (g * ((j == target) - p_j) - h * p_j * (log p_j + entropy)),  p = exp(z - lse)
// From the row's own sums log p = (l - peak) * scale - log(sum), which is right however large the logits are; from a stored lse,
// which fp32 has rounded, log p = l * scale - lse.  The hardware's exp2 has no results below 2^-126; a type that has them
// gets them from the square of half the exponent's power.
template<int T, bool PEAK>
struct RowGradient {
    float peak, rest, scale, entropy, g, h;
    int target;

    template<int V>
    __device__ __forceinline__ void apply(const float (&l)[V], int e, float (&d)[V]) const
    {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float logp = fmaf(PEAK ? l[k] - peak : l[k], scale, -rest);
            float p;
            if constexpr (T == PXH_F16) {
                p = __builtin_amdgcn_exp2f(logp * kLog2e);
            } else {
                const float root = __builtin_amdgcn_exp2f(logp * (0.5f * kLog2e));
                p = root * root;
            }
            d[k] = -g * p;
            if (h != 0.0f) d[k] -= h * p * (fmaxf(logp, kFar) + entropy);
        }
        if (static_cast<uint32_t>(target - e) < static_cast<uint32_t>(V)) {
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (e + k == target) d[k] += g;
        }
    }
};

template<int T, bool PEAK>
__device__ __forceinline__ RowGradient<T, PEAK> gradient_of(const TokenArgs& a, long long row, int target, float peak, float rest,
                                                            float entropy)
{
    RowGradient<T, PEAK> r;
    r.peak = peak;
    r.rest = rest;
    r.scale = a.scale;
    r.entropy = entropy;
    r.target = target;
    // the factor that z has of l is taken into the row's own
    r.g = a.d_logp && target >= 0 ? a.d_logp[row] * a.scale : 0.0f;
    r.h = a.d_entropy ? a.d_entropy[row] * a.scale : 0.0f;
    if (rest == -INFINITY) {        // no distribution: every probability 0, and no gradient
        r.rest = INFINITY;
        r.peak = r.g = r.h = 0.0f;
    }
    return r;
}

// A workgroup takes one part of a row.
constexpr int kGradientSteps = 4;

template<int T>
__global__ __launch_bounds__(kBlock) void token_gradient_kernel(TokenArgs a, FastDiv parts)
{
    constexpr int V = kVec<T>;
    uint32_t row, part;
    parts.divmod(blockIdx.x, row, part);
    const auto r = gradient_of<T, false>(a, row, target_of(a, row), 0.0f, a.lse_in[row], a.d_entropy ? a.entropy_in[row] : 0.0f);
    const char* logits = static_cast<const char*>(a.logits) + row * a.stride * kSize<T>;
    char* out = static_cast<char*>(a.dlogits) + row * a.d_stride * kSize<T>;
#pragma unroll
    for (int s = 0; s < kGradientSteps; ++s) {
        const int e = ((part * kGradientSteps + s) * kBlock + threadIdx.x) * V;
        if (e >= a.vocab) break;
        float l[V], d[V];
        load_row<T, V>(logits, e, a.vocab).get(l);
        r.template apply<V>(l, e, d);
        Raw<T, V> raw;
        raw.set(d);
        store_row<T, V>(out, e, a.vocab, raw);
    }
}

// ---------------------------------------------------------------- forward and gradient at once
// A workgroup per row, which stays in registers, K vectors a lane, between its sums and its gradient (K == 0: a row of any
// length, read again).  A lane writes the values that it has read, so the gradient may take the logits' place.
template<int T, bool ENTROPY, int LANES, int K>
__global__ __launch_bounds__(LANES) void token_train_kernel(TokenArgs a)
{
    constexpr int V = kVec<T>;
    __shared__ Sums slots[LANES / kWave];
    const long long row = blockIdx.x;
    const char* logits = static_cast<const char*>(a.logits) + row * a.stride * kSize<T>;
    char* out = static_cast<char*>(a.dlogits) + row * a.d_stride * kSize<T>;
    const float c = a.scale * kLog2e;
    const int target = target_of(a, row);
    const float given = target < 0 ? 0.0f : load_one<T>(logits, target);        // before it is overwritten
    Raw<T, V> kept[K ? K : 1];
    Sums s = nothing();
    if constexpr (K > 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int e = (k * LANES + threadIdx.x) * V;
            kept[k] = load_row<T, V>(logits, e < a.vocab ? e : a.vocab, a.vocab, -INFINITY);
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float l[V];
            kept[k].get(l);
#pragma unroll
            for (int i = 0; i < V; ++i) s.peak = fmaxf(s.peak, l[i]);
        }
        const float ref = s.reference();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float l[V];
            kept[k].get(l);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float u = (l[i] - ref) * c;
                const float e = __builtin_amdgcn_exp2f(u);
                s.sum += e;
                if (ENTROPY) s.weighted = fmaf(e, fmaxf(u, kFar), s.weighted);
            }
        }
    } else {
        for (int e = threadIdx.x * V; e < a.vocab; e += LANES * V) {
            float l[V];
            load_row<T, V>(logits, e, a.vocab, -INFINITY).get(l);
            s.add(l, c);
        }
    }
    s = group_join<LANES>(s, c, slots);
    const RowResult r = finish_row(a, row, s, target, given, threadIdx.x == 0);
    const auto gradient = gradient_of<T, true>(a, row, target, s.peak, r.log_sum, r.entropy);
    const auto write = [&](int e, const Raw<T, V>& raw) {
        float l[V], d[V];
        raw.get(l);
        gradient.template apply<V>(l, e, d);
        Raw<T, V> o;
        o.set(d);
        store_row<T, V>(out, e, a.vocab, o);
    };
    if constexpr (K > 0) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int e = (k * LANES + threadIdx.x) * V;
            if (e < a.vocab) write(e, kept[k]);
        }
    } else {
        for (int e = threadIdx.x * V; e < a.vocab; e += LANES * V) write(e, load_row<T, V>(logits, e, a.vocab));
    }
}

template<int T, bool ENTROPY>
int launch_train(const char* who, const TokenArgs& a, hipStream_t s)
{
    const dim3 grid(static_cast<unsigned>(a.rows));
    const int vectors = a.vocab / kVec<T> + (a.vocab % kVec<T> != 0);
    if (vectors <= 256) hipLaunchKernelGGL((token_train_kernel<T, ENTROPY, 256, 1>), grid, dim3(256), 0, s, a);
    else if (vectors <= 1024) hipLaunchKernelGGL((token_train_kernel<T, ENTROPY, 256, 4>), grid, dim3(256), 0, s, a);
    else if (vectors <= 4096) hipLaunchKernelGGL((token_train_kernel<T, ENTROPY, 512, 8>), grid, dim3(512), 0, s, a);
    else if (vectors <= 8192) hipLaunchKernelGGL((token_train_kernel<T, ENTROPY, 1024, 8>), grid, dim3(1024), 0, s, a);
    else if (vectors <= 16384) hipLaunchKernelGGL((token_train_kernel<T, ENTROPY, 1024, 16>), grid, dim3(1024), 0, s, a);
    else if (vectors <= 20480) hipLaunchKernelGGL((token_train_kernel<T, ENTROPY, 1024, 20>), grid, dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((token_train_kernel<T, true, 1024, 0>), grid, dim3(1024), 0, s, a);
    return check_launch(who);
}

template<int T>
int launch_forward(const char* who, const TokenArgs& a, hipStream_t s)
{
    if (a.vocab <= 8192) hipLaunchKernelGGL((token_logprobs_kernel<T, 256>), dim3(static_cast<unsigned>(a.rows)), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((token_logprobs_kernel<T, 1024>), dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, s, a);
    return check_launch(who);
}

template<int T>
int launch_gradient(const char* who, const TokenArgs& a, hipStream_t s)
{
    const int per = kGradientSteps * kBlock * kVec<T>;
    const int parts = a.vocab / per + (a.vocab % per != 0);
    hipLaunchKernelGGL((token_gradient_kernel<T>), dim3(static_cast<unsigned>(a.rows) * parts), dim3(kBlock), 0, s, a, FastDiv(parts));
    return check_launch(who);
}

// Runs `launch` over as many rows at a time as one grid takes.
template<typename F>
int by_rows(const TokenArgs& a, int type, const F& launch)
{
    const size_t size = size_of(type);
    const long long most = 1 << 20;
    long long per = (1ll << 31) / (static_cast<long long>(a.vocab) / 1024 + 1) / 1024;
    if (per > most) per = most;
    if (per < 1) per = 1;
    for (long long done = 0; done < a.rows; done += per) {
        TokenArgs p = a;
        p.rows = a.rows - done < per ? a.rows - done : per;
        p.logits = static_cast<const char*>(a.logits) + done * a.stride * size;
        p.targets = a.targets ? static_cast<const char*>(a.targets) + done * (a.wide ? 8 : 4) : nullptr;
        p.dlogits = a.dlogits ? static_cast<char*>(a.dlogits) + done * a.d_stride * size : nullptr;
        for (float** f: { &p.logp, &p.entropy, &p.lse })
            if (*f) *f += done;
        for (const float** f: { &p.d_logp, &p.d_entropy, &p.lse_in, &p.entropy_in })
            if (*f) *f += done;
        if (a.top) {
            p.top_logp += done * a.top;
            p.top_ids += done * a.top;
        }
        if (int rc = launch(p)) return rc;
    }
    return PXH_OK;
}

// What the entry points refuse alike.
int check_tokens(const char* who, const void* logits, int type, int wide, long long rows, int vocab, long long stride, float scale)
{
    if (type != PXH_F32 && type != PXH_BF16 && type != PXH_F16) return fail_invalid("%s: type %d is not fp32, bf16 or half", who, type);
    if (wide != 0 && wide != 1) return fail_invalid("%s: wide_targets is 0 or 1 (got %d)", who, wide);
    if (rows < 0) return fail_invalid("%s: %lld rows", who, rows);
    if (vocab <= 0 || vocab > 1 << 30) return fail_invalid("%s: rows of %d logits", who, vocab);
    if (!(scale > 0.0f && scale < INFINITY)) return fail_invalid("%s: scale %g", who, static_cast<double>(scale));
    if (rows > 0 && !logits) return fail_invalid("%s: null pointer", who);
    if (rows > 0 && stride < vocab) return fail_invalid("%s: rows of %d logits that overlap", who, vocab);
    return PXH_OK;
}

}  // namespace
}  // namespace pxh

using namespace pxh;

extern "C" {

size_t pxh_token_logprobs_workspace_bytes(long long rows, int vocab, int top)
{
    (void) rows; (void) vocab; (void) top;
    return 0;
}

int pxh_token_logprobs_forward(const void* logits, const void* targets, float* logp, float* entropy, float* lse,
                               float* top_logp, int* top_ids, int type, int wide_targets, long long rows, int vocab,
                               long long stride, int top, float scale, void* workspace, size_t workspace_bytes, void* stream)
{
    const char* who = "pxh_token_logprobs_forward";
    if (int rc = check_tokens(who, logits, type, wide_targets, rows, vocab, stride, scale)) return rc;
    if (!targets != !logp) return fail_invalid("%s: targets and logp go together", who);
    if (top < 0 || top > PXH_MOST_ALTERNATIVES || top > vocab)
        return fail_invalid("%s: %d alternatives of %d (at most %d)", who, top, vocab, PXH_MOST_ALTERNATIVES);
    if (top && rows > 0 && (!top_logp || !top_ids)) return fail_invalid("%s: null pointer", who);
    TokenArgs a{};
    a.logits = logits; a.targets = targets; a.logp = logp; a.entropy = entropy; a.lse = lse;
    a.top_logp = top_logp; a.top_ids = top_ids; a.rows = rows; a.stride = stride; a.vocab = vocab; a.wide = wide_targets;
    a.top = top; a.scale = scale;
    hipStream_t s = as_stream(stream);
    int rc = PXH_OK;
    dispatch_type(type, [&]<int T>() { rc = by_rows(a, T, [&](const TokenArgs& p) { return launch_forward<T>(who, p, s); }); });
    return rc;
}

int pxh_token_logprobs_backward(const void* logits, const void* targets, const float* lse, const float* entropy,
                                const float* d_logp, const float* d_entropy, void* dlogits, int type, int wide_targets,
                                long long rows, int vocab, long long stride, long long d_stride, float scale, void* stream)
{
    const char* who = "pxh_token_logprobs_backward";
    if (int rc = check_tokens(who, logits, type, wide_targets, rows, vocab, stride, scale)) return rc;
    if (!targets && d_logp) return fail_invalid("%s: a gradient of logp without targets", who);
    if (rows > 0 && (!lse || !dlogits || (d_entropy && !entropy))) return fail_invalid("%s: null pointer", who);
    if (rows > 0 && d_stride < vocab) return fail_invalid("%s: rows of %d logits that overlap", who, vocab);
    TokenArgs a{};
    a.logits = logits; a.targets = targets; a.lse_in = lse; a.entropy_in = entropy; a.d_logp = d_logp; a.d_entropy = d_entropy;
    a.dlogits = dlogits; a.rows = rows; a.stride = stride; a.d_stride = d_stride; a.vocab = vocab; a.wide = wide_targets; a.scale = scale;
    hipStream_t s = as_stream(stream);
    int rc = PXH_OK;
    dispatch_type(type, [&]<int T>() { rc = by_rows(a, T, [&](const TokenArgs& p) { return launch_gradient<T>(who, p, s); }); });
    return rc;
}

int pxh_token_logprobs_forward_train(const void* logits, const void* targets, const float* d_logp, const float* d_entropy,
                                     void* dlogits, float* logp, float* entropy, float* lse, int type, int wide_targets,
                                     long long rows, int vocab, long long stride, long long d_stride, float scale, void* stream)
{
    const char* who = "pxh_token_logprobs_forward_train";
    if (int rc = check_tokens(who, logits, type, wide_targets, rows, vocab, stride, scale)) return rc;
    if (!targets && (d_logp || logp)) return fail_invalid("%s: logp or its gradient without targets", who);
    if (rows > 0 && !dlogits) return fail_invalid("%s: null pointer", who);
    if (rows > 0 && d_stride < vocab) return fail_invalid("%s: rows of %d logits that overlap", who, vocab);
    TokenArgs a{};
    a.logits = logits; a.targets = targets; a.d_logp = d_logp; a.d_entropy = d_entropy; a.dlogits = dlogits; a.logp = logp;
    a.entropy = entropy; a.lse = lse; a.rows = rows; a.stride = stride; a.d_stride = d_stride; a.vocab = vocab;
    a.wide = wide_targets; a.scale = scale;
    hipStream_t s = as_stream(stream);
    int rc = PXH_OK;
    dispatch_type(type, [&]<int T>() {
        rc = by_rows(a, T, [&](const TokenArgs& p) {
            return entropy || d_entropy ? launch_train<T, true>(who, p, s) : launch_train<T, false>(who, p, s);
        });
    });
    return rc;
}

}
