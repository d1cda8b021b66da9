// Log probabilities of given tokens, entropy, the most probable alternatives, and the gradient of the logits.
#include "stream.h"
#include "tokens.h"
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

    // Adds the sums of o, whose peak is not above this one's.
    __device__ __forceinline__ void take(const Sums& o, float c)
    {
        const float t = (o.peak - reference()) * c;
        const float f = __builtin_amdgcn_exp2f(t);
        weighted += f * fmaf(fmaxf(t, kFar), o.sum, o.weighted);
        sum += o.sum * f;
    }

    // V more values
    template<int V>
    __device__ __forceinline__ void add(const float (&l)[V], float c)
    {
        Sums r{ peak, 0.0f, 0.0f };
#pragma unroll
        for (int k = 0; k < V; ++k) r.peak = fmaxf(r.peak, l[k]);
        r.take(*this, c);
        const float ref = r.reference();
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float u = (l[k] - ref) * c;
            const float e = __builtin_amdgcn_exp2f(u);
            r.sum += e;
            r.weighted = fmaf(e, fmaxf(u, kFar), r.weighted);
        }
        *this = r;
    }
};

__device__ __forceinline__ Sums nothing() { return Sums{ -INFINITY, 0.0f, 0.0f }; }

// Over a workgroup; the result in every lane.  The maximum first, then the sums relative to it: an exponential per lane.
template<int LANES>
__device__ __forceinline__ Sums group_join(Sums s, float c, Sums* slots)
{
    static_assert(LANES == kWave || LANES == 4 * kWave || LANES == 8 * kWave || LANES == 16 * kWave, "waves in part of a row of lanes");
    Sums w{ wave_max_by_rows(s.peak), 0.0f, 0.0f };
    w.take(s, c);
    w.sum = wave_sum_by_rows(w.sum);
    w.weighted = wave_sum_by_rows(w.weighted);
    if constexpr (LANES > kWave) {
        if ((threadIdx.x & (kWave - 1)) == 0) slots[threadIdx.x / kWave] = w;
        __syncthreads();
        // a wave's sums to a lane, and over as many lanes of a row of 16 as there are waves
        constexpr int kWaves = LANES / kWave;
        const Sums o = slots[threadIdx.x % kWaves];
        Sums all{ o.peak, 0.0f, 0.0f };
        all.peak = fmaxf(all.peak, lane_in_row<0xB1>(all.peak));
        all.peak = fmaxf(all.peak, lane_in_row<0x4E>(all.peak));
        if constexpr (kWaves > 4) all.peak = fmaxf(all.peak, lane_in_row<0x141>(all.peak));
        if constexpr (kWaves > 8) all.peak = fmaxf(all.peak, lane_in_row<0x140>(all.peak));
        all.take(o, c);
        const auto over_waves = [](float v) {
            v += lane_in_row<0xB1>(v);
            v += lane_in_row<0x4E>(v);
            if constexpr (kWaves > 4) v += lane_in_row<0x141>(v);
            if constexpr (kWaves > 8) v += lane_in_row<0x140>(v);
            return v;
        };
        all.sum = over_waves(all.sum);
        all.weighted = over_waves(all.weighted);
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
    float2* row_sums;       // nullable: the rows' largest logits and sums
    long long rows, stride, d_stride;
    int vocab, wide, top;
    float scale;
    float order_scale;      // what the logits are ordered times: the scale, or one, so that none meet in a rounded product
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
    float peak;                         // times the scale

    // of an alternative, from its logit times the scale: as that of the given token it is right where lse has lost the logarithm of the
    // sum beside huge logits
    __device__ __forceinline__ float logp(float z) const { return (z - peak) - log_sum; }
};

// What a row's sums say, with the given token's place (or -1) and logit.
__device__ __forceinline__ RowResult finish_row(const TokenArgs& a, long long row, const Sums& s, int target, float given, bool writes)
{
    // nothing but minus infinities; beside a NaN, which is above nothing, the sum is one
    const bool empty = s.peak == -INFINITY && s.sum == 0.0f;
    const float log_sum = logf(s.sum);
    RowResult r;
    r.log_sum = log_sum;
    r.peak = s.peak * a.scale;
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

// ---------------------------------------------------------------- alternatives
// One number that orders by value, then by the lowest index: the value's bits in their order in the upper half.  A NaN is below
// everything, and 0 is no value at all.
__device__ __forceinline__ uint32_t order_of(float z)
{
    const uint32_t bits = __float_as_uint(z + 0.0f);        // one zero
    return z != z ? 0u : (bits & 0x80000000u) ? ~bits : bits | 0x80000000u;
}

__device__ __forceinline__ unsigned long long key_of(float z, uint32_t index)
{
    return (static_cast<unsigned long long>(order_of(z)) << 32) | ~index;
}

__device__ __forceinline__ float value_of(unsigned long long key)
{
    const uint32_t order = static_cast<uint32_t>(key >> 32);
    if (order == 0) return __builtin_nanf("");
    return __uint_as_float((order & 0x80000000u) ? order & 0x7fffffffu : ~order);
}

constexpr uint32_t kNumber = 0x00800000u;       // the least order of a number: that of minus infinity is one less
// for 64 of 65536 normal values 270 pass on average, more than 512 in a row of 50, and more than 1024 in one of 100000
constexpr int kCandidates = 1024;

struct Selection {
    union {
        uint32_t orders[1024];                  // of the lanes, wave by wave
        unsigned long long list[kCandidates];
    };
    unsigned long long best[kWave];
    unsigned long long floor, most;
    uint32_t low;
    int count;
    bool mixed;
};

template<int CTRL>
__device__ __forceinline__ uint32_t max_in_row(uint32_t v)
{
    const uint32_t o = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), CTRL, 0xF, 0xF, true));
    return v > o ? v : o;
}

__device__ __forceinline__ uint32_t wave_max_of(uint32_t v)
{
    v = max_in_row<0x140>(max_in_row<0x141>(max_in_row<0x4E>(max_in_row<0xB1>(v))));
    const auto of_lane = [&](int lane) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), lane)); };
    return max(max(of_lane(0), of_lane(16)), max(of_lane(32), of_lane(48)));
}

__device__ __forceinline__ unsigned long long key_of_lane(unsigned long long key, int lane)
{
    const uint32_t low = __builtin_amdgcn_readlane(static_cast<int>(key), lane), high = __builtin_amdgcn_readlane(static_cast<int>(key >> 32), lane);
    return static_cast<unsigned long long>(high) << 32 | low;
}

// The key of a value that is no number, or 0.
__device__ __forceinline__ unsigned long long key_of_masked(float z, uint32_t index) { return z > -INFINITY ? 0ull : key_of(z, index); }

// The k largest keys of a workgroup, largest first: put(place, key), key 0 where there are fewer.  `best` is the largest order of
// the lane's keys, or less than kNumber where none is a number's; largest() is its largest key; above(floor, f) calls f with those of its
// keys that are not below `floor`, and may with others of its order; each(f) calls f with all keys of the workgroup, some by every lane; masked(i) is the
// key of the i-th of `values` values by their places, or 0 where that is a number.  OWN: largest() is of the keys that above() goes through.
// The lanes' maxima, in 64 columns (the lanes at one place in their waves), are as many different values, so the k-th largest of those
// is not above the k-th largest of all: only the lanes that reach it look at their values again, and little more than k values pass
// (8 of 16384 normal ones: 9 on average).  They are ranked by counting.
// Where many values are equal, too many would pass, or do: the columns' floor is then formed once more from whole keys, of which the
// lowest places are the largest, and what passes lies in the first vectors of a few columns (8 of 50001 values of one level: 57).
// Minus infinity never passes: where fewer than k values are numbers, the other places go to the first that are masked, of which
// there are enough among the first k.  Only where a NaN is among those, or too much passes all the same, does each place take a pass.
template<int LANES, bool OWN, typename Largest, typename Above, typename Each, typename Masked, typename Put>
__device__ __forceinline__ void select_largest(int k, int values, uint32_t best, const Largest& largest, const Above& above, const Each& each,
                                               const Masked& masked, const Put& put, Selection& s)
{
    static_assert(LANES % kWave == 0 && LANES <= 1024, "whole waves");
    const int lane = threadIdx.x % kWave;
    const bool first_wave = threadIdx.x < kWave;
    s.orders[threadIdx.x] = best;
    __syncthreads();
    if (first_wave) {
        uint32_t mine = best;
#pragma unroll
        for (int w = 1; w < LANES / kWave; ++w) mine = max(mine, s.orders[w * kWave + lane]);
        uint32_t low = 0;
        if (k <= 8) {
            // the k-th largest of different ones, which is no larger, or 0 where there are fewer: round by round
            uint32_t left = mine;
            for (int j = 0; j < k; ++j) {
                low = wave_max_of(left);
                left = left == low ? 0u : left;
            }
            if (static_cast<int>(__popcll(__ballot(mine >= max(low, kNumber)))) > 2 * k + 8) {
                // far more of them: once more, with those that are equal
                left = mine;
                for (int need = k; need > 0;) {
                    low = wave_max_of(left);
                    if (low < kNumber) break;
                    need -= __popcll(__ballot(left == low));
                    left = left == low ? 0u : left;
                }
            }
        } else {
            int larger = 0;
#pragma unroll
            for (int j = 0; j < kWave; ++j) larger += static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(mine), j)) > mine;
            low = ~wave_max_of(larger < k ? ~mine : 0u);
        }
        low = max(low, kNumber);
        const int reach = __popcll(__ballot(mine >= low));
        s.best[lane] = 0;
        if (lane == 0) {
            if (reach < k) low = kNumber;
            s.floor = static_cast<unsigned long long>(low) << 32;
            s.count = 0;
            s.low = reach == kWave && k < kWave ? 0 : low;      // every column reaches it: there may be any number of them
        }
    }
    __syncthreads();
    int n = kCandidates + 1;
    const auto pass = [&]<bool EXACT>(unsigned long long floor, bool reaches) {
        if (reaches)
            above(floor, [&](unsigned long long key) {
                if (EXACT && key < floor) return;
                const int at = atomicAdd(&s.count, 1);
                if (at < kCandidates) s.list[at] = key;
            });
        __syncthreads();
        n = __builtin_amdgcn_readfirstlane(s.count);
    };
    if (const uint32_t low = __builtin_amdgcn_readfirstlane(s.low)) pass.template operator()<false>(static_cast<unsigned long long>(low) << 32, !OWN || best >= low);
    if (n > 12 * k + 24) {           // few as they are, they are ranked sooner than looked for again
        const unsigned long long mine = !OWN || best >= static_cast<uint32_t>(s.floor >> 32) ? largest() : 0ull;
        if (mine) atomicMax(&s.best[lane], mine);
        __syncthreads();
        if (first_wave) {
            const unsigned long long column = s.best[lane];
            int larger = 0;
            for (int j = 0; j < kWave; ++j) larger += key_of_lane(column, j) > column;
            const unsigned long long at = __ballot(column != 0 && larger == k - 1);
            if (lane == 0) s.count = 0;
            if (at != 0) {
                const unsigned long long kth = key_of_lane(column, __ffsll(at) - 1);
                if (lane == 0) s.floor = kth;
            }
        }
        __syncthreads();
        const unsigned long long floor = key_of_lane(s.floor, 0);
        pass.template operator()<true>(floor, !OWN || mine >= floor);
    }
    if (n <= kCandidates) {
        for (int t = threadIdx.x; t < n; t += LANES) {
            const unsigned long long key = s.list[t];
            int larger = 0;
            for (int j = 0; j < n; ++j) larger += s.list[j] > key;
            if (larger < k) put(larger, key);
        }
        if (n >= k) return;
        if (first_wave) {
            const unsigned long long key = lane < min(k, values) ? masked(lane) : 0ull;
            const bool infinity = static_cast<uint32_t>(key >> 32) == kNumber - 1;
            const unsigned long long infinite = __ballot(infinity);
            const bool mixed = __ballot(key != 0 && !infinity) != 0;
            if (lane == 0) s.mixed = mixed;
            if (!mixed) {
                const int place = n + __popcll(infinite & ((1ull << lane) - 1));
                if (infinity && place < k) put(place, key);
                for (int t = n + __popcll(infinite) + lane; t < k; t += kWave) put(t, 0ull);
            }
        }
        __syncthreads();
        if (!s.mixed) return;
    }
    unsigned long long before = ~0ull;
    for (int place = 0; place < k; ++place) {
        __syncthreads();
        if (threadIdx.x == 0) s.most = 0;
        __syncthreads();
        unsigned long long mine = 0;
        each([&](unsigned long long key) {
            if (key < before && key > mine) mine = key;
        });
        atomicMax(&s.most, mine);
        __syncthreads();
        before = s.most;
        if (threadIdx.x == 0) put(place, before);
    }
}

// ---------------------------------------------------------------- a part of a row
// Vectors first .. first + count of a row, K to a lane, and of the row's last values, which fill no vector, one to each of the
// first lanes of the part that has them.  What is not there is minus infinity.
constexpr int kMostVectors = 8;         // vectors of a lane
// ... of one of 512 for a row that 1024 would hold otherwise: held to 80 registers, so that three such workgroups share a unit and not two
// (4096 x 50001 half with three alternatives, when it was taken, 92.6 -> 84.6 us; 16 vectors are 85 registers, two workgroups, and 101.7)
constexpr int kThirdVectors = 14;

// SETTLES: rows of 16-bit values off a 4-byte boundary are read from one value further on (below).  For the lanes of 14 vectors, where every
// other row is: half with three alternatives, 4096 x 32777 59.0 -> 57.6 us, x 40001 67.9 -> 62.4, x 50001 83.2 -> 76.3, x 57345 94.1 -> 83.3;
// at the short end with few rows it loses (1100 x 32777 bf16 16.4 -> 17.9, x 57351 35.9 -> 33.0).  The other forms lose (8000 x 17001
// 55.5 -> 58, 300 x 50001 14.8 -> 16.2).
template<int T, int LANES, int K, bool NT, bool SETTLES = false>
struct Part {
    static constexpr bool kSettles = SETTLES && kSize<T> == 2;
    static constexpr int V = kVec<T>;
    Raw<T, V> kept[K];
    float extra, peak;          // peak: the largest of the lane's values, from sums()
    int first, count, extra_at;
    uint32_t before;            // lane k: lane 0's first value in step k, where `odd`
    bool odd;

    __device__ __forceinline__ bool has(int k) const { return k * LANES + static_cast<int>(threadIdx.x) < count; }
    __device__ __forceinline__ int at(int k) const { return (first + k * LANES + static_cast<int>(threadIdx.x)) * V; }

    // of the part's values, in a row of `vocab`
    __device__ __forceinline__ int end(int vocab) const { return (first + count) * V + V > vocab ? vocab : (first + count) * V; }

    __device__ __forceinline__ void load(const char* row, int vocab, int first_vector, int vectors)
    {
        constexpr uint32_t nothing = T == PXH_F32 ? 0xff800000u : T == PXH_BF16 ? 0xff80ff80u : 0xfc00fc00u;
        const int whole = vocab / V;
        first = first_vector;
        count = min(vectors, whole - first_vector);
        // before the vectors, which are waited for in their order (8000 x 17000 bf16 with five alternatives 106 -> 94 us), and without a
        // branch, whose end would wait for all loads
        extra_at = whole * V + static_cast<int>(threadIdx.x);
        if (first_vector + vectors < whole || extra_at >= vocab) extra_at = -1;
        extra = load_one<T>(row, extra_at < 0 ? 0 : extra_at);
        if (extra_at < 0) extra = -INFINITY;
        const char* place = row;
        if constexpr (kSettles) {
            // Vectors off a 4-byte boundary are slow to load: one value further on they are not, and that value is the neighbour's to give.
            // The last one reads the first of the values that fill no vector, so there have to be some.
            odd = (reinterpret_cast<uintptr_t>(row) & 2) && whole * V < vocab;
            const int lane = threadIdx.x % kWave, of = lane * LANES + static_cast<int>(threadIdx.x) - lane;
            before = global_memory<uint16_t>(row)[odd && lane < K && of < count ? (first + of) * V : 0];
            place += odd ? 2 : 0;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
#pragma unroll
            for (int i = 0; i < Raw<T, V>::kWords; ++i) kept[k].w[i] = nothing;
            if (has(k)) kept[k] = load_raw_at<T, V, NT>(place + (static_cast<size_t>(first) + k * LANES) * 16, threadIdx.x * 16u);
        }
        if constexpr (kSettles)
            if (odd) settle();
    }

    // Values 1 to 8 of a vector become 0 to 7: the first is the last one of the lane in front, and lane 0's is in `before`.
    __device__ __forceinline__ void settle()
    {
        constexpr int kBehind = 0x138;          // every lane the value of the lane in front; lane 0 keeps the old one
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (k * LANES >= count) break;
            uint32_t (&w)[4] = kept[k].w;
            const uint32_t given = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(before), k)) << 16;
            const uint32_t front = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(static_cast<int>(given), static_cast<int>(w[3]), kBehind, 0xF, 0xF, false));
            if (!has(k)) continue;
            w[3] = __builtin_amdgcn_alignbit(w[3], w[2], 16);
            w[2] = __builtin_amdgcn_alignbit(w[2], w[1], 16);
            w[1] = __builtin_amdgcn_alignbit(w[1], w[0], 16);
            w[0] = __builtin_amdgcn_alignbit(w[0], front, 16);
        }
    }

    // Between two passes over the values: as fp32 numbers, which the compiler would keep from the first, they take twice the
    // registers that they were read into (8 vectors of bf16: 169 in place of 60, two waves to a unit in place of eight).
    __device__ __forceinline__ void again()
    {
        typedef uint32_t words __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int k = 0; k < K; ++k) {
            words w = __builtin_bit_cast(words, kept[k]);
            asm volatile("" : "+v"(w));
            kept[k] = __builtin_bit_cast(Raw<T, V>, w);
        }
    }

    // The lane's number, so that the compiler does not keep a place for each value, or the eight or fourteen masks of the lanes that have a
    // vector, from one look at them to the next: with more than 80 scalar registers a wave, one workgroup of 1024 lanes has a unit and not
    // two (300 x 50001 bf16 with three alternatives 19.1 us in place of 14.1)
    __device__ __forceinline__ int lane_again() const
    {
        int lane = threadIdx.x;
        asm volatile("" : "+v"(lane));
        return lane;
    }

    // The sums of the lane's values.  An exponent is one fused multiply-add, l * c - peak * c (which a half-precision value enters
    // without being converted first), where the rounding of peak * c is less than 2^-4: it is the same in all of the lane's
    // exponents, and taken out of the sums at the end.  Beyond that, in rows of huge values, (l - peak) * c, value by value
    // from memory: two ways through the registers would hold them twice.
    template<bool ENTROPY>
    __device__ __forceinline__ Sums sums(const char* row, float c)
    {
        peak = largest();
        again();
        Sums s{ peak, 0.0f, 0.0f };
        const float ref = s.reference();
        const float shift = ref * c;
        if (!__all(fabsf(shift) < 0x1p20f)) return far_sums(row, c);
        const auto add = [&](float l) {
            const float u = fmaf(l, c, -shift);
            const float e = __builtin_amdgcn_exp2f(u);
            s.sum += e;
            if (ENTROPY) s.weighted = fmaf(e, fmaxf(u, kFar), s.weighted);
        };
        add(extra);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (k * LANES >= count) break;
            float l[V];
            kept[k].get(l);
#pragma unroll
            for (int i = 0; i < V; ++i) add(l[i]);
            __builtin_amdgcn_sched_barrier(0);
        }
        const float off = fmaf(ref, c, -shift), f = __builtin_amdgcn_exp2f(-off);
        s.weighted = f * fmaf(-off, s.sum, s.weighted);
        s.sum *= f;
        return s;
    }

    // The largest of one vector.
    __device__ __forceinline__ float largest_of(const Raw<T, V>& raw) const
    {
        if constexpr (T == PXH_F16) {
            typedef _Float16 two __attribute__((ext_vector_type(2)));
            two pair = __builtin_bit_cast(two, raw.w[0]);
#pragma unroll
            for (int i = 1; i < Raw<T, V>::kWords; ++i) pair = __builtin_elementwise_max(pair, __builtin_bit_cast(two, raw.w[i]));
            return fmaxf(static_cast<float>(pair.x), static_cast<float>(pair.y));
        } else {
            float l[V];
            raw.get(l);
            float most = l[0];
#pragma unroll
            for (int i = 1; i < V; ++i) most = fmaxf(most, l[i]);
            return most;
        }
    }

    __device__ __forceinline__ float largest() const
    {
        float most = extra;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (k * LANES >= count) break;
            most = fmaxf(most, largest_of(kept[k]));
            __builtin_amdgcn_sched_barrier(0);          // a vector at a time, in few registers
        }
        return most;
    }

    __device__ __forceinline__ Sums far_sums(const char* row, float c) const
    {
        Sums s{ extra, extra == -INFINITY ? 0.0f : 1.0f, 0.0f };
        for (int k = 0; k < K && has(k); ++k)
            for (int i = 0; i < V; ++i) s.template add<1>({ load_one<T>(row, at(k) + i) }, c);
        return s;
    }

    // The largest key of the lane's values, one of which is a number: the first place of the peak.
    __device__ __forceinline__ unsigned long long largest_key(float scale)
    {
        again();
        const float z = peak * scale;
        const int lane = lane_again(), place = (first + lane) * V;
        int index = -1;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!__any(index < 0)) break;
            if (index >= 0 || k * LANES + lane >= count) continue;
            float l[V];
            kept[k].get(l);
#pragma unroll
            for (int i = V - 1; i >= 0; --i)
                if (l[i] * scale == z) index = place + k * LANES * V + i;
            __builtin_amdgcn_sched_barrier(0);
        }
        return key_of(z, index < 0 ? extra_at : index);
    }

    // f with the keys of all values whose order is not below that of `floor`, which is a number's; of those that are equal to it, some of those
    // behind its place may be left out.  A vector at a time: one whose largest value is not enough is passed over
    template<typename F>
    __device__ __forceinline__ void above(float scale, unsigned long long floor, const F& f)
    {
        again();
        const float least = value_of(floor);
        const uint32_t last = ~static_cast<uint32_t>(floor);
        const int lane = lane_again(), place = (first + lane) * V;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (k * LANES + lane >= count) continue;
            const float most = largest_of(kept[k]) * scale;
            if (!(most > least || (most == least && static_cast<uint32_t>(place + k * LANES * V) <= last))) continue;
            float l[V];
            kept[k].get(l);
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (l[i] * scale >= least) f(key_of(l[i] * scale, place + k * LANES * V + i));
        }
        if (extra_at >= 0 && extra * scale >= least) f(key_of(extra * scale, extra_at));
    }

    // f with the keys of all values of the part, read from memory one by one
    template<typename F>
    __device__ __forceinline__ void each(const char* row, int vocab, float scale, const F& f) const
    {
        for (int e = first * V + static_cast<int>(threadIdx.x); e < end(vocab); e += LANES) f(key_of(load_one<T>(row, e) * scale, e));
    }
};

// ---------------------------------------------------------------- forward
// A workgroup takes one part of a row into its registers; a row of several parts is put together by a second launch from
// their sums and their largest values.  4096 x 50001 half with entropy and three alternatives: 410 MB in 74.5 us, 5.5 TB/s.  The
// arithmetic alone, 8.5 instructions a value counting an exponential as four, is 44 us; it waits for the row's maximum, so that the
// next row's loads, another workgroup's, have to cover it.
struct Parts {
    unsigned long long* keys;       // [rows][parts][top]
    Sums* sums;                     // [rows][parts]
    int parts, vectors;             // parts of a row, vectors of a part
    FastDiv by_parts;
};

template<int T, bool ENTROPY, int LANES, int K, bool NT>
__global__ __launch_bounds__(LANES, K == kThirdVectors ? 6 : 1) void token_logprobs_kernel(TokenArgs a, Parts p)
{
    __shared__ Sums slots[LANES / kWave];
    __shared__ Selection selection;
    uint32_t row, part;
    p.by_parts.divmod(blockIdx.x, row, part);
    const char* logits = static_cast<const char*>(a.logits) + row * a.stride * kSize<T>;
    const float c = a.scale * kLog2e;
    const bool whole = p.parts == 1;
    const int target = whole ? target_of(a, row) : -1;
    const float given = load_one<T>(logits, target < 0 ? 0 : target);
    Part<T, LANES, K, NT, K == kThirdVectors> mine;
    mine.load(logits, a.vocab, static_cast<int>(part) * p.vectors, p.vectors);
    const Sums s = group_join<LANES>(mine.template sums<ENTROPY>(logits, c), c, slots);
    RowResult result{};
    if (whole) {
        result = finish_row(a, row, s, target, given, threadIdx.x == 0);
        if (a.row_sums && threadIdx.x == 0) a.row_sums[row] = make_float2(s.peak, s.sum);
    } else if (threadIdx.x == 0) {
        p.sums[blockIdx.x] = s;
    }
    if (a.top) {
        // a lane of NaNs has minus infinity for its peak, which need not be a value of the row: no floor comes from there
        const float peak = mine.peak * a.order_scale;
        const auto put = [&](int place, unsigned long long key) {
            if (whole) {
                a.top_ids[static_cast<long long>(row) * a.top + place] = static_cast<int>(~static_cast<uint32_t>(key));
                a.top_logp[static_cast<long long>(row) * a.top + place] = result.logp(value_of(key));
            } else {
                p.keys[static_cast<size_t>(blockIdx.x) * a.top + place] = key;
            }
        };
        const int begin = mine.first * kVec<T>;
        const auto largest = [&] { return mine.largest_key(a.order_scale); };
        const auto above = [&](unsigned long long floor, const auto& f) { mine.above(a.order_scale, floor, f); };
        const auto each = [&](const auto& f) { mine.each(logits, a.vocab, a.order_scale, f); };
        const auto masked = [&](int i) { return key_of_masked(load_one<T>(logits, begin + i) * a.order_scale, begin + i); };
        select_largest<LANES, true>(a.top, mine.end(a.vocab) - begin, peak > -INFINITY ? order_of(peak) : 0u, largest, above, each, masked, put, selection);
    }
}

// A row's parts put together by one wave: at most 64 of them, and as many keys.
template<int T>
__global__ __launch_bounds__(kBlock) void token_join_few_kernel(TokenArgs a, Parts p)
{
    const int lane = threadIdx.x % kWave;
    const long long row = static_cast<long long>(blockIdx.x) * (kBlock / kWave) + threadIdx.x / kWave;
    if (row >= a.rows) return;                  // a whole wave, and none waits for another
    const float c = a.scale * kLog2e;
    const int target = target_of(a, row);
    const float given = load_one<T>(static_cast<const char*>(a.logits) + row * a.stride * kSize<T>, target < 0 ? 0 : target);
    const int n = p.parts * a.top;
    const unsigned long long mine = lane < n ? p.keys[row * n + lane] : 0;
    Sums s = nothing();
    if (lane < p.parts) s = p.sums[row * p.parts + lane];
    s = group_join<kWave>(s, c, nullptr);
    const RowResult result = finish_row(a, row, s, target, given, lane == 0);
    if (a.row_sums && lane == 0) a.row_sums[row] = make_float2(s.peak, s.sum);
    int larger = 0;
    for (int j = 0; j < n; ++j) larger += key_of_lane(mine, j) > mine;
    if (lane < n && larger < a.top) {
        a.top_ids[row * a.top + larger] = static_cast<int>(~static_cast<uint32_t>(mine));
        a.top_logp[row * a.top + larger] = result.logp(value_of(mine));
    }
}

template<int T>
__global__ __launch_bounds__(kBlock) void token_join_kernel(TokenArgs a, Parts p)
{
    __shared__ Sums slots[kBlock / kWave];
    __shared__ Selection selection;
    const long long row = blockIdx.x;
    const float c = a.scale * kLog2e;
    const int target = target_of(a, row);
    const float given = target < 0 ? 0.0f : load_one<T>(static_cast<const char*>(a.logits) + row * a.stride * kSize<T>, target);
    Sums s = nothing();
    for (int k = threadIdx.x; k < p.parts; k += kBlock) {
        const Sums o = p.sums[row * p.parts + k];
        Sums r{ fmaxf(s.peak, o.peak), 0.0f, 0.0f };
        r.take(s, c);
        r.take(o, c);
        s = r;
    }
    s = group_join<kBlock>(s, c, slots);
    const RowResult result = finish_row(a, row, s, target, given, threadIdx.x == 0);
    if (a.row_sums && threadIdx.x == 0) a.row_sums[row] = make_float2(s.peak, s.sum);
    if (a.top) {
        const unsigned long long* keys = p.keys + static_cast<size_t>(row) * p.parts * a.top;
        const int n = p.parts * a.top;
        unsigned long long best = 0;
        // by places, so that the columns have the parts' first ones; where those are equal, by parts, whose first has the lowest places
        const auto each = [&](const auto& f) {
            for (int k = threadIdx.x; k < n; k += kBlock) {
                uint32_t place, part;
                p.by_parts.divmod(k, place, part);
                if (const unsigned long long key = keys[part * a.top + place]) f(key);
            }
        };
        each([&](unsigned long long key) { best = max(best, key); });
        const auto first_keys = [&] {
            unsigned long long most = 0;
            for (int k = threadIdx.x; k < n; k += kBlock) most = max(most, keys[k]);
            return most >> 32 < kNumber ? 0ull : most;
        };
        const char* logits = static_cast<const char*>(a.logits) + row * a.stride * kSize<T>;
        const auto above = [&](unsigned long long floor, const auto& f) {
            each([&](unsigned long long key) {
                if (key >> 32 >= floor >> 32) f(key);
            });
        };
        const auto masked = [&](int i) { return key_of_masked(load_one<T>(logits, i) * a.order_scale, i); };
        const auto put = [&](int place, unsigned long long key) {
            a.top_ids[row * a.top + place] = static_cast<int>(~static_cast<uint32_t>(key));
            a.top_logp[row * a.top + place] = result.logp(value_of(key));
        };
        select_largest<kBlock, false>(a.top, a.vocab, static_cast<uint32_t>(best >> 32), first_keys, above, each, masked, put, selection);
    }
}

// ---------------------------------------------------------------- gradient
//   d_j = scale * (g * ((j == target) - p_j) - h * p_j * (log p_j + entropy)),  p = exp(z - lse)
// From the row's own sums log p = (l - peak) * scale - log(sum), which is right however large the logits are; from a stored lse,
// which fp32 has rounded, log p = l * scale - lse.  The hardware's exp2 has no results below 2^-126; a type that has them
// gets them from the square of half the exponent's power.
// A 16-bit gradient of logp alone takes its exponent from one fused multiply-add, l * c - shift, where the shift is below 2^10 and
// its rounding, below 2^-14, far less than the result's own: 8.5 instructions a value in place of 13 (an exponential counts four).
template<int T, bool PEAK>
struct RowGradient {
    float peak, rest, scale, entropy, g, h, c, shift;
    int target;
    bool quick;

    // QUICK where `quick` says so
    template<int V, bool QUICK>
    __device__ __forceinline__ void apply(const float (&l)[V], int e, float (&d)[V]) const
    {
        if constexpr (T != PXH_F32 && QUICK) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                if constexpr (T == PXH_F16) {
                    d[k] = -g * __builtin_amdgcn_exp2f(fmaf(l[k], c, -shift));
                } else {
                    const float root = __builtin_amdgcn_exp2f(fmaf(l[k], c, -shift));
                    d[k] = -g * root * root;
                }
            }
            hit<V>(e, d);
            return;
        }
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
        hit<V>(e, d);
    }

    // the given token's own part
    template<int V>
    __device__ __forceinline__ void hit(int e, float (&d)[V]) const
    {
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
    r.c = a.scale * (T == PXH_F16 ? kLog2e : 0.5f * kLog2e);
    r.shift = fmaf(r.peak, a.scale, r.rest) * (T == PXH_F16 ? kLog2e : 0.5f * kLog2e);
    r.quick = __builtin_amdgcn_readfirstlane(r.h == 0.0f && fabsf(r.shift) < 0x1p10f);
    return r;
}

// A workgroup takes one part of a row: 1000 x 100001 fp32 with the entropy's gradient is 800 MB in 137 us, 5.8 TB/s where a copy has
// 6.6.  Past the caches in short parts (1000 x 100001 fp32: 149 us with four steps through the caches, 144
// with four past them, 137 with two), within them in longer ones (512 x 32768 bf16: 11.5 us, and 13 past them).
template<bool NT>
constexpr int kGradientSteps = NT ? 2 : 4;

// A row's vectors begin at its first 16-byte boundary (4096 x 50001 half with the entropy's gradient 138 -> 134 us).  The passes that sum over a row
// begin at its first value, so that a row's results do not depend on its address (on the number of rows they do, by the last bits: the
// lanes of a row and its parts are chosen by it).
template<int T, bool NT>
__global__ __launch_bounds__(kBlock) void token_gradient_kernel(TokenArgs a, FastDiv parts)
{
    constexpr int V = kVec<T>;
    uint32_t row, part;
    parts.divmod(blockIdx.x, row, part);
    const auto r = gradient_of<T, false>(a, row, target_of(a, row), 0.0f, a.lse_in[row], a.d_entropy ? a.entropy_in[row] : 0.0f);
    const char* logits = static_cast<const char*>(a.logits) + row * a.stride * kSize<T>;
    char* out = static_cast<char*>(a.dlogits) + row * a.d_stride * kSize<T>;
    const int head = min(static_cast<int>(-reinterpret_cast<uintptr_t>(logits) & 15) / kSize<T>, a.vocab);
    const int whole = (a.vocab - head) / V;
    const auto write = [&]<bool QUICK>() {
#pragma unroll
        for (int s = 0; s < kGradientSteps<NT>; ++s) {
            const int v = (part * kGradientSteps<NT> + s) * kBlock + threadIdx.x;
            if (v >= whole) break;
            float l[V], d[V];
            load_raw<T, V, NT>(logits, head + v * V).get(l);
            r.template apply<V, QUICK>(l, head + v * V, d);
            Raw<T, V> raw;
            raw.set(d);
            store_raw<T, V, NT>(out, head + v * V, raw);
        }
        // what fills no vector
        int e = threadIdx.x;
        if (e >= head) e += whole * V;
        if (part == 0 && e < a.vocab) {
            float d[1];
            r.template apply<1, QUICK>({ load_one<T>(logits, e) }, e, d);
            store_one<T>(out, e, d[0]);
        }
    };
    if (T != PXH_F32 && r.quick) write.template operator()<true>();
    else write.template operator()<false>();
}

// ---------------------------------------------------------------- forward and gradient at once
// A workgroup per row, which stays in registers between its sums and its gradient.  A lane writes the values that it has read, so the
// gradient may take the logits' place.  1024 lanes of 8 vectors are held to 64 registers, so that two rows share a unit and not one
// (2000 x 65536 bf16 110 -> 102 us).
template<int T, bool ENTROPY, int LANES, int K, bool NT>
__global__ __launch_bounds__(LANES, LANES == 1024 && K == 8 ? 8 : 1) void token_train_kernel(TokenArgs a)
{
    constexpr int V = kVec<T>;
    __shared__ Sums slots[LANES / kWave];
    const long long row = blockIdx.x;
    const char* logits = static_cast<const char*>(a.logits) + row * a.stride * kSize<T>;
    char* out = static_cast<char*>(a.dlogits) + row * a.d_stride * kSize<T>;
    const float c = a.scale * kLog2e;
    const int target = target_of(a, row);
    const float given = load_one<T>(logits, target < 0 ? 0 : target);       // before it is overwritten
    Part<T, LANES, K, NT> mine;
    mine.load(logits, a.vocab, 0, a.vocab);
    const Sums s = group_join<LANES>(mine.template sums<ENTROPY>(logits, c), c, slots);
    const RowResult r = finish_row(a, row, s, target, given, threadIdx.x == 0);
    const auto gradient = gradient_of<T, true>(a, row, target, s.peak, r.log_sum, r.entropy);
    mine.again();
    const auto write = [&]<bool QUICK>() {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!mine.has(k)) continue;
            float l[V], d[V];
            mine.kept[k].get(l);
            gradient.template apply<V, QUICK>(l, mine.at(k), d);
            Raw<T, V> o;
            o.set(d);
            store_raw_at<T, V>(out + static_cast<size_t>(k) * LANES * 16, threadIdx.x * 16u, o);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (mine.extra_at >= 0) {
            float d[1];
            gradient.template apply<1, QUICK>({ mine.extra }, mine.extra_at, d);
            store_one<T>(out, mine.extra_at, d[0]);
        }
    };
    if (T != PXH_F32 && gradient.quick) write.template operator()<true>();
    else write.template operator()<false>();
}

// The same for a gradient of logp alone over rows of up to 4096 vectors: not the values stay in registers but their powers, so that
// there is one exponential a value and not two (13 instructions a value of bf16 in place of 17, counting an exponential as four;
// 8192 x 32768: 203 -> 192 us; with loads past the caches 189.6, 1074 MB at 5.7 TB/s).  A type with results below 2^-126 keeps
// their roots.
template<int T, bool ENTROPY, int LANES, int K, bool NT>
__global__ __launch_bounds__(LANES) void token_powers_kernel(TokenArgs a)
{
    constexpr int V = kVec<T>;
    constexpr bool kRoots = T != PXH_F16;
    __shared__ Sums slots[LANES / kWave];
    const long long row = blockIdx.x;
    const char* logits = static_cast<const char*>(a.logits) + row * a.stride * kSize<T>;
    char* out = static_cast<char*>(a.dlogits) + row * a.d_stride * kSize<T>;
    const float c = a.scale * kLog2e;
    const int target = target_of(a, row);
    const float given = load_one<T>(logits, target < 0 ? 0 : target);       // before it is overwritten
    float power[K][V], last;
    float peak, shift, off;
    Sums s;
    bool near;
    {
        Part<T, LANES, K, NT> mine;
        mine.load(logits, a.vocab, 0, a.vocab);
        last = mine.extra;
        peak = mine.largest();
        s = Sums{ peak, 0.0f, 0.0f };
        const float ref = s.reference();
        shift = ref * c;
        near = __all(fabsf(shift) < 0x1p20f);       // as in sums()
        off = fmaf(ref, c, -shift);
        if (near) {
            const float c1 = kRoots ? 0.5f * c : c, shift1 = kRoots ? 0.5f * shift : shift;
            const auto take = [&](float l) {
                const float u = fmaf(l, c1, -shift1);
                const float r = __builtin_amdgcn_exp2f(u);
                const float e = kRoots ? r * r : r;
                s.sum += e;
                if (ENTROPY) s.weighted = fmaf(e, fmaxf(u, kFar), s.weighted);
                return r;
            };
            last = take(last);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (k * LANES >= mine.count) break;
                float l[V];
                mine.kept[k].get(l);
#pragma unroll
                for (int i = 0; i < V; ++i) power[k][i] = take(l[i]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (kRoots) s.weighted *= 2.0f;
            const float f = __builtin_amdgcn_exp2f(-off);
            s.weighted = f * fmaf(-off, s.sum, s.weighted);
            s.sum *= f;
        } else {
            s = mine.far_sums(logits, c);
        }
    }
    s = group_join<LANES>(s, c, slots);
    const RowResult r = finish_row(a, row, s, target, given, threadIdx.x == 0);
    const auto gradient = gradient_of<T, true>(a, row, target, s.peak, r.log_sum, r.entropy);
    const int count = a.vocab / V;
    const int extra_at = count * V + static_cast<int>(threadIdx.x) < a.vocab ? count * V + static_cast<int>(threadIdx.x) : -1;
    if (near) {
        // p = power * 2^((lane's peak - row's peak) * c - off) / sum
        float f = peak == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(((peak - s.peak) * c - off) * (kRoots ? 0.5f : 1.0f));
        const float scaled = gradient.g == 0.0f ? 0.0f : -gradient.g / s.sum;
        if (!kRoots) f *= scaled;
        const auto result = [&](float r) {
            const float q = r * f;
            return kRoots ? scaled * q * q : q;
        };
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (k * LANES + static_cast<int>(threadIdx.x) >= count) continue;
            float d[V];
#pragma unroll
            for (int i = 0; i < V; ++i) d[i] = result(power[k][i]);
            gradient.template hit<V>((k * LANES + static_cast<int>(threadIdx.x)) * V, d);
            Raw<T, V> o;
            o.set(d);
            store_raw_at<T, V>(out + static_cast<size_t>(k) * LANES * 16, threadIdx.x * 16u, o);
        }
        if (extra_at >= 0) {
            float d[1] = { result(last) };
            gradient.template hit<1>(extra_at, d);
            store_one<T>(out, extra_at, d[0]);
        }
    } else {
        for (int v = threadIdx.x; v < count; v += LANES) {
            float l[V], d[V];
            load_raw<T, V>(logits, static_cast<size_t>(v) * V).get(l);
            gradient.template apply<V, false>(l, v * V, d);
            Raw<T, V> o;
            o.set(d);
            store_raw<T, V>(out, static_cast<size_t>(v) * V, o);
        }
        if (extra_at >= 0) {
            float d[1];
            gradient.template apply<1, false>({ last }, extra_at, d);
            store_one<T>(out, extra_at, d[0]);
        }
    }
}

// Rows that no workgroup's registers hold are read twice.
template<int T>
__global__ __launch_bounds__(1024) void token_train_long_kernel(TokenArgs a)
{
    constexpr int V = kVec<T>;
    __shared__ Sums slots[1024 / kWave];
    const long long row = blockIdx.x;
    const char* logits = static_cast<const char*>(a.logits) + row * a.stride * kSize<T>;
    char* out = static_cast<char*>(a.dlogits) + row * a.d_stride * kSize<T>;
    const float c = a.scale * kLog2e;
    const int target = target_of(a, row);
    const float given = target < 0 ? 0.0f : load_one<T>(logits, target);        // before it is overwritten
    Sums s = nothing();
    for (int e = threadIdx.x * V; e < a.vocab; e += 1024 * V) {
        float l[V];
        load_row<T, V>(logits, e, a.vocab, -INFINITY).get(l);
        s.add(l, c);
    }
    s = group_join<1024>(s, c, slots);
    const RowResult r = finish_row(a, row, s, target, given, threadIdx.x == 0);
    const auto gradient = gradient_of<T, true>(a, row, target, s.peak, r.log_sum, r.entropy);
    for (int e = threadIdx.x * V; e < a.vocab; e += 1024 * V) {
        float l[V], d[V];
        load_row<T, V>(logits, e, a.vocab).get(l);
        gradient.template apply<V, false>(l, e, d);
        Raw<T, V> o;
        o.set(d);
        store_row<T, V>(out, e, a.vocab, o);
    }
}

// The logits past the caches where they and the gradient do not fit (8192 x 32768 bf16 192 -> 187 us; 512 x 32768 would lose 8 %).
template<int T, bool ENTROPY, bool NT>
int launch_train(const char* who, const TokenArgs& a, hipStream_t s)
{
    const dim3 grid(static_cast<unsigned>(a.rows));
    const int vectors = a.vocab / kVec<T>;
    if (!a.d_entropy && vectors <= 4096) {
        if (vectors <= 256) hipLaunchKernelGGL((token_powers_kernel<T, ENTROPY, 256, 1, NT>), grid, dim3(256), 0, s, a);
        else if (vectors <= 1024) hipLaunchKernelGGL((token_powers_kernel<T, ENTROPY, 256, 4, NT>), grid, dim3(256), 0, s, a);
        else if (vectors <= 2048) hipLaunchKernelGGL((token_powers_kernel<T, ENTROPY, 512, 4, NT>), grid, dim3(512), 0, s, a);
        else hipLaunchKernelGGL((token_powers_kernel<T, ENTROPY, 512, 8, NT>), grid, dim3(512), 0, s, a);
        return check_launch(who);
    }
    if (vectors <= 256) hipLaunchKernelGGL((token_train_kernel<T, ENTROPY, 256, 1, NT>), grid, dim3(256), 0, s, a);
    else if (vectors <= 1024) hipLaunchKernelGGL((token_train_kernel<T, ENTROPY, 256, 4, NT>), grid, dim3(256), 0, s, a);
    else if (vectors <= 4096) hipLaunchKernelGGL((token_train_kernel<T, ENTROPY, 512, 8, NT>), grid, dim3(512), 0, s, a);
    else if (vectors <= 8192) hipLaunchKernelGGL((token_train_kernel<T, ENTROPY, 1024, 8, NT>), grid, dim3(1024), 0, s, a);
    else if (vectors <= 16384) hipLaunchKernelGGL((token_train_kernel<T, ENTROPY, 1024, 16, NT>), grid, dim3(1024), 0, s, a);
    else if (vectors <= 20480) hipLaunchKernelGGL((token_train_kernel<T, ENTROPY, 1024, 20, NT>), grid, dim3(1024), 0, s, a);
    else hipLaunchKernelGGL((token_train_long_kernel<T>), grid, dim3(1024), 0, s, a);
    return check_launch(who);
}

// Whether tensors of the logits' size, `tensors` of them, go past the caches.
inline bool streams(const TokenArgs& a, int type, int tensors)
{
    return static_cast<size_t>(a.rows) * static_cast<size_t>(a.vocab) * size_of(type) * tensors >= kStreamingBytes;
}

// Workgroups that fill the machine four times over: from there on a workgroup takes as much as its registers hold.
constexpr long long kEnoughParts = 1024;

// Lanes of the workgroup that takes a whole row, without a second launch, or 0.  1024 up to 4096 vectors whatever the rows (8 x 32768 bf16
// 8.0 us in parts, 5.0 whole; 256 x 32768 with five alternatives 14.2 and 9.4), and up to the 8192 that they hold from 64 rows on
// (256 x 65536 with eight 18.2 and 13.5; 16 x 65536 9.9 and 11.1).  Where there are rows enough for all units, as few as hold it: what
// waits for a row's maximum, and for its alternatives, is then less of the machine (4096 x 32768 with five alternatives 1024 lanes 65 us,
// 512 52; 8000 x 16000 97 and, with 256, 52; 300 x 50001 1024 lanes 15.2, 512 17.7).
inline int lanes_for_whole_rows(long long rows, long long vectors)
{
    if (vectors <= kBlock || vectors > 1024 * kMostVectors) return 0;
    if (rows >= kEnoughParts) {
        if (vectors <= kBlock * kMostVectors) return 0;
        if (vectors <= 512 * kThirdVectors) return 512;
    }
    return vectors <= 512 * kMostVectors || rows >= 64 ? 1024 : 0;
}

// Parts of a row of `vectors`, with up to `k` vectors to a lane.
inline int parts_of(long long vectors, int k) { return static_cast<int>((vectors + kBlock * k - 1) / (kBlock * k)); }

int vectors_per_lane(long long rows, long long vectors)
{
    int k = kMostVectors;
    while (k > 1 && rows * parts_of(vectors, k) < kEnoughParts) k /= 2;
    return k;
}

template<int T, bool ENTROPY>
int launch_forward(const char* who, const TokenArgs& a, void* workspace, hipStream_t s)
{
    const int vectors = a.vocab < kVec<T> ? 1 : a.vocab / kVec<T>;      // the values behind the last one go with it
    Parts p{};
    const bool past = streams(a, T, 1);
    if (const int lanes = lanes_for_whole_rows(a.rows, vectors)) {
        p.parts = 1;
        p.vectors = vectors;
        const dim3 grid(static_cast<unsigned>(a.rows)), block(lanes);
        const auto launch = [&](auto* kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, a, p); };
        if (lanes == 512 && vectors > 512 * kMostVectors)
            launch(past ? &token_logprobs_kernel<T, ENTROPY, 512, kThirdVectors, true> : &token_logprobs_kernel<T, ENTROPY, 512, kThirdVectors, false>);
        else if (lanes == 512) launch(past ? &token_logprobs_kernel<T, ENTROPY, 512, kMostVectors, true> : &token_logprobs_kernel<T, ENTROPY, 512, kMostVectors, false>);
        else launch(past ? &token_logprobs_kernel<T, ENTROPY, 1024, kMostVectors, true> : &token_logprobs_kernel<T, ENTROPY, 1024, kMostVectors, false>);
        return check_launch(who);
    }
    // parts of 4096 vectors where they are enough, else of as many as make enough of them
    const bool large = a.rows * parts_of(vectors, 2 * kMostVectors) >= kEnoughParts && vectors > kBlock * kMostVectors;
    const int k = large ? 2 * kMostVectors : vectors_per_lane(a.rows, vectors);
    p.parts = parts_of(vectors, k);
    p.vectors = (vectors + p.parts - 1) / p.parts;
    p.parts = (vectors + p.vectors - 1) / p.vectors;
    p.by_parts = FastDiv(p.parts);
    const size_t groups = static_cast<size_t>(a.rows) * p.parts;
    p.keys = static_cast<unsigned long long*>(workspace);
    p.sums = reinterpret_cast<Sums*>(static_cast<char*>(workspace) + groups * a.top * sizeof(unsigned long long));
    const auto launch = [&](auto* kernel, int lanes) { hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(groups)), dim3(lanes), 0, s, a, p); };
    switch (k) {
    case 1: launch(&token_logprobs_kernel<T, ENTROPY, kBlock, 1, false>, kBlock); break;
    case 2: launch(&token_logprobs_kernel<T, ENTROPY, kBlock, 2, false>, kBlock); break;
    case 4: launch(&token_logprobs_kernel<T, ENTROPY, kBlock, 4, false>, kBlock); break;
    // past the caches where the logits do not fit (4096 x 50001 half: 101.5 -> 99.5 us)
    case kMostVectors:
        launch(past ? &token_logprobs_kernel<T, ENTROPY, kBlock, kMostVectors, true> : &token_logprobs_kernel<T, ENTROPY, kBlock, kMostVectors, false>, kBlock);
        break;
    default: launch(past ? &token_logprobs_kernel<T, ENTROPY, 512, kMostVectors, true> : &token_logprobs_kernel<T, ENTROPY, 512, kMostVectors, false>, 512);
    }
    if (int rc = check_launch(who)) return rc;
    if (p.parts == 1) return PXH_OK;
    if (p.parts <= kWave && p.parts * a.top <= kWave)
        hipLaunchKernelGGL((token_join_few_kernel<T>), dim3(grid_for(a.rows, kBlock / kWave)), dim3(kBlock), 0, s, a, p);
    else hipLaunchKernelGGL((token_join_kernel<T>), dim3(static_cast<unsigned>(a.rows)), dim3(kBlock), 0, s, a, p);
    return check_launch(who);
}

template<int T, bool NT>
int launch_gradient(const char* who, const TokenArgs& a, hipStream_t s)
{
    const int per = kGradientSteps<NT> * kBlock * kVec<T>;
    const int parts = a.vocab / per + (a.vocab % per != 0);
    hipLaunchKernelGGL((token_gradient_kernel<T, NT>), dim3(static_cast<unsigned>(a.rows) * parts), dim3(kBlock), 0, s, a, FastDiv(parts));
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
        if (a.row_sums) p.row_sums += done;
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

size_t token_rows_workspace_bytes(long long rows, int vocab, int top) { return pxh_token_logprobs_workspace_bytes(rows, vocab, top); }

int token_rows(const char* who, const void* logits, int type, long long rows, int vocab, long long stride, int top, float scale,
               float* values, int* ids, float2* sums, void* workspace, hipStream_t s)
{
    TokenArgs a{};
    a.logits = logits; a.top_logp = values; a.top_ids = ids; a.row_sums = sums; a.rows = rows; a.stride = stride; a.vocab = vocab;
    a.top = top; a.scale = scale; a.order_scale = 1.0f;
    int rc = PXH_OK;
    dispatch_type(type, [&]<int T>() { rc = by_rows(a, T, [&](const TokenArgs& p) { return launch_forward<T, false>(who, p, workspace, s); }); });
    return rc;
}

}  // namespace pxh

using namespace pxh;

extern "C" {

size_t pxh_token_logprobs_workspace_bytes(long long rows, int vocab, int top)
{
    if (rows <= 0 || vocab <= 0 || top < 0) return 0;
    // fp32 has the most vectors; a row whose parts are not the largest possible is one of few
    const long long vectors = vocab < 4 ? 1 : vocab / 4;
    const long long most = rows * parts_of(vectors, 1), least = rows * parts_of(vectors, kMostVectors);
    const long long few = most < 2 * kEnoughParts ? most : 2 * kEnoughParts;
    return static_cast<size_t>(least > few ? least : few) * (static_cast<size_t>(top) * sizeof(unsigned long long) + sizeof(Sums));
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
    a.top = top; a.scale = a.order_scale = scale;
    hipStream_t s = as_stream(stream);
    int rc = PXH_OK;
    if (rows == 0) return PXH_OK;
    void* ws = nullptr;
    if ((rc = resolve_workspace(workspace, workspace_bytes, pxh_token_logprobs_workspace_bytes(rows, vocab, top), &ws, s))) return rc;
    dispatch_type(type, [&]<int T>() {
        rc = by_rows(a, T, [&](const TokenArgs& p) {
            return entropy ? launch_forward<T, true>(who, p, ws, s) : launch_forward<T, false>(who, p, ws, s);
        });
    });
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
    dispatch_type(type, [&]<int T>() { rc = by_rows(a, T, [&](const TokenArgs& p) { return streams(a, T, 2) ? launch_gradient<T, true>(who, p, s) : launch_gradient<T, false>(who, p, s); }); });
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
            const bool past = streams(a, T, 2);
            if (entropy || d_entropy) return past ? launch_train<T, true, true>(who, p, s) : launch_train<T, true, false>(who, p, s);
            return past ? launch_train<T, false, true>(who, p, s) : launch_train<T, false, false>(who, p, s);
        });
    });
    return rc;
}

}
