// A gated linear recurrence over sequences of tokens, its gradients, and the step for one new token of each sequence.
//   z = 1 / (1 + exp(-update));  h[t] = h[t - 1] + z * (x - h[t - 1]);  y = h, or with a gate h * gate / (1 + exp(-gate))
#include "rows.h"
#include "stream.h"

namespace pxh {
namespace {

// A range of tokens takes a state s to (1 - Z) * s + H.  1 - z is never kept: of a z of 2^-13 it has only half the digits in fp32, which
// thousands of tokens would add up, while Z = z + z' - z z' has them all.  Z == 1 says that what was in front of the range is forgotten:
// the state behind it is H, or no number where s is infinite or none.  A range in which a sequence begins has nothing in front of
// it (kWhole): the state behind it is H to the bit.
struct Range {
    float z, h;
};

constexpr float kWhole = 2.0f;

__device__ __forceinline__ float behind(float s, Range r)
{
    const float by = r.z == 1.0f ? fmaf(0.0f, s, r.h) : s + fmaf(-r.z, s, r.h);
    return r.z == kWhole ? r.h : by;
}

__device__ __forceinline__ Range joined(Range first, Range then)
{
    const float z = then.z == 1.0f ? 1.0f : first.z + fmaf(-then.z, first.z, then.z);
    return Range{ first.z == kWhole || then.z == kWhole ? kWhole : z, behind(first.h, then) };
}

// z = 1 / (1 + e) with e = exp(-u), and 1 - z to all its digits: e z where z is near 1.  16-bit values: the hardware's exp2 of the
// product, an error of 2^-24 |u| and less.  An update of minus infinity has z = 0.
template<int T>
__device__ __forceinline__ void gate_of(float u, float& z, float& rest)
{
    float e;
    if constexpr (T == PXH_F32) {
        const float a = u < -87.0f ? -87.0f : u > 110.0f ? 110.0f : u;
        e = exp_by_exp2(-a);
        z = u < -87.0f ? 0.0f : quotient(1.0f, 1.0f + e);
    } else {
        e = __builtin_amdgcn_exp2f(u * -1.44269504f);
        z = __builtin_amdgcn_rcpf(1.0f + e);
    }
    rest = z < 0.5f ? 1.0f - z : e * z;
}

// h times the gate's factor o s.
template<int T>
__device__ __forceinline__ float gated(float h, float o)
{
    float s, rest;
    gate_of<T>(o, s, rest);
    return h * (o * s);
}

// A result, rounded to fp32 before it is rounded to the type: the compiler would round some products and sums to half at once, here and not there,
// and a chunk at a row's end would not have the bits of the others, nor a step those of the forward pass.
template<int T, int V>
__device__ __forceinline__ Raw<T, V> result_of(const float (&x)[V])
{
    float v[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        v[k] = x[k];
        if constexpr (T == PXH_F16) asm("" : "+v"(v[k]));
    }
    Raw<T, V> r;
    r.set(v);
    return r;
}

// What goes past the caches.
enum { kNone, kResults, kAll };

// Channels of a lane, four bytes of a row: 16 tokens of a few tensors and what is formed of them fit the registers.  And of a workgroup.
template<int T>
constexpr int kChannels = 4 / kSize<T>;
template<int T>
constexpr int kTileOf = kChannels<T> * kWave;
constexpr int kSaved = PXH_SCAN_SAVED;  // tokens from one saved state to the next

// Tokens of a wave, waves of a workgroup, one behind the other along the tokens, and chunks (workgroups) of a group.
template<int STEPS, int WAVES, int GROUP>
struct Shape {
    static constexpr int kSteps = STEPS, kWaves = WAVES, kGroup = GROUP, kChunk = STEPS * WAVES, kLanes = WAVES * kWave;
    static constexpr uint32_t kAll = (1u << STEPS) - 1;
    static_assert(kSaved % STEPS == 0 && kChunk % kSaved == 0, "a saved state is in front of a wave's tokens");
};
// Two workgroups of eight waves to a unit.  Chunks of 64 tokens pay twice for what a chunk costs whatever its length (a number, a word, a
// look back: 8 x 4096 x 2048 bf16 with a gate 139 us where 128 take 116).  The gradients keep three values for each that they read:
// waves of 16 tokens spill (430 us, and 193).
using Forward = Shape<16, 8, 8>;
using Backward = Shape<8, 8, 4>;

// Where sequences begin: starts[sequences + 1], or all of one length.  Of fewer than kFew sequences a wave's lanes keep all places, asked for
// before the workgroup knows its chunk.
constexpr int kFew = kWave - 1;
struct Sequences {
    const int* starts;
    FastDiv length;
    int count, rows;

    __device__ __forceinline__ bool few() const { return starts && count < kFew; }
    __device__ __forceinline__ int kept() const
    {
        const int lane = threadIdx.x % kWave;
        return few() && lane <= count ? starts[lane] : 0x7fffffff;
    }
};

// States of sequences: a row of `width` fp32 for each slot.
struct Slots {
    const int* of;          // [sequences], or null: a sequence's own number
    int count;
};

// The place of sequence s in the states, or -1 where none is kept.
__device__ __forceinline__ int slot_of(const Slots& slots, int s)
{
    const int slot = slots.of ? slots.of[s] : s;
    return slot >= 0 && slot < slots.count ? slot : -1;
}

// What the wave has to know of its tokens first .. first + STEPS: a bit each, for those that begin a sequence, end one, and lie in
// one; lane i knows the sequence of token i.
struct Borders {
    uint32_t begins, ends, active;
    int sequence;
};

// The last of n ascending places that is not behind t, or -1.
__device__ __forceinline__ int last_in_front(const int* starts, int n, int t)
{
    int low = 0;
    while (n > 0) {
        const int half = n / 2;
        if (starts[low + half] <= t) {
            low += half + 1;
            n -= half + 1;
        } else {
            n = half;
        }
    }
    return low - 1;
}

// The same for one t of the whole wave, 64 places at a time: 4000 sequences are two trips to memory, where halves are twelve.
__device__ __forceinline__ int last_in_front_of_wave(const int* starts, int n, int t)
{
    const int lane = threadIdx.x % kWave;
    int low = 0;
    while (n > 0) {
        const int step = (n + kWave - 1) / kWave, at = lane * step;
        const int passed = __popcll(__ballot(at < n && starts[low + at] <= t));
        if (passed == 0) break;
        low += (passed - 1) * step + 1;
        n = min(step - 1, n - (passed - 1) * step - 1);
    }
    return low - 1;
}

// `kept`: the lane's place, as Sequences keeps it.  All lanes of the wave.
template<int STEPS>
__device__ __forceinline__ Borders borders_of(const Sequences& q, int kept, int first)
{
    const int lane = threadIdx.x % kWave;
    const int t = first + lane;
    const bool mine = lane < STEPS && t < q.rows;
    bool begins = false, ends = false, active = false;
    int s = 0;
    if (q.starts) {
        int begin = 0, end = 0;
        if (q.few()) {
            s = -1;
#pragma unroll
            for (int half = kWave / 2; half; half /= 2) s = __shfl(kept, s + half) <= t ? s + half : s;
            begin = __shfl(kept, max(s, 0));
            end = __shfl(kept, s + 1);
        } else {
            const int low = max(last_in_front_of_wave(q.starts, q.count + 1, first), 0);
            const int among = last_in_front_of_wave(q.starts + low, q.count + 1 - low, first + STEPS - 1) + 1;
            s = low + last_in_front(q.starts + low, among, t);
            if (s >= 0 && s < q.count) {
                begin = q.starts[s];
                end = q.starts[s + 1];
            }
        }
        active = mine && s >= 0 && s < q.count;
        begins = active && begin == t;
        ends = active && (end == t + 1 || t + 1 == q.rows);
        s = active ? s : 0;
    } else if (mine) {
        uint32_t which, place;
        q.length.divmod(t, which, place);
        s = static_cast<int>(which);
        active = true;
        begins = place == 0;
        ends = place + 1 == q.length.d;
    }
    return Borders{ static_cast<uint32_t>(__ballot(begins)), static_cast<uint32_t>(__ballot(ends)), static_cast<uint32_t>(__ballot(active)), s };
}

// Whether tokens first .. first + n are all there and of one sequence, which may begin with the first and end with the last of them: then
// most of what a workgroup has to look at, token by token, is not there.
struct Whole {
    bool there, begins, ends;
    int sequence;
};

__device__ __forceinline__ Whole within_one(const Sequences& q, int kept, int first, int n)
{
    if (first + n > q.rows) return Whole{ false, false, false, 0 };
    if (!q.starts) {
        uint32_t which, place;
        q.length.divmod(first, which, place);
        return Whole{ place + n <= q.length.d, place == 0, place + n == q.length.d, static_cast<int>(which) };
    }
    const int s = q.few() ? __popcll(__ballot(kept <= first)) - 1 : last_in_front_of_wave(q.starts, q.count + 1, first);
    if (s < 0 || s >= q.count) return Whole{ false, false, false, 0 };
    const int begin = q.few() ? __builtin_amdgcn_readlane(kept, s) : q.starts[s], end = q.few() ? __builtin_amdgcn_readlane(kept, s + 1) : q.starts[s + 1];
    return Whole{ end >= first + n, begin == first, end == first + n || first + n == q.rows, s };
}

// ---------------------------------------------------------------- from chunk to chunk
// Workgroups take numbers, chunk by chunk along the tokens (for the gradients against them).  Each leaves what its chunk does to a
// state, channel by channel, as one 64-bit word; the last one of a group of chunks leaves one for all of them, and once it knows the state in
// front of the group, the state behind it as a whole range.  A chunk waits for the words of those in front of it in its group, which
// wait for nobody, and for the state in front of the group: the words of up to kWindow groups, until one of them is whole and none nearer is
// missing.  So the state has to go from hand to hand only once for kWindow groups.  A state is always put together in the same way,
// whichever words were there first: the same call gives the same bits.
// A workgroup waits for lower numbers only, which are running or done: the lowest of those running waits for none.  The bound on the looks
// makes the exit unconditional all the same (a second or two); where it was reached (two launches at once on one workspace, which the
// interface forbids) the states are NaN.
constexpr unsigned long long kNotThere = ~0ull;     // no range: a Z that is no number is left as 1, with its H
// (65536 x 256 bf16, channels that remember: every chunk handing its state on 173 us, groups of 4 49, of 8 36.  Eight words more than the gradients
// have registers for: 8 x 4096 x 2048 with a gate 193 us with groups of 4, 244 with groups of 8)
constexpr int kWindow = 4;
constexpr uint32_t kLooks = 1u << 20;

// The chunks of the call: segments of as many chunks each, of which none needs another segment's.  Where all sequences have the same length, of
// whole chunks, they are the segments, and numbers go round them: chunks that run together then wait for few of each other.
struct Exchange {
    unsigned long long* words;      // [segments * per][width]; null where no chunk needs another's
    unsigned long long* groups;     // [segments * groups_per][width]
    uint32_t* counter;
    uint32_t per, groups_per;       // of a segment
    FastDiv by_tiles, by_segments;
};

struct Place {
    uint32_t segment, chunk, tile;  // chunk: of the segment, in the order in which they wait for each other
};

__device__ __forceinline__ unsigned long long word_of(Range r)
{
    return static_cast<unsigned long long>(__float_as_uint(r.z != r.z ? 1.0f : r.z)) << 32 | __float_as_uint(r.h);
}

__device__ __forceinline__ Range range_of(unsigned long long w)
{
    return Range{ __uint_as_float(static_cast<uint32_t>(w >> 32)), __uint_as_float(static_cast<uint32_t>(w)) };
}

__device__ __forceinline__ void leave_word(unsigned long long* at, Range r)
{
    __hip_atomic_store(at, word_of(r), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ unsigned long long see_word(const unsigned long long* at)
{
    return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// What the `count` chunks (fewer than GROUP) whose words begin at `words` do to a state, of one channel (there: one that exists); all lanes of
// the wave.
template<int GROUP>
__device__ __forceinline__ Range of_group(const unsigned long long* words, uint32_t count, size_t width, bool there)
{
    unsigned long long w[GROUP - 1];
    uint32_t looks = kLooks;
    for (; looks; --looks) {
        bool missing = false;
#pragma unroll
        for (int d = 0; d < GROUP - 1; ++d) {
            w[d] = 0;                                   // a range of no tokens
            if (there && static_cast<uint32_t>(d) < count) w[d] = see_word(words + d * width);
        }
#pragma unroll
        for (int d = 0; d < GROUP - 1; ++d) missing = missing || w[d] == kNotThere;
        if (!__any(missing)) break;
        __builtin_amdgcn_s_sleep(1);
    }
    Range all = range_of(w[0]);
#pragma unroll
    for (int d = 1; d < GROUP - 1; ++d) all = joined(all, range_of(w[d]));
    return looks ? all : Range{ kWhole, __builtin_nanf("") };
}

// The state in front of the group whose word is at `word`, the group'th of its segment, of one channel; all lanes of the wave.
__device__ __forceinline__ float look_back(const unsigned long long* word, uint32_t group, size_t width, bool there)
{
    unsigned long long w[kWindow];
    int found = -1;
    for (uint32_t looks = kLooks; looks; --looks) {
#pragma unroll
        for (int d = 0; d < kWindow; ++d) {
            w[d] = word_of(Range{ kWhole, 0.0f });       // in front of the first group
            if (there && group > static_cast<uint32_t>(d)) w[d] = see_word(word - (d + 1) * width);
        }
        bool whole = true;
        found = -1;
#pragma unroll
        for (int d = 0; d < kWindow; ++d) {
            whole = whole && w[d] != kNotThere;
            if (whole && found < 0 && range_of(w[d]).z == kWhole) found = d;
        }
        if (!__any(found < 0)) break;
        __builtin_amdgcn_s_sleep(1);
    }
    float s = __builtin_nanf("");
#pragma unroll
    for (int d = kWindow - 1; d >= 0; --d) {
        if (d < found) s = behind(s, range_of(w[d]));
        else if (d == found) s = range_of(w[d]).h;
    }
    return s;
}

template<int WAVES, int TILE>
struct ScanShared {
    Range ranges[WAVES][TILE];
    Range in_front[TILE];               // the chunks of the group in front of this one
    float states[TILE];                 // in front of the group
    float begun[TILE];                  // what the sequence begins with that begins with the chunk
    float passed[WAVES][TILE];         // from wave to wave
    uint32_t number, fresh;             // fresh: no state reaches the chunk
};

template<int WAVES, int TILE>
__device__ __forceinline__ Place take_number(const Exchange& x, ScanShared<WAVES, TILE>& lds)
{
    uint32_t number = blockIdx.x;
    if (x.words) {
        if (threadIdx.x == 0) lds.number = atomicAdd(x.counter, 1u);
        __syncthreads();
        number = __builtin_amdgcn_readfirstlane(lds.number);
    }
    Place p;
    uint32_t rest;
    x.by_tiles.divmod(number, rest, p.tile);
    x.by_segments.divmod(rest, p.chunk, p.segment);
    return p;
}

// From the waves' ranges, in the order `order(0 .. WAVES - 1)`, of which the wave is number `turn`, and the chunks in front of the workgroup's: the
// state in front of the wave, of its lane's channels.
template<int GROUP, int WAVES, int TILE, int V, typename Order>
__device__ __forceinline__ void join_waves(const Exchange& x, ScanShared<WAVES, TILE>& lds, const Place& p, int width, int turn, const Order& order,
                                           float (&s)[V])
{
    __syncthreads();
    const int c = threadIdx.x % TILE, lane = threadIdx.x % kWave;
    const int e = static_cast<int>(p.tile) * TILE + c;
    const bool there = e < width;
    if (x.words) {
        const size_t pitch = static_cast<size_t>(width);
        const uint32_t group = p.chunk / GROUP, place = p.chunk % GROUP;
        const bool fresh = p.chunk == 0 || lds.fresh, last = p.chunk + 1 == x.per, ends_group = place == GROUP - 1 && !last;
        unsigned long long* const of_groups = x.groups + (static_cast<size_t>(p.segment) * x.groups_per + group) * pitch + e;
        Range all{ 0.0f, 0.0f };
        if (threadIdx.x < TILE) {            // whole waves
#pragma unroll
            for (int w = 0; w < WAVES; ++w) all = joined(all, lds.ranges[order(w)][c]);
            if (fresh) all.z = kWhole;
            unsigned long long* const word = x.words + (static_cast<size_t>(p.segment) * x.per + p.chunk) * pitch + e;
            if (there && !ends_group && !last) leave_word(word, all);
            Range front{ fresh ? kWhole : 0.0f, fresh ? lds.begun[c] : 0.0f };
            if (!fresh && place) front = of_group<GROUP>(word - place * pitch, place, pitch, there);
            lds.in_front[c] = front;
            all = joined(front, all);
            if (there && ends_group) leave_word(of_groups, all);
        } else if (threadIdx.x < 2 * TILE) {
            lds.states[c] = fresh ? 0.0f : look_back(of_groups, group, pitch, there);
        }
        __syncthreads();
        if (threadIdx.x < TILE && there && ends_group && all.z != kWhole) leave_word(of_groups, Range{ kWhole, behind(lds.states[c], all) });
    }
#pragma unroll
    for (int k = 0; k < V; ++k) s[k] = x.words ? behind(lds.states[lane * V + k], lds.in_front[lane * V + k]) : lds.begun[lane * V + k];
    for (int w = 0; w < turn; ++w) {
#pragma unroll
        for (int k = 0; k < V; ++k) s[k] = behind(s[k], lds.ranges[order(w)][lane * V + k]);
    }
}

// ---- the launch in front: empties the words, and hands the states of sequences without tokens on.
__global__ __launch_bounds__(kBlock) void scan_start_kernel(unsigned long long* words, size_t count, uint32_t* counter, Sequences q, Slots slots, const float* from,
                                                            float* to, int width)
{
    const size_t i = static_cast<size_t>(blockIdx.x) * kBlock + threadIdx.x;
    const size_t lanes = static_cast<size_t>(gridDim.x) * kBlock;
    if (i == 0 && counter) *counter = 0;
    for (size_t k = i; k < count; k += lanes) words[k] = kNotThere;
    if (!to) return;
    for (int s = blockIdx.x; s < q.count; s += gridDim.x) {
        if (q.starts && q.starts[s] != q.starts[s + 1]) continue;
        const int slot = slot_of(slots, s);
        if (slot < 0) continue;
        for (int e = threadIdx.x; e < width; e += kBlock)
            to[static_cast<size_t>(slot) * width + e] = from ? from[static_cast<size_t>(slot) * width + e] : 0.0f;
    }
}

// V channels of a row of fp32 states.
template<int V>
__device__ __forceinline__ void load_state(const float* states, int slot, int e, int width, float (&s)[V])
{
#pragma unroll
    for (int k = 0; k < V; ++k) s[k] = states && slot >= 0 && e + k < width ? states[static_cast<size_t>(slot) * width + e + k] : 0.0f;
}

template<bool NT = false, int V>
__device__ __forceinline__ void store_state(float* states, int slot, int e, int width, const float (&s)[V])
{
    if (slot < 0 || e >= width) return;
    Raw<PXH_F32, V> r;
    r.set(s);
    store_row<PXH_F32, V, NT>(states + static_cast<size_t>(slot) * width, e, width, r);
}

// Channels of a lane in rows of a tensor: a place that is the workgroup's and a byte offset of the lane's own, one for all rows.
struct Columns {
    int tile_first, e, width;       // the workgroup's first channel and the lane's
    bool inside;                    // the workgroup's channels are all there
};

// The wave's tokens of a tensor, a word a lane; tokens behind the last row repeat it, channels behind the last one are zeros.  No
// branch around a load: a lane at the end of a row reads the row's last word, and takes what is its own.
template<int T, int STEPS, bool NT>
__device__ __forceinline__ void load_tokens(const void* p, long long stride, int first, int rows, const Columns& c, Raw<T, kChannels<T>> (&r)[STEPS])
{
    constexpr int V = kChannels<T>;
    const int last = rows - 1 - first;                  // of the wave's tokens; where none is there, all are the last row
    const char* row = row_of<T>(p, last < 0 ? rows - 1 : first, stride);
    const size_t step = static_cast<size_t>(stride) * kSize<T>;
    if (c.inside) {
        row += static_cast<size_t>(c.tile_first) * kSize<T>;
        const uint32_t offset = static_cast<uint32_t>(c.e - c.tile_first) * kSize<T>;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            r[i] = load_raw_at<T, V, NT>(row, offset);
            row += i < last ? step : 0;
        }
    } else if (c.width >= V) {
        const int at = min(c.e, c.width - V), beyond = c.e - at;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            r[i] = load_raw<T, V, NT>(row, at);
            row += i < last ? step : 0;
        }
#pragma unroll
        for (int i = 0; i < STEPS; ++i) r[i].w[0] = beyond == 0 ? r[i].w[0] : V == 2 && beyond == 1 ? r[i].w[0] >> 16 : 0u;
    } else {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            float x[V] = {};
            const float only = load_one<T>(row, 0);
            x[0] = c.e == 0 ? only : 0.0f;
            r[i].set(x);
            row += i < last ? step : 0;
        }
    }
}

// Values as they were read, to be unpacked again: unpacked they would be kept, in twice the registers.
template<int T, int STEPS>
__device__ __forceinline__ void as_read(Raw<T, kChannels<T>> (&r)[STEPS])
{
    if constexpr (T != PXH_F32) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) asm volatile("" : "+v"(r[i].w[0]));
    }
}

// The rows of a tensor that a wave writes, one behind the other or against the tokens.
template<int T, bool NT>
struct Writer {
    static constexpr int kV = kChannels<T>;
    char* row;
    long long step;
    const Columns& c;

    __device__ __forceinline__ Writer(void* p, long long stride, int first, const Columns& columns, bool against = false)
        : row(row_of<T>(static_cast<char*>(p) + (columns.inside ? static_cast<size_t>(columns.tile_first) * kSize<T> : 0), first, stride)),
          step(stride * kSize<T> * (against ? -1 : 1)), c(columns) {}

    // RARE: not of all tokens, or not all channels
    template<bool RARE>
    __device__ __forceinline__ void put(bool active, const float (&v)[kV])
    {
        const Raw<T, kV> r = result_of<T>(v);
        if (!RARE || active) {
            if (!RARE || c.inside) store_raw_at<T, kV, NT>(row, static_cast<uint32_t>(c.e - c.tile_first) * kSize<T>, r);
            else if (c.e < c.width) store_row<T, kV, NT>(row, c.e, c.width, r);
        }
        row += step;
    }
};

// ---------------------------------------------------------------- forward
struct ScanArgs {
    const void* x;
    const void* update;
    const void* gate;
    void* y;
    const float* state;
    float* final;
    float* saved;               // [rows / kSaved, rounded up][width]: in front of every kSaved-th token
    long long x_stride, update_stride, gate_stride, y_stride;
    Sequences q;
    Slots slots;
    Exchange exchange;
    int width;
};

// A workgroup takes a chunk of tokens of kTile channels, a wave a few of them, which stay in registers as z and x between the pass that finds
// what they do to a state and the one that forms the states: one trip to memory.
// 8 x 4096 x 2048 bf16 with a gate and what is saved 111 us: 108 in this kernel, in which 578 MB move (5.4 TB/s) and the vector units have work for
// 53; of sequences of 256 tokens, where a chunk waits for one other at most, 99.  Without a gate 91, and 82 where the caches hold some of it
// from the call before.  30011 x 2561 half in 31 sequences 142: 618 MB where 461 would do, for the lines that two tiles share, as rows begin
// off them (2560 values wide 112).  75 scalar registers (53 in fp32) are kept in lanes of vector registers; what that costs is not known.
template<int T, bool GATE, int PAST>
__global__ __launch_bounds__(Forward::kLanes, 4) void scan_kernel(ScanArgs a)
{
    constexpr int kSteps = Forward::kSteps, kChunk = Forward::kChunk, kV = kChannels<T>, kTile = kTileOf<T>;
    __shared__ ScanShared<Forward::kWaves, kTile> lds;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const int kept = a.q.kept();
    const Place place = take_number(a.exchange, lds);
    if (place.chunk >= a.exchange.per) return;              // a counter that another launch takes numbers from
    const int chunk_first = static_cast<int>(place.segment * a.exchange.per + place.chunk) * kChunk, first = chunk_first + wave * kSteps;
    const int tile_first = static_cast<int>(place.tile) * kTile, e = tile_first + lane * kV;
    const Columns columns{ tile_first, e, a.width, tile_first + kTile <= a.width };
    Raw<T, kV> x[kSteps], u[kSteps], o[GATE ? kSteps : 1];
    load_tokens<T, kSteps, PAST == kAll>(a.x, a.x_stride, first, a.q.rows, columns, x);
    load_tokens<T, kSteps, PAST == kAll>(a.update, a.update_stride, first, a.q.rows, columns, u);
    if constexpr (GATE) load_tokens<T, kSteps, PAST == kAll>(a.gate, a.gate_stride, first, a.q.rows, columns, o);
    const Whole whole = columns.inside ? within_one(a.q, kept, chunk_first, kChunk) : Whole{ false, false, false, 0 };
    const auto pass = [&]<bool RARE>() {
        Borders b{ 0, 0, Forward::kAll, 0 };
        if constexpr (RARE) b = borders_of<kSteps>(a.q, kept, first);
        const bool begins_here = !RARE && whole.begins && wave == 0;
        if (threadIdx.x == 0) lds.fresh = RARE ? b.begins & 1 : whole.begins;
        float z[kSteps][kV];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            float v[kV], rest;
            u[i].get(v);
#pragma unroll
            for (int k = 0; k < kV; ++k) gate_of<T>(v[k], z[i][k], rest);
        }
        float h[kV] = {}, Z[kV] = {};
        if (begins_here && a.state) load_state(a.state, slot_of(a.slots, whole.sequence), e, a.width, h);
        if (wave == 0) {
#pragma unroll
            for (int k = 0; k < kV; ++k) lds.begun[lane * kV + k] = h[k];
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const bool begins = RARE && (b.begins >> i & 1), active = !RARE || (b.active >> i & 1);
            if (begins) load_state(a.state, a.state ? slot_of(a.slots, __builtin_amdgcn_readlane(b.sequence, i)) : -1, e, a.width, h);
            float v[kV];
            x[i].get(v);
#pragma unroll
            for (int k = 0; k < kV; ++k) {
                if (RARE) z[i][k] = active ? z[i][k] : 0.0f;
                const float ahead = active ? v[k] - h[k] : 0.0f;
                Z[k] += fmaf(-z[i][k], Z[k], z[i][k]);
                h[k] = fmaf(z[i][k], ahead, h[k]);
            }
            if (begins) {
                // the second pass takes the state from here: by then `final`, which may be `state`, may have been written
#pragma unroll
                for (int k = 0; k < kV; ++k) {
                    Z[k] = 1.0f;
                    z[i][k] = h[k];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kV; ++k) lds.ranges[wave][lane * kV + k] = Range{ begins_here || (RARE && b.begins) ? kWhole : Z[k], h[k] };
        join_waves<Forward::kGroup>(a.exchange, lds, place, a.width, wave, [](int w) { return w; }, h);
        as_read(x);
        if (a.saved && first % kSaved == 0 && first < a.q.rows) store_state<PAST != kNone>(a.saved, first / kSaved, e, a.width, h);
        Writer<T, PAST != kNone> y(a.y, a.y_stride, first, columns);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const bool begins = RARE && (b.begins >> i & 1), active = !RARE || (b.active >> i & 1);
            float v[kV];
            x[i].get(v);
#pragma unroll
            for (int k = 0; k < kV; ++k) {
                const float ahead = active ? v[k] - h[k] : 0.0f;
                h[k] = begins ? z[i][k] : fmaf(z[i][k], ahead, h[k]);
                v[k] = h[k];
            }
            if constexpr (GATE) {
                float w[kV];
                o[i].get(w);
#pragma unroll
                for (int k = 0; k < kV; ++k) v[k] = gated<T>(h[k], w[k]);
            }
            y.template put<RARE>(active, v);
            if (RARE && a.final && (b.ends >> i & 1))
                store_state(a.final, slot_of(a.slots, __builtin_amdgcn_readlane(b.sequence, i)), e, a.width, h);
        }
        if (!RARE && a.final && whole.ends && wave == Forward::kWaves - 1) store_state(a.final, slot_of(a.slots, whole.sequence), e, a.width, h);
    };
    if (whole.there) pass.template operator()<false>();
    else pass.template operator()<true>();
}

// ---------------------------------------------------------------- backward
//   G[t] = dy * g + (1 - z[t + 1]) * G[t + 1], g = gate / (1 + exp(-gate));  dx = z G;  dupdate = G (x - h[t - 1]) z (1 - z)
//   dgate = dy h s (1 + gate (1 - s)), s = 1 / (1 + exp(-gate))
// Along the tokens from the saved states for h, then against them for G: the carry C = (1 - z) G goes through a range as a state does.
// 8 x 4096 x 2048 bf16 with a gate 189 us: 183 in this kernel, in which 993 MB move (5.4 TB/s) and the vector units have work for 99.  Half as many
// tokens to a workgroup as forward, for want of registers, and the same waits.  30011 x 2561 half in 31 sequences 255: 1056 MB where 788 would do.
struct ScanBackwardArgs {
    const void* dy;
    const void* x;
    const void* update;
    const void* gate;
    const float* saved;
    void* dx;
    void* dupdate;
    void* dgate;
    const float* state;
    const float* d_final;
    float* d_state;
    long long dy_stride, x_stride, update_stride, gate_stride, dx_stride, dupdate_stride, dgate_stride;
    Sequences q;
    Slots slots;
    Exchange exchange;
    int width;
};

template<int T, bool GATE, int PAST>
__global__ __launch_bounds__(Backward::kLanes, 4) void scan_backward_kernel(ScanBackwardArgs a)
{
    constexpr int kSteps = Backward::kSteps, kWaves = Backward::kWaves, kChunk = Backward::kChunk, kV = kChannels<T>, kTile = kTileOf<T>;
    __shared__ ScanShared<kWaves, kTile> lds;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
    const int kept = a.q.kept();
    const Place place = take_number(a.exchange, lds);
    if (place.chunk >= a.exchange.per) return;              // a counter that another launch takes numbers from
    const int chunk_first = static_cast<int>((place.segment + 1) * a.exchange.per - 1 - place.chunk) * kChunk, first = chunk_first + wave * kSteps;
    const int tile_first = static_cast<int>(place.tile) * kTile, e = tile_first + lane * kV;
    const Columns columns{ tile_first, e, a.width, tile_first + kTile <= a.width };
    Raw<T, kV> x[kSteps], u[kSteps], dy[kSteps], o[GATE ? kSteps : 1];
    load_tokens<T, kSteps, PAST == kAll>(a.update, a.update_stride, first, a.q.rows, columns, u);
    load_tokens<T, kSteps, PAST == kAll>(a.x, a.x_stride, first, a.q.rows, columns, x);
    load_tokens<T, kSteps, PAST == kAll>(a.dy, a.dy_stride, first, a.q.rows, columns, dy);
    if constexpr (GATE) load_tokens<T, kSteps, PAST == kAll>(a.gate, a.gate_stride, first, a.q.rows, columns, o);
    float h[kV];
    load_state(a.saved, first % kSaved == 0 && first < a.q.rows ? first / kSaved : -1, e, a.width, h);
    const Whole whole = columns.inside ? within_one(a.q, kept, chunk_first, kChunk) : Whole{ false, false, false, 0 };
    const auto pass = [&]<bool RARE>() {
        Borders b{ 0, 0, Backward::kAll, 0 };
        if constexpr (RARE) b = borders_of<kSteps>(a.q, kept, first);
        if (wave == kWaves - 1) {
            if (lane == 0) lds.fresh = b.ends >> (kSteps - 1) & 1;
#pragma unroll
            for (int k = 0; k < kV; ++k) lds.begun[lane * kV + k] = 0.0f;
        }
        const auto begin = [&](int i) {
            if (b.begins >> i & 1) load_state(a.state, a.state ? slot_of(a.slots, __builtin_amdgcn_readlane(b.sequence, i)) : -1, e, a.width, h);
        };
        float z[kSteps][kV], w[kSteps][kV], g[kSteps][kV];         // w: z (1 - z), then times x - h
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            float v[kV];
            u[i].get(v);
#pragma unroll
            for (int k = 0; k < kV; ++k) {
                float rest;
                gate_of<T>(v[k], z[i][k], rest);
                w[i][k] = z[i][k] * rest;
            }
        }
        if (RARE && b.active != Backward::kAll) {
            // tokens of no sequence leave everything as it is
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const bool active = b.active >> i & 1;
#pragma unroll
                for (int k = 0; k < kV; ++k) z[i][k] = active ? z[i][k] : 0.0f;
#pragma unroll
                for (int k = 0; k < Raw<T, kV>::kWords; ++k) {
                    x[i].w[k] = active ? x[i].w[k] : 0u;
                    dy[i].w[k] = active ? dy[i].w[k] : 0u;
                    if constexpr (GATE) o[i].w[k] = active ? o[i].w[k] : 0u;
                }
            }
        }
        if constexpr (kSteps < kSaved) {
            // a state is saved for every few waves: the others have theirs from the one in front
#pragma unroll
            for (int part = 0; part + 1 < kSaved / kSteps; ++part) {
                if (wave % (kSaved / kSteps) == part) {
                    float was[kV];
#pragma unroll
                    for (int k = 0; k < kV; ++k) was[k] = h[k];
#pragma unroll
                    for (int i = 0; i < kSteps; ++i) {
                        if (RARE) begin(i);
                        float v[kV];
                        x[i].get(v);
#pragma unroll
                        for (int k = 0; k < kV; ++k) h[k] = fmaf(z[i][k], v[k] - h[k], h[k]);
                    }
#pragma unroll
                    for (int k = 0; k < kV; ++k) {
                        lds.passed[wave + 1][lane * kV + k] = h[k];
                        h[k] = was[k];
                    }
                }
                __syncthreads();
                as_read(x);
                if (wave % (kSaved / kSteps) == part + 1) {
#pragma unroll
                    for (int k = 0; k < kV; ++k) h[k] = lds.passed[wave][lane * kV + k];
                }
            }
        }
        Writer<T, PAST != kNone> out(a.dgate, a.dgate_stride, first, columns);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            if (RARE) begin(i);
            float d[kV];
            x[i].get(d);
            dy[i].get(g[i]);
#pragma unroll
            for (int k = 0; k < kV; ++k) {
                const float ahead = d[k] - h[k];
                w[i][k] *= ahead;
                h[k] = fmaf(z[i][k], ahead, h[k]);
            }
            if constexpr (GATE) {
                float p[kV], dgate[kV];
                o[i].get(p);
#pragma unroll
                for (int k = 0; k < kV; ++k) {
                    float s, rest;
                    gate_of<T>(p[k], s, rest);
                    dgate[k] = g[i][k] * h[k] * (s * fmaf(p[k], rest, 1.0f));
                    g[i][k] *= p[k] * s;
                }
                out.template put<RARE>(b.active >> i & 1, dgate);
                __builtin_amdgcn_sched_barrier(0);      // a token's gate after the other's: all at once they want more registers than there are
            }
            if (RARE && a.d_final && (b.ends >> i & 1)) {
                float more[kV];
                load_state(a.d_final, slot_of(a.slots, __builtin_amdgcn_readlane(b.sequence, i)), e, a.width, more);
#pragma unroll
                for (int k = 0; k < kV; ++k) g[i][k] += more[k];
            }
        }
        float C[kV] = {}, Z[kV] = {};
#pragma unroll
        for (int i = kSteps - 1; i >= 0; --i) {
            const bool ends = RARE && (b.ends >> i & 1);
#pragma unroll
            for (int k = 0; k < kV; ++k) {
                const float G = ends ? g[i][k] : g[i][k] + C[k];
                C[k] = fmaf(-z[i][k], G, G);
                Z[k] = ends ? 1.0f : Z[k] + fmaf(-z[i][k], Z[k], z[i][k]);
            }
        }
#pragma unroll
        for (int k = 0; k < kV; ++k) lds.ranges[wave][lane * kV + k] = Range{ RARE && b.ends ? kWhole : Z[k], C[k] };
        join_waves<Backward::kGroup>(a.exchange, lds, place, a.width, kWaves - 1 - wave, [](int k) { return kWaves - 1 - k; }, C);
        Writer<T, PAST != kNone> out_x(a.dx, a.dx_stride, first + kSteps - 1, columns, true), out_u(a.dupdate, a.dupdate_stride, first + kSteps - 1, columns, true);
#pragma unroll
        for (int i = kSteps - 1; i >= 0; --i) {
            const bool ends = RARE && (b.ends >> i & 1), active = !RARE || (b.active >> i & 1);
            float dx[kV], du[kV];
#pragma unroll
            for (int k = 0; k < kV; ++k) {
                const float G = ends ? g[i][k] : g[i][k] + C[k];
                dx[k] = z[i][k] * G;
                du[k] = w[i][k] * G;
                C[k] = G - dx[k];
            }
            out_x.template put<RARE>(active, dx);
            out_u.template put<RARE>(active, du);
            if (RARE && a.d_state && (b.begins >> i & 1))
                store_state(a.d_state, slot_of(a.slots, __builtin_amdgcn_readlane(b.sequence, i)), e, a.width, C);
        }
    };
    if (whole.there && !whole.begins && !whole.ends) pass.template operator()<false>();
    else pass.template operator()<true>();
}

// ---------------------------------------------------------------- one token of each sequence
struct StepArgs {
    const char* x;
    const char* update;
    const char* gate;
    char* y;
    float* state;
    long long x_stride, update_stride, gate_stride, y_stride;
    Slots slots;
    uint32_t items;
    FastDiv by_row;
    int width;
};

template<int T, bool GATE>
__global__ __launch_bounds__(kBlock) void scan_step_kernel(StepArgs a)
{
    constexpr int V = 4;
    const uint32_t item = blockIdx.x * kBlock + threadIdx.x;
    if (item >= a.items) return;
    uint32_t row, vector;
    a.by_row.divmod(item, row, vector);
    const int e = static_cast<int>(vector) * V;
    float x[V], u[V], o[V] = {}, h[V] = {};
    load_row<T, V>(row_of<T>(a.x, row, a.x_stride), e, a.width).get(x);
    load_row<T, V>(row_of<T>(a.update, row, a.update_stride), e, a.width).get(u);
    if constexpr (GATE) load_row<T, V>(row_of<T>(a.gate, row, a.gate_stride), e, a.width).get(o);
    const int slot = slot_of(a.slots, static_cast<int>(row));
    float* const state = a.state + static_cast<size_t>(slot < 0 ? 0 : slot) * a.width;
    if (slot >= 0) load_row<PXH_F32, V>(state, e, a.width).get(h);
#pragma unroll
    for (int k = 0; k < V; ++k) {
        float z, rest;
        gate_of<T>(u[k], z, rest);
        h[k] = fmaf(z, x[k] - h[k], h[k]);
    }
    if (slot >= 0) {
        Raw<PXH_F32, V> r;
        r.set(h);
        store_row<PXH_F32, V>(state, e, a.width, r);
    }
    if constexpr (GATE) {
#pragma unroll
        for (int k = 0; k < V; ++k) h[k] = gated<T>(h[k], o[k]);
    }
    store_row<T, V>(row_of<T>(a.y, row, a.y_stride), e, a.width, result_of<T>(h));
}

// ---------------------------------------------------------------- host
size_t chunks_of(long long rows, int chunk) { return (static_cast<size_t>(rows) + chunk - 1) / chunk; }

constexpr int kLine = 128;             // bytes

// Words of chunks and groups: a segment of two chunks and more has half as many groups at most.
size_t words_of(size_t chunks, int width) { return (chunks + chunks / 2 + 1) * static_cast<size_t>(width); }

// The words' counter in front of them.
constexpr size_t kCounterBytes = 256;

// What goes past the caches: nothing where `tensors` of the tokens' size fit them, else the results (8 x 4096 x 2048 bf16 without a gate, no chunk waiting for
// another, 79 -> 61 us), and, where rows begin with lines, so that no line is read for two tiles, what is read (its gradients with a gate 194 -> 188 us,
// 65536 x 1024 in one sequence 169 -> 167; rows that do not: 30080 x 2561 half 238 -> 244).
int past_caches(long long rows, int width, int type, int tensors, long long strides)
{
    if (static_cast<size_t>(rows) * static_cast<size_t>(width) * size_of(type) * tensors < kStreamingBytes) return kNone;
    return strides * static_cast<long long>(size_of(type)) % kLine ? kResults : kAll;
}

// pick(constant) for one of the two or three that a kernel is built for.
template<typename F>
auto for_past(int past, const F& pick)
{
    return past == kAll ? pick.template operator()<kAll>() : past == kResults ? pick.template operator()<kResults>() : pick.template operator()<kNone>();
}

int check_scan(const char* who, int type, long long rows, int width, int sequences, const int* starts, const int* slots, int slot_count, bool states)
{
    if (type != PXH_F32 && type != PXH_BF16 && type != PXH_F16) return fail_invalid("%s: type %d is not fp32, bf16 or half", who, type);
    if (rows < 0 || rows > 1 << 30) return fail_invalid("%s: %lld rows", who, rows);
    if (width <= 0 || width > 1 << 24) return fail_invalid("%s: rows of %d values", who, width);
    if (sequences < 0 || sequences > 1 << 30 || (sequences == 0 && rows > 0)) return fail_invalid("%s: %d sequences", who, sequences);
    if (!starts && sequences > 0 && rows % sequences) return fail_invalid("%s: %lld rows are not %d sequences of one length", who, rows, sequences);
    if (slots && !states) return fail_invalid("%s: slots without states", who);
    if (states && slot_count < 0) return fail_invalid("%s: %d slots", who, slot_count);
    if (states && !slots && slot_count < sequences) return fail_invalid("%s: states of %d slots for %d sequences", who, slot_count, sequences);
    return PXH_OK;
}

// Distances that sequences side by side are kept away from, of rows and of sequences.
constexpr long long kRowsApart = 4096, kSequencesApart = 8 << 20;

// Sequences of the call, and the words that its chunks exchange (none where every chunk begins and ends with a sequence).  Sequences of one
// length and of whole chunks are segments, side by side: gradients of 8 x 4096 x 2048 bf16 with a gate 195 -> 184 us, without 154 -> 136, forward without one
// 83.8 -> 81.8, with one 8 x 3968 x 2048 107 -> 102.5, 8 x 4224 x 2048 113 -> 108, 16 x 4096 x 1024 117 -> 107, 64 x 512 x 2048 108 -> 100.  Not so forward with a
// gate where rows lie multiples of 4 kB apart and sequences multiples of 8 MB (`row_bytes`, the distances of the rows that are read, or-ed; 0 where that does not
// matter): 8 x 4096 x 2048 112 -> 116, 16 x 2048 x 2048 109 -> 117, 16 x 2048 x 4096 197 -> 224, 8 x 4096 x 1024 fp32 104 -> 114, columns of a product three times as
// wide 111 -> 116.  There they go one behind the other, which costs the longer ones of such distances some (8 x 8192 x 2048 194 -> 203).  The gradients have no such
// distance: of 71 shapes one loses more than 5 % with a gate (8 x 2048 x 2048 fp32 177 -> 202) and four without, and others at the same distances win as much.
// Where groups of chunks begin with sequences either way, the bits are the same either way: rows at another distance have the same results.
template<typename S>
int start_scan(const char* who, long long row_bytes, int type, long long rows, int width, int sequences, const int* starts, const Slots& slots, const float* from, float* to,
               void* workspace, size_t workspace_bytes, Sequences& q, Exchange& x, uint32_t& groups, hipStream_t s)
{
    const long long length = starts || sequences == 0 ? 0 : rows / sequences;
    q = Sequences{ starts, FastDiv(length > 0 ? static_cast<uint32_t>(length) : 1), sequences, static_cast<int>(rows) };
    constexpr int kChunk = S::kChunk;
    const size_t chunks = chunks_of(rows, kChunk), tile = 4 / size_of(type) * kWave, tiles = (static_cast<size_t>(width) + tile - 1) / tile;
    if (chunks * tiles * S::kLanes >= 1ull << 32) return fail_invalid("%s: too many rows of too many values", who);
    groups = static_cast<uint32_t>(chunks * tiles);
    const bool meet = row_bytes && row_bytes % kRowsApart == 0 && length * row_bytes % kSequencesApart == 0 && length % (kChunk * S::kGroup) == 0;
    const bool apart = !meet && length > 0 && length % kChunk == 0 && sequences > 1;
    const size_t segments = apart ? sequences : 1, per = chunks / segments, groups_per = (per + S::kGroup - 1) / S::kGroup;
    x = Exchange{ nullptr, nullptr, nullptr, static_cast<uint32_t>(per), static_cast<uint32_t>(groups_per), FastDiv(static_cast<uint32_t>(tiles)),
                  FastDiv(static_cast<uint32_t>(segments)) };
    size_t count = 0;
    if (per > 1 && (starts || kChunk % length)) {
        void* ws = nullptr;
        count = segments * (per + groups_per) * static_cast<size_t>(width);
        if (int rc = resolve_workspace(workspace, workspace_bytes, kCounterBytes + words_of(chunks, width) * sizeof(unsigned long long), &ws, s)) return rc;
        x.counter = static_cast<uint32_t*>(ws);
        x.words = reinterpret_cast<unsigned long long*>(static_cast<char*>(ws) + kCounterBytes);
        x.groups = x.words + chunks * static_cast<size_t>(width);
    }
    // sequences may be without tokens where their lengths are given, or where there are none at all
    if (to == from || sequences == 0 || !(starts || length == 0)) to = nullptr;
    if (count || to) {
        size_t blocks = (count + 4 * kBlock - 1) / (4 * kBlock);
        if (to && blocks < static_cast<size_t>(sequences)) blocks = sequences;
        if (blocks > 2048) blocks = 2048;
        hipLaunchKernelGGL(scan_start_kernel, dim3(static_cast<unsigned>(blocks)), dim3(kBlock), 0, s, x.words, count, x.counter, q, slots, from, to, width);
        return check_launch(who);
    }
    return PXH_OK;
}

}  // namespace
}  // namespace pxh

using namespace pxh;

extern "C" {

size_t pxh_gated_scan_workspace_bytes(long long rows, int width)
{
    if (rows <= 0 || width <= 0) return 0;
    return kCounterBytes + words_of(chunks_of(rows, Forward::kChunk < Backward::kChunk ? Forward::kChunk : Backward::kChunk), width) * sizeof(unsigned long long);
}

int pxh_gated_scan_forward(const void* x, const void* update, const void* gate, void* y, const int* starts, const float* state, float* final,
                           const int* slots, float* saved, int type, long long rows, int width, int sequences, int slot_count, long long x_stride,
                           long long update_stride, long long gate_stride, long long y_stride, void* workspace, size_t workspace_bytes, void* stream)
{
    const char* who = "pxh_gated_scan_forward";
    if (int rc = check_scan(who, type, rows, width, sequences, starts, slots, slot_count, state || final)) return rc;
    if (rows > 0 && (!x || !update || !y)) return fail_invalid("%s: null pointer", who);
    if (rows > 1 && (x_stride < width || update_stride < width || y_stride < width || (gate && gate_stride < width)))
        return fail_invalid("%s: rows of %d values that overlap", who, width);
    ScanArgs a{ x, update, gate, y, state, final, saved, x_stride, update_stride, gate_stride, y_stride, {}, Slots{ slots, slot_count }, {}, width };
    uint32_t groups;
    hipStream_t s = as_stream(stream);
    const long long row_bytes = gate ? (x_stride | update_stride | gate_stride) * static_cast<long long>(size_of(type)) : 0;
    if (int rc = start_scan<Forward>(who, row_bytes, type, rows, width, sequences, starts, a.slots, state, final, workspace, workspace_bytes, a.q, a.exchange, groups, s)) return rc;
    if (rows == 0) return PXH_OK;
    dispatch_type(type, [&]<int T>() {
        // (without a gate what is read stays: 8 x 4096 x 2048 bf16 81 us, and 91)
        const int past = past_caches(rows, width, type, gate ? 4 : 3, x_stride | update_stride | gate_stride);
        const auto kernel = gate ? for_past(past, []<int PAST>() { return &scan_kernel<T, true, PAST>; })
                                 : past != kNone ? &scan_kernel<T, false, kResults> : &scan_kernel<T, false, kNone>;
        hipLaunchKernelGGL(kernel, dim3(groups), dim3(Forward::kLanes), 0, s, a);
    });
    return check_launch(who);
}

int pxh_gated_scan_backward(const void* dy, const void* x, const void* update, const void* gate, const float* saved, void* dx, void* dupdate,
                            void* dgate, const int* starts, const float* state, const float* d_final, float* d_state, const int* slots, int type,
                            long long rows, int width, int sequences, int slot_count, long long dy_stride, long long x_stride,
                            long long update_stride, long long gate_stride, long long dx_stride, long long dupdate_stride,
                            long long dgate_stride, void* workspace, size_t workspace_bytes, void* stream)
{
    const char* who = "pxh_gated_scan_backward";
    if (int rc = check_scan(who, type, rows, width, sequences, starts, slots, slot_count, state || d_final || d_state)) return rc;
    if (!gate != !dgate) return fail_invalid("%s: gate and dgate go together", who);
    if (rows > 0 && (!dy || !x || !update || !saved || !dx || !dupdate)) return fail_invalid("%s: null pointer", who);
    if (rows > 1 && (dy_stride < width || x_stride < width || update_stride < width || dx_stride < width || dupdate_stride < width
                     || (gate && (gate_stride < width || dgate_stride < width))))
        return fail_invalid("%s: rows of %d values that overlap", who, width);
    ScanBackwardArgs a{ dy, x, update, gate, saved, dx, dupdate, dgate, state, d_final, d_state, dy_stride, x_stride, update_stride, gate_stride,
                        dx_stride, dupdate_stride, dgate_stride, {}, Slots{ slots, slot_count }, {}, width };
    uint32_t groups;
    hipStream_t s = as_stream(stream);
    if (int rc = start_scan<Backward>(who, 0, type, rows, width, sequences, starts, a.slots, d_final, d_state, workspace, workspace_bytes, a.q, a.exchange, groups, s))
        return rc;
    if (rows == 0) return PXH_OK;
    dispatch_type(type, [&]<int T>() {
        const int past = past_caches(rows, width, type, gate ? 7 : 5, x_stride | update_stride | dy_stride | (gate ? gate_stride : 0));
        const auto kernel = gate ? for_past(past, []<int PAST>() { return &scan_backward_kernel<T, true, PAST>; })
                                 : for_past(past, []<int PAST>() { return &scan_backward_kernel<T, false, PAST>; });
        hipLaunchKernelGGL(kernel, dim3(groups), dim3(Backward::kLanes), 0, s, a);
    });
    return check_launch(who);
}

int pxh_gated_scan_step(const void* x, const void* update, const void* gate, void* y, float* state, const int* slots, int type, long long rows,
                        int width, int slot_count, long long x_stride, long long update_stride, long long gate_stride, long long y_stride, void* stream)
{
    const char* who = "pxh_gated_scan_step";
    if (int rc = check_scan(who, type, rows, width, static_cast<int>(rows), nullptr, slots, slot_count, true)) return rc;
    if (rows == 0) return PXH_OK;
    if (!x || !update || !y || (!state && slot_count > 0)) return fail_invalid("%s: null pointer", who);
    if (rows > 1 && (x_stride < width || update_stride < width || y_stride < width || (gate && gate_stride < width)))
        return fail_invalid("%s: rows of %d values that overlap", who, width);
    const int vectors = (width + 3) / 4;
    if (rows * vectors >= (1ll << 31) - kBlock) return fail_invalid("%s: too many rows of too many values", who);
    const StepArgs a{ static_cast<const char*>(x), static_cast<const char*>(update), static_cast<const char*>(gate), static_cast<char*>(y), state, x_stride,
                      update_stride, gate_stride, y_stride, Slots{ slots, slot_count }, static_cast<uint32_t>(rows * vectors), FastDiv(vectors), width };
    const dim3 grid(grid_for(a.items, kBlock)), block(kBlock);
    hipStream_t s = as_stream(stream);
    dispatch_type(type, [&]<int T>() {
        if (gate) hipLaunchKernelGGL((scan_step_kernel<T, true>), grid, block, 0, s, a);
        else hipLaunchKernelGGL((scan_step_kernel<T, false>), grid, block, 0, s, a);
    });
    return check_launch(who);
}

}
