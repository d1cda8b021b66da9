// Beam search: the best continuations over beams and vocabulary, and tensors with a row for each beam in the beams' new order.
#include "tokens.h"
#include "rows.h"

namespace pxh {
namespace {

// ---------------------------------------------------------------- selection
// A beam's continuations are ordered as its logits are, so the `count` best of all beams are among the `count` largest logits of each: those
// are found row by row (as the alternatives of a token), and a workgroup for each item puts its beams' together.  Scores are formed and compared
// in 64 bits from the logits as they are, so that in a beam the larger logit always comes first; a beam's sum of exponentials is of fp32, and
// continuations of different beams that are nearer than its error (some vocab / 64 roundings) may change places.
// The rows' launch is bound by the logits (512 x 50001 half 16.5 us, 3.1 TB/s), this one by its trips to memory, ids, then logits: 5.2 us for 64
// items of 8 beams with 8 continuations, 3.2 for one of 4 with 4.
constexpr int kMostBeams = 64;

struct SelectArgs {
    const void* logits;
    const float* scores;                // [batch][beams]
    const unsigned char* ended;
    const int* ids;                     // [batch * beams][per]
    const float2* sums;
    float* out_scores;                  // [batch][count]
    int* parents;
    int* tokens;
    long long stride;
    int vocab, beams, count, per, end_token;
    float scale;
};

// One number that orders scores, 0 for what is no candidate: minus infinity, as it is left or before, and what is no number.
__device__ __forceinline__ unsigned long long order_of(double score)
{
    if (!(static_cast<float>(score) > -INFINITY)) return 0;
    const unsigned long long bits = static_cast<unsigned long long>(__double_as_longlong(score + 0.0));
    return bits >> 63 ? ~bits : bits | 1ull << 63;
}

__device__ __forceinline__ double score_of(unsigned long long order)
{
    return __longlong_as_double(static_cast<long long>(order >> 63 ? order & ~(1ull << 63) : ~order));
}

template<int T>
__global__ __launch_bounds__(kBlock) void beam_select_kernel(SelectArgs a)
{
    // beams * per scores, each beam's descending, then a count of the candidates of all
    extern __shared__ unsigned long long orders[];
    __shared__ int candidates;
    const long long item = blockIdx.x;
    const int n = a.beams * a.per;
    if (threadIdx.x == 0) candidates = 0;
    for (int c = threadIdx.x; c < n; c += kBlock) {
        const int beam = c / a.per, place = c - beam * a.per;
        const long long row = item * a.beams + beam;
        const double so_far = a.scores[row];
        double score = so_far;
        if (a.ended && a.ended[row]) {
            if (place > 0) score = -INFINITY;
        } else {
            const float2 s = a.sums[row];
            const int token = a.ids[row * a.per + place];
            if (token >= 0 && token < a.vocab) {            // a row of no numbers has none
                // times the scale in 64 bits: neighbouring logits would meet in a product of 32, and large ones be infinite
                const double below = static_cast<double>(load_one<T>(row_of<T>(a.logits, row, a.stride), token)) - static_cast<double>(s.x);
                score += below * static_cast<double>(a.scale) - log(static_cast<double>(s.y));
            } else {
                score = -INFINITY;
            }
        }
        orders[c] = order_of(score);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < n; c += kBlock) {
        const unsigned long long own = orders[c];
        if (own == 0) continue;
        atomicAdd(&candidates, 1);
        const int beam = c / a.per;
        int rank = 0;
        if (n <= kBlock) {
            // few: how many come first, of equal ones those in front
#pragma unroll 8
            for (int o = 0; o < n; ++o) rank += orders[o] > own || (orders[o] == own && o < c);
        } else {
            rank = c - beam * a.per;
            for (int b = 0; b < a.beams && rank < a.count; ++b) {
                if (b == beam) continue;
                // how many of beam b's come first: of equal ones those of the lower beam
                const unsigned long long* list = orders + b * a.per;
                const unsigned long long least = b < beam ? own : own + 1;
                int low = 0, left = a.per;
                while (left > 0) {
                    const int half = left / 2;
                    if (list[low + half] >= least) {
                        low += half + 1;
                        left -= half + 1;
                    } else {
                        left = half;
                    }
                }
                rank += low;
            }
        }
        if (rank >= a.count) continue;
        const long long row = item * a.beams + beam, out = item * a.count + rank;
        a.out_scores[out] = static_cast<float>(score_of(own));
        a.parents[out] = beam;
        a.tokens[out] = a.ended && a.ended[row] ? a.end_token : a.ids[row * a.per + (c - beam * a.per)];
    }
    __syncthreads();
    for (int k = candidates + threadIdx.x; k < a.count; k += kBlock) {
        a.out_scores[item * a.count + k] = -INFINITY;
        a.parents[item * a.count + k] = -1;
        a.tokens[item * a.count + k] = -1;
    }
}

constexpr size_t align256(size_t b) { return (b + 255) & ~static_cast<size_t>(255); }

// What a workspace holds: the rows' largest logits, their sums, and what finding them needs.
struct Space {
    size_t values, sums, rows, bytes;
    Space(long long count, int vocab, int per)
    {
        const size_t list = align256(static_cast<size_t>(count) * per * 4);
        values = list;
        sums = 2 * list;
        rows = sums + align256(static_cast<size_t>(count) * sizeof(float2));
        bytes = rows + token_rows_workspace_bytes(count, vocab, per);
    }
};

// ---------------------------------------------------------------- reordering
// In place: a workgroup takes columns of all beams of one item, each lane up to kHeld pieces of 16 bytes, which it reads from the parent's
// row and, when all of the workgroup have read, writes.  Rows that stay where they are are neither read nor written for themselves.
// Parents, then rows, then stores, one behind the other: nine tensors of one item of 4 beams 3.6 us, five of 64 items of 8 beams 6.3 (18 MB); 16
// tensors of 1024 rows of 16 kB 53 (537 MB if every row moved; three of four do).  Eight pieces a lane: 8.1 and 55.
constexpr int kHeld = 4, kMostTensors = 32;

struct Tensor {
    char* data;
    long long stride, bytes;            // from row to row, and of a row
    unsigned first;                     // the tensor's first workgroup
    unsigned parts;                     // workgroups of an item
};

struct ReorderArgs {
    Tensor tensors[kMostTensors];
    const int* parents;
    int count, batch, beams, columns;   // columns: pieces of a row that a workgroup takes
    FastDiv by_columns;
};

__global__ __launch_bounds__(kBlock) void beam_reorder_kernel(ReorderArgs a)
{
    // the last tensor that begins no further behind: all of them looked at in one trip
    const int lane = threadIdx.x % kWave;
    const int which = __popcll(__ballot(lane < a.count && blockIdx.x >= a.tensors[lane < a.count ? lane : 0].first)) - 1;
    const Tensor& t = a.tensors[which];
    const unsigned at = blockIdx.x - t.first;
    const long long item = at / t.parts;
    const long long first = static_cast<long long>(at % t.parts) * a.columns * 16;
    char* const rows = t.data + item * a.beams * t.stride;
    const int* const parents = a.parents + item * a.beams;
    const int pieces = a.beams * a.columns;
    typedef uint32_t words __attribute__((ext_vector_type(4), aligned(1)));
    // all parents first, then all rows: one trip to memory each
    int beam[kHeld], parent[kHeld];
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        const int piece = j * kBlock + threadIdx.x;
        beam[j] = piece < pieces ? static_cast<int>(a.by_columns.div(piece)) : 0;
        parent[j] = parents[beam[j]];
    }
    words held[kHeld];
    long long byte[kHeld];
    bool moves[kHeld];
    // a row's last piece is read as its last 16 bytes, and what is the piece's own is written
    const long long last = t.bytes - 16;
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        const int piece = j * kBlock + threadIdx.x;
        byte[j] = first + static_cast<long long>(piece - beam[j] * a.columns) * 16;
        moves[j] = piece < pieces && byte[j] < t.bytes && parent[j] != beam[j] && parent[j] >= 0 && parent[j] < a.beams;
        const char* const from = rows + (moves[j] ? parent[j] : 0) * t.stride;
        if (last >= 0) {
            if (moves[j]) held[j] = *global_memory<words>(from + (byte[j] < last ? byte[j] : last));
        } else if (moves[j]) {
            uint32_t w[4] = {};
            for (int k = 0; k < t.bytes; ++k) w[k / 4] |= static_cast<uint32_t>(*global_memory<unsigned char>(from + k)) << (8 * (k & 3));
            held[j] = words{ w[0], w[1], w[2], w[3] };
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kHeld; ++j) {
        if (!moves[j]) continue;
        char* const to = rows + beam[j] * t.stride + byte[j];
        if (byte[j] <= last) {
            *global_memory<words>(to) = held[j];
            continue;
        }
        const int left = static_cast<int>(t.bytes - byte[j]), skip = last >= 0 ? 16 - left : 0;
        for (int k = 0; k < left; ++k) *global_memory<unsigned char>(to + k) = static_cast<unsigned char>(held[j][(k + skip) / 4] >> (8 * ((k + skip) & 3)));
    }
}

}  // namespace
}  // namespace pxh

using namespace pxh;

extern "C" {

size_t pxh_beam_select_workspace_bytes(int batch, int beams, int vocab, int count)
{
    if (batch <= 0 || beams <= 0 || vocab <= 0 || count <= 0) return 0;
    return Space(static_cast<long long>(batch) * beams, vocab, count < vocab ? count : vocab).bytes;
}

int pxh_beam_select(const void* logits, const float* scores, const unsigned char* ended, float* out_scores, int* parents, int* tokens, int type,
                    int batch, int beams, int vocab, long long stride, int count, int end_token, float scale, void* workspace,
                    size_t workspace_bytes, void* stream)
{
    const char* who = "pxh_beam_select";
    if (type != PXH_F32 && type != PXH_BF16 && type != PXH_F16) return fail_invalid("%s: type %d is not fp32, bf16 or half", who, type);
    if (batch < 0 || batch > 1 << 20) return fail_invalid("%s: %d items", who, batch);
    if (beams < 1 || beams > kMostBeams) return fail_invalid("%s: %d beams (1 to %d)", who, beams, kMostBeams);
    if (count < 1 || count > PXH_MOST_ALTERNATIVES) return fail_invalid("%s: %d continuations (1 to %d)", who, count, PXH_MOST_ALTERNATIVES);
    if (vocab <= 0 || vocab > 1 << 30) return fail_invalid("%s: rows of %d logits", who, vocab);
    if (!(scale > 0.0f && scale < INFINITY)) return fail_invalid("%s: scale %g", who, static_cast<double>(scale));
    if (batch == 0) return PXH_OK;
    if (!logits || !scores || !out_scores || !parents || !tokens) return fail_invalid("%s: null pointer", who);
    const long long rows = static_cast<long long>(batch) * beams;
    if (rows > 1 && stride < vocab) return fail_invalid("%s: rows of %d logits that overlap", who, vocab);
    const int per = count < vocab ? count : vocab;
    const Space space(rows, vocab, per);
    hipStream_t s = as_stream(stream);
    void* ws = nullptr;
    if (int rc = resolve_workspace(workspace, workspace_bytes, space.bytes, &ws, s)) return rc;
    char* const base = static_cast<char*>(ws);
    int* const ids = reinterpret_cast<int*>(base);
    float2* const sums = reinterpret_cast<float2*>(base + space.sums);
    if (int rc = token_rows(who, logits, type, rows, vocab, stride, per, scale, reinterpret_cast<float*>(base + space.values), ids, sums,
                            base + space.rows, s))
        return rc;
    const SelectArgs a{ logits, scores, ended, ids, sums, out_scores, parents, tokens, stride, vocab, beams, count, per, end_token, scale };
    dispatch_type(type, [&]<int T>() {
        hipLaunchKernelGGL((beam_select_kernel<T>), dim3(batch), dim3(kBlock), static_cast<size_t>(beams) * per * 8, s, a);
    });
    return check_launch(who);
}

int pxh_beam_reorder(int count, void* const* tensors, const long long* row_bytes, const long long* strides, const int* parents, int batch, int beams,
                     void* stream)
{
    const char* who = "pxh_beam_reorder";
    if (count < 0 || (count > 0 && (!tensors || !row_bytes || !strides))) return fail_invalid("%s: %d tensors", who, count);
    if (batch < 0 || batch > 1 << 20) return fail_invalid("%s: %d items", who, batch);
    if (beams < 1 || beams > kMostBeams) return fail_invalid("%s: %d beams (1 to %d)", who, beams, kMostBeams);
    if (batch == 0 || count == 0) return PXH_OK;
    if (!parents) return fail_invalid("%s: null pointer", who);
    const int columns = kHeld * kBlock / beams;
    const long long width = static_cast<long long>(columns) * 16;
    // everything is looked at before the first launch
    for (int i = 0; i < count; ++i) {
        if (row_bytes[i] < 0 || row_bytes[i] > 1ll << 40) return fail_invalid("%s: rows of %lld bytes", who, row_bytes[i]);
        if (row_bytes[i] && !tensors[i]) return fail_invalid("%s: null pointer", who);
        if (strides[i] < row_bytes[i]) return fail_invalid("%s: rows of %lld bytes that overlap", who, row_bytes[i]);
        if ((row_bytes[i] + width - 1) / width * batch >= 1 << 23) return fail_invalid("%s: %d rows of %lld bytes", who, batch * beams, row_bytes[i]);
        for (int j = 0; j < i && row_bytes[i]; ++j)
            if (tensors[j] == tensors[i] && row_bytes[j]) return fail_invalid("%s: tensors %d and %d are the same", who, j, i);
    }
    ReorderArgs a{};
    a.by_columns = FastDiv(columns);
    a.parents = parents;
    a.batch = batch;
    a.beams = beams;
    a.columns = columns;
    unsigned groups = 0;
    const auto launch = [&] {
        if (!groups) return static_cast<int>(PXH_OK);
        hipLaunchKernelGGL(beam_reorder_kernel, dim3(groups), dim3(kBlock), 0, as_stream(stream), a);
        a.count = 0;
        groups = 0;
        return check_launch(who);
    };
    for (int i = 0; i < count; ++i) {
        if (row_bytes[i] == 0) continue;
        const long long parts = (row_bytes[i] + width - 1) / width;
        const unsigned more = static_cast<unsigned>(parts * batch);
        if (a.count == kMostTensors || groups + more >= 1u << 24)
            if (int rc = launch()) return rc;
        a.tensors[a.count++] = Tensor{ static_cast<char*>(tensors[i]), strides[i], row_bytes[i], groups, static_cast<unsigned>(parts) };
        groups += more;
    }
    return launch();
}

}
