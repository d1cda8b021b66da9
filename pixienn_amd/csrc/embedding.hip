// Rows of a table looked up by token, with a scale, and the gradient of the table.
#include "rows.h"
#include "stream.h"

#include <type_traits>

namespace pxh {
namespace {

// The token of place i; `vocab` for one outside the vocabulary.
__device__ __forceinline__ uint32_t token_at(const void* tokens, bool wide, long long i, int vocab)
{
    const long long t = wide ? static_cast<const long long*>(tokens)[i] : static_cast<const int*>(tokens)[i];
    return t >= 0 && t < vocab ? static_cast<uint32_t>(t) : static_cast<uint32_t>(vocab);
}

// ---------------------------------------------------------------- forward
//   y[r] = scale * table[token[r]], zeros for a token outside the vocabulary
struct LookupArgs {
    const char* table;
    const void* tokens;
    char* y;
    long long table_stride, y_stride;
    uint32_t items;             // vectors of all rows
    FastDiv by_row;             // vectors of a row
    int vocab, width;
    float scale;
    bool wide;
};

template<int T, bool NT>
__global__ __launch_bounds__(kBlock) void embedding_kernel(LookupArgs a)
{
    constexpr int V = kVec<T>;
    const uint32_t item = blockIdx.x * kBlock + threadIdx.x;
    if (item >= a.items) return;
    uint32_t row, vector;
    a.by_row.divmod(item, row, vector);
    const int e = static_cast<int>(vector) * V;
    const uint32_t token = token_at(a.tokens, a.wide, row, a.vocab);
    float x[V] = {};
    if (token < static_cast<uint32_t>(a.vocab)) {
        load_row<T, V>(row_of<T>(a.table, token, a.table_stride), e, a.width).get(x);
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] *= a.scale;
    }
    Raw<T, V> r;
    r.set(x);
    store_row<T, V, NT>(row_of<T>(a.y, row, a.y_stride), e, a.width, r);
}

// ---------------------------------------------------------------- backward
//   d[v] (+)= scale * the sum over the rows r with token[r] = v of dy[r], in the rows' order
// The rows are sorted by token, those of one token in their own order; then every 32 consecutive ones are added up run by run, runs that go
// on beyond their 32 in a launch behind it, part after part.  No order depends on which workgroup comes first.

// -- sorting: tiles of 2048 rows by one workgroup each, then up to 32 sorted tiles at a time into one.
constexpr int kTile = 2048, kSortLanes = 1024, kFanIn = 32;
constexpr uint32_t kNoToken = ~0u;          // behind the last row: larger than any token

// Bitonic sorting of 2048 keys, two to a lane: the token above the place in the tile, all of them different.
template<typename Key>
__device__ __forceinline__ void compare(Key& a, Key& b, bool up)
{
    if ((a > b) == up) {
        const Key t = a;
        a = b;
        b = t;
    }
}

template<typename Key>
__global__ __launch_bounds__(kSortLanes) void sort_tile_kernel(const void* tokens, bool wide, long long rows, int vocab, uint32_t* sorted_tokens,
                                                               uint32_t* sorted_rows)
{
    constexpr int kShift = sizeof(Key) == 4 ? 11 : 32;
    __shared__ Key keys[kTile];
    const long long first = static_cast<long long>(blockIdx.x) * kTile;
    const int lane = threadIdx.x;
    Key k[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const long long i = first + 2 * lane + j;
        // rows that are not there come last, in a tile of which only what is there is kept
        const Key token = i < rows ? token_at(tokens, wide, i, vocab) : static_cast<Key>(~static_cast<Key>(0)) >> kShift;
        k[j] = token << kShift | static_cast<Key>(2 * lane + j);
    }
#pragma unroll
    for (int size = 2; size <= kTile; size *= 2) {
        const bool up = (2 * lane & size) == 0;
        int step = size / 2;
        // steps across waves
        if (step >= 2 * kWave) {
            __syncthreads();
            keys[2 * lane] = k[0];
            keys[2 * lane + 1] = k[1];
            for (; step >= 2 * kWave; step /= 2) {
                __syncthreads();
                // lane-th pair of places `step` apart
                const int low = (lane & (step - 1)) | ((lane & ~(step - 1)) << 1);
                Key a = keys[low], b = keys[low + step];
                compare(a, b, (low & size) == 0);
                keys[low] = a;
                keys[low + step] = b;
            }
            __syncthreads();
            k[0] = keys[2 * lane];
            k[1] = keys[2 * lane + 1];
        }
        for (; step >= 2; step /= 2) {
            const bool lower = (2 * lane & step) == 0;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const Key other = __shfl_xor(k[j], step / 2, kWave);
                const bool takes_less = lower == up;
                k[j] = (other < k[j]) == takes_less ? other : k[j];
            }
        }
        compare(k[0], k[1], up);
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const long long i = first + 2 * lane + j;
        if (i >= rows) continue;
        sorted_tokens[i] = static_cast<uint32_t>(k[j] >> kShift);
        sorted_rows[i] = static_cast<uint32_t>(first) + (static_cast<uint32_t>(k[j]) & (kTile - 1));
    }
}

// Places of sorted[0 .. n) that hold less than `token`, or, with OR_EQUAL, not more.
template<bool OR_EQUAL>
__device__ __forceinline__ uint32_t places_below(const uint32_t* sorted, uint32_t n, uint32_t token)
{
    uint32_t low = 0;
    while (n > 0) {
        const uint32_t half = n / 2;
        const uint32_t t = sorted[low + half];
        if (OR_EQUAL ? t <= token : t < token) {
            low += half + 1;
            n -= half + 1;
        } else {
            n = half;
        }
    }
    return low;
}

// Up to kFanIn neighbouring tiles of `tile` rows into one: a row's place is the number of rows in front of it in each.
__global__ __launch_bounds__(kBlock) void merge_tiles_kernel(const uint32_t* tokens, const uint32_t* rows, uint32_t* out_tokens, uint32_t* out_rows,
                                                             uint32_t count, uint32_t tile)
{
    const uint32_t i = blockIdx.x * kBlock + threadIdx.x;
    if (i >= count) return;
    const uint32_t own = i / tile, first = own / kFanIn * kFanIn;
    const uint32_t tiles = count / tile + (count % tile != 0);
    const uint32_t last = first + kFanIn < tiles ? first + kFanIn : tiles;
    const uint32_t token = tokens[i];
    uint32_t place = first * tile + (i - own * tile);
    for (uint32_t t = first; t < own; ++t) place += places_below<true>(tokens + t * tile, tile, token);
    for (uint32_t t = own + 1; t < last; ++t) place += places_below<false>(tokens + t * tile, count - t * tile < tile ? count - t * tile : tile, token);
    out_tokens[place] = token;
    out_rows[place] = rows[i];
}

// -- sums
constexpr int kRun = 32;            // sorted rows that a workgroup adds up

struct TableGradientArgs {
    const char* dy;
    char* d;
    const uint32_t* tokens;         // sorted
    const uint32_t* rows;
    float* partial;                 // [chunks][2][width]: of the run that goes on from the chunk before, of the one that goes on behind it
    long long dy_stride, d_stride;
    uint32_t count, chunks;         // rows, and every kRun of them
    int vocab, width, column_groups;
    float scale;
    bool accumulate;
};

template<int T, int D, int V>
__device__ __forceinline__ void write_sum(const TableGradientArgs& a, uint32_t token, int e, const float (&sum)[V])
{
    constexpr int kPart = V * kSize<D> > 16 ? 16 / kSize<D> : V;
    char* const d = row_of<D>(a.d, token, a.d_stride);
#pragma unroll
    for (int q = 0; q < V; q += kPart) {
        if (e + q >= a.width) break;
        float x[kPart] = {};
        if (a.accumulate) load_row<D, kPart>(d, e + q, a.width).get(x);
#pragma unroll
        for (int k = 0; k < kPart; ++k) x[k] = fmaf(a.scale, sum[q + k], x[k]);
        Raw<D, kPart> r;
        r.set(x);
        store_row<D, kPart>(d, e + q, a.width, r);
    }
}

// The first workgroups add up kRun sorted rows each (times column groups), the others, where the gradient is overwritten, write zeros to
// kZeroRows rows of the table each, where no row has their token.
constexpr int kZeroRows = 32;

template<int T, int D, int LANES>
__global__ __launch_bounds__(LANES) void table_gradient_kernel(TableGradientArgs a, FastDiv by_columns)
{
    constexpr int V = kVec<T>, kAhead = 8;
    __shared__ uint32_t tokens[kRun + 2], rows[kRun];
    uint32_t part, group;
    by_columns.divmod(blockIdx.x, part, group);
    const int e = static_cast<int>(group * LANES + threadIdx.x) * V;
    if (part >= a.chunks) {
        const uint32_t first = (part - a.chunks) * kZeroRows;
        if (threadIdx.x < kZeroRows) {
            const uint32_t token = first + threadIdx.x;
            bool empty = token < static_cast<uint32_t>(a.vocab);
            if (empty && a.count) {
                const uint32_t at = places_below<false>(a.tokens, a.count, token);
                empty = at == a.count || a.tokens[at] != token;
            }
            rows[threadIdx.x] = empty;
        }
        __syncthreads();
        if (e >= a.width) return;
        constexpr int kPart = V * kSize<D> > 16 ? 16 / kSize<D> : V;
        for (int i = 0; i < kZeroRows; ++i) {
            if (!rows[i]) continue;
            char* const d = row_of<D>(a.d, first + i, a.d_stride);
#pragma unroll
            for (int q = 0; q < V; q += kPart)
                if (e + q < a.width) store_row<D, kPart>(d, e + q, a.width, Raw<D, kPart>{});
        }
        return;
    }
    const uint32_t first = part * kRun;
    const int n = static_cast<int>(a.count - first < static_cast<uint32_t>(kRun) ? a.count - first : kRun);
    // tokens[0] and tokens[n + 1]: those of the neighbours
    for (int i = threadIdx.x; i < kRun + 2; i += LANES) {
        const long long at = static_cast<long long>(first) + i - 1;
        tokens[i] = at >= 0 && at < a.count ? a.tokens[at] : kNoToken;
        if (i >= 1 && i <= n) rows[i - 1] = a.rows[at];
    }
    __syncthreads();
    if (e >= a.width) return;
    float sum[V] = {};
    uint32_t begin = 0;             // place of the run's first row in the chunk
    for (int base = 0; base < n; base += kAhead) {
        Raw<T, V> x[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int i = min(base + j, n - 1);
            x[j] = load_row<T, V>(row_of<T>(a.dy, rows[i], a.dy_stride), e, a.width);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int i = base + j;
            if (i >= n) break;
            float v[V];
            x[j].get(v);
#pragma unroll
            for (int k = 0; k < V; ++k) sum[k] += v[k];
            const uint32_t token = tokens[i + 1];
            const bool ends = tokens[i + 2] != token;
            if (!ends && i + 1 < n) continue;
            const bool goes_on_from = begin == 0 && tokens[0] == token;
            if (token < static_cast<uint32_t>(a.vocab)) {
                if (ends && !goes_on_from) {
                    write_sum<T, D, V>(a, token, e, sum);
                } else {
                    float* const partial = a.partial + (static_cast<size_t>(part) * 2 + !goes_on_from) * a.width;
#pragma unroll
                    for (int q = 0; q < V; q += 4) {
                        Raw<PXH_F32, 4> r;
#pragma unroll
                        for (int k = 0; k < 4; ++k) r.w[k] = __float_as_uint(sum[q + k]);
                        if (e + q < a.width) store_row<PXH_F32, 4>(partial, e + q, a.width, r);
                    }
                }
            }
            begin = i + 1;
#pragma unroll
            for (int k = 0; k < V; ++k) sum[k] = 0.0f;
        }
    }
}

// The runs that go on beyond a chunk, by the workgroup of the chunk in which they begin: 256 columns to a workgroup, whose waves share
// the chunks.
constexpr int kJoinLanes = 1024, kJoinColumns = 256;

template<int D>
__global__ __launch_bounds__(kJoinLanes) void table_join_kernel(TableGradientArgs a, FastDiv by_columns)
{
    constexpr int kWaves = kJoinLanes / kWave;
    __shared__ float sums[kWaves][kJoinColumns];
    uint32_t part, group;
    by_columns.divmod(blockIdx.x, part, group);
    const uint32_t first = part * kRun, next = first + kRun;
    if (next >= a.count) return;
    const uint32_t token = a.tokens[next];
    if (token >= static_cast<uint32_t>(a.vocab) || a.tokens[next - 1] != token) return;
    if (a.tokens[first] == token && first > 0 && a.tokens[first - 1] == token) return;       // begins further in front
    // its end: the last chunk that has rows of it
    const uint32_t end = next + places_below<true>(a.tokens + next, a.count - next, token);
    const uint32_t last = (end - 1) / kRun;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int e = static_cast<int>(group) * kJoinColumns + lane * 4;
    float sum[4] = {};
    if (e < a.width) {
        // part's second row of sums, then the first one of the chunks behind it
        const auto row = [&](uint32_t c) { return a.partial + (static_cast<size_t>(c) * 2 + (c == part)) * a.width; };
        constexpr int kAhead = 4;
        uint32_t c = part + wave;
        for (; c + (kAhead - 1) * kWaves <= last; c += kAhead * kWaves) {
            Raw<PXH_F32, 4> x[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) x[j] = load_row<PXH_F32, 4>(row(c + j * kWaves), e, a.width);
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) sum[k] += __uint_as_float(x[j].w[k]);
        }
        for (; c <= last; c += kWaves) {
            const Raw<PXH_F32, 4> x = load_row<PXH_F32, 4>(row(c), e, a.width);
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[k] += __uint_as_float(x.w[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) sums[wave][lane * 4 + k] = sum[k];
    __syncthreads();
    if (wave != 0 || e >= a.width) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k] = 0.0f;
    for (int w = 0; w < kWaves; ++w)
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] += sums[w][lane * 4 + k];
    write_sum<D, D, 4>(a, token, e, sum);
}

constexpr size_t align256(size_t b) { return (b + 255) & ~static_cast<size_t>(255); }

// What a workspace holds: two lists of sorted tokens and rows, and the partial sums.
struct Space {
    size_t list, partial, bytes;
    Space(long long rows, int width)
    {
        list = align256(static_cast<size_t>(rows) * 4);
        partial = 4 * list;
        const size_t chunks = (static_cast<size_t>(rows) + kRun - 1) / kRun;
        bytes = partial + align256(chunks * 2 * static_cast<size_t>(width) * sizeof(float));
    }
};

template<int T, int D, int LANES>
void launch_sums(const TableGradientArgs& a, uint32_t groups, hipStream_t s)
{
    hipLaunchKernelGGL((table_gradient_kernel<T, D, LANES>), dim3(groups), dim3(LANES), 0, s, a, FastDiv(a.column_groups));
}

template<int T, int D>
int launch_gradient(const char* who, TableGradientArgs a, hipStream_t s)
{
    const int vectors = (a.width + kVec<T> - 1) / kVec<T>;
    const int lanes = vectors <= 64 ? 64 : vectors <= 128 ? 128 : 256;
    a.column_groups = (vectors + lanes - 1) / lanes;
    const long long zero_groups = a.accumulate ? 0 : (static_cast<long long>(a.vocab) + kZeroRows - 1) / kZeroRows;
    const long long groups = (a.chunks + zero_groups) * a.column_groups;
    if (groups * lanes >= 1ll << 32 || groups >= 1ll << 31) return fail_invalid("%s: too many rows of too many values", who);
    if (groups == 0) return PXH_OK;
    const auto go = lanes == 64 ? &launch_sums<T, D, 64> : lanes == 128 ? &launch_sums<T, D, 128> : &launch_sums<T, D, 256>;
    go(a, static_cast<uint32_t>(groups), s);
    if (int rc = check_launch(who)) return rc;
    if (a.chunks <= 1) return PXH_OK;
    const int columns = (a.width + kJoinColumns - 1) / kJoinColumns;
    const long long joins = static_cast<long long>(a.chunks - 1) * columns;
    if (joins * kJoinLanes >= 1ll << 32) return fail_invalid("%s: too many rows of too many values", who);
    hipLaunchKernelGGL((table_join_kernel<D>), dim3(static_cast<uint32_t>(joins)), dim3(kJoinLanes), 0, s, a, FastDiv(columns));
    return check_launch(who);
}

int check_embedding(const char* who, int type, int wide, long long rows, int vocab, int width)
{
    if (type != PXH_F32 && type != PXH_BF16 && type != PXH_F16) return fail_invalid("%s: type %d is not fp32, bf16 or half", who, type);
    if (wide != 0 && wide != 1) return fail_invalid("%s: wide_tokens is 0 or 1 (got %d)", who, wide);
    if (rows < 0 || rows >= 1 << 30) return fail_invalid("%s: %lld rows", who, rows);
    if (vocab <= 0 || vocab > 1 << 30) return fail_invalid("%s: a table of %d rows", who, vocab);
    if (width <= 0 || width > 1 << 24) return fail_invalid("%s: rows of %d values", who, width);
    return PXH_OK;
}

}  // namespace
}  // namespace pxh

using namespace pxh;

extern "C" {

int pxh_embedding_forward(const void* table, const void* tokens, void* y, int type, int wide_tokens, long long rows, int vocab, int width,
                          long long table_stride, long long y_stride, float scale, void* stream)
{
    const char* who = "pxh_embedding_forward";
    if (int rc = check_embedding(who, type, wide_tokens, rows, vocab, width)) return rc;
    if (rows == 0) return PXH_OK;
    if (!table || !tokens || !y) return fail_invalid("%s: null pointer", who);
    if ((table_stride < width && vocab > 1) || (y_stride < width && rows > 1)) return fail_invalid("%s: rows of %d values that overlap", who, width);
    int rc = PXH_OK;
    dispatch_type(type, [&]<int T>() {
        const int vectors = (width + kVec<T> - 1) / kVec<T>;
        const long long most = ((1ll << 31) - kBlock) / vectors;
        const bool past = static_cast<size_t>(rows) * static_cast<size_t>(width) * kSize<T> * 2 >= kStreamingBytes;
        for (long long done = 0; done < rows && !rc; done += most) {
            const long long part = rows - done < most ? rows - done : most;
            const LookupArgs a{ static_cast<const char*>(table), static_cast<const char*>(tokens) + done * (wide_tokens ? 8 : 4),
                                row_of<T>(y, done, y_stride), table_stride, y_stride, static_cast<uint32_t>(part * vectors), FastDiv(vectors), vocab,
                                width, scale, wide_tokens != 0 };
            const dim3 grid(grid_for(a.items, kBlock)), block(kBlock);
            if (past) hipLaunchKernelGGL((embedding_kernel<T, true>), grid, block, 0, as_stream(stream), a);
            else hipLaunchKernelGGL((embedding_kernel<T, false>), grid, block, 0, as_stream(stream), a);
            rc = check_launch(who);
        }
    });
    return rc;
}

size_t pxh_embedding_workspace_bytes(long long rows, int width)
{
    if (rows <= 0 || width <= 0) return 0;
    return Space(rows, width).bytes;
}

int pxh_embedding_backward(const void* dy, const void* tokens, void* d, int type, int d_type, int wide_tokens, long long rows, int vocab,
                           int width, long long dy_stride, long long d_stride, float scale, int accumulate, void* workspace,
                           size_t workspace_bytes, void* stream)
{
    const char* who = "pxh_embedding_backward";
    if (int rc = check_embedding(who, type, wide_tokens, rows, vocab, width)) return rc;
    if (d_type != type && d_type != PXH_F32) return fail_invalid("%s: the gradient is of the type of dy or fp32 (got type %d)", who, d_type);
    if (!d || (rows > 0 && (!dy || !tokens))) return fail_invalid("%s: null pointer", who);
    if ((rows > 1 && dy_stride < width) || (vocab > 1 && d_stride < width)) return fail_invalid("%s: rows of %d values that overlap", who, width);
    hipStream_t s = as_stream(stream);
    TableGradientArgs a{};
    a.dy = static_cast<const char*>(dy);
    a.d = static_cast<char*>(d);
    a.dy_stride = dy_stride;
    a.d_stride = d_stride;
    a.count = static_cast<uint32_t>(rows);
    a.chunks = (a.count + kRun - 1) / kRun;
    a.vocab = vocab;
    a.width = width;
    a.scale = scale;
    a.accumulate = accumulate != 0;
    if (rows > 0) {
        const Space space(rows, width);
        void* ws = nullptr;
        if (int rc = resolve_workspace(workspace, workspace_bytes, space.bytes, &ws, s)) return rc;
        char* const base = static_cast<char*>(ws);
        uint32_t* lists[4];
        for (int i = 0; i < 4; ++i) lists[i] = reinterpret_cast<uint32_t*>(base + i * space.list);
        a.partial = reinterpret_cast<float*>(base + space.partial);
        const uint32_t tiles = (a.count + kTile - 1) / kTile;
        // token and place of the tile in 32 bits
        if (vocab < (1 << 21) - 1)
            hipLaunchKernelGGL((sort_tile_kernel<uint32_t>), dim3(tiles), dim3(kSortLanes), 0, s, tokens, wide_tokens != 0, rows, vocab, lists[0], lists[1]);
        else
            hipLaunchKernelGGL((sort_tile_kernel<unsigned long long>), dim3(tiles), dim3(kSortLanes), 0, s, tokens, wide_tokens != 0, rows, vocab, lists[0], lists[1]);
        if (int rc = check_launch(who)) return rc;
        int from = 0;
        for (unsigned long long tile = kTile; tile < a.count; tile *= kFanIn) {
            const int to = 2 - from;
            hipLaunchKernelGGL(merge_tiles_kernel, dim3(grid_for(a.count, kBlock)), dim3(kBlock), 0, s, lists[from], lists[from + 1], lists[to],
                               lists[to + 1], a.count, static_cast<uint32_t>(tile));
            if (int rc = check_launch(who)) return rc;
            from = to;
        }
        a.tokens = lists[from];
        a.rows = lists[from + 1];
    }
    int rc = PXH_OK;
    dispatch_type(type, [&]<int T>() {
        if (d_type == T) rc = launch_gradient<T, T>(who, a, s);
        else rc = launch_gradient<T, PXH_F32>(who, a, s);
    });
    return rc;
}

}
