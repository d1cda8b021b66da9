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
// A vector a lane, rows one behind the other: bound by what is written and by the table's rows that the caches do not hold.  16384 x 4096
// bf16 of a text's tokens 30.4 us: 134 MB written and 76 MB read, a row of the table once however many places have its token (7.0 TB/s).
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
// The rows are sorted by token, those of one token in their own order; then every 4 to 32 consecutive ones are added up run by run, runs that go
// on beyond those in a launch behind it, part after part.  No order depends on which workgroup comes first.
// What comes out of the workspace is looked at before it is a place: where another call writes to the same one at the same time, which the
// interface forbids, the results have no meaning, but nothing beyond the tensors and the workspace is touched.
// 16384 x 2048 bf16 into 32768 rows: sorting 11.5 us (with 64 MB of zeros), merging 5.3, sums and the other zeros 29.6 (153 MB at 5.2 TB/s), what
// goes on from chunk to chunk 7.5; 53 us in all, with tensors that no cache holds (floor 31).  4099 x 1025 fp32 added to 10007 rows: places 7.6,
// sums 9.6, chunk to chunk 5.7, 23 in all (floor 8): three launches, each a few trips to memory one behind the other.

// -- zeros.  Sorting keeps a few units busy for some microseconds, in which the others write zeros to the table's last rows, whether
// a row has their token or not; the rows in front of those wait for the sums, which know which of them have none.
struct Zeros {
    char* d;
    long long first, rows, stride_bytes, row_bytes;
    FastDiv by_row;             // pieces of 16 bytes of a row
    uint32_t groups;            // workgroups, each of kZeroPieces pieces a lane
    bool past;                  // the caches
};

constexpr int kZeroPieces = 8;

template<int LANES>
__device__ __forceinline__ void write_zeros(const Zeros& z, uint32_t group)
{
    typedef uint32_t words __attribute__((ext_vector_type(4), aligned(1)));
    const uint32_t base = group * (LANES * kZeroPieces) + threadIdx.x;
#pragma unroll
    for (int j = 0; j < kZeroPieces; ++j) {
        uint32_t row, piece;
        z.by_row.divmod(base + j * LANES, row, piece);
        if (row >= z.rows) return;
        char* const at = z.d + (z.first + row) * z.stride_bytes + static_cast<size_t>(piece) * 16;
        const long long left = z.row_bytes - static_cast<long long>(piece) * 16;
        if (left >= 16) {
            if (z.past) __builtin_nontemporal_store(words{}, global_memory<words>(at));
            else *global_memory<words>(at) = words{};
        } else {
            for (long long k = 0; k < left; k += 2) *global_memory<uint16_t>(at + k) = 0;
        }
    }
}

// -- sorting: tiles of 2048 rows by one workgroup each, then several sorted tiles at a time into one: all 32 of up to 65536
// rows (65536 x 512 62 us for the whole call, and 66 with eight at a time), of more rows eight (2^20 x 64 265 us, and 385).
constexpr int kTile = 2048, kSortLanes = 1024, kFanIn = 8, kMostTiles = 32;
constexpr uint32_t kNoToken = ~0u;          // behind the last row: larger than any token

// Few rows: a row's place is the number of rows in front of it, those of a lower token and those of the same one further in front, counted one by
// one.  A workgroup takes kRanked rows; all tokens are in LDS, in kShares shares of a multiple of four, each counted for the kRanked rows by as many lanes.
constexpr int kRanked = 16, kRankLanes = 1024, kShares = kRankLanes / kRanked;

__global__ __launch_bounds__(kRankLanes) void rank_kernel(const void* tokens, bool wide, uint32_t rows, int vocab, uint32_t share, uint32_t* sorted_tokens,
                                                          uint32_t* sorted_rows, uint32_t groups, Zeros zeros)
{
    if (blockIdx.x >= groups) {
        write_zeros<kRankLanes>(zeros, blockIdx.x - groups);
        return;
    }
    extern __shared__ uint32_t all[];               // [kShares][share]
    __shared__ uint32_t places[kRanked];
    if (threadIdx.x < kRanked) places[threadIdx.x] = 0;
    for (uint32_t i = threadIdx.x; i < share * kShares; i += kRankLanes) all[i] = i < rows ? token_at(tokens, wide, i, vocab) : kNoToken;
    __syncthreads();
    const uint32_t row = blockIdx.x * kRanked + threadIdx.x % kRanked, from = threadIdx.x / kRanked * share;
    const uint32_t token = all[row < rows ? row : 0];
    // those in front count up to the token, those behind below it
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    uint32_t count = 0;
    const uint32_t first = blockIdx.x * kRanked;
    if (first < from + share && first + kRanked > from) {
        for (uint32_t j = from; j < from + share; ++j) count += all[j] < token + (j < row);
    } else {
        const uint32_t below = token + (from < first);
#pragma unroll 4
        for (uint32_t j = from; j < from + share; j += 4) {
            const words w = *reinterpret_cast<const words*>(all + j);
#pragma unroll
            for (int k = 0; k < 4; ++k) count += w[k] < below;
        }
    }
#pragma unroll
    for (int over = kRanked; over < kWave; over *= 2) count += __shfl_xor(count, over, kWave);
    if (static_cast<int>(threadIdx.x) % kWave < kRanked) atomicAdd(places + threadIdx.x % kRanked, count);
    __syncthreads();
    if (threadIdx.x >= kRanked || row >= rows) return;
    sorted_tokens[places[threadIdx.x]] = token;
    sorted_rows[places[threadIdx.x]] = row;
}

// Bitonic sorting of 2048 keys, two to a lane: the token above the place in the tile, all of them different.  66 steps one behind the
// other, of which 56 stay in a wave: 11.5 us with the zeros beside it, whatever the number of tiles.
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
                                                               uint32_t* sorted_rows, uint32_t tiles, Zeros zeros)
{
    if (blockIdx.x >= tiles) {
        write_zeros<kSortLanes>(zeros, blockIdx.x - tiles);
        return;
    }
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

// Places of sorted[0 .. n) that hold less than `token`.
__device__ __forceinline__ uint32_t places_below(const uint32_t* sorted, uint32_t n, uint32_t token)
{
    uint32_t low = 0;
    while (n > 0) {
        const uint32_t half = n / 2;
        if (sorted[low + half] < token) {
            low += half + 1;
            n -= half + 1;
        } else {
            n = half;
        }
    }
    return low;
}

// `fan` neighbouring tiles into one: a row's place is the number of rows in front of it in each, of those of the same token in the tiles in
// front too.  A workgroup takes kMerged rows of one tile, and kFanIn tiles at a time into LDS (a step of a search in memory that another
// XCD has written waits 0.7 us); each of its four parts searches two of them for every row.
constexpr int kMerged = 256, kMergeLanes = 1024, kParts = kMergeLanes / kMerged;

__global__ __launch_bounds__(kMergeLanes) void merge_tiles_kernel(const uint32_t* tokens, const uint32_t* rows, uint32_t* out_tokens, uint32_t* out_rows,
                                                                  uint32_t count, uint32_t fan)
{
    __shared__ uint32_t lists[kFanIn][kTile];
    __shared__ uint32_t counts[kParts][kMerged];
    const uint32_t begin = blockIdx.x * kMerged, own = begin / kTile, first = own / fan * fan;
    const uint32_t tiles = count / kTile + (count % kTile != 0);
    const uint32_t last = first + fan < tiles ? first + fan : tiles;
    const uint32_t part = threadIdx.x / kMerged, i = begin + threadIdx.x % kMerged;
    const uint32_t token = tokens[i < count ? i : 0], row = rows[i < count ? i : 0];
    uint32_t below = 0;
    for (uint32_t t = first; t < last; t += kFanIn) {
        __syncthreads();
        const uint32_t base = t * kTile;
        // all of them asked for before the first is waited for; the list's memory goes on to the next 64 words
        constexpr int kLoads = kFanIn * kTile / (4 * kMergeLanes);
        typedef uint32_t words __attribute__((ext_vector_type(4)));
        words w[kLoads];
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const uint32_t at = base + (j * kMergeLanes + threadIdx.x) * 4;
            w[j] = *reinterpret_cast<const words*>(tokens + (at < count ? at : 0));
        }
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const uint32_t at = (j * kMergeLanes + threadIdx.x) * 4;
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) w[j][k] = base + at + k < count ? w[j][k] : kNoToken;
            *reinterpret_cast<words*>(&lists[0][0] + at) = w[j];
        }
        __syncthreads();
        // step by step in all of the part's lists at once; a list that is not there holds kNoToken, and nothing below a token
        constexpr int kOwn = kFanIn / kParts;
        uint32_t low[kOwn] = {};
        const auto look = [&](uint32_t step) {
            uint32_t seen[kOwn];
#pragma unroll
            for (int j = 0; j < kOwn; ++j) seen[j] = lists[part * kOwn + j][low[j] + step - 1];
#pragma unroll
            for (int j = 0; j < kOwn; ++j) low[j] += (t + part * kOwn + j < own ? seen[j] <= token : seen[j] < token) ? step : 0;
        };
#pragma unroll
        for (uint32_t step = kTile / 2; step; step /= 2) look(step);
        look(1);
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
            const uint32_t list = t + part * kOwn + j;
            below += list < last && list != own ? low[j] : 0;
        }
    }
    counts[part][threadIdx.x % kMerged] = below;
    __syncthreads();
    if (part != 0 || i >= count) return;
    uint32_t place = first * kTile + (i - own * kTile);
#pragma unroll
    for (int k = 0; k < kParts; ++k) place += counts[k][threadIdx.x];
    if (place >= count) return;             // lists that another call writes
    out_tokens[place] = token;
    out_rows[place] = row;
}

// kFanIn larger tiles into one, in memory, step by step in all tiles at once.
__global__ __launch_bounds__(kBlock) void merge_large_kernel(const uint32_t* tokens, const uint32_t* rows, uint32_t* out_tokens, uint32_t* out_rows,
                                                             uint32_t count, uint32_t tile)
{
    const uint32_t i = blockIdx.x * kBlock + threadIdx.x;
    if (i >= count) return;
    const uint32_t own = i / tile, first = own / kFanIn * kFanIn;
    const uint32_t token = tokens[i];
    uint32_t low[kFanIn] = {}, n[kFanIn];
#pragma unroll
    for (uint32_t j = 0; j < kFanIn; ++j) {
        const unsigned long long begin = static_cast<unsigned long long>(first + j) * tile;
        n[j] = first + j == own || begin >= count ? 0 : count - begin < tile ? static_cast<uint32_t>(count - begin) : tile;
    }
    const auto look = [&](uint32_t step) {
        uint32_t seen[kFanIn];
#pragma unroll
        for (uint32_t j = 0; j < kFanIn; ++j) {
            const uint32_t at = low[j] + step - 1;
            seen[j] = at < n[j] ? tokens[(first + j) * tile + at] : kNoToken;
        }
#pragma unroll
        for (uint32_t j = 0; j < kFanIn; ++j) low[j] += (first + j < own ? seen[j] <= token : seen[j] < token) ? step : 0;
    };
    for (uint32_t step = tile / 2; step; step /= 2) look(step);
    look(1);
    uint32_t place = first * tile + (i - own * tile);
#pragma unroll
    for (int j = 0; j < kFanIn; ++j) place += low[j];
    if (place >= count) return;             // lists that another call writes
    out_tokens[place] = token;
    out_rows[place] = rows[i];
}

// -- sums
constexpr int kMostRun = 32, kLeastRun = 4;             // sorted rows that a workgroup adds up

struct TableGradientArgs {
    const char* dy;
    char* d;
    const uint32_t* tokens;         // sorted
    const uint32_t* rows;
    float* partial;                 // [chunks][2][width]: of the run that goes on from the chunk before, of the one that goes on behind it
    long long dy_stride, d_stride;
    uint32_t count, chunks;         // rows, and every `run` of them
    int run;
    uint32_t open;                  // the table's first rows, which hold no zeros yet
    int vocab, width, column_groups;
    float scale;
    bool accumulate;
    bool past;                      // rows, sums and zeros past the caches
};

// V values of a row of the gradient, as many of them as one access takes at a time.
template<int D, int V>
struct TableRow {
    static constexpr int kPart = V * kSize<D> > 16 ? 16 / kSize<D> : V, kParts = V / kPart;
    Raw<D, kPart> r[kParts];

    __device__ __forceinline__ void load(const TableGradientArgs& a, uint32_t token, int e)
    {
        const char* const d = row_of<D>(a.d, token, a.d_stride);
#pragma unroll
        for (int q = 0; q < kParts; ++q)
            if (e + q * kPart < a.width) r[q] = load_row<D, kPart>(d, e + q * kPart, a.width);
    }

    // the row with scale * sum added to what it holds
    template<bool NT>
    __device__ __forceinline__ void write(const TableGradientArgs& a, uint32_t token, int e, const float (&sum)[V])
    {
        char* const d = row_of<D>(a.d, token, a.d_stride);
#pragma unroll
        for (int q = 0; q < kParts; ++q) {
            if (e + q * kPart >= a.width) break;
            float x[kPart];
            r[q].get(x);
#pragma unroll
            for (int k = 0; k < kPart; ++k) x[k] = fmaf(a.scale, sum[q * kPart + k], x[k]);
            r[q].set(x);
            store_row<D, kPart, NT>(d, e + q * kPart, a.width, r[q]);
        }
    }
};

// Bound by the memory: eight rows of a run are asked for at once, and as many workgroups run as units hold.
// The first workgroups add up a run of sorted rows each (times column groups), the others, where the gradient is overwritten, write zeros to
// kZeroRows rows of the table each, where no row has their token.
constexpr int kZeroRows = 32;

template<int T, int D, bool ADDS, bool NT>
__global__ __launch_bounds__(kBlock) void table_gradient_kernel(TableGradientArgs a, FastDiv by_columns)
{
    constexpr int V = kVec<T>, kAhead = 8;
    __shared__ uint32_t tokens[kMostRun + 2], rows[kMostRun];
    uint32_t part, group;
    by_columns.divmod(blockIdx.x, part, group);
    const int e = static_cast<int>(group * blockDim.x + threadIdx.x) * V;
    if (part >= a.chunks) {
        const uint32_t first = (part - a.chunks) * kZeroRows;
        if (threadIdx.x < kZeroRows) {
            const uint32_t token = first + threadIdx.x;
            bool empty = token < a.open;
            if (empty && a.count) {
                const uint32_t at = places_below(a.tokens, a.count, token);
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
                if (e + q < a.width) store_row<D, kPart, NT>(d, e + q, a.width, Raw<D, kPart>{});
        }
        return;
    }
    const uint32_t first = part * a.run;
    const int n = static_cast<int>(a.count - first < static_cast<uint32_t>(a.run) ? a.count - first : a.run);
    // tokens[0] and tokens[n + 1]: those of the neighbours
    for (int i = threadIdx.x; i < a.run + 2; i += blockDim.x) {
        const long long at = static_cast<long long>(first) + i - 1;
        tokens[i] = at >= 0 && at < a.count ? a.tokens[at] : kNoToken;
        if (i >= 1 && i <= n) rows[i - 1] = min(a.rows[at], a.count - 1);
    }
    __syncthreads();
    if (e >= a.width) return;
    float sum[V] = {};
    int begin = 0;                  // place of the run's first row in the chunk
    for (int base = 0; base < n; base += kAhead) {
        Raw<T, V> x[kAhead];
        TableRow<D, V> old[ADDS ? kAhead : 1];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int i = min(base + j, n - 1);
            x[j] = load_row<T, V, NT>(row_of<T>(a.dy, rows[i], a.dy_stride), e, a.width);
            // what the run is added to, asked for with it
            if (ADDS && tokens[i + 2] != tokens[i + 1] && tokens[i + 1] < static_cast<uint32_t>(a.vocab)) old[ADDS ? j : 0].load(a, tokens[i + 1], e);
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
                    if (!ADDS) old[0] = TableRow<D, V>{};
                    old[ADDS ? j : 0].template write<NT && !ADDS>(a, token, e, sum);
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
// the chunks.  Most chunks have none: 7.5 us of 16384 x 2048, 5.7 of 4099 x 1025, a launch and two trips to memory (where all of 16384 rows
// have one token the call takes 10 us more).
constexpr int kJoinLanes = 256, kJoinColumns = 256;

template<int D>
__global__ __launch_bounds__(kJoinLanes) void table_join_kernel(TableGradientArgs a, FastDiv by_columns)
{
    constexpr int kWaves = kJoinLanes / kWave;
    __shared__ float sums[kWaves][kJoinColumns];
    uint32_t part, group;
    by_columns.divmod(blockIdx.x, part, group);
    const uint32_t first = part * a.run, next = first + a.run;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    if (next >= a.count) return;
    // the run's last chunk: those whose first row is of the token, looked at by as many lanes at once
    const uint32_t in_front = first > 0 ? a.tokens[first - 1] : kNoToken, begin = a.tokens[first], before = a.tokens[next - 1];
    const auto is_of = [&](uint32_t c, uint32_t token) { return c < a.chunks && a.tokens[c * a.run] == token; };
    bool mine = is_of(part + 1 + lane, before);
    const uint32_t token = before;
    if (token >= static_cast<uint32_t>(a.vocab) || !__builtin_amdgcn_readfirstlane(mine)) return;
    if (begin == token && in_front == token) return;       // begins further in front
    uint32_t last = part;
    for (;;) {
        const unsigned long long no = ~__ballot(mine);
        const int run = no ? __ffsll(no) - 1 : kWave;
        last += run;
        if (run < kWave) break;
        mine = is_of(last + 1 + lane, token);
    }
    const int e = static_cast<int>(group) * kJoinColumns + lane * 4;
    float sum[4] = {};
    if (e < a.width) {
        // part's second row of sums, then the first one of the chunks behind it
        const auto row = [&](uint32_t c) { return a.partial + (static_cast<size_t>(c) * 2 + (c == part)) * a.width; };
        constexpr int kAhead = 8;
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
    const int waves = last - part + 1 < static_cast<uint32_t>(kWaves) ? static_cast<int>(last - part + 1) : kWaves;
    for (int w = 1; w < waves; ++w)
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[k] += sums[w][lane * 4 + k];
    TableRow<D, 4> d{};
    if (a.accumulate) d.load(a, token, e);
    d.template write<false>(a, token, e, sum);
}

// What the machine writes while it sorts, from the table's end, whose tokens are the rare ones where they are numbered by their frequency (16384 x
// 2048 bf16 into 32768 rows 62 us without, 53 so; 65536 x 512 into 32768 rows of fp32 63 and 57).
constexpr long long kZerosDuringSort = 64ll << 20;

// Counted up to here, sorted in tiles and merged beyond: one launch for two, and work that grows with the square of the rows (64 rows 14.6 -> 9.5 us
// for the whole call, 4099 27.5 -> 22.6, 7000 30.3 -> 28.2, but 8192 30.7 -> 32.4).
constexpr uint32_t kMostRanked = 7168;

// Workgroups for the columns of a row.
int column_groups_of(int width, int type)
{
    const int v = 16 / static_cast<int>(size_of(type)), vectors = (width + v - 1) / v;
    return (vectors + kBlock - 1) / kBlock;
}

// Rows of a run: as few as still leave no more than kEnoughChunks workgroups, five to a unit (16384 x 2048 bf16 into 32768 rows with 1024 of
// them 53 us, with 512 56; x 4096, where each takes half the columns, with 1024 92 and with 2048 97.  All of one token it costs: 73, and 61).
constexpr size_t kEnoughChunks = 1280;
int run_of(long long rows, int groups)
{
    int run = kMostRun;
    while (run > kLeastRun && (rows + run / 2 - 1) / (run / 2) * groups <= static_cast<long long>(kEnoughChunks)) run /= 2;
    return run;
}

constexpr size_t align256(size_t b) { return (b + 255) & ~static_cast<size_t>(255); }

// What a workspace holds: two lists of sorted tokens and rows, and the partial sums.
struct Space {
    size_t list, partial, bytes;
    Space(long long rows, int width)
    {
        list = align256(static_cast<size_t>(rows) * 4);
        partial = 4 * list;
        // the fewest rows to a run are those of a call that makes few of them
        const size_t chunks = (static_cast<size_t>(rows) + kMostRun - 1) / kMostRun, short_chunks = (static_cast<size_t>(rows) + kLeastRun - 1) / kLeastRun;
        const size_t most = short_chunks < kEnoughChunks ? short_chunks : kEnoughChunks;
        bytes = partial + align256((chunks > most ? chunks : most) * 2 * static_cast<size_t>(width) * sizeof(float));
    }
};

// Workgroups that add up the runs and write zeros, with their lanes, and those that put together what goes on from chunk to chunk.
struct Grids {
    long long sums, joins;
    int lanes, join_columns;

    Grids(const TableGradientArgs& a, int type)
    {
        // the vectors of a row in equal parts of at most kBlock (1025 fp32 values: 257 vectors are twice 192 lanes, not 256 and one)
        const int v = 16 / static_cast<int>(size_of(type)), vectors = (a.width + v - 1) / v;
        lanes = ((vectors + a.column_groups - 1) / a.column_groups + kWave - 1) / kWave * kWave;
        sums = (a.chunks + (static_cast<long long>(a.open) + kZeroRows - 1) / kZeroRows) * a.column_groups;
        join_columns = (a.width + kJoinColumns - 1) / kJoinColumns;
        joins = a.chunks > 1 ? static_cast<long long>(a.chunks - 1) * join_columns : 0;
    }
    bool too_many() const { return sums * lanes >= 1ll << 32 || sums >= 1ll << 31 || joins * kJoinLanes >= 1ll << 32; }
};

template<int T, int D>
int launch_gradient(const char* who, TableGradientArgs a, const Grids& grids, hipStream_t s)
{
    if (grids.sums == 0) return PXH_OK;
    const auto kernel = a.accumulate ? a.past ? &table_gradient_kernel<T, D, true, true> : &table_gradient_kernel<T, D, true, false>
                        : a.past ? &table_gradient_kernel<T, D, false, true> : &table_gradient_kernel<T, D, false, false>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<uint32_t>(grids.sums)), dim3(grids.lanes), 0, s, a, FastDiv(a.column_groups));
    if (int rc = check_launch(who)) return rc;
    if (grids.joins == 0) return PXH_OK;
    hipLaunchKernelGGL((table_join_kernel<D>), dim3(static_cast<uint32_t>(grids.joins)), dim3(kJoinLanes), 0, s, a, FastDiv(grids.join_columns));
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
    a.column_groups = column_groups_of(width, type);
    a.run = run_of(rows, a.column_groups);
    a.chunks = (a.count + a.run - 1) / a.run;
    a.vocab = vocab;
    a.width = width;
    a.scale = scale;
    a.accumulate = accumulate != 0;
    // what is read and written does not fit the caches (131072 x 1024 bf16 into 50001 rows 133 us through them, 119 past them)
    a.past = (static_cast<size_t>(rows) * size_of(type) + (accumulate ? 0 : static_cast<size_t>(vocab)) * size_of(d_type)) * static_cast<size_t>(width) >= kStreamingBytes;
    a.open = a.accumulate ? 0 : static_cast<uint32_t>(vocab);
    // zeros for a launch that takes some microseconds on a few units: `bytes` of them, from the rows that have none yet
    const long long row_bytes = static_cast<long long>(width) * size_of(d_type), pieces = (row_bytes + 15) / 16;
    const auto zeros = [&](long long bytes, int lanes) {
        const long long some = bytes / row_bytes < a.open ? bytes / row_bytes : a.open;
        a.open -= static_cast<uint32_t>(some);
        return Zeros{ a.d, a.open, some, d_stride * static_cast<long long>(size_of(d_type)), row_bytes, FastDiv(static_cast<uint32_t>(pieces)),
                      grid_for(static_cast<size_t>(some) * pieces, static_cast<size_t>(lanes) * kZeroPieces), a.past };
    };
    static_assert(kRankLanes == kSortLanes, "zeros are written by as many lanes");
    const Zeros during = rows > 0 ? zeros(kZerosDuringSort, kSortLanes) : Zeros{};
    // looked at before the first launch
    const Grids grids(a, type);
    if (grids.too_many()) return fail_invalid("%s: too many rows of too many values", who);
    if (rows > 0) {
        const Space space(rows, width);
        void* ws = nullptr;
        if (int rc = resolve_workspace(workspace, workspace_bytes, space.bytes, &ws, s)) return rc;
        char* const base = static_cast<char*>(ws);
        uint32_t* lists[4];
        for (int i = 0; i < 4; ++i) lists[i] = reinterpret_cast<uint32_t*>(base + i * space.list);
        a.partial = reinterpret_cast<float*>(base + space.partial);
        const uint32_t tiles = (a.count + kTile - 1) / kTile;
        if (a.count <= kMostRanked) {
            const uint32_t groups = (a.count + kRanked - 1) / kRanked, share = (a.count + 4 * kShares - 1) / (4 * kShares) * 4;
            hipLaunchKernelGGL(rank_kernel, dim3(groups + during.groups), dim3(kRankLanes), share * kShares * sizeof(uint32_t), s, tokens, wide_tokens != 0,
                               a.count, vocab, share, lists[0], lists[1], groups, during);
            if (int rc = check_launch(who)) return rc;
            a.tokens = lists[0];
            a.rows = lists[1];
        } else {
            // token and place of the tile in 32 bits
            const auto sort = vocab < (1 << 21) - 1 ? &sort_tile_kernel<uint32_t> : &sort_tile_kernel<unsigned long long>;
            hipLaunchKernelGGL(sort, dim3(tiles + during.groups), dim3(kSortLanes), 0, s, tokens, wide_tokens != 0, rows, vocab, lists[0], lists[1], tiles, during);
            if (int rc = check_launch(who)) return rc;
            const uint32_t fan = tiles <= kMostTiles ? kMostTiles : kFanIn;
            int from = 0;
            for (unsigned long long tile = kTile; tile < a.count; tile *= tile == kTile ? fan : kFanIn) {
                const int to = 2 - from;
                if (tile == kTile) {
                    hipLaunchKernelGGL(merge_tiles_kernel, dim3(grid_for(a.count, kMerged)), dim3(kMergeLanes), 0, s, lists[from], lists[from + 1], lists[to],
                                       lists[to + 1], a.count, fan);
                } else {
                    hipLaunchKernelGGL(merge_large_kernel, dim3(grid_for(a.count, kBlock)), dim3(kBlock), 0, s, lists[from], lists[from + 1], lists[to],
                                       lists[to + 1], a.count, static_cast<uint32_t>(tile));
                }
                if (int rc = check_launch(who)) return rc;
                from = to;
            }
            a.tokens = lists[from];
            a.rows = lists[from + 1];
        }
    }
    int rc = PXH_OK;
    dispatch_type(type, [&]<int T>() {
        if (d_type == T) rc = launch_gradient<T, T>(who, a, grids, s);
        else rc = launch_gradient<T, PXH_F32>(who, a, grids, s);
    });
    return rc;
}

}
