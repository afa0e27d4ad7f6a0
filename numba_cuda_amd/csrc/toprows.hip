// nbh_rows_top: the k largest entries of each row of logits with their indices, and the row's log-sum-exp.
//
// Entries are compared as 64-bit integers, (an integer that orders like the value) << 32 | ~index: no two
// are equal, so ties and NaN need no cases of their own.  One pass over the data: a workgroup streams a
// stretch of a row in chunks and appends to a list in LDS whatever exceeds a threshold that at least k
// entries reach.
//   * The first threshold comes from the first chunk: of the maxima of its 16-byte vectors (1024 of them),
//     the k-th largest, or a value below it, found by bisection on the integers.
//   * Afterwards a vector whose maximum does not exceed the threshold costs its maximum and a comparison;
//     the list grows by few entries per chunk.
//   * A list that runs full is cut to its k best (bisection again), which raises the threshold; entries
//     that found no room are offered again.  Rows sorted upwards or with masses of equal entries get there
//     again and again and stay right.
// The remaining list is sorted in LDS.  Few rows are split over workgroups, whose lists a second launch
// joins.
#include "rows.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kVecs = 4;                 // 16-byte vectors per lane and chunk
constexpr int kJoinCap = 4096;           // entries the joining workgroup holds

struct Top {
    const char *in;
    int64_t stride, vocab, slice, row0;
    int splits, k;
    char *values;
    int64_t values_stride;
    char *indices;
    int64_t indices_stride;
    float *lse;
    float temperature, scale;
    uint64_t *parts;                     // splits lists of k per row, when rows are split
    nbh_softmax *part_stats;
};

// Orders like the value; NaN above all, -0 as +0.
__device__ __forceinline__ uint32_t key_of(float x)
{
    const uint32_t bits = __float_as_uint(x + 0.0f);
    return x != x ? 0xffffffffu : bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u);
}
// A float `t` such that !(x <= t) holds for every x whose key exceeds `key` (and, if t is NaN, for all).
__device__ __forceinline__ float float_below(uint32_t key)
{
    if (key < 0x007fffffu)               // below -inf's key: nothing may be passed over
        return __uint_as_float(0x7fc00000u);
    if (key == 0x7fffffffu)              // between the largest negative number and zero: would read -0
        return __uint_as_float(0x80000001u);
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ uint64_t entry_of(float x, int64_t index)
{
    return (uint64_t)key_of(x) << 32 | (uint32_t)~(uint32_t)index;
}
__device__ __forceinline__ int64_t index_of(uint64_t entry) { return (uint32_t)~(uint32_t)entry; }

// What a workgroup shares besides the list itself.
struct Shared {
    int count;                           // entries offered since the list was last cut
    int full[2];                         // by turn: somebody found no room
    int tally[2][kWaves];                // by turn: counts of a bisection step
    nbh_softmax stats[kWaves];
};

// Sum over the workgroup of a number every lane of a wavefront agrees on.  One barrier: the next step
// writes the other row.
__device__ __forceinline__ int group_sum(int of_wave, Shared &sh, int &turn)
{
    if ((threadIdx.x & 63) == 0)
        sh.tally[turn][threadIdx.x >> 6] = of_wave;
    __syncthreads();
    int sum = 0;
    for (int w = 0; w < kWaves; ++w)
        sum += sh.tally[turn][w];
    turn ^= 1;
    return sum;
}

// Cuts the list (`have` entries, more than k) to its k best; returns a threshold exactly they exceed.
template <int CAP>
__device__ uint64_t cut_list(uint64_t *list, int have, int k, Shared &sh, int &turn)
{
    uint64_t mine[CAP / kThreads];
    for (int i = 0; i < CAP / kThreads; ++i) {
        const int at = i * kThreads + threadIdx.x;
        mine[i] = at < have ? list[at] : 0;
    }
    uint64_t low = 1, high = ~0ull;      // at least k entries reach `low`
    while (low < high) {
        const uint64_t mid = high - (high - low) / 2;
        int reach = 0;
        for (int i = 0; i < CAP / kThreads; ++i)
            reach += __popcll(__ballot(mine[i] >= mid));
        reach = group_sum(reach, sh, turn);
        if (reach >= k)
            low = mid;
        else
            high = mid - 1;
        if (reach == k)
            break;
    }
    __syncthreads();                     // everybody has read the list
    if (threadIdx.x == 0)
        sh.count = 0;
    __syncthreads();
    for (int i = 0; i < CAP / kThreads; ++i)
        if (mine[i] >= low)
            list[atomicAdd(&sh.count, 1)] = mine[i];
    __syncthreads();
    return low - 1;
}

// The k best of the list, sorted downwards in its front (missing ones read 0).
template <int CAP>
__device__ void sort_list(uint64_t *list, int have, int k, Shared &sh, int &turn)
{
    int size = 2;
    while (size < k)
        size *= 2;
    if (have > 2 * size) {
        cut_list<CAP>(list, have, k, sh, turn);
        have = k;
    }
    while (size < have)
        size *= 2;
    for (int i = have + threadIdx.x; i < size; i += kThreads)
        list[i] = 0;
    for (int run = 2; run <= size; run *= 2)
        for (int step = run / 2; step; step /= 2) {
            __syncthreads();
            for (int i = threadIdx.x; i < size / 2; i += kThreads) {
                const int a = 2 * i - (i & (step - 1)), b = a + step;
                const uint64_t x = list[a], y = list[b];
                if ((x < y) == ((a & run) == 0)) {
                    list[a] = y;
                    list[b] = x;
                }
            }
        }
    __syncthreads();
}

template <typename E>
__device__ void write_row(const Top &a, int64_t row, const uint64_t *list, nbh_softmax stats)
{
    typedef typename E::item item;
    const item *in = reinterpret_cast<const item *>(a.in + row * a.stride);
    item *values = reinterpret_cast<item *>(a.values + row * a.values_stride);
    int32_t *indices = reinterpret_cast<int32_t *>(a.indices + row * a.indices_stride);
    for (int i = threadIdx.x; i < a.k; i += kThreads) {
        const int64_t index = index_of(list[i]);
        values[i] = in[index];
        indices[i] = (int32_t)index;
    }
    if (a.lse && threadIdx.x == 0)
        a.lse[row] = nbh_softmax_lse(stats, a.temperature);
}

template <typename E, bool LSE, int CAP>
__global__ __launch_bounds__(kThreads) void top_rows(Top a)
{
    typedef typename E::item item;
    constexpr int kItems = E::items, kChunk = kThreads * kVecs * kItems;
    __shared__ uint64_t list[CAP];
    __shared__ Shared sh;
    const int64_t row = a.row0 + blockIdx.x / a.splits;
    const int split = blockIdx.x % a.splits;
    const item *in = reinterpret_cast<const item *>(a.in + row * a.stride);
    const int64_t begin = split * a.slice, end = a.vocab < begin + a.slice ? a.vocab : begin + a.slice;

    if (threadIdx.x == 0) {
        sh.count = 0;
        sh.full[0] = sh.full[1] = 0;
    }
    __syncthreads();
    int turn = 0, full_turn = 0;
    nbh_softmax stats = nbh_softmax_empty();
    uint64_t threshold = 0;              // entries above it belong into the list
    for (int64_t at = begin; at < end; at += kChunk) {
        float f[kVecs][kItems], peak[kVecs];
        for (int j = 0; j < kVecs; ++j) {
            const int64_t v = at + (j * kThreads + threadIdx.x) * kItems;
            nbh_row_load<E, true>(in, v, end, -INFINITY, f[j]);
        }
        for (int j = 0; j < kVecs; ++j) {
            peak[j] = f[j][0];
            for (int i = 1; i < kItems; ++i)
                peak[j] = __builtin_elementwise_maximum(peak[j], f[j][i]);
            if (LSE)
                nbh_softmax_add(stats, f[j], a.scale);
        }
        if (at == begin) {
            uint32_t peaks[kVecs];
            for (int j = 0; j < kVecs; ++j)
                peaks[j] = at + (j * kThreads + threadIdx.x) * kItems < end ? key_of(peak[j]) : 0u;
            uint32_t low = 1, high = ~0u;
            while (low < high) {         // at least k vectors reach `low`, or all there are
                const uint32_t mid = high - (high - low) / 2;
                int reach = 0;
                for (int j = 0; j < kVecs; ++j)
                    reach += __popcll(__ballot(peaks[j] >= mid));
                reach = group_sum(reach, sh, turn);
                if (reach >= a.k)
                    low = mid;
                else
                    high = mid - 1;
                if (reach >= a.k && reach <= a.k + a.k / 8)
                    break;
            }
            threshold = ((uint64_t)low << 32) - 1;
        }
        // entries of this lane still to be offered, one bit each
        uint32_t pending = 0;
        {
            const uint32_t key = (uint32_t)(threshold >> 32);
            const float below = float_below(key);
            for (int j = 0; j < kVecs; ++j)
                if (!(peak[j] <= below))
                    for (int i = 0; i < kItems; ++i)
                        if (key_of(f[j][i]) > key && at + (j * kThreads + threadIdx.x) * kItems + i < end)
                            pending |= 1u << (j * kItems + i);
        }
        for (;;) {
            if (pending)
                for (int j = 0; j < kVecs; ++j)
                    for (int i = 0; i < kItems; ++i) {
                        const uint32_t bit = 1u << (j * kItems + i);
                        if (!(pending & bit))
                            continue;
                        const uint64_t entry =
                            entry_of(f[j][i], at + (j * kThreads + threadIdx.x) * kItems + i);
                        if (entry > threshold) {
                            const int place = atomicAdd(&sh.count, 1);
                            if (place >= CAP) {
                                sh.full[full_turn] = 1;
                                continue;
                            }
                            list[place] = entry;
                        }
                        pending &= ~bit;
                    }
            __syncthreads();
            const int full = sh.full[full_turn];
            full_turn ^= 1;
            if (!full)
                break;
            threshold = cut_list<CAP>(list, CAP, a.k, sh, turn);
            if (threadIdx.x == 0)
                sh.full[full_turn ^ 1] = 0;
            __syncthreads();
        }
    }
    const int have = sh.count < CAP ? sh.count : CAP;
    __syncthreads();
    sort_list<CAP>(list, have, a.k, sh, turn);
    if (LSE)
        stats = nbh_softmax_group<kThreads>(stats, a.scale, sh.stats);
    if (a.splits == 1) {
        write_row<E>(a, row, list, stats);
        return;
    }
    uint64_t *part = a.parts + ((row - a.row0) * a.splits + split) * a.k;
    for (int i = threadIdx.x; i < a.k; i += kThreads)
        part[i] = i < have ? list[i] : 0;
    if (LSE && threadIdx.x == 0)
        a.part_stats[(row - a.row0) * a.splits + split] = stats;
}

template <typename E, bool LSE>
__global__ __launch_bounds__(kThreads) void top_join(Top a)
{
    __shared__ uint64_t list[kJoinCap];
    __shared__ Shared sh;
    const int64_t at = blockIdx.x, row = a.row0 + at;
    const int have = a.splits * a.k;
    for (int i = threadIdx.x; i < have; i += kThreads)
        list[i] = a.parts[at * have + i];
    nbh_softmax stats = nbh_softmax_empty();
    if (LSE)
        for (int s = 0; s < a.splits; ++s)
            stats = nbh_softmax_join(stats, a.part_stats[at * a.splits + s], a.scale);
    __syncthreads();
    int turn = 0;
    sort_list<kJoinCap>(list, have, a.k, sh, turn);
    write_row<E>(a, row, list, stats);
}

// Stretches a row is split into.  Workgroups for four per compute unit; a stretch is at least one chunk
// and the joined lists fit the joining workgroup.
struct Split {
    int splits;
    int64_t slice;
};
Split split_of(int64_t rows, int64_t vocab, int64_t k, int dtype)
{
    const int64_t chunk = (int64_t)kThreads * kVecs * (dtype == NBH_ROW_F32 ? 4 : 8);
    const int64_t chunks = (vocab + chunk - 1) / chunk;
    int64_t splits = (1024 + rows - 1) / rows;
    if (splits > kJoinCap / k)
        splits = kJoinCap / k;
    if (splits > chunks)
        splits = chunks;
    const int64_t each = (chunks + splits - 1) / splits;
    return {(int)((chunks + each - 1) / each), each * chunk};
}

template <typename E, bool LSE>
int launch_top(Top a, int64_t rows, hipStream_t stream)
{
    const int64_t most = NBH_ROW_MOST_GROUPS / a.splits;
    const int64_t all = rows;
    for (a.row0 = 0; a.row0 < all; a.row0 += most) {
        const int64_t now = all - a.row0 < most ? all - a.row0 : most;
        const dim3 grid((unsigned)(now * a.splits));
        if (a.k <= 512)
            top_rows<E, LSE, 2048><<<grid, dim3(kThreads), 0, stream>>>(a);
        else
            top_rows<E, LSE, 4096><<<grid, dim3(kThreads), 0, stream>>>(a);
        if (a.splits > 1)
            top_join<E, LSE><<<dim3((unsigned)now), dim3(kThreads), 0, stream>>>(a);
        if (const int status = nbh_launch_status())
            return status;
    }
    return 0;
}
template <typename E>
int launch_top(const Top &a, int64_t rows, hipStream_t stream)
{
    return a.lse ? launch_top<E, true>(a, rows, stream) : launch_top<E, false>(a, rows, stream);
}

}  // namespace

extern "C" size_t nbh_rows_top_workspace(int64_t rows, int64_t vocab, int64_t k, int dtype)
{
    if (rows <= 0 || vocab <= 0 || vocab > INT32_MAX || k <= 0 || k > vocab || k > NBH_ROW_TOP_MOST || dtype < 0 ||
        dtype > NBH_ROW_BF16)
        return 0;
    const Split s = split_of(rows, vocab, k, dtype);
    return s.splits == 1 ? 0 : (size_t)rows * s.splits * ((size_t)k * sizeof(uint64_t) + sizeof(nbh_softmax));
}

extern "C" int nbh_rows_top(const void *logits, int64_t rows, int64_t vocab, int64_t stride, int dtype, int64_t k,
                            void *values, int64_t values_stride, int32_t *indices, int64_t indices_stride, float *lse,
                            double temperature, void *workspace, size_t workspace_bytes, nbh_stream_t stream)
{
    if (rows < 0 || vocab < 0 || vocab > INT32_MAX || dtype < 0 || dtype > NBH_ROW_BF16 || k < 1 || k > vocab ||
        k > NBH_ROW_TOP_MOST || !nbh_row_temperature(temperature))
        return (int)hipErrorInvalidValue;
    if (rows == 0)
        return 0;
    if (!logits || !values || !indices)
        return (int)hipErrorInvalidValue;
    const Split split = split_of(rows, vocab, k, dtype);
    const size_t need = nbh_rows_top_workspace(rows, vocab, k, dtype);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)))
        return (int)hipErrorInvalidValue;
    Top a = {};
    a.in = (const char *)logits;
    a.stride = stride;
    a.vocab = vocab;
    a.slice = split.slice;
    a.splits = split.splits;
    a.k = (int)k;
    a.values = (char *)values;
    a.values_stride = values_stride;
    a.indices = (char *)indices;
    a.indices_stride = indices_stride;
    a.lse = lse;
    a.temperature = (float)temperature;
    a.scale = (float)(1.4426950408889634 / temperature);
    a.parts = (uint64_t *)workspace;
    a.part_stats = (nbh_softmax *)((char *)workspace + (size_t)rows * split.splits * k * sizeof(uint64_t));

    const hipStream_t s = nbh_hip_stream(stream);
    nbh_stream_report report(s);
    switch (dtype) {
    case NBH_ROW_F32:
        return launch_top<nbh_row_f32>(a, rows, s);
    case NBH_ROW_F16:
        return launch_top<nbh_row_f16>(a, rows, s);
    default:
        return launch_top<nbh_row_bf16>(a, rows, s);
    }
}
