// nbh_rows_top: the k largest entries of each row of logits with their indices, and the row's log-sum-exp.
//
// Entries are compared as 64-bit integers, (an integer that orders like the value) << 32 | ~index: no two
// are equal, so ties and NaN need no cases of their own.  The row is read once:
//   * The entries are split into groups (what a lane reads in a number of chunks), whose maxima are kept.
//     The k-th largest of the maxima is a value that at least k entries reach, and hardly more: with m
//     groups about -m ln(1 - k / m).  Bisection on the integers finds it, or one a little below, in a few
//     counts.
//   * The groups whose maximum reaches it, about k, are listed in LDS and read again, a vector per lane;
//     what reaches it there is appended to another list, whose order does not matter, and that is sorted:
//     short ones by counting how many entries exceed each, others by a bitonic network.
//   * Where too many entries reach it (masses of equal ones, rows sorted by blocks) the bound is raised by
//     bisection over all entries, and if it ends on a value that too many share, over their indices.
// Many rows: one workgroup does all of that for a row.  Few rows: a first launch spreads the groups'
// maxima and the statistics of the log-sum-exp over the device, a second one does the rest.
#include "rows.h"

namespace {

constexpr int kAhead = kNbhAhead;
constexpr int kSlots = 8;                // groups per lane that the one-launch kernel remembers
constexpr int kMaximaThreads = 256;      // first launch of two
constexpr int kMostGroups = 16384;       // groups per row of the two-launch path
constexpr int kFinishThreads = 512;

struct Top {
    const char *in;
    int64_t stride, vocab, row0;
    int k;
    char *values;
    int64_t values_stride;
    char *indices;
    int64_t indices_stride;
    float *lse;
    float temperature, scale;
    int splits, parts;                   // two launches: workgroups per row, groups per lane of theirs
    int64_t slice;                       // entries per workgroup
    uint32_t *maxima;                    // [row][split][part][lane], as keys, 0 for an empty group
    nbh_softmax *part_stats;             // [row][split]
};

// Orders like the value; NaN above all, -0 as +0.  No value has key 0.
__device__ __forceinline__ uint32_t key_of(float x)
{
    const uint32_t bits = __float_as_uint(x + 0.0f);
    return x != x ? 0xffffffffu : bits ^ ((uint32_t)((int32_t)bits >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t entry_of(float x, int64_t index)
{
    return (uint64_t)key_of(x) << 32 | (uint32_t)~(uint32_t)index;
}
// The value again, but for the sign of a zero and the bits of a NaN.
__device__ __forceinline__ float value_of(uint64_t entry)
{
    const uint32_t key = (uint32_t)(entry >> 32);
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ int64_t index_of(uint64_t entry) { return (uint32_t)~(uint32_t)entry; }

// What a workgroup of T lanes shares besides the list itself.
template <int T> struct Shared {
    int groups;                          // groups to be read again, or that would have been
    int count;                           // entries appended, or that would have been
    int tally[2][T / 64];                // by turn: counts of a bisection step
    uint32_t ends[2][T / 64];
    nbh_softmax stats[T / 64];
};

// Sum over the workgroup of a number every lane of a wavefront agrees on.  One barrier: the next step
// writes the other row.
template <int T> __device__ __forceinline__ int group_sum(int of_wave, Shared<T> &sh, int &turn)
{
    if ((threadIdx.x & 63) == 0)
        sh.tally[turn][threadIdx.x >> 6] = of_wave;
    __syncthreads();
    int sum = 0;
    for (int w = 0; w < T / 64; ++w)
        sum += sh.tally[turn][w];
    turn ^= 1;
    return sum;
}

// A key that at least k of the groups' maxima reach (P of them in every lane, 0 for none), or 1 if there
// are not that many; `top` is the largest.
template <int T, int P>
__device__ uint32_t bound_of(const uint32_t (&peaks)[P], int k, Shared<T> &sh, int &turn, uint32_t &top)
{
    uint32_t high = 0, low = ~0u;
#pragma unroll
    for (int g = 0; g < P; ++g) {
        high = peaks[g] > high ? peaks[g] : high;
        low = peaks[g] && peaks[g] < low ? peaks[g] : low;
    }
    for (int step = 32; step; step >>= 1) {
        const uint32_t h = __shfl_xor(high, step), l = __shfl_xor(low, step);
        high = h > high ? h : high;
        low = l < low ? l : low;
    }
    int there = 0;
#pragma unroll
    for (int g = 0; g < P; ++g)
        there += __popcll(__ballot(peaks[g] != 0));
    if ((threadIdx.x & 63) == 0) {
        sh.ends[0][threadIdx.x >> 6] = high;
        sh.ends[1][threadIdx.x >> 6] = low;
    }
    there = group_sum(there, sh, turn);
    for (int w = 0; w < T / 64; ++w) {
        high = sh.ends[0][w] > high ? sh.ends[0][w] : high;
        low = sh.ends[1][w] < low ? sh.ends[1][w] : low;
    }
    top = high;
    if (there < k)
        return 1;
    while (low < high) {
        const uint32_t mid = high - (high - low) / 2;
        int reach = 0;
#pragma unroll
        for (int g = 0; g < P; ++g)
            reach += __popcll(__ballot(peaks[g] >= mid));
        reach = group_sum(reach, sh, turn);
        if (reach >= k)
            low = mid;
        else
            high = mid - 1;
        if (reach >= k && reach <= k + (k < 64 ? 8 : k / 8))
            break;
    }
    return low;
}

// Appends what reaches `bound` of the entries at .. at + items.
template <typename E, int T, int CAP>
__device__ __forceinline__ void append(const typename E::item *in, int64_t at, int64_t end, uint64_t bound,
                                       uint64_t *list, Shared<T> &sh)
{
    if (at >= end)
        return;
    float f[E::items];
    nbh_row_load<E, false>(in, at, end, -INFINITY, f);
    if (key_of(nbh_row_most(f)) < (uint32_t)(bound >> 32))
        return;
    for (int i = 0; i < E::items; ++i) {
        const uint64_t entry = entry_of(f[i], at + i);
        if (entry >= bound && at + i < end) {
            const int place = atomicAdd(&sh.count, 1);
            if (place < CAP)
                list[place] = entry;
        }
    }
}

// More than CAP of the row's n entries reach the key `low`, none exceeds the key `high`: a bound that at
// least k and at most CAP entries reach.
template <typename E, int T, int CAP>
__device__ uint64_t raised_bound(const typename E::item *in, int64_t n, uint32_t low, uint32_t high, int k,
                                 Shared<T> &sh, int &turn)
{
    auto count = [&](auto reaches) {
        int mine = 0;
        for (int64_t at = (int64_t)threadIdx.x * E::items; at < n; at += T * E::items) {
            float f[E::items];
            nbh_row_load<E, false>(in, at, n, -INFINITY, f);
            for (int i = 0; i < E::items; ++i)
                mine += at + i < n && reaches(f[i], at + i);
        }
        for (int step = 32; step; step >>= 1)
            mine += __shfl_xor(mine, step);
        return group_sum(mine, sh, turn);
    };
    int reach = CAP + 1;
    while (low < high && reach > CAP) {
        const uint32_t mid = high - (high - low) / 2;
        const int now = count([&](float x, int64_t) { return key_of(x) >= mid; });
        if (now >= k) {
            low = mid;
            reach = now;
        } else {
            high = mid - 1;
        }
    }
    uint64_t from = (uint64_t)low << 32, to = from | 0xffffffffu;
    while (from < to && reach > CAP) {   // low is the k-th largest value, and too many share it
        const uint64_t mid = to - (to - from) / 2;
        const int now = count([&](float x, int64_t index) { return entry_of(x, index) >= mid; });
        if (now >= k) {
            from = mid;
            reach = now;
        } else {
            to = mid - 1;
        }
    }
    return from;
}

// Writes the k best of the list (at least k entries) in order.  The list has been written before a
// barrier and has room for two entries more.
template <typename E, int T>
__device__ void write_ranked(const Top &a, int64_t row, uint64_t *list, int have)
{
    typedef typename E::item item;
    const item *in = reinterpret_cast<const item *>(a.in + row * a.stride);
    item *values = reinterpret_cast<item *>(a.values + row * a.values_stride);
    int32_t *indices = reinterpret_cast<int32_t *>(a.indices + row * a.indices_stride);
    auto put = [&](int rank, uint64_t entry) {
        const int64_t index = index_of(entry);
        const float value = value_of(entry);
        values[rank] = value == 0.0f || value != value ? in[index] : E::put(value);
        indices[rank] = (int32_t)index;
    };
    if (have <= 256) {
        // a lane per entry counts what exceeds it: have / 2 reads of LDS, the same address in all lanes
        if (threadIdx.x == 0)
            list[have] = 0;
        __syncthreads();
        if ((int)threadIdx.x < have) {
            const uint64_t mine = list[threadIdx.x];
            int rank = 0;
            for (int i = 0; i < have; i += 2) {
                const ulonglong2 two = *reinterpret_cast<const ulonglong2 *>(list + i);
                rank += (two.x > mine) + (two.y > mine);
            }
            if (rank < a.k)
                put(rank, mine);
        }
        return;
    }
    int size = 512;
    while (size < have)
        size *= 2;
    for (int i = have + threadIdx.x; i < size; i += T)
        list[i] = 0;
    __syncthreads();
    for (int run = 2; run <= size; run *= 2)
        for (int step = run / 2; step; step /= 2) {
            for (int i = threadIdx.x; i < size / 2; i += T) {
                const int at = 2 * i - (i & (step - 1)), other = at + step;
                const uint64_t x = list[at], y = list[other];
                if ((x < y) == ((at & run) == 0)) {
                    list[at] = y;
                    list[other] = x;
                }
            }
            // Pairs at most 64 apart stay within the 128 entries of a wavefront, whose LDS accesses are in
            // order, until the next step reaches further.
            if (step > 64 || (step == 1 && run >= 128))
                __syncthreads();
            else
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    __syncthreads();
    for (int i = threadIdx.x; i < a.k; i += T)
        put(i, list[i]);
}

// One workgroup per row.
template <typename E, bool LSE, int T, int CAP> __global__ __launch_bounds__(T) void top_rows(Top a)
{
    typedef typename E::item item;
    constexpr int kItems = E::items, kChunk = kAhead * T * kItems;
    __shared__ __align__(16) uint64_t list[CAP + 2];
    __shared__ uint32_t maxima[kSlots * T];
    __shared__ int again[CAP];
    __shared__ Shared<T> sh;
    const int64_t row = a.row0 + blockIdx.x;
    const item *in = reinterpret_cast<const item *>(a.in + row * a.stride);
    const int64_t n = a.vocab;
    // chunks per group, a power of two
    int shift = 0;
    while ((n + kChunk - 1) / kChunk > (int64_t)kSlots << shift)
        ++shift;
    int turn = 0;
    if (threadIdx.x == 0)
        sh.groups = sh.count = 0;

    // -- groups' maxima, and the statistics of the log-sum-exp.  For the bound a lane's maximum will do up
    // to k = T / 4, else the maxima of the four vectors of its chunks.
    const bool fine = a.k > T / 4;
    nbh_softmax stats = nbh_softmax_empty();
    float peak[kAhead], slot = -INFINITY;
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        peak[j] = -INFINITY;
    nbh_row_stream<E, T, false>(in, 0, n, [&](int64_t at, const nbh_u32x4(&raw)[kAhead]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            float f[kItems];
            E::unpack(raw[j], f);
            const float most = nbh_row_most(f);
            peak[j] = __builtin_elementwise_maximum(peak[j], most);
            slot = __builtin_elementwise_maximum(slot, most);
            if (LSE)
                nbh_softmax_add(stats, f, most, a.scale);
        }
        const int64_t chunk = at / kChunk;
        maxima[(chunk >> shift) * T + threadIdx.x] = key_of(slot);
        if (((chunk + 1) & ((1 << shift) - 1)) == 0)
            slot = -INFINITY;
    });
    uint32_t peaks[kAhead], top;
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        peaks[j] = (j * T + (int64_t)threadIdx.x) * kItems < n ? key_of(peak[j]) : 0u;
    uint32_t key;
    if (fine) {
        key = bound_of<T>(peaks, a.k, sh, turn, top);
    } else {
        uint32_t lane[1] = {0u};
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            lane[0] = peaks[j] > lane[0] ? peaks[j] : lane[0];
        key = bound_of<T>(lane, a.k, sh, turn, top);
    }

    // -- what reaches it
    uint64_t bound = (uint64_t)key << 32;
    for (;;) {
        const int64_t group = (int64_t)kChunk << shift;
        for (int g = threadIdx.x; (g / T) * group < n; g += T)
            if (maxima[g] >= (uint32_t)(bound >> 32)) {
                const int place = atomicAdd(&sh.groups, 1);
                if (place < CAP)
                    again[place] = g;
            }
        __syncthreads();
        if (sh.groups <= CAP) {
            const int vectors = kAhead << shift;     // of a group
            for (int i = threadIdx.x; i < sh.groups * vectors; i += T) {
                const int g = again[i / vectors], v = i % vectors;
                append<E, T, CAP>(in, (g / T) * group + (v * T + g % T) * (int64_t)kItems, n, bound, list, sh);
            }
            __syncthreads();
            if (sh.count <= CAP)
                break;
        }
        bound = raised_bound<E, T, CAP>(in, n, (uint32_t)(bound >> 32), top, a.k, sh, turn);
        __syncthreads();
        if (threadIdx.x == 0)
            sh.groups = sh.count = 0;
        __syncthreads();
    }
    if (LSE) {
        stats = nbh_softmax_group<T>(stats, a.scale, sh.stats);
        if (threadIdx.x == 0)
            a.lse[row] = nbh_softmax_lse(stats, a.temperature, a.scale);
    }
    write_ranked<E, T>(a, row, list, sh.count);
}

// First launch of two: the maxima of the lanes (or of the four vectors of their chunks) of a stretch.
template <typename E, bool LSE> __global__ __launch_bounds__(kMaximaThreads) void top_maxima(Top a)
{
    constexpr int T = kMaximaThreads, kItems = E::items;
    __shared__ nbh_softmax room[T / 64];
    const int64_t at = blockIdx.x / a.splits, row = a.row0 + at;
    const int split = blockIdx.x % a.splits;
    const typename E::item *in = reinterpret_cast<const typename E::item *>(a.in + row * a.stride);
    const int64_t begin = split * a.slice, end = a.vocab < begin + a.slice ? a.vocab : begin + a.slice;
    nbh_softmax stats = nbh_softmax_empty();
    float peak[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
        peak[j] = -INFINITY;
    nbh_row_stream<E, T, false>(in, begin, end, [&](int64_t, const nbh_u32x4(&raw)[kAhead]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            float f[kItems];
            E::unpack(raw[j], f);
            const float most = nbh_row_most(f);
            peak[j] = __builtin_elementwise_maximum(peak[j], most);
            if (LSE)
                nbh_softmax_add(stats, f, most, a.scale);
        }
    });
    uint32_t *out = a.maxima + (blockIdx.x * (int64_t)a.parts) * T + threadIdx.x;
    uint32_t lane = 0;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
        const uint32_t key = begin + (j * T + (int64_t)threadIdx.x) * kItems < end ? key_of(peak[j]) : 0u;
        lane = key > lane ? key : lane;
        if (a.parts > 1)
            out[j * T] = key;
    }
    if (a.parts == 1)
        out[0] = lane;
    if (LSE) {
        stats = nbh_softmax_group<T>(stats, a.scale, room);
        if (threadIdx.x == 0)
            a.part_stats[at * a.splits + split] = stats;
    }
}

// Second launch: a workgroup per row, P groups per lane.
template <typename E, bool LSE, int P> __global__ __launch_bounds__(kFinishThreads) void top_finish(Top a)
{
    typedef typename E::item item;
    constexpr int T = kFinishThreads, kItems = E::items, M = kMaximaThreads, CAP = 4096;
    constexpr int kChunk = kAhead * M * kItems;
    __shared__ __align__(16) uint64_t list[CAP + 2];
    __shared__ int again[CAP];
    __shared__ Shared<T> sh;
    const int64_t row = a.row0 + blockIdx.x;
    const item *in = reinterpret_cast<const item *>(a.in + row * a.stride);
    const int groups = a.splits * a.parts * M;
    const uint32_t *maxima = a.maxima + blockIdx.x * (int64_t)groups;
    int turn = 0;
    if (threadIdx.x == 0)
        sh.groups = sh.count = 0;
    uint32_t peaks[P], top;
#pragma unroll
    for (int g = 0; g < P; ++g) {
        const int at = g * T + threadIdx.x;
        peaks[g] = at < groups ? maxima[at] : 0u;
    }
    if (LSE && threadIdx.x < 64) {
        static_assert(kMostGroups / M <= 64, "a lane per stretch");
        const int lane = threadIdx.x;
        nbh_softmax stats = lane < a.splits ? a.part_stats[blockIdx.x * (int64_t)a.splits + lane] : nbh_softmax_empty();
        for (int step = 32; step; step >>= 1) {
            const nbh_softmax other = {__shfl_xor(stats.peak, step), __shfl_xor(stats.sum, step)};
            stats = nbh_softmax_join(stats, other, a.scale);
        }
        if (lane == 0)
            a.lse[row] = nbh_softmax_lse(stats, a.temperature, a.scale);
    }
    uint64_t bound = (uint64_t)bound_of<T>(peaks, a.k, sh, turn, top) << 32;
    const int chunks = (int)(a.slice / kChunk), vectors = chunks * (a.parts > 1 ? 1 : kAhead);       // of a group
    for (;;) {
#pragma unroll
        for (int g = 0; g < P; ++g)
            if (peaks[g] && peaks[g] >= (uint32_t)(bound >> 32)) {
                const int place = atomicAdd(&sh.groups, 1);
                if (place < CAP)
                    again[place] = g * T + threadIdx.x;
            }
        __syncthreads();
        if (sh.groups <= CAP) {
            for (int64_t i = threadIdx.x; i < (int64_t)sh.groups * vectors; i += T) {
                const int g = again[i / vectors], v = (int)(i % vectors);
                const int lane = g % M, part = g / M % a.parts, split = g / M / a.parts;
                const int64_t begin = split * a.slice, end = a.vocab < begin + a.slice ? a.vocab : begin + a.slice;
                const int64_t at = a.parts > 1 ? begin + v * (int64_t)kChunk + (part * M + lane) * kItems
                                               : begin + (v * (int64_t)M + lane) * kItems;
                append<E, T, CAP>(in, at, end, bound, list, sh);
            }
            __syncthreads();
            if (sh.count <= CAP)
                break;
        }
        bound = raised_bound<E, T, CAP>(in, a.vocab, (uint32_t)(bound >> 32), top, a.k, sh, turn);
        __syncthreads();
        if (threadIdx.x == 0)
            sh.groups = sh.count = 0;
        __syncthreads();
    }
    write_ranked<E, T>(a, row, list, sh.count);
}

// Workgroups per row: one from 256 rows on (a compute unit each), or where a row is a chunk or less; else
// enough for four per compute unit, with at most kMostGroups groups.  Four groups per lane where k is more
// than a quarter of the groups would otherwise be.
struct Split {
    int splits, parts;
    int64_t slice;
};
Split split_of(int64_t rows, int64_t vocab, int64_t k, int dtype)
{
    const int64_t chunk = (int64_t)kMaximaThreads * kAhead * (dtype == NBH_ROW_F32 ? 4 : 8);
    const int64_t chunks = (vocab + chunk - 1) / chunk;
    if (rows >= 256 || chunks == 1)
        return {1, 1, vocab};
    int64_t splits = (1024 + rows - 1) / rows;
    if (splits > chunks)
        splits = chunks;
    if (splits > kMostGroups / kMaximaThreads)
        splits = kMostGroups / kMaximaThreads;
    int parts = k > splits * kMaximaThreads / 4 ? kAhead : 1;
    if (parts * splits > kMostGroups / kMaximaThreads)
        parts = 1;
    const int64_t each = (chunks + splits - 1) / splits;
    return {(int)((chunks + each - 1) / each), parts, each * chunk};
}

template <typename E, bool LSE> int launch_top(Top a, int64_t rows, hipStream_t stream)
{
    const int64_t most = NBH_ROW_MOST_GROUPS / a.splits;
    for (a.row0 = 0; a.row0 < rows; a.row0 += most) {
        const int64_t now = rows - a.row0 < most ? rows - a.row0 : most;
        const dim3 grid((unsigned)now);
        if (a.splits == 1) {
            // 256 lanes make 1024 groups, which serve up to k = 256; larger workgroups wait longer at
            // their barriers (4096 x 65536 bfloat16, k = 64: 124 us, with 512 lanes 140 us)
            if (a.k <= 256)
                top_rows<E, LSE, 256, 1024><<<grid, dim3(256), 0, stream>>>(a);
            else
                top_rows<E, LSE, 512, 4096><<<grid, dim3(512), 0, stream>>>(a);
        } else {
            top_maxima<E, LSE><<<dim3((unsigned)(now * a.splits)), dim3(kMaximaThreads), 0, stream>>>(a);
            const int groups = a.splits * a.parts * kMaximaThreads;
            if (groups <= 8 * kFinishThreads)
                top_finish<E, LSE, 8><<<grid, dim3(kFinishThreads), 0, stream>>>(a);
            else
                top_finish<E, LSE, kMostGroups / kFinishThreads><<<grid, dim3(kFinishThreads), 0, stream>>>(a);
        }
        if (const int status = nbh_launch_status())
            return status;
    }
    return 0;
}
template <typename E> int launch_top(const Top &a, int64_t rows, hipStream_t stream)
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
    return s.splits == 1 ? 0
                         : (size_t)rows * s.splits *
                               ((size_t)s.parts * kMaximaThreads * sizeof(uint32_t) + sizeof(nbh_softmax));
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
    a.k = (int)k;
    a.values = (char *)values;
    a.values_stride = values_stride;
    a.indices = (char *)indices;
    a.indices_stride = indices_stride;
    a.lse = lse;
    a.temperature = (float)temperature;
    a.scale = (float)(1.4426950408889634 / a.temperature);
    a.splits = split.splits;
    a.parts = split.parts;
    a.slice = split.slice;
    a.maxima = (uint32_t *)workspace;
    a.part_stats = (nbh_softmax *)(a.maxima + (size_t)rows * split.splits * split.parts * kMaximaThreads);

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
