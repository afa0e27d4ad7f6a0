// nbh_rows_top: the k largest entries of each row of logits with their indices, and the row's log-sum-exp.
//
// Entries are compared as 64-bit integers, (an integer that orders like the value) << 32 | ~index: no two
// are equal, so ties and NaN need no cases of their own.  A workgroup reads a stretch of a row once and
// keeps the maximum of each 16-byte vector:
//   * The maxima of the lanes (or of the parts of a lane, for large k) are maxima of disjoint groups, so the
//     k-th largest of them is a value that at least k entries reach, and hardly more: with m groups about
//     -m ln(1 - k / m).  Bisection on the integers finds it, or one a little below, in a few counts.
//   * The vectors whose maximum reaches it are read again (about k of them), what reaches it in them is
//     appended to a list in LDS, whose order does not matter, and the list is sorted: short ones by
//     counting how many entries exceed each, others by a bitonic network.
//   * Where too many entries reach it (masses of equal ones, rows sorted by blocks) the bound is raised by
//     bisection over all entries, and if it ends on a value that too many share, over their indices.
// Rows longer than a stretch, and few rows, are split over workgroups, whose lists a second launch joins.
#include "rows.h"

namespace {

constexpr int kJoinThreads = 256;
constexpr int kJoinCap = 4096;           // entries the joining workgroup holds at a time

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
// A float `t` such that !(x < t) holds for every x whose key reaches `key` (and, if t is NaN, for all).
__device__ __forceinline__ float float_at(uint32_t key)
{
    if (key <= 0x007fffffu)              // -inf's key or below
        return __uint_as_float(0xff800000u);
    return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}
__device__ __forceinline__ uint64_t entry_of(float x, int64_t index)
{
    return (uint64_t)key_of(x) << 32 | (uint32_t)~(uint32_t)index;
}
__device__ __forceinline__ int64_t index_of(uint64_t entry) { return (uint32_t)~(uint32_t)entry; }

// What a workgroup of T lanes shares besides the list itself.
template <int T> struct Shared {
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

// Cuts the list (`have` entries, more than k) to its k best, in any order.
template <int T, int CAP> __device__ void cut_list(uint64_t *list, int have, int k, Shared<T> &sh, int &turn)
{
    uint64_t mine[CAP / T];
    for (int i = 0; i < CAP / T; ++i) {
        const int at = i * T + threadIdx.x;
        mine[i] = at < have ? list[at] : 0;
    }
    uint64_t low = 1, high = ~0ull;      // at least k entries reach `low`, fewer `high` + 1
    while (low < high) {
        const uint64_t mid = high - (high - low) / 2;
        int reach = 0;
        for (int i = 0; i < CAP / T; ++i)
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
    for (int i = 0; i < CAP / T; ++i)
        if (mine[i] >= low)
            list[atomicAdd(&sh.count, 1)] = mine[i];
    __syncthreads();
}

// Calls put(rank, entry) for the k best of the list, rank 0 the largest; fewer if there are fewer.  The
// list has been written before a barrier and has room for two entries more.
template <int T, int CAP, typename F>
__device__ void rank_list(uint64_t *list, int have, int k, Shared<T> &sh, int &turn, F put)
{
    if (have <= T) {
        // every lane counts what exceeds its entry: have / 2 reads of LDS, the same address in all lanes
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
            if (rank < k)
                put(rank, mine);
        }
        return;
    }
    int size = 2;
    while (size < k)
        size *= 2;
    if (have > 2 * size) {
        cut_list<T, CAP>(list, have, k, sh, turn);
        have = sh.count;
    }
    while (size < have)
        size *= 2;
    for (int i = have + threadIdx.x; i < size; i += T)
        list[i] = 0;
    for (int run = 2; run <= size; run *= 2)
        for (int step = run / 2; step; step /= 2) {
            __syncthreads();
            for (int i = threadIdx.x; i < size / 2; i += T) {
                const int a = 2 * i - (i & (step - 1)), b = a + step;
                const uint64_t x = list[a], y = list[b];
                if ((x < y) == ((a & run) == 0)) {
                    list[a] = y;
                    list[b] = x;
                }
            }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < k && i < have; i += T)
        put(i, list[i]);
}

template <typename E> struct Out {
    typedef typename E::item item;
    const item *in;
    item *values;
    int32_t *indices;
    __device__ Out(const Top &a, int64_t row)
        : in(reinterpret_cast<const item *>(a.in + row * a.stride)),
          values(reinterpret_cast<item *>(a.values + row * a.values_stride)),
          indices(reinterpret_cast<int32_t *>(a.indices + row * a.indices_stride))
    {
    }
    __device__ void operator()(int rank, uint64_t entry) const
    {
        const int64_t index = index_of(entry);
        values[rank] = in[index];
        indices[rank] = (int32_t)index;
    }
};

// T lanes take V vectors each; the maxima of P parts of a lane's vectors are its groups' maxima.
template <typename E, bool LSE, int T, int V, int P, int CAP>
__global__ __launch_bounds__(T, 4) void top_rows(Top a)
{
    typedef typename E::item item;
    constexpr int kItems = E::items, kAhead = 4;
    __shared__ __align__(16) uint64_t list[CAP + 2];
    __shared__ float maxima[V * T];
    __shared__ Shared<T> sh;
    const int64_t row = a.row0 + blockIdx.x / a.splits;
    const int split = blockIdx.x % a.splits;
    const int64_t begin = split * a.slice;
    const item *in = reinterpret_cast<const item *>(a.in + row * a.stride) + begin;
    const int n = (int)(a.vocab - begin < a.slice ? a.vocab - begin : a.slice);
    int turn = 0;

    if (threadIdx.x == 0)
        sh.count = 0;
    // -- the vectors' maxima, and the statistics of the log-sum-exp
    nbh_softmax stats = nbh_softmax_empty();
    float peak[P];
#pragma unroll
    for (int g = 0; g < P; ++g)
        peak[g] = -INFINITY;
    {
        // four loads are on their way while four others are looked at
        nbh_u32x4 raw[kAhead], next[kAhead];
        auto ask = [&](nbh_u32x4(&to)[kAhead], int at) {
            if ((at + kAhead * T) * kItems <= n) {
#pragma unroll
                for (int j = 0; j < kAhead; ++j)
                    to[j] = E::template load<false>(in + (at + j * T + threadIdx.x) * kItems);
            } else {
#pragma unroll
                for (int j = 0; j < kAhead; ++j)
                    to[j] = nbh_row_load_raw<E, false>(in, (at + j * T + threadIdx.x) * kItems, n, E::lowest);
            }
        };
        ask(raw, 0);
#pragma unroll 1
        for (int at = 0; at * kItems < n; at += kAhead * T) {
            if (V > kAhead)
                ask(next, at + kAhead * T);
            float part = -INFINITY;      // of this lane's four vectors
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                float f[kItems];
                E::unpack(raw[j], f);
                float most = f[0];
#pragma unroll
                for (int i = 1; i < kItems; ++i)
                    most = __builtin_elementwise_maximum(most, f[i]);
                maxima[at + j * T + threadIdx.x] = most;
                if (V == kAhead && P > 1)
                    peak[j % P] = __builtin_elementwise_maximum(peak[j % P], most);
                part = __builtin_elementwise_maximum(part, most);
                if (LSE)
                    nbh_softmax_add(stats, f, a.scale);
            }
            if (V > kAhead || P == 1) {
#pragma unroll
                for (int g = 0; g < P; ++g)
                    if (at / (kAhead * T) % P == g)
                        peak[g] = __builtin_elementwise_maximum(peak[g], part);
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                raw[j] = next[j];
        }
    }
    uint32_t peaks[P];
    uint32_t high = 0, low = ~0u;
#pragma unroll
    for (int g = 0; g < P; ++g) {
        // the group's first vector
        const bool there = ((V > kAhead ? g * kAhead : g) * T + (int)threadIdx.x) * kItems < n;
        peaks[g] = there ? key_of(peak[g]) : 0u;
        high = peaks[g] > high ? peaks[g] : high;
        low = peaks[g] < low ? peaks[g] : low;
    }
    // -- the bound: at least k of the maxima reach `low`, or it is below them all
    for (int step = 32; step; step >>= 1) {
        const uint32_t h = __shfl_xor(high, step), l = __shfl_xor(low, step);
        high = h > high ? h : high;
        low = l < low ? l : low;
    }
    if ((threadIdx.x & 63) == 0) {
        sh.ends[0][threadIdx.x >> 6] = high;
        sh.ends[1][threadIdx.x >> 6] = low;
    }
    __syncthreads();
    for (int w = 0; w < T / 64; ++w) {
        high = sh.ends[0][w] > high ? sh.ends[0][w] : high;
        low = sh.ends[1][w] < low ? sh.ends[1][w] : low;
    }
    const uint32_t top = high;
    if (low == 0 || a.k > T * P)
        low = 1;                         // groups without entries, or fewer groups than entries wanted
    if (a.k <= T * P)
        while (low < high) {
            const uint32_t mid = high - (high - low) / 2;
            int reach = 0;
#pragma unroll
            for (int g = 0; g < P; ++g)
                reach += __popcll(__ballot(peaks[g] >= mid));
            reach = group_sum(reach, sh, turn);
            if (reach >= a.k)
                low = mid;
            else
                high = mid - 1;
            if (reach >= a.k && reach <= a.k + a.k / 8)
                break;
        }

    // -- what reaches it
    uint64_t bound = (uint64_t)low << 32;
    for (int attempt = 0;; ++attempt) {
        const uint32_t key = (uint32_t)(bound >> 32);
        const float from = float_at(key);
        float lane = peak[0];
#pragma unroll
        for (int g = 1; g < P; ++g)
            lane = __builtin_elementwise_maximum(lane, peak[g]);
        // a lane sees its own maxima only
        for (int v = threadIdx.x; !(lane < from) && v * kItems < n; v += T) {
            if (maxima[v] < from)
                continue;
            const int first = v * kItems;
            float f[kItems];
            nbh_row_load<E, false>(in, first, n, -INFINITY, f);
            for (int i = 0; i < kItems; ++i) {
                const uint64_t entry = entry_of(f[i], begin + first + i);
                if (entry >= bound && first + i < n) {
                    const int place = atomicAdd(&sh.count, 1);
                    if (place < CAP)
                        list[place] = entry;
                }
            }
        }
        __syncthreads();
        if (sh.count <= CAP)
            break;
        // Too many.  Raise the bound: first the value, until at most CAP entries reach it or it is the
        // k-th largest, then the index, likewise.  (Two attempts: the second one's list is never too long.)
        auto count = [&](auto reaches) {
            int mine = 0;
            for (int at = threadIdx.x * kItems; at < n; at += T * kItems) {      // from memory: this is rare
                float f[kItems];
                nbh_row_load<E, false>(in, at, n, -INFINITY, f);
                for (int i = 0; i < kItems; ++i)
                    mine += at + i < n && reaches(f[i], begin + at + i);
            }
            for (int step = 32; step; step >>= 1)
                mine += __shfl_xor(mine, step);
            return group_sum(mine, sh, turn);
        };
        uint32_t low = key, high = top;  // at least k entries reach `low`
        int reach = CAP + 1;
        while (low < high && reach > CAP) {
            const uint32_t mid = high - (high - low) / 2;
            const int now = count([&](float x, int64_t) { return key_of(x) >= mid; });
            if (now >= a.k) {
                low = mid;
                reach = now;
            } else {
                high = mid - 1;
            }
        }
        bound = (uint64_t)low << 32;
        if (reach > CAP) {               // low is the k-th largest value, and too many share it
            uint64_t from = bound, to = bound | 0xffffffffu;
            while (from < to && reach > CAP) {
                const uint64_t mid = to - (to - from) / 2;
                const int now = count([&](float x, int64_t index) { return entry_of(x, index) >= mid; });
                if (now >= a.k) {
                    from = mid;
                    reach = now;
                } else {
                    to = mid - 1;
                }
            }
            bound = from;
        }
        if (threadIdx.x == 0)
            sh.count = 0;
        __syncthreads();
    }
    const int have = sh.count;
    if (LSE)
        stats = nbh_softmax_group<T>(stats, a.scale, sh.stats);
    if (a.splits == 1) {
        rank_list<T, CAP>(list, have, a.k, sh, turn, Out<E>(a, row));
        if (LSE && threadIdx.x == 0)
            a.lse[row] = nbh_softmax_lse(stats, a.temperature);
        return;
    }
    uint64_t *part = a.parts + ((row - a.row0) * a.splits + split) * a.k;
    rank_list<T, CAP>(list, have, a.k, sh, turn, [&](int rank, uint64_t entry) { part[rank] = entry; });
    for (int i = have + threadIdx.x; i < a.k; i += T)
        part[i] = 0;
    if (LSE && threadIdx.x == 0)
        a.part_stats[(row - a.row0) * a.splits + split] = stats;
}

template <typename E, bool LSE> __global__ __launch_bounds__(kJoinThreads) void top_join(Top a)
{
    constexpr int T = kJoinThreads;
    __shared__ __align__(16) uint64_t list[kJoinCap + 2];
    __shared__ Shared<T> sh;
    const int64_t at = blockIdx.x, row = a.row0 + at;
    const int64_t all = (int64_t)a.splits * a.k;
    if (LSE && threadIdx.x == 0) {
        nbh_softmax stats = nbh_softmax_empty();
        for (int s = 0; s < a.splits; ++s)
            stats = nbh_softmax_join(stats, a.part_stats[at * a.splits + s], a.scale);
        a.lse[row] = nbh_softmax_lse(stats, a.temperature);
    }
    int turn = 0, have = 0;
    for (int64_t next = 0; next < all;) {
        const int more = (int)(all - next < kJoinCap - have ? all - next : kJoinCap - have);
        for (int i = threadIdx.x; i < more; i += T)
            list[have + i] = a.parts[at * all + next + i];
        __syncthreads();
        next += more;
        have += more;
        if (next < all) {                // the list is full: keep its k best, all but the last list are whole
            cut_list<T, kJoinCap>(list, have, a.k, sh, turn);
            have = a.k;
        }
    }
    rank_list<T, kJoinCap>(list, have, a.k, sh, turn, Out<E>(a, row));
}

// Stretches a row is split into: 128 KiB on 512 lanes where rows alone make a workgroup or more per compute
// unit, else 16 KiB on 256 lanes, unless
// their lists would not fit the joining workgroup at once.
struct Split {
    bool large;
    int splits;
    int64_t slice;
};
Split split_of(int64_t rows, int64_t vocab, int64_t k, int dtype)
{
    const int64_t items = dtype == NBH_ROW_F32 ? 4 : 8;
    const int64_t small = 256 * 4 * items, large = 512 * 16 * items;
    const int64_t many = (vocab + small - 1) / small, few = (vocab + large - 1) / large;
    const bool use_large = many > 1 && (rows * few >= 256 || many * k > kJoinCap);
    const int64_t splits = use_large ? few : many;
    return {use_large, (int)splits, use_large ? large : small};
}

template <typename E, bool LSE>
int launch_top(Top a, int64_t rows, bool large, hipStream_t stream)
{
    const int64_t most = NBH_ROW_MOST_GROUPS / a.splits;
    const int64_t all = rows;
    for (a.row0 = 0; a.row0 < all; a.row0 += most) {
        const int64_t now = all - a.row0 < most ? all - a.row0 : most;
        const dim3 grid((unsigned)(now * a.splits));
        if (large && a.k <= 256)
            top_rows<E, LSE, 512, 16, 1, 2048><<<grid, dim3(512), 0, stream>>>(a);
        else if (large)
            top_rows<E, LSE, 512, 16, 4, 4096><<<grid, dim3(512), 0, stream>>>(a);
        else if (a.k <= 128)
            top_rows<E, LSE, 256, 4, 1, 2048><<<grid, dim3(256), 0, stream>>>(a);
        else
            top_rows<E, LSE, 256, 4, 4, 4096><<<grid, dim3(256), 0, stream>>>(a);
        if (a.splits > 1)
            top_join<E, LSE><<<dim3((unsigned)now), dim3(kJoinThreads), 0, stream>>>(a);
        if (const int status = nbh_launch_status())
            return status;
    }
    return 0;
}
template <typename E>
int launch_top(const Top &a, int64_t rows, bool large, hipStream_t stream)
{
    return a.lse ? launch_top<E, true>(a, rows, large, stream) : launch_top<E, false>(a, rows, large, stream);
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
        return launch_top<nbh_row_f32>(a, rows, split.large, s);
    case NBH_ROW_F16:
        return launch_top<nbh_row_f16>(a, rows, split.large, s);
    default:
        return launch_top<nbh_row_bf16>(a, rows, split.large, s);
    }
}
