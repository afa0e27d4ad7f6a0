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
//     short ones by counting how many entries exceed each, others by buckets of their values, or where
//     those are too uneven by a bitonic network.
//   * Where too many entries reach it (masses of equal ones, rows sorted by blocks) the bound is raised, once:
//     by bisection over all entries, and if it ends on a value that too many share, to the first of them.
// Short rows: one workgroup does all of that for a row.  Long ones: a first launch of small workgroups in the
// order of memory finds the groups' maxima and the statistics of the log-sum-exp, a second one does the rest.
// For many rows one launch is faster, as one row's bisection hides behind another's reading: 4096 x 65536
// bfloat16, k = 64, 116 us (537 MB at 4.6 TB/s; 676 MB leave the L2 caches, with the lines read again), in two
// launches 103 + 53.  Few long rows end with the second launch's latency: 16 x 131072 float16, k = 512, 5 + 19 us;
// 64 x 100003 bfloat16, k = 50, 9 + 11 us.
#include "rows.h"

namespace {

constexpr int kAhead = kNbhAhead;
constexpr int kSlots = 8;                // groups per lane that the one-launch kernel remembers
constexpr int kPieceVecs = 8;            // first launch of two: a wavefront takes 8 KiB at a time
constexpr int kMostGroups = 16384;       // groups per row of the two-launch path

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
    int tiles, pieces;                   // two launches: workgroups per row, pieces of 8 KiB for each
    uint32_t *maxima;                    // [row][tile][lane], as keys, 0 for an empty group
    nbh_softmax *part_stats;             // [row][tile]
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

// Appends what reaches `bound` of the entries at .. at + items, the 16 bytes `raw`.
template <typename E, int T, int CAP>
__device__ __forceinline__ void append(nbh_u32x4 raw, int64_t at, int64_t end, uint64_t bound, uint64_t *list,
                                       Shared<T> &sh)
{
    float f[E::items];
    E::unpack(raw, f);
    if (at >= end || at + E::items <= 0 || key_of(nbh_row_most(f)) < (uint32_t)(bound >> 32))
        return;
#pragma unroll
    for (int i = 0; i < E::items; ++i) {
        const uint64_t entry = entry_of(f[i], at + i);
        if (entry >= bound && at + i >= 0 && at + i < end) {
            const int place = atomicAdd(&sh.count, 1);
            if (place < CAP)
                list[place] = entry;
        }
    }
}

// Too many of the row's n entries reach the key `low`, none exceeds the key `high`: a bound that at least k
// and at most CAP entries reach.
template <typename E, int T, int CAP>
__device__ uint64_t raised_bound(const typename E::item *in, int64_t n, uint32_t low, uint32_t high, int k,
                                 Shared<T> &sh, int &turn)
{
    constexpr int kItems = E::items;
    auto sum = [&](int mine) {
        for (int step = 32; step; step >>= 1)
            mine += __shfl_xor(mine, step);
        return group_sum(mine, sh, turn);
    };
    auto count = [&](uint32_t key) {     // of all entries, those that reach it
        int mine = 0;
        for (int64_t at = (int64_t)threadIdx.x * kItems; at < n; at += T * kItems) {
            float f[kItems];
            nbh_row_load<E, false>(in, at, n, -INFINITY, f);
            for (int i = 0; i < kItems; ++i)
                mine += at + i < n && key_of(f[i]) >= key;
        }
        return sum(mine);
    };
    // The value: by bisection, unless `low` is the k-th largest already, as where all but a few entries
    // are masked.
    int above = low < high ? count(low + 1) : 0;             // entries that exceed `high` in what follows
    if (above >= k) {
        above = 0;
        while (low < high) {
            const uint32_t mid = high - (high - low) / 2;
            const int now = count(mid);
            if (now >= k && now <= CAP)
                return (uint64_t)mid << 32;
            if (now >= k) {
                low = mid;
            } else {
                high = mid - 1;
                above = now;
            }
        }
    }
    // `above` < k entries exceed `low` and too many equal it: those with the lowest indices, in the order of
    // memory.
    int need = k - above;
    for (int64_t first = 0; first < n; first += T * kItems) {
        const int64_t at = first + threadIdx.x * kItems;
        uint32_t equal = 0;              // bit i: entry at + i
        if (at < n) {
            float f[kItems];
            nbh_row_load<E, false>(in, at, n, -INFINITY, f);
            for (int i = 0; i < kItems; ++i)
                equal |= at + i < n && key_of(f[i]) == low ? 1u << i : 0u;
        }
        const int here = sum(__popc(equal));
        if (here < need) {
            need -= here;
            continue;
        }
        int from = 0, to = T * kItems - 1;                   // the entry that makes them enough
        while (from < to) {
            const int mid = from + (to - from) / 2, mine = mid - (int)threadIdx.x * kItems;
            const uint32_t upto = mine < 0 ? 0u : mine >= kItems ? ~0u : (2u << mine) - 1;
            if (sum(__popc(equal & upto)) >= need)
                to = mid;
            else
                from = mid + 1;
        }
        return (uint64_t)low << 32 | (uint32_t)~(uint32_t)(first + from);
    }
    return (uint64_t)low << 32;          // not reached: the row holds k entries
}

// Lists group g to be read again.
template <int T, int CAP> __device__ __forceinline__ void list_group(int g, int *again, Shared<T> &sh)
{
    const int at = atomicAdd(&sh.groups, 1);
    if (at < CAP)
        again[at] = g;
}

// Brings at least k and at most CAP entries that reach a bound into the list, sh.count of them: first those
// that reach `bound`; if they turn out to be too many, those that reach a raised one, which are not.
// `reaching(key)` lists the groups whose maxima reach the key; `place(g, v)`: first entry of vector v of
// group g.  Code that a workgroup runs once costs the fetching of its instructions: small loops, not
// unrolled ones.
template <typename E, int T, int CAP, typename Reaching, typename Place>
__device__ __forceinline__ void collect(const typename E::item *in, int64_t n, uint64_t bound, uint32_t top, int k,
                                        uint64_t *list, int *again, Shared<T> &sh, int &turn, int groups, int vectors,
                                        Reaching reaching, Place place)
{
#pragma unroll 1
    for (int attempt = 0; attempt < 2; ++attempt) {
        reaching((uint32_t)(bound >> 32));
        __syncthreads();
        const int listed = sh.groups;
        // With the raised bound many groups may share its value, but few of their entries its indices:
        // then all groups are gone through.
        const bool all = listed > CAP;
        if (!all || attempt) {
            const uint32_t vecs = (uint32_t)(all ? groups : listed) * vectors;
            // the next vector is on its way while the last is looked at
            uint32_t i = threadIdx.x;
            int64_t at = i < vecs ? place(all ? i / vectors : again[i / vectors], i % vectors) : n;
            nbh_u32x4 raw = nbh_row_load_raw<E, false>(in, at, n, E::lowest);
#pragma unroll 1
            for (; i < vecs; i += T) {
                const uint32_t next = i + T;
                const int64_t ahead =
                    next < vecs ? place(all ? next / vectors : again[next / vectors], next % vectors) : n;
                const nbh_u32x4 coming = nbh_row_load_raw<E, false>(in, ahead, n, E::lowest);
                append<E, T, CAP>(raw, at, n, bound, list, sh);
                raw = coming;
                at = ahead;
            }
        }
        __syncthreads();
        if (attempt || (!all && sh.count <= CAP))
            return;
        bound = raised_bound<E, T, CAP>(in, n, (uint32_t)(bound >> 32), top, k, sh, turn);
        __syncthreads();
        if (threadIdx.x == 0)
            sh.groups = sh.count = 0;
        __syncthreads();
    }
}

// Ranks the list's entries by counting them into 1024 buckets of equal width between the smallest and the
// largest key: put(rank, entry).  False, and nothing done, where a bucket is too crowded to be searched.
// Where the keys are of both signs, the widths are equal in the values: nearly all of the keys between lie about
// zero (512 of 1024, 4096 rows of bfloat16: 122 us by keys, 60 by values).  `counts` holds 1024 integers; the
// list's order changes.
constexpr int kBuckets = 1024, kCrowd = 64;
template <int T, int CAP, typename F>
__device__ bool rank_by_buckets(uint64_t *list, int have, int *counts, Shared<T> &sh, F put)
{
    constexpr int kEach = CAP / T, kOf = kBuckets / T;
    uint64_t mine[kEach];
    uint32_t low = ~0u, high = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int at = i * T + threadIdx.x;
        mine[i] = at < have ? list[at] : 0;
        const uint32_t key = (uint32_t)(mine[i] >> 32);
        if (at < have) {
            low = key < low ? key : low;
            high = key > high ? key : high;
        }
    }
    for (int step = 32; step; step >>= 1) {
        const uint32_t l = __shfl_xor(low, step), h = __shfl_xor(high, step);
        low = l < low ? l : low;
        high = h > high ? h : high;
    }
    if ((threadIdx.x & 63) == 0) {
        sh.ends[0][threadIdx.x >> 6] = high;
        sh.ends[1][threadIdx.x >> 6] = low;
    }
    for (int i = threadIdx.x; i < kBuckets; i += T)
        counts[i] = 0;
    __syncthreads();
    for (int w = 0; w < T / 64; ++w) {
        high = sh.ends[0][w] > high ? sh.ends[0][w] : high;
        low = sh.ends[1][w] < low ? sh.ends[1][w] : low;
    }
    const int bits = 32 - __clz((int)(high - low)), shift = bits > 10 ? bits - 10 : 0;
    const float least = fmaxf(value_of((uint64_t)low << 32), -1e38f);
    const float most = fminf(value_of((uint64_t)high << 32), 1e38f);      // NaN: 1e38
    const bool linear = low < 0x80000000u && high > 0x80000000u && most - least > 1e-30f;
    const float steep = linear ? kBuckets / (most - least) : 0.0f;
    auto bucket_of = [&](uint64_t entry) {                   // rises with the entry
        if (!linear)
            return (int)(((uint32_t)(entry >> 32) - low) >> shift);
        const float value = fmaxf(fminf(value_of(entry), most), least);
        const int bucket = (int)((value - least) * steep);
        return bucket < kBuckets ? bucket : kBuckets - 1;
    };
    int bucket[kEach], place[kEach];     // of an entry, and its place within the bucket
    bool crowded = false;
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        if (mine[i]) {
            bucket[i] = bucket_of(mine[i]);
            place[i] = atomicAdd(&counts[bucket[i]], 1);
            crowded |= place[i] >= kCrowd;
        }
    if (__syncthreads_or(crowded))
        return false;
    // a bucket's count becomes the number of entries in the buckets above it; lane t has the buckets
    // kBuckets - 1 - t kOf downwards
    int own[kOf], sum = 0;
#pragma unroll
    for (int i = 0; i < kOf; ++i) {
        own[i] = counts[kBuckets - 1 - (threadIdx.x * kOf + i)];
        sum += own[i];
    }
    int upto = sum;
    for (int step = 1; step < 64; step *= 2) {
        const int other = __shfl_up(upto, step);
        if ((int)(threadIdx.x & 63) >= step)
            upto += other;
    }
    if ((threadIdx.x & 63) == 63)
        sh.tally[0][threadIdx.x >> 6] = upto;
    __syncthreads();
    int above = upto - sum;
    for (int w = 0; w < (int)threadIdx.x >> 6; ++w)
        above += sh.tally[0][w];
#pragma unroll
    for (int i = 0; i < kOf; ++i) {
        counts[kBuckets - 1 - (threadIdx.x * kOf + i)] = above;
        above += own[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        if (mine[i])
            list[counts[bucket[i]] + place[i]] = mine[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEach; ++i)
        if (mine[i]) {
            const int first = counts[bucket[i]], end = bucket[i] ? counts[bucket[i] - 1] : have;
            int rank = first;
            for (int at = first; at < end; ++at)
                rank += list[at] > mine[i];
            put(rank, mine[i]);
        }
    return true;
}

// Writes the k best of the list (at least k entries) in order.  The list has been written before a
// barrier and has room for two entries more; `counts` holds CAP integers, at least 1024 of them if CAP exceeds 256.
template <typename E, int T, int CAP>
__device__ void write_ranked(const Top &a, int64_t row, uint64_t *list, int have, int *counts, Shared<T> &sh)
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
    auto put_best = [&](int rank, uint64_t entry) {
        if (rank < a.k)
            put(rank, entry);
    };
    if (CAP <= 256 || have <= 256) {
        // a lane per entry counts what exceeds it: have / 2 reads of LDS, the same address in all lanes
        if (threadIdx.x == 0)
            list[have] = 0;
        __syncthreads();
        for (int at = threadIdx.x; at < have; at += T) {
            const uint64_t mine = list[at];
            int rank = 0;
            for (int i = 0; i < have; i += 2) {
                const ulonglong2 two = *reinterpret_cast<const ulonglong2 *>(list + i);
                rank += (two.x > mine) + (two.y > mine);
            }
            put_best(rank, mine);
        }
        return;
    }
    if (rank_by_buckets<T, CAP>(list, have, counts, sh, put_best))
        return;
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
    nbh_row_stream<E, T, false>(in, 0, n, [&](int64_t at, const nbh_u32x4(&raw)[kAhead])
                                __attribute__((always_inline)) {
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
    const uint64_t bound = (uint64_t)key << 32;
    const int64_t group = (int64_t)kChunk << shift;
    const int groups = (int)((n + group - 1) / group) * T, vectors = kAhead << shift;       // of a group
    collect<E, T, CAP>(
        in, n, bound, top, a.k, list, again, sh, turn, groups, vectors,
        [&](uint32_t key) {
            for (int g = threadIdx.x; g < groups; g += T)
                if (maxima[g] >= key)
                    list_group<T, CAP>(g, again, sh);
        },
        [&](int g, int v) { return (g / T) * group + (v * T + g % T) * (int64_t)kItems; });
    if (LSE) {
        stats = nbh_softmax_group<T>(stats, a.scale, sh.stats);
        if (threadIdx.x == 0)
            a.lse[row] = nbh_softmax_lse(stats, a.temperature, a.scale);
    }
    write_ranked<E, T, CAP>(a, row, list, sh.count < CAP ? sh.count : CAP, again, sh);
}

// The largest of each eight lanes, in all eight.
__device__ __forceinline__ uint32_t most_of_eight(uint32_t key)
{
    uint32_t other = __builtin_amdgcn_mov_dpp(key, 0xb1, 0xf, 0xf, true);        // quad_perm 1, 0, 3, 2
    key = other > key ? other : key;
    other = __builtin_amdgcn_mov_dpp(key, 0x4e, 0xf, 0xf, true);                 // quad_perm 2, 3, 0, 1
    key = other > key ? other : key;
    other = __builtin_amdgcn_mov_dpp(key, 0x141, 0xf, 0xf, true);                // the half row mirrored
    return other > key ? other : key;
}

// First launch of two, a wavefront per workgroup: a group is the 128 bytes that eight lanes read together
// (of each of the workgroup's pieces), so that reading it again is reading a cache line.  Lane 8 i + j
// keeps the maximum of the lanes 8 i .. 8 i + 7 in vector j.
template <typename E, bool LSE> __global__ __launch_bounds__(64) void top_maxima(Top a)
{
    constexpr int kItems = E::items, kPiece = 64 * kPieceVecs * kItems;
    const int64_t at = blockIdx.x / a.tiles, row = a.row0 + at;
    const int tile = blockIdx.x % a.tiles, lane = threadIdx.x;
    const typename E::item *in = reinterpret_cast<const typename E::item *>(a.in + row * a.stride);
    int64_t first = (int64_t)tile * a.pieces * kPiece - nbh_row_before<E>(in);
    nbh_softmax stats = nbh_softmax_empty();
    uint32_t mine = 0;
    for (int piece = 0; piece < a.pieces && first < a.vocab; ++piece, first += kPiece) {
        nbh_u32x4 raw[kPieceVecs];
        const bool full = first >= 0 && first + kPiece <= a.vocab;
        if (full) {
#pragma unroll
            for (int j = 0; j < kPieceVecs; ++j)
                raw[j] = E::template load<true>(in + first + (j * 64 + lane) * kItems);
        } else {
#pragma unroll
            for (int j = 0; j < kPieceVecs; ++j)
                raw[j] = nbh_row_load_raw<E, true>(in, first + (j * 64 + lane) * kItems, a.vocab, E::lowest);
        }
#pragma unroll
        for (int j = 0; j < kPieceVecs; ++j) {
            float f[kItems];
            E::unpack(raw[j], f);
            const float most = nbh_row_most(f);
            const int64_t v = first + (j * 64 + lane) * kItems;
            uint32_t key = key_of(most);
            if (!full && (v >= a.vocab || v + kItems <= 0))
                key = 0;
            key = most_of_eight(key);
            if ((lane & 7) == j)
                mine = key > mine ? key : mine;
            if (LSE)
                nbh_softmax_add(stats, f, most, a.scale);
        }
    }
    a.maxima[blockIdx.x * (int64_t)64 + lane] = mine;
    if (LSE) {
        stats = nbh_softmax_wave(stats, a.scale);
        if (lane == 0)
            a.part_stats[blockIdx.x] = stats;
    }
}

// Second launch: a workgroup per row, up to P groups per lane.
template <typename E, bool LSE, int T, int P, int CAP> __global__ __launch_bounds__(T) void top_finish(Top a)
{
    typedef typename E::item item;
    constexpr int kItems = E::items, kPiece = 64 * kPieceVecs * kItems;
    __shared__ __align__(16) uint64_t list[CAP + 2];
    __shared__ int again[CAP];
    __shared__ Shared<T> sh;
    const int64_t row = a.row0 + blockIdx.x;
    const item *in = reinterpret_cast<const item *>(a.in + row * a.stride);
    const int before = nbh_row_before<E>(in);
    const int groups = a.tiles * 64;
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
        nbh_softmax stats = nbh_softmax_empty();
        for (int s = threadIdx.x; s < a.tiles; s += 64)
            stats = nbh_softmax_join(stats, a.part_stats[blockIdx.x * (int64_t)a.tiles + s], a.scale);
        stats = nbh_softmax_wave(stats, a.scale);
        if (threadIdx.x == 0)
            a.lse[row] = nbh_softmax_lse(stats, a.temperature, a.scale);
    }
    const uint64_t bound = (uint64_t)bound_of<T>(peaks, a.k, sh, turn, top) << 32;
    collect<E, T, CAP>(
        in, a.vocab, bound, top, a.k, list, again, sh, turn, groups, 8 * a.pieces,
        [&](uint32_t key) {
#pragma unroll
            for (int g = 0; g < P; ++g)
                if (peaks[g] && peaks[g] >= key)
                    list_group<T, CAP>(g * T + threadIdx.x, again, sh);
        },
        [&](int g, int v) {
            const int64_t piece = (int64_t)(g / 64) * a.pieces + v / 8;
            const int lane = g % 64 / 8 * 8 + v % 8, j = g % 8;
            return piece * kPiece - before + (j * 64 + lane) * kItems;
        });
    write_ranked<E, T, CAP>(a, row, list, sh.count < CAP ? sh.count : CAP, again, sh);
}

// Workgroups of the first launch per row and their pieces; 0 tiles: one launch.  `spare`: entries before a
// row's beginning that its first vector may hold.
// Two launches where a few workgroups would read long rows for themselves.  Measured, k = 50, one against
// two: rows of 256 KiB, 1 row 17 and 16 us, 64 rows 19 and 18, 200 rows 20 and 23; rows of 512 KiB, 1 row 26
// and 16, 64 rows 28 and 21, 200 rows 32 and 31; rows of 128 KiB, 1 row 13 and 16.
struct Spread {
    int tiles, pieces;
};
Spread spread_of(int64_t rows, int64_t vocab, int dtype, int spare)
{
    const int64_t piece = 64 * kPieceVecs * (dtype == NBH_ROW_F32 ? 4 : 8);
    // (the number of pieces per workgroup does not depend on `spare`: a workspace for the largest serves all)
    const int64_t all = (vocab + spare + piece - 1) / piece, most = (vocab + 7 + piece - 1) / piece;
    if (rows >= 128 || vocab <= 20 * piece)
        return {0, 0};
    const int64_t pieces = (most + kMostGroups / 64 - 1) / (kMostGroups / 64);
    return {(int)((all + pieces - 1) / pieces), (int)pieces};
}

// Lanes of the one-launch kernel.  A lane's four vectors give as many maxima for the bound, so T lanes serve well
// up to k = T; larger workgroups wait longer at their barriers and fewer rows are under way at a time.  A call of
// one row finishes sooner with more lanes.  Measured, bfloat16:
//   k <= 64, rows of up to 16 KiB, 64 and 256 lanes: k = 50, 4096 x 1024 21 and 42 us, 4096 x 8192 28 and 35, 2048 x
//   8192 21 and 22, 1500 x 8192 19 and 17, 64 x 8192 16 and 11; rows of 32 KiB, 4096 of them 44 and 45, of 64 KiB
//   80 and 65.
//   k <= 256, 256 and 512 lanes: k = 64, 4096 x 65536 124 and 140; k = 200, 4096 x 1024 118 and 214.
//   k = 500, 256 and 512 lanes: 512 x 8192 21 and 25, 4096 x 8192 66 and 168; 512 x 32768 34 and 29, 1024 x 32768
//   44 and 50, 4096 x 32768 118 and 180, 1024 x 50021 57 and 66, 512 x 131072 66 and 51 (k = 300: 2048 x 131072
//   159 and 143).
//   k = 1000: 4096 x 1024 117 and 214, 4096 x 8192 222 and 391, 4096 x 32768 799 and 265 (k = 700: 395 and 214).
//   k > 512, few short rows: 45 x 1822, k = 981, 40 and 19, 512 x 8192, k = 700, 38 and 29, 900 x 8192, k = 600,
//   41 and 48, 900 x 4096, k = 1000, 60 and 64.
int lanes_of(int64_t rows, int64_t vocab, int64_t bytes, int k)
{
    const bool brief = vocab * bytes <= (16 << 10);
    if (brief && k <= 64 && rows >= 2048)
        return 64;
    if (k <= 256 || (brief && (k <= 512 || rows > 512)) ||
        (k <= 512 && rows >= 1024 && vocab * bytes <= (128 << 10)))
        return 256;
    return 512;
}

template <typename E, bool LSE> int launch_top(Top a, int64_t rows, hipStream_t stream)
{
    const int lanes = lanes_of(rows, a.vocab, sizeof(typename E::item), a.k);
    const int64_t most = NBH_ROW_MOST_GROUPS / (a.tiles ? a.tiles : 1);
    for (a.row0 = 0; a.row0 < rows; a.row0 += most) {
        const int64_t now = rows - a.row0 < most ? rows - a.row0 : most;
        const dim3 grid((unsigned)now);
        if (a.tiles == 0) {
            if (lanes == 64)
                top_rows<E, LSE, 64, 256><<<grid, dim3(64), 0, stream>>>(a);
            else if (lanes == 256)
                top_rows<E, LSE, 256, 1024><<<grid, dim3(256), 0, stream>>>(a);
            else
                top_rows<E, LSE, 512, 4096><<<grid, dim3(512), 0, stream>>>(a);
        } else {
            top_maxima<E, LSE><<<dim3((unsigned)(now * a.tiles)), dim3(64), 0, stream>>>(a);
            if (a.tiles * 64 > 4096)
                top_finish<E, LSE, 512, kMostGroups / 512, 4096><<<grid, dim3(512), 0, stream>>>(a);
            else if (a.k > 128)
                top_finish<E, LSE, 1024, 4, 4096><<<grid, dim3(1024), 0, stream>>>(a);
            else
                top_finish<E, LSE, 512, 8, 1024><<<grid, dim3(512), 0, stream>>>(a);
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
    const Spread s = spread_of(rows, vocab, dtype, 7);
    return (size_t)rows * s.tiles * (64 * sizeof(uint32_t) + sizeof(nbh_softmax));
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
    const Spread spread = spread_of(rows, vocab, dtype, nbh_row_spare(logits, stride, dtype));
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
    a.tiles = spread.tiles;
    a.pieces = spread.pieces;
    a.maxima = (uint32_t *)workspace;
    a.part_stats = (nbh_softmax *)(a.maxima + (size_t)rows * spread.tiles * 64);

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
