// nbh_rows_distill: distillation from a teacher's top logits, forward, backward or both at once.
//
//   lse = log sum exp(s / T);  p_j from the teacher's k entries;  P = sum p_j
//   loss = sum p_j (log p_j - (s[i_j] / T - lse))
//   grad[v] = grad_loss / T * (P exp(s[v] / T - lse) - sum over i_j = v of p_j)
//
// One workgroup per row: its first wavefront brings the teacher's entries to LDS while the others begin
// the pass over the row that gives its maximum and sum together; a second pass, backwards, so that it finds
// the end of the first in the caches, writes the gradient as a * 2^((s - m) * c) for every entry, and behind
// a barrier the few entries the teacher names are written again with their p_j taken off.  The loss
// alone, and few rows, are spread: small workgroups in the order of memory for the statistics, then a launch
// that joins them and does the rest.  A large gradient by itself is a copy with arithmetic: a launch prepares two
// numbers for each row, small workgroups in memory order do the copy, a last launch writes the named entries.
//
// Bound by memory: the loss reads a row once (2048 x 50021 float16: 36 + 6 us, 205 MB at 5.8 TB/s in the first
// launch), the gradient reads and writes it (1024 x 100003 float32: 10 + 139 + 5 us, 819 MB at 5.9 TB/s in the
// second).  Both at once read it once and the part that was not kept again (4096 x 131072 bfloat16: 414 us; 1.33 GB
// read and 1.08 GB written leave or enter the L2 caches, 5.8 TB/s); beside the traffic there are two exponentials
// per entry, some 0.28 ms of the vector units' time.
#include "rows.h"

namespace {

constexpr int kStatsThreads = 64, kStatsVecs = 8;      // 8 KiB per workgroup
constexpr float kLog2e = 1.44269502f, kLog2eRest = 1.92596299e-8f;       // log2(e) and its rounding
constexpr float kLn2 = 0.693147180559945309f;

// exp(s / T - lse) P grad_loss / T = whole * nbh_softmax_term(s, peak, scale, shift) for a row; 0 where `zero`.
struct Plan {
    float peak, whole, shift;
    int zero;
};
// An entry of the gradient that the teacher names: its index (-1: none) and value.
struct Named {
    int32_t index;
    float value;
};

struct Distill {
    const char *student;
    int64_t stride, vocab, slice, row0;
    int splits, k, index_bytes, values_dtype;
    const char *values, *indices;
    int64_t values_stride, indices_stride;
    const float *teacher_lse, *grad_loss;
    int64_t grad_loss_stride;
    float grad_loss_value;
    float temperature, scale, scale_rest;    // log2(e) / temperature, and what its rounding took off
    float *loss, *lse;
    char *grad;
    int64_t grad_stride;
    nbh_softmax *parts;                  // per row and stretch
    float *targets;                      // per row: the student's values at the teacher's k indices
    Plan *plans;                         // per row
    Named *named;                        // per row and teacher's entry
    int tiles;                           // workgroups per row of distill_stats or distill_flat
};

// The statistics of 8 KiB of a row per workgroup, in the order of memory, one pair of numbers per wavefront.
// 2048 x 50021 float16: 35.8 us; 4 KiB per wavefront 39.4, 16 KiB 40.7, two wavefronts 39.6, four 45.
template <typename E>
__global__ __launch_bounds__(kStatsThreads) void distill_stats(Distill a)
{
    constexpr int T = kStatsThreads, kItems = E::items;
    const int64_t at = blockIdx.x / a.tiles, row = a.row0 + at;
    const int tile = blockIdx.x % a.tiles;
    const typename E::item *in = reinterpret_cast<const typename E::item *>(a.student + row * a.stride);
    const int64_t first = (int64_t)tile * T * kStatsVecs * kItems - nbh_row_before<E>(in);
    nbh_u32x4 raw[kStatsVecs];
    if (first >= 0 && first + T * kStatsVecs * kItems <= a.vocab) {
#pragma unroll
        for (int j = 0; j < kStatsVecs; ++j)
            raw[j] = E::template load<true>(in + first + (j * T + threadIdx.x) * kItems);
    } else {
#pragma unroll
        for (int j = 0; j < kStatsVecs; ++j)
            raw[j] = nbh_row_load_raw<E, true>(in, first + (j * T + (int)threadIdx.x) * kItems, a.vocab, E::lowest);
    }
    nbh_softmax stats = nbh_softmax_empty();
    nbh_row_stats<E>(stats, raw, a.scale);
    stats = nbh_softmax_wave(stats, a.scale);
    if ((threadIdx.x & 63) == 0)
        a.parts[(at * a.tiles + tile) * (T / 64) + threadIdx.x / 64] = stats;
    // The loss needs these of the whole row, and the gradient may be written over the row while another
    // stretch's workgroup still works on the loss: they are set aside.
    if (a.targets && tile == 0)
        for (int j = threadIdx.x; j < a.k; j += T) {
            const int64_t index = nbh_row_int(a.indices + row * a.indices_stride, a.index_bytes, j);
            a.targets[at * a.k + j] = index >= 0 && index < a.vocab ? E::get(in[index]) : 0.0f;
        }
}
// What they add up to; every wavefront for itself.
__device__ __forceinline__ nbh_softmax joined_stats(const Distill &a, int64_t at)
{
    const int parts = a.tiles * (kStatsThreads / 64);
    nbh_softmax stats = nbh_softmax_empty();
    for (int i = threadIdx.x & 63; i < parts; i += 64)
        stats = nbh_softmax_join(stats, a.parts[at * parts + i], a.scale);
    return nbh_softmax_wave(stats, a.scale);
}

__device__ __forceinline__ float wave_add(float x)
{
    for (int step = 32; step; step >>= 1)
        x += __shfl_xor(x, step);
    return x;
}
__device__ __forceinline__ float wave_max(float x)
{
    for (int step = 32; step; step >>= 1)
        x = fmaxf(x, __shfl_xor(x, step));
    return x;
}

__device__ __forceinline__ float teacher_value(const Distill &a, int64_t row, int j)
{
    const char *p = a.values + row * a.values_stride;
    switch (a.values_dtype) {
    case NBH_ROW_F32:
        return reinterpret_cast<const float *>(p)[j];
    case NBH_ROW_F16:
        return (float)reinterpret_cast<const _Float16 *>(p)[j];
    default:
        return nbh_row_bf16::get(reinterpret_cast<const uint16_t *>(p)[j]);
    }
}

// What a launch does; kParts: the statistics come from distill_stats.
constexpr int kLoss = 1, kGrad = 2, kParts = 4;

// The teacher's entries of a row in LDS: index (-1: absent), p, log p, and the student's value there.
struct Teacher {
    int32_t *index;
    float *p, *log_p, *student;
    int32_t *table;                      // at least 2 k slots, for the search for repeated indices
    float mass;
    int some, repeated;

    static __host__ __device__ int slots(int k)
    {
        int n = 2;
        while (n < 2 * k)
            n *= 2;
        return n;
    }
    static size_t bytes(int k) { return (size_t)k * 16 + (size_t)slots(k) * 4; }
    __device__ void place(char *lds, int k)
    {
        index = reinterpret_cast<int32_t *>(lds);
        p = reinterpret_cast<float *>(index + k);
        log_p = p + k;
        student = log_p + k;
        table = reinterpret_cast<int32_t *>(student + k);
    }
};

// One wavefront's work: no barriers, its LDS accesses are in order.  `begin` .. `end`: the part of the row
// whose values are wanted (elsewhere another workgroup may be writing the gradient over them already).
template <typename E, int WHAT>
__device__ __forceinline__ void load_teacher(const Distill &a, int64_t row, int64_t begin, int64_t end, Teacher &t)
{
    const typename E::item *in = reinterpret_cast<const typename E::item *>(a.student + row * a.stride);
    const int lane = threadIdx.x & 63;
    const int slots = Teacher::slots(a.k);
    if (WHAT & kGrad)
        for (int i = lane; i < slots; i += 64)
            t.table[i] = -1;
    float peak = -FLT_MAX;
    int some = 0;
    for (int j = lane; j < a.k; j += 64) {
        const int64_t at = nbh_row_int(a.indices + row * a.indices_stride, a.index_bytes, j);
        const float value = teacher_value(a, row, j);
        const bool present = at >= 0 && at < a.vocab && value != -INFINITY;
        t.index[j] = present ? (int32_t)at : -1;
        t.log_p[j] = value;
        if (present) {
            t.student[j] = (WHAT & (kParts | kGrad)) == (kParts | kGrad) ? a.targets[(row - a.row0) * a.k + j]
                           : at >= begin && at < end                     ? E::get(in[at])
                                                                         : 0.0f;
            peak = fmaxf(peak, fminf(value, FLT_MAX));
            some = 1;
        }
    }
    // p = exp(value / T - norm), or relative to the peak and then divided by the sum
    const float norm = a.teacher_lse ? a.teacher_lse[row] : 0.0f;
    if (!a.teacher_lse)
        peak = wave_max(peak);
    float sum = 0.0f;
    for (int j = lane; j < a.k; j += 64) {
        const float z = a.teacher_lse ? t.log_p[j] / a.temperature - norm : (t.log_p[j] - peak) / a.temperature;
        t.log_p[j] = z;
        t.p[j] = t.index[j] >= 0 ? expf(z) : 0.0f;
        sum += t.p[j];
    }
    sum = wave_add(sum);
    t.mass = sum;
    if (!a.teacher_lse) {
        const float log_sum = logf(sum);
        float mass = 0.0f;
        for (int j = lane; j < a.k; j += 64) {
            t.log_p[j] -= log_sum;
            t.p[j] = t.index[j] >= 0 ? t.p[j] / sum : 0.0f;
            mass += t.p[j];
        }
        t.mass = wave_add(mass);
    }
    t.some = __any(some);
    int repeated = 0;
    if (WHAT & kGrad)
        for (int j = lane; j < a.k; j += 64)
            if (t.index[j] >= 0) {
                uint32_t slot = (uint32_t)t.index[j] * 2654435761u;
                for (int tries = 0; tries < slots; ++tries, ++slot) {
                    const int32_t was = atomicCAS(&t.table[slot & (slots - 1)], -1, t.index[j]);
                    repeated |= was == t.index[j];
                    if (was == -1 || was == t.index[j])
                        break;
                }
            }
    t.repeated = __any(repeated);
}

// The student's side of a row: q(v) = base * nbh_softmax_term(s, peak, scale, shift).
struct Student {
    float peak, base, log_sum;           // log_sum: log2 of the sum relative to the peak
    float shift;
};
__device__ __forceinline__ Student student_of(nbh_softmax stats)
{
    return {stats.peak == -INFINITY ? 0.0f : stats.peak, stats.sum == 0.0f ? 0.0f : 1.0f / stats.sum, log2f(stats.sum),
            0.0f};
}
__device__ __forceinline__ Student student_of_lse(const Distill &a, float lse)
{
    // T * lse rounded to float32 takes the place of the peak; what the roundings of it, of its product
    // with the scale, and of the scale itself take off goes into the factor.  Where the product is not near, the
    // first of them may be hundreds of powers of two, which only together with the difference s - peak make an
    // ordinary exponent.
    const float peak = lse * a.temperature, product = peak * a.scale;
    if (lse == -INFINITY)
        return {0.0f, 0.0f, 0.0f, 0.0f};
    if (nbh_softmax_near(product)) {
        const float high = lse * kLog2e, low = fmaf(lse, kLog2e, -high) + lse * kLog2eRest;
        return {peak, exp2f((product - high) - low + peak * a.scale_rest), 0.0f, 0.0f};
    }
    const float rest = __builtin_isfinite(peak) ? fmaf(lse, a.temperature, -peak) : 0.0f;
    // the same for the whole row: in a scalar register
    return {peak, 1.0f, 0.0f, __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(rest * a.scale)))};
}

// One wavefront's work.  (Called, not inlined, it would leave the arguments in scratch memory.)
__device__ __forceinline__ float loss_of(const Distill &a, const Teacher &t, Student s)
{
    const float product = s.peak * a.scale;
    float loss = 0.0f;
    for (int j = threadIdx.x & 63; j < a.k; j += 64)
        if (t.index[j] >= 0 && t.p[j] != 0.0f) {
            const float x = t.student[j];
            float log_q = x;
            if (x != -INFINITY)
                log_q = nbh_softmax_near(product) && fabsf(x) < 1e30f
                            ? (fmaf(x, a.scale, -product) - s.log_sum) * kLn2
                            : (x - s.peak) / a.temperature - s.log_sum * kLn2;
            loss += t.p[j] * (t.log_p[j] - log_q);
        }
    loss = wave_add(loss);
    return t.some ? loss : 0.0f;
}

__device__ __forceinline__ float factor_of(const Distill &a, int64_t row)
{
    const float grad_loss =
        a.grad_loss ? *reinterpret_cast<const float *>((const char *)a.grad_loss + row * a.grad_loss_stride)
                    : a.grad_loss_value;
    return grad_loss / a.temperature;
}

// The gradient at the teacher's entry j; index -1 if there is none, or an earlier entry of the same index
// answers for it.
__device__ __forceinline__ Named named_of(const Distill &a, const Teacher &t, int j, Student s, float whole,
                                          float factor)
{
    const int32_t index = t.index[j];
    if (index < 0)
        return {-1, 0.0f};
    float own = t.p[j];
    if (t.repeated) {                    // the first of them takes all their shares, in order
        for (int i = 0; i < j; ++i)
            if (t.index[i] == index)
                return {-1, 0.0f};
        for (int i = j + 1; i < a.k; ++i)
            if (t.index[i] == index)
                own += t.p[i];
    }
    return {index, whole * nbh_softmax_term(t.student[j], s.peak, a.scale, s.shift) - factor * own};
}

// With 512 lanes the loss and the gradient together keep the beginning of the row, 96 KiB of it in registers and
// 64 KiB in LDS, so that only what lies behind is read again, from the caches.  Two such workgroups fill a compute
// unit.  4096 x 131072 bfloat16: nothing kept 460 us (2.07 GB of reads leave the L2 caches instead of 1.07), 32 KiB
// in LDS 446, 64 KiB 442, and in registers 32 KiB 435, 64 KiB 430, 96 KiB 423; one workgroup per compute unit with
// 128 KiB in LDS 473.
template <int T, int WHAT> struct Kept {
    static constexpr bool some = T == 512 && WHAT == (kLoss | kGrad);
    static constexpr int held = some ? 3 : 0, stored = some ? 2 : 0, waves = some ? 4 : 1;
};
template <typename E, int T, int WHAT>
__global__ __launch_bounds__(T, (Kept<T, WHAT>::waves)) void distill_rows(Distill a)
{
    typedef typename E::item item;
    typedef Kept<T, WHAT> Keep;
    constexpr int kItems = E::items;
    constexpr int64_t kChunk = kNbhAhead * T * kItems;
    extern __shared__ char lds[];
    __shared__ nbh_softmax room[T / 64];
    __shared__ float mass;
    __shared__ int some, repeated;
    __shared__ nbh_u32x4 store[Keep::some ? Keep::stored * kNbhAhead * T : 1];
    nbh_u32x4 hold[Keep::some ? Keep::held * kNbhAhead : 1];
    Teacher teacher;
    teacher.place(lds, a.k);

    // the loss alone takes one workgroup per row, whatever the statistics took
    constexpr bool kWhole = WHAT == (kLoss | kParts);
    const int64_t row = a.row0 + (kWhole ? blockIdx.x : blockIdx.x / a.splits);
    const int split = kWhole ? 0 : blockIdx.x % a.splits;
    const item *in = reinterpret_cast<const item *>(a.student + row * a.stride);
    const int64_t begin = split * a.slice, end = a.vocab < begin + a.slice ? a.vocab : begin + a.slice;
    // entries 0 .. held are in `hold`, held .. kept in `store`
    const int64_t held = a.vocab >= Keep::held * kChunk ? Keep::held * kChunk : 0;
    const int64_t chunks = (a.vocab - held) / kChunk;
    const int64_t kept = held + (chunks < Keep::stored ? chunks : Keep::stored) * kChunk;

    if (threadIdx.x < 64) {
        load_teacher<E, WHAT>(a, row, WHAT & kLoss ? 0 : begin, WHAT & kLoss ? a.vocab : end, teacher);
        if (threadIdx.x == 0) {
            mass = teacher.mass;
            some = teacher.some;
            repeated = teacher.repeated;
        }
    }
    Student student;
    if (WHAT & kLoss) {
        nbh_softmax stats;
        if (WHAT & kParts) {
            stats = joined_stats(a, row - a.row0);
            __syncthreads();
        } else {
            stats = nbh_softmax_empty();
            if (Keep::some && held) {
#pragma unroll
                for (int j = 0; j < Keep::held * kNbhAhead; ++j)
                    hold[j] = E::template load<false>(in + (j * T + threadIdx.x) * kItems);
                // (not through a reference to `hold`: that leaves it in scratch memory)
#pragma unroll
                for (int j = 0; j < Keep::held * kNbhAhead; ++j) {
                    float f[kItems];
                    E::unpack(hold[j], f);
                    nbh_softmax_add(stats, f, nbh_row_most(f), a.scale);
                }
            }
            nbh_row_stream<E, T, false>(
                in, held, a.vocab, [&](int64_t at, const nbh_u32x4(&raw)[kNbhAhead]) __attribute__((always_inline)) {
                    if (at < kept) {
#pragma unroll
                        for (int j = 0; j < kNbhAhead; ++j)
                            store[((at - held) / kChunk * kNbhAhead + j) * T + threadIdx.x] = raw[j];
                    }
                    nbh_row_stats<E>(stats, raw, a.scale);
                });
            stats = nbh_softmax_group<T>(stats, a.scale, room);
        }
        student = student_of(stats);
        if (a.lse && split == 0 && threadIdx.x == 0)
            a.lse[row] = nbh_softmax_lse(stats, a.temperature, a.scale);
        if (split == 0 && threadIdx.x < 64) {
            const float loss = loss_of(a, teacher, student);
            if (threadIdx.x == 0)
                a.loss[row] = loss;
        }
    } else {
        student = student_of_lse(a, a.lse[row]);
        __syncthreads();
    }
    if (!(WHAT & kGrad))
        return;

    item *out = reinterpret_cast<item *>(a.grad + row * a.grad_stride);
    const float factor = factor_of(a, row);
    if (!some || factor == 0.0f) {
        float zero[kItems] = {};
        for (int64_t at = begin + threadIdx.x * kItems; at < end; at += T * kItems)
            nbh_row_store<E, true>(out, at, end, zero);
        return;
    }
    const float whole = factor * mass * student.base, product = student.peak * a.scale;
    const bool near = nbh_softmax_near(product);
    auto write = [&](int64_t at, const nbh_u32x4(&raw)[kNbhAhead]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kNbhAhead; ++j) {
            float f[kItems];
            E::unpack(raw[j], f);
            if (near) {
#pragma unroll
                for (int i = 0; i < kItems; ++i)
                    f[i] = whole * nbh_exp2(fmaf(f[i], a.scale, -product));
            } else {
                for (int i = 0; i < kItems; ++i)
                    f[i] = whole * nbh_exp2((f[i] - student.peak) * a.scale - student.shift);
            }
            nbh_row_store<E, true>(out, at + (j * T + threadIdx.x) * kItems, end, f);
        }
    };
    nbh_row_stream<E, T, true, true>(in, begin + kept, end, write);
    if (Keep::some) {
        for (int64_t at = kept; at > held;) {
            at -= kChunk;
            nbh_u32x4 raw[kNbhAhead];
#pragma unroll
            for (int j = 0; j < kNbhAhead; ++j)
                raw[j] = store[((at - held) / kChunk * kNbhAhead + j) * T + threadIdx.x];
            write(at, raw);
        }
        if (held) {
#pragma unroll
            for (int chunk = 0; chunk < Keep::held; ++chunk) {
                nbh_u32x4 raw[kNbhAhead];
#pragma unroll
                for (int j = 0; j < kNbhAhead; ++j)
                    raw[j] = hold[chunk * kNbhAhead + j];
                write(chunk * kChunk, raw);
            }
        }
    }
    __syncthreads();
    teacher.repeated = repeated;
    for (int j = threadIdx.x; j < a.k; j += T)
        if (teacher.index[j] >= begin && teacher.index[j] < end) {
            const Named n = named_of(a, teacher, j, student, whole, factor);
            if (n.index >= 0)
                out[n.index] = E::put(n.value);
        }
}

// The gradient in three launches.  First: a wavefront per row.
template <typename E> __global__ __launch_bounds__(64) void distill_plan(Distill a)
{
    extern __shared__ char lds[];
    const int64_t row = a.row0 + blockIdx.x;
    Teacher teacher;
    teacher.place(lds, a.k);
    load_teacher<E, kGrad>(a, row, 0, a.vocab, teacher);
    const Student student = student_of_lse(a, a.lse[row]);
    const float factor = factor_of(a, row);
    const bool zero = !teacher.some || factor == 0.0f;
    const float whole = factor * teacher.mass * student.base;
    if (threadIdx.x == 0)
        a.plans[row - a.row0] = {student.peak, whole, student.shift, zero};
    for (int j = threadIdx.x; j < a.k; j += 64)
        a.named[(row - a.row0) * a.k + j] = zero ? Named{-1, 0.0f} : named_of(a, teacher, j, student, whole, factor);
}
// Second: small workgroups in the order of memory, a vector per lane (1024 x 100003 float32: 139 us; with two
// vectors 161, with four 149, four wavefronts 140).
constexpr int kFlatThreads = 64, kFlatVecs = 1;
template <typename E> __global__ __launch_bounds__(kFlatThreads) void distill_flat(Distill a)
{
    typedef typename E::item item;
    constexpr int kItems = E::items, T = kFlatThreads, V = kFlatVecs;
    const int64_t row = blockIdx.x / a.tiles;
    const item *in = reinterpret_cast<const item *>(a.student + (a.row0 + row) * a.stride);
    item *out = reinterpret_cast<item *>(a.grad + (a.row0 + row) * a.grad_stride);
    const int64_t first = (int64_t)(blockIdx.x % a.tiles) * T * V * kItems - nbh_row_before<E>(in);
    const Plan plan = a.plans[row];
    nbh_u32x4 raw[V];
    const bool full = first >= 0 && first + T * V * kItems <= a.vocab;
    if (full) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            raw[j] = E::template load<true>(in + first + (j * T + threadIdx.x) * kItems);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            raw[j] = nbh_row_load_raw<E, true>(in, first + (j * T + (int)threadIdx.x) * kItems, a.vocab, 0);
    }
    const float product = plan.peak * a.scale;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float f[kItems];
        E::unpack(raw[j], f);
        if (plan.zero) {
            for (int i = 0; i < kItems; ++i)
                f[i] = 0.0f;
        } else if (nbh_softmax_near(product)) {
            for (int i = 0; i < kItems; ++i)
                f[i] = plan.whole * nbh_exp2(fmaf(f[i], a.scale, -product));
        } else {
            for (int i = 0; i < kItems; ++i)
                f[i] = plan.whole * nbh_exp2((f[i] - plan.peak) * a.scale - plan.shift);
        }
        const int64_t at = first + (j * T + (int)threadIdx.x) * kItems;
        if (full)
            nbh_store16<sizeof(item), true>(out + at, E::pack(f));
        else
            nbh_row_store<E, true>(out, at, a.vocab, f);
    }
}
// Third: a lane per entry the teacher names.
template <typename E> __global__ __launch_bounds__(256) void distill_named(Distill a, int64_t rows)
{
    const int64_t i = blockIdx.x * (int64_t)256 + threadIdx.x;
    if (i >= rows * a.k)
        return;
    const Named n = a.named[i];
    if (n.index >= 0)
        reinterpret_cast<typename E::item *>(a.grad + (a.row0 + i / a.k) * a.grad_stride)[n.index] = E::put(n.value);
}

// How a call is spread.
//   kRows     one workgroup per row does everything; for the gradient by itself `splits` of them, each a
//             stretch of `slice` entries
//   kInParts  a launch of small workgroups for the statistics, then a wavefront per row for the loss alone, or
//             with the gradient `splits` workgroups per row, four per compute unit
//   kFlat     the gradient by itself in three launches
// Measured, one launch against the two of kInParts for the loss, k = 32, bfloat16: 4 x 32768 14 and 18 us,
// 256 x 131072 19 and 20, 4096 x 32768 53 and 52, 1024 x 131072 53 and 50; float32: 4 x 131072 20 and 17,
// 256 x 131072 28 and 29, 4096 x 32768 96 and 90.  For both, bfloat16: 4 x 32768 16 and 20, 4 x 131072 22 and
// 20, 64 x 131072 23 and 22, 256 x 131072 35 and 47; float32: 4 x 131072 25 and 20, 64 x 131072 28 and 27.  One
// launch against the three of kFlat, float32: 256 x 32768 16 and 24, 256 x 131072 52 and 51, 1024 x 100003 193
// and 157.
// Rows of up to 16 KiB, a chunk of the row kernel, are always kRows with a wavefront each: what a workgroup does
// once per row takes longer than the row, and this way most of the rows of a call are under way together.
// bfloat16, 64, 256 and 512 lanes: loss 4096 x 1024 13, 22 and 40 us, 4096 x 8192 20, 22 and 43, 4096 x 16384 35,
// 35 and 36; gradient 4096 x 1024 16, 30 and 53, 4096 x 8192 33, 34 and 53; both 4096 x 1024 19, 42 and 78, 4096 x
// 8192 40, 40 and 74.  In several launches: loss 131072 x 1024 280 instead of 171, 16384 x 8192 70 instead of 59,
// gradient 288 instead of 234 and 153 instead of 137.
// Both at once, 256 and 512 lanes: 4096 x 16384 67 and 97, 4096 x 32768 125 and 130, 512 x 16384 17 and 17, 256 x
// 32768 18 and 17, 4096 x 50021 242 and 224, 4096 x 65536 239 and 206.  Many entries of the teacher take a wavefront
// long, which more rows under way hide better, unless the row is longer than what 512 lanes keep of it; of more than
// 512 entries LDS leaves room for one workgroup of 512 only.  k = 64, 150, 250, 300, 350, 400 and 512:
//   4096 x 65536 bfloat16   239 256 276 291 311 331 359 and 206 264 304 321 349 387 451
//   1024 x 50021 float16     61  66  71  73  76  79  83 and  53  61  69  71  76  80  89
//   600 x 32768 float32      39  45  48  50  52  54  59 and  35  44  51  53  57  62  70
//   2048 x 65536 float32    234 246 259 268 275 284 308 and 209 231 255 263 275 288 309
//   1024 x 131072 bfloat16  121 131 141 146 152 157 164 and  97 110 124 128 138 147 160
//   512 x 65536 bfloat16     35  41  44  45  48  50  54 and  27  33  37  39  42  45  49
//   k = 600 4096 x 65536 371 and 627, 1000 457 and 906, 1024 x 131072 205 and 287, 256 x 131072 77 and 71.
enum Way { kRows, kInParts, kFlat };
struct Spread {
    Way way;
    int tiles, lanes, splits;            // lanes of the row kernel
    int64_t slice;
};
// `spare`: entries before a row's beginning that its first vector may hold
Spread spread_of(int64_t rows, int64_t vocab, int64_t k, int dtype, int what, int spare)
{
    const int64_t items = dtype == NBH_ROW_F32 ? 4 : 8;
    const int64_t chunk = 256 * kNbhAhead * items;           // 16 KiB, a step of the row kernel
    const int64_t tile = kStatsThreads * kStatsVecs * items;
    const int64_t flat = kFlatThreads * kFlatVecs * items;
    const int64_t chunks = vocab ? (vocab + chunk - 1) / chunk : 1;
    const bool small = chunks == 1, large = !small && rows * vocab >= ((int64_t)128 << 20) / 16 * items;
    const int tiles = (int)((vocab + spare + tile - 1) / tile);
    // kFlat needs a launch to hold a row (whatever `spare` is: the workspace goes by the largest); from 2^29
    // entries of four bytes or 2^30 of two on, one does not.
    if (what == kGrad && large && vocab + 7 <= (int64_t)NBH_ROW_MOST_GROUPS * flat)
        return {kFlat, (int)((vocab + spare + flat - 1) / flat), 0, 1, vocab};
    if (what == kLoss)
        return {large || (rows < 256 && chunks > 24) ? kInParts : kRows, tiles, small ? 64 : 256, 1, vocab};
    if (what == (kLoss | kGrad) && (rows >= 128 || chunks <= 12)) {
        const bool more = (rows > 512 && (chunks <= 4 || (k > 300 && chunks <= 10))) || (k > 512 && rows > 256);
        return {kRows, tiles, small ? 64 : more ? 256 : 512, 1, vocab};
    }
    int64_t splits = (1024 + rows - 1) / rows;
    if (splits > chunks)
        splits = chunks;
    const int64_t each = (chunks + splits - 1) / splits;
    return {what == kGrad ? kRows : kInParts, tiles, small ? 64 : 256, (int)((chunks + each - 1) / each),
            each * chunk};
}

template <typename E>
int launch_distill(Distill a, Way way, int lanes, int64_t rows, int what, hipStream_t stream)
{
    const size_t bytes = Teacher::bytes(a.k);
    const int64_t most = NBH_ROW_MOST_GROUPS / (way == kRows ? a.splits : a.tiles);
    for (a.row0 = 0; a.row0 < rows; a.row0 += most) {
        const int64_t now = rows - a.row0 < most ? rows - a.row0 : most;
        const dim3 each((unsigned)now), split((unsigned)(now * a.splits)), tiled((unsigned)(now * a.tiles));
        if (way == kFlat) {
            distill_plan<E><<<each, dim3(64), bytes, stream>>>(a);
            distill_flat<E><<<tiled, dim3(kFlatThreads), 0, stream>>>(a);
            if (a.k)
                distill_named<E><<<dim3((unsigned)((now * a.k + 255) / 256)), dim3(256), 0, stream>>>(a, now);
        } else if (way == kInParts) {
            distill_stats<E><<<tiled, dim3(kStatsThreads), 0, stream>>>(a);
            if (what == kLoss)
                distill_rows<E, 64, kLoss | kParts><<<each, dim3(64), bytes, stream>>>(a);
            else
                distill_rows<E, 256, kLoss | kGrad | kParts><<<split, dim3(256), bytes, stream>>>(a);
        } else if (what == kGrad) {
            if (lanes == 64)
                distill_rows<E, 64, kGrad><<<split, dim3(64), bytes, stream>>>(a);
            else
                distill_rows<E, 256, kGrad><<<split, dim3(256), bytes, stream>>>(a);
        } else if (what == kLoss) {
            if (lanes == 64)
                distill_rows<E, 64, kLoss><<<each, dim3(64), bytes, stream>>>(a);
            else
                distill_rows<E, 256, kLoss><<<each, dim3(256), bytes, stream>>>(a);
        } else {
            if (lanes == 64)
                distill_rows<E, 64, kLoss | kGrad><<<each, dim3(64), bytes, stream>>>(a);
            else if (lanes == 256)
                distill_rows<E, 256, kLoss | kGrad><<<each, dim3(256), bytes, stream>>>(a);
            else
                distill_rows<E, 512, kLoss | kGrad><<<each, dim3(512), bytes, stream>>>(a);
        }
        if (const int status = nbh_launch_status())
            return status;
    }
    return 0;
}

}  // namespace

extern "C" size_t nbh_rows_distill_workspace(int64_t rows, int64_t vocab, int64_t k, int dtype, int what)
{
    if (rows <= 0 || vocab < 0 || vocab > INT32_MAX || k < 0 || k > NBH_ROW_TOP_MOST || dtype < 0 ||
        dtype > NBH_ROW_BF16 || what < kLoss || what > (kLoss | kGrad))
        return 0;
    const Spread s = spread_of(rows, vocab, k, dtype, what, 7);
    if (s.way == kFlat)
        return (size_t)rows * (sizeof(Plan) + (size_t)k * sizeof(Named));
    if (s.way == kInParts)
        return (size_t)rows * ((size_t)s.tiles * (kStatsThreads / 64) * sizeof(nbh_softmax) +
                               (what & kGrad ? (size_t)k * sizeof(float) : 0));
    return 0;
}

extern "C" int nbh_rows_distill(const struct nbh_rows_distill_args *p, nbh_stream_t stream)
{
    if (!p || p->struct_bytes != (int64_t)sizeof(*p) || p->rows < 0 || p->vocab < 0 || p->vocab > INT32_MAX ||
        p->dtype < 0 || p->dtype > NBH_ROW_BF16 || p->values_dtype < 0 || p->values_dtype > NBH_ROW_BF16 || p->k < 0 ||
        p->k > NBH_ROW_TOP_MOST || (p->index_bytes != 4 && p->index_bytes != 8) || !nbh_row_temperature(p->temperature) ||
        p->what < NBH_DISTILL_LOSS || p->what > (NBH_DISTILL_LOSS | NBH_DISTILL_GRAD))
        return (int)hipErrorInvalidValue;
    if (p->rows == 0)
        return 0;
    const bool loss = p->what & NBH_DISTILL_LOSS, grad = p->what & NBH_DISTILL_GRAD;
    if ((p->vocab && !p->student) || (p->k && (!p->values || !p->indices)) || (loss && !p->loss) ||
        (!loss && !p->lse) || (grad && p->vocab && !p->grad))
        return (int)hipErrorInvalidValue;
    const size_t need = nbh_rows_distill_workspace(p->rows, p->vocab, p->k, (int)p->dtype, (int)p->what);
    if (need && (!p->workspace || p->workspace_bytes < (int64_t)need || ((uintptr_t)p->workspace & 15)))
        return (int)hipErrorInvalidValue;
    const Spread spread = spread_of(p->rows, p->vocab, p->k, (int)p->dtype, (int)p->what,
                                    nbh_row_spare(p->student, p->stride, (int)p->dtype));
    Distill a = {};
    a.student = (const char *)p->student;
    a.stride = p->stride;
    a.vocab = p->vocab;
    a.slice = spread.slice;
    a.splits = spread.splits;
    a.k = (int)p->k;
    a.index_bytes = (int)p->index_bytes;
    a.values_dtype = (int)p->values_dtype;
    a.values = (const char *)p->values;
    a.indices = (const char *)p->indices;
    a.values_stride = p->values_stride;
    a.indices_stride = p->indices_stride;
    a.teacher_lse = p->teacher_lse;
    a.grad_loss = p->grad_loss;
    a.grad_loss_stride = p->grad_loss_stride;
    a.grad_loss_value = (float)p->grad_loss_value;
    a.temperature = (float)p->temperature;
    a.scale = (float)(1.4426950408889634 / a.temperature);
    a.scale_rest = (float)(1.4426950408889634 / a.temperature - a.scale);
    a.loss = p->loss;
    a.lse = p->lse;
    a.grad = (char *)p->grad;
    a.grad_stride = p->grad_stride;
    a.parts = (nbh_softmax *)p->workspace;
    a.tiles = spread.tiles;
    if (grad)
        a.targets = (float *)(a.parts + p->rows * spread.tiles * (kStatsThreads / 64));
    a.plans = (Plan *)p->workspace;
    a.named = (Named *)(a.plans + p->rows);

    const hipStream_t s = nbh_hip_stream(stream);
    nbh_stream_report report(s);
    switch (p->dtype) {
    case NBH_ROW_F32:
        return launch_distill<nbh_row_f32>(a, spread.way, spread.lanes, p->rows, (int)p->what, s);
    case NBH_ROW_F16:
        return launch_distill<nbh_row_f16>(a, spread.way, spread.lanes, p->rows, (int)p->what, s);
    default:
        return launch_distill<nbh_row_bf16>(a, spread.way, spread.lanes, p->rows, (int)p->what, s);
    }
}
