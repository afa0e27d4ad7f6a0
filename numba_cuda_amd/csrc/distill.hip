// nbh_rows_distill: distillation from a teacher's top logits, forward, backward or both at once.
//
//   lse = log sum exp(s / T);  p_j from the teacher's k entries;  P = sum p_j
//   loss = sum p_j (log p_j - (s[i_j] / T - lse))
//   grad[v] = grad_loss / T * (P exp(s[v] / T - lse) - sum over i_j = v of p_j)
//
// One workgroup per row: the teacher's entries go to LDS, one pass over the row gives its maximum and
// sum together, the second writes the gradient as a * 2^((s - m) * c) for every entry, and behind a
// barrier the few entries the teacher names are written again with their p_j taken off.  The row's second
// reading comes out of the caches.  Few rows are split over workgroups: a launch for the statistics of the
// stretches, then one that joins them and works on the stretches.
#include "rows.h"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr float kLog2e = 1.44269502f, kLog2eRest = 1.92596299e-8f;       // log2(e) and its rounding
constexpr float kLn2 = 0.693147180559945309f;

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
};

template <typename E>
__global__ __launch_bounds__(kThreads) void distill_stats(Distill a)
{
    __shared__ nbh_softmax room[kWaves];
    const int64_t row = a.row0 + blockIdx.x / a.splits;
    const int split = blockIdx.x % a.splits;
    const typename E::item *in = reinterpret_cast<const typename E::item *>(a.student + row * a.stride);
    const int64_t begin = split * a.slice, end = a.vocab < begin + a.slice ? a.vocab : begin + a.slice;
    const nbh_softmax stats =
        nbh_softmax_group<kThreads>(nbh_row_stats<E, kThreads, false>(in, begin, end, a.scale), a.scale, room);
    if (threadIdx.x == 0)
        a.parts[(row - a.row0) * a.splits + split] = stats;
    // The loss needs these of the whole row, and the gradient may be written over the row while another
    // stretch's workgroup still works on the loss: they are set aside.
    if (split == 0)
        for (int j = threadIdx.x; j < a.k; j += kThreads) {
            const int64_t at = nbh_row_int(a.indices + row * a.indices_stride, a.index_bytes, j);
            a.targets[(row - a.row0) * a.k + j] = at >= 0 && at < a.vocab ? E::get(in[at]) : 0.0f;
        }
}

// The sum of x over the workgroup, in every lane; the barriers also order what was written to LDS before.
__device__ __forceinline__ float group_add(float x, float *room)
{
    for (int step = 32; step; step >>= 1)
        x += __shfl_xor(x, step);
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
        room[threadIdx.x >> 6] = x;
    __syncthreads();
    x = room[0];
    for (int w = 1; w < kWaves; ++w)
        x += room[w];
    return x;
}
__device__ __forceinline__ float group_max(float x, float *room)
{
    for (int step = 32; step; step >>= 1)
        x = fmaxf(x, __shfl_xor(x, step));
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
        room[threadIdx.x >> 6] = x;
    __syncthreads();
    x = room[0];
    for (int w = 1; w < kWaves; ++w)
        x = fmaxf(x, room[w]);
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

// What one launch of the row kernel does
constexpr int kLoss = 1, kGrad = 2, kParts = 4;      // kParts: statistics come from distill_stats

template <typename E, int WHAT>
__global__ __launch_bounds__(kThreads) void distill_rows(Distill a)
{
    typedef typename E::item item;
    constexpr int kItems = E::items;
    extern __shared__ char lds[];        // index, p and log p, and the table that finds repeated indices
    __shared__ nbh_softmax room[kWaves];
    __shared__ float add_room[kWaves];
    __shared__ int repeated;
    int32_t *const index = reinterpret_cast<int32_t *>(lds);
    float *const p = reinterpret_cast<float *>(index + a.k), *const log_p = p + a.k;
    int32_t *const table = reinterpret_cast<int32_t *>(log_p + a.k);

    // the loss alone takes one workgroup per row, whatever the statistics took
    constexpr bool kWhole = WHAT == (kLoss | kParts);
    const int64_t row = a.row0 + (kWhole ? blockIdx.x : blockIdx.x / a.splits);
    const int split = kWhole ? 0 : blockIdx.x % a.splits;
    const item *in = reinterpret_cast<const item *>(a.student + row * a.stride);
    const int64_t begin = split * a.slice, end = a.vocab < begin + a.slice ? a.vocab : begin + a.slice;

    // -- the teacher's entries
    float peak = -FLT_MAX;
    int some = 0;
    for (int j = threadIdx.x; j < a.k; j += kThreads) {
        const int64_t at = nbh_row_int(a.indices + row * a.indices_stride, a.index_bytes, j);
        const float t = teacher_value(a, row, j);
        const bool present = at >= 0 && at < a.vocab && t != -INFINITY;
        index[j] = present ? (int32_t)at : -1;
        log_p[j] = t;
        if (present) {
            peak = fmaxf(peak, fminf(t, FLT_MAX));
            some = 1;
        }
    }
    float mass = 0.0f;
    if (a.teacher_lse) {
        const float norm = a.teacher_lse[row];
        for (int j = threadIdx.x; j < a.k; j += kThreads) {
            log_p[j] = log_p[j] / a.temperature - norm;
            p[j] = index[j] >= 0 ? expf(log_p[j]) : 0.0f;
            mass += p[j];
        }
        mass = group_add(mass, add_room);
    } else {
        peak = group_max(peak, add_room);
        float sum = 0.0f;
        for (int j = threadIdx.x; j < a.k; j += kThreads) {
            log_p[j] = (log_p[j] - peak) / a.temperature;
            p[j] = index[j] >= 0 ? expf(log_p[j]) : 0.0f;
            sum += p[j];
        }
        sum = group_add(sum, add_room);
        const float norm = logf(sum);
        for (int j = threadIdx.x; j < a.k; j += kThreads) {
            log_p[j] -= norm;
            p[j] = index[j] >= 0 ? p[j] / sum : 0.0f;
            mass += p[j];
        }
        mass = group_add(mass, add_room);
    }
    some = __syncthreads_or(some);

    // -- the student's statistics: exp(s / T - lse) = base * 2^(s * scale - peak * scale)
    float peak_s, base, log_sum = 0.0f;
    if (WHAT & kLoss) {
        nbh_softmax stats;
        if (WHAT & kParts) {
            stats = a.parts[(row - a.row0) * a.splits];
            for (int s = 1; s < a.splits; ++s)
                stats = nbh_softmax_join(stats, a.parts[(row - a.row0) * a.splits + s], a.scale);
        } else {
            stats = nbh_softmax_group<kThreads>(nbh_row_stats<E, kThreads, false>(in, 0, a.vocab, a.scale), a.scale,
                                                room);
        }
        peak_s = stats.peak == -INFINITY ? 0.0f : stats.peak;
        base = stats.sum == 0.0f ? 0.0f : 1.0f / stats.sum;
        log_sum = log2f(stats.sum);
        if (a.lse && split == 0 && threadIdx.x == 0)
            a.lse[row] = nbh_softmax_lse(stats, a.temperature, a.scale);
    } else {
        const float lse = a.lse[row];
        // T * lse rounded to float32 takes the place of the largest value; what the roundings of it, of
        // its product with the scale, and of the scale itself take off goes into the factor.
        peak_s = lse * a.temperature;
        const float product = peak_s * a.scale;
        if (nbh_softmax_near(product)) {
            const float high = lse * kLog2e, low = fmaf(lse, kLog2e, -high) + lse * kLog2eRest;
            base = exp2f((product - high) - low + peak_s * a.scale_rest);
        } else {
            const float rest = __builtin_isfinite(peak_s) ? fmaf(lse, a.temperature, -peak_s) : 0.0f;
            base = expf(-rest / a.temperature);
        }
        if (lse == -INFINITY)
            peak_s = base = 0.0f;
    }
    const float product = peak_s * a.scale;
    const bool near = nbh_softmax_near(product);

    // -- loss
    if ((WHAT & kLoss) && split == 0) {
        float loss = 0.0f;
        for (int j = threadIdx.x; j < a.k; j += kThreads)
            if (index[j] >= 0 && p[j] != 0.0f) {
                const float s = WHAT & kParts ? a.targets[(row - a.row0) * a.k + j] : E::get(in[index[j]]);
                float log_q = s;
                if (s != -INFINITY)
                    log_q = near && fabsf(s) < 1e30f
                                ? (fmaf(s, a.scale, -product) - log_sum) * kLn2
                                : (s - peak_s) / a.temperature - log_sum * kLn2;
                loss += p[j] * (log_p[j] - log_q);
            }
        loss = group_add(loss, add_room);
        if (threadIdx.x == 0)
            a.loss[row] = some ? loss : 0.0f;
    }
    if (!(WHAT & kGrad))
        return;

    // -- gradient
    item *out = reinterpret_cast<item *>(a.grad + row * a.grad_stride);
    const float factor =
        (a.grad_loss ? *reinterpret_cast<const float *>((const char *)a.grad_loss + row * a.grad_loss_stride)
                     : a.grad_loss_value) /
        a.temperature;
    if (!some || factor == 0.0f) {
        float zero[kItems] = {};
        for (int64_t at = begin + threadIdx.x * kItems; at < end; at += kThreads * kItems)
            nbh_row_store<E, true>(out, at, end, zero);
        return;
    }
    // which of the teacher's indices occur more than once (none, as a rule): a table of at least 2 k slots
    int slots = 2;
    while (slots < 2 * a.k)
        slots *= 2;
    for (int i = threadIdx.x; i < slots; i += kThreads)
        table[i] = -1;
    if (threadIdx.x == 0)
        repeated = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < a.k; j += kThreads)
        if (index[j] >= 0) {
            uint32_t slot = (uint32_t)index[j] * 2654435761u;
            for (int tries = 0; tries < slots; ++tries, ++slot) {
                const int32_t was = atomicCAS(&table[slot & (slots - 1)], -1, index[j]);
                if (was == index[j])
                    repeated = 1;
                if (was == -1 || was == index[j])
                    break;
            }
        }
    __syncthreads();
    // the student's values at the teacher's entries, before they are written over
    const float whole = factor * mass * base;
    for (int j = threadIdx.x; j < a.k; j += kThreads) {
        if (index[j] < begin || index[j] >= end)
            continue;
        float own = p[j];
        if (repeated) {                  // the first of them takes all their shares, in order
            bool first = true;
            for (int i = 0; i < j && first; ++i)
                first = index[i] != index[j];
            for (int i = j + 1; i < a.k && first; ++i)
                if (index[i] == index[j])
                    own += p[i];
            if (!first) {
                log_p[j] = 0.0f;
                continue;
            }
        }
        const float s = E::get(in[index[j]]);
        log_p[j] = whole * nbh_softmax_term(s, peak_s, a.scale) - factor * own;
    }
    __syncthreads();
    nbh_row_stream<E, kThreads, false, true>(in, begin, end, [&](int64_t at, const nbh_u32x4(&raw)[kNbhAhead]) __attribute__((always_inline)) {
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
                    f[i] = whole * nbh_exp2((f[i] - peak_s) * a.scale);
            }
            nbh_row_store<E, true>(out, at + (j * kThreads + threadIdx.x) * kItems, end, f);
        }
    });
    __syncthreads();
    for (int j = threadIdx.x; j < a.k; j += kThreads) {
        if (index[j] < begin || index[j] >= end)
            continue;
        if (repeated) {
            bool first = true;
            for (int i = 0; i < j && first; ++i)
                first = index[i] != index[j];
            if (!first)
                continue;
        }
        out[index[j]] = E::put(log_p[j]);
    }
}

// Stretches of a row: one workgroup per row from 1024 rows on, else workgroups for four per compute unit.
struct Split {
    int splits;
    int64_t slice;
};
Split split_of(int64_t rows, int64_t vocab, int dtype)
{
    const int64_t chunk = (int64_t)kThreads * kNbhAhead * (dtype == NBH_ROW_F32 ? 4 : 8);
    const int64_t chunks = vocab ? (vocab + chunk - 1) / chunk : 1;
    int64_t splits = (1024 + rows - 1) / rows;
    if (splits > chunks)
        splits = chunks;
    const int64_t each = (chunks + splits - 1) / splits;
    return {(int)((chunks + each - 1) / each), each * chunk};
}

template <typename E>
int launch_distill(Distill a, int64_t rows, int what, hipStream_t stream)
{
    int slots = 2;
    while (slots < 2 * a.k)
        slots *= 2;
    const size_t bytes = (size_t)a.k * 12 + (size_t)slots * 4;
    const int64_t most = NBH_ROW_MOST_GROUPS / a.splits;
    for (a.row0 = 0; a.row0 < rows; a.row0 += most) {
        const int64_t now = rows - a.row0 < most ? rows - a.row0 : most;
        const dim3 block(kThreads);
        dim3 grid((unsigned)(now * a.splits));
        if (what == kGrad) {
            distill_rows<E, kGrad><<<grid, block, bytes, stream>>>(a);
        } else if (a.splits == 1) {
            if (what == kLoss)
                distill_rows<E, kLoss><<<grid, block, bytes, stream>>>(a);
            else
                distill_rows<E, kLoss | kGrad><<<grid, block, bytes, stream>>>(a);
        } else {
            distill_stats<E><<<grid, block, 0, stream>>>(a);
            if (what == kLoss)
                distill_rows<E, kLoss | kParts><<<dim3((unsigned)now), block, bytes, stream>>>(a);
            else
                distill_rows<E, kLoss | kGrad | kParts><<<grid, block, bytes, stream>>>(a);
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
        dtype > NBH_ROW_BF16 || !(what & NBH_DISTILL_LOSS))
        return 0;
    const Split s = split_of(rows, vocab, dtype);
    return s.splits == 1 ? 0 : (size_t)rows * (s.splits * sizeof(nbh_softmax) + (size_t)k * sizeof(float));
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
    const Split split = split_of(p->rows, p->vocab, (int)p->dtype);
    Distill a = {};
    a.student = (const char *)p->student;
    a.stride = p->stride;
    a.vocab = p->vocab;
    a.slice = split.slice;
    a.splits = split.splits;
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
    a.targets = (float *)(a.parts + p->rows * split.splits);

    const hipStream_t s = nbh_hip_stream(stream);
    nbh_stream_report report(s);
    switch (p->dtype) {
    case NBH_ROW_F32:
        return launch_distill<nbh_row_f32>(a, p->rows, (int)p->what, s);
    case NBH_ROW_F16:
        return launch_distill<nbh_row_f16>(a, p->rows, (int)p->what, s);
    default:
        return launch_distill<nbh_row_bf16>(a, p->rows, (int)p->what, s);
    }
}
