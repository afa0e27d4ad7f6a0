// Helpers of the kernels that work on the rows of a 2-d array of logits (logits.hip, toprows.hip,
// distill.hip): 16-byte vectors of float32, float16 or bfloat16 at any element alignment, and the
// running maximum and sum of a softmax.
#pragma once

#include <float.h>

#include "common.h"

typedef float nbh_f32x4 __attribute__((ext_vector_type(4)));
typedef float nbh_f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 nbh_f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 nbh_bf16x2 __attribute__((ext_vector_type(2)));

// Workgroups of one launch: with up to 1024 lanes each they stay below 2^32 lanes.  A row of 2^31 entries makes
// 2^20 tiles of the statistics' 2048 float32 entries, fewer of every other kernel but the gradient's in the order of
// memory, which takes 256 entries and is for rows that fit a launch.
#define NBH_ROW_MOST_GROUPS (1 << 21)

// Element types.  `items` elements make 16 bytes; arithmetic is float32 throughout, stores round once,
// to nearest even.
struct nbh_row_f32 {
    typedef float item;
    static constexpr int items = 4;
    static constexpr uint32_t lowest = 0xff800000u;      // bits of -inf
    template <bool NT> static __device__ __forceinline__ nbh_u32x4 load(const item *p) { return nbh_load16<4, NT>(p); }
    static __device__ __forceinline__ uint32_t bits(item x) { return __float_as_uint(x); }
    static __device__ __forceinline__ float get(item x) { return x; }
    static __device__ __forceinline__ item put(float x) { return x; }
    static __device__ __forceinline__ void unpack(nbh_u32x4 v, float (&f)[4])
    {
        for (int i = 0; i < 4; ++i)
            f[i] = __uint_as_float(v[i]);
    }
    static __device__ __forceinline__ nbh_u32x4 pack(const float (&f)[4])
    {
        nbh_u32x4 v;
        for (int i = 0; i < 4; ++i)
            v[i] = __float_as_uint(f[i]);
        return v;
    }
};
struct nbh_row_f16 {
    typedef _Float16 item;
    static constexpr int items = 8;
    static constexpr uint32_t lowest = 0xfc00u;
    template <bool NT> static __device__ __forceinline__ nbh_u32x4 load(const item *p) { return nbh_load16<2, NT>(p); }
    static __device__ __forceinline__ uint32_t bits(item x) { return __builtin_bit_cast(uint16_t, x); }
    static __device__ __forceinline__ float get(item x) { return (float)x; }
    static __device__ __forceinline__ item put(float x) { return (item)x; }
    static __device__ __forceinline__ void unpack(nbh_u32x4 v, float (&f)[8])
    {
        for (int i = 0; i < 4; ++i) {
            const nbh_f16x2 h = __builtin_bit_cast(nbh_f16x2, (uint32_t)v[i]);
            f[2 * i] = (float)h[0];
            f[2 * i + 1] = (float)h[1];
        }
    }
    static __device__ __forceinline__ nbh_u32x4 pack(const float (&f)[8])
    {
        nbh_u32x4 v;
        for (int i = 0; i < 4; ++i) {
            const nbh_f16x2 h = {(_Float16)f[2 * i], (_Float16)f[2 * i + 1]};
            v[i] = __builtin_bit_cast(uint32_t, h);
        }
        return v;
    }
};
struct nbh_row_bf16 {
    typedef uint16_t item;
    static constexpr int items = 8;
    static constexpr uint32_t lowest = 0xff80u;
    template <bool NT> static __device__ __forceinline__ nbh_u32x4 load(const item *p) { return nbh_load16<2, NT>(p); }
    static __device__ __forceinline__ uint32_t bits(item x) { return x; }
    static __device__ __forceinline__ float get(item x) { return __uint_as_float((uint32_t)x << 16); }
    static __device__ __forceinline__ item put(float x)
    {
        return __builtin_bit_cast(uint16_t, (__bf16)x);
    }
    static __device__ __forceinline__ void unpack(nbh_u32x4 v, float (&f)[8])
    {
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(v[i] << 16);
            f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ nbh_u32x4 pack(const float (&f)[8])
    {
        nbh_u32x4 v;
        for (int i = 0; i < 4; ++i) {
            const nbh_f32x2 two = {f[2 * i], f[2 * i + 1]};
            v[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(two, nbh_bf16x2));
        }
        return v;
    }
};

// The two-byte types four at a time, for results of four bytes: a wavefront's stores are then whole lines.
typedef uint32_t nbh_u32x2 __attribute__((ext_vector_type(2)));
typedef nbh_u32x2 nbh_u32x2_any __attribute__((aligned(2)));
template <typename E> struct nbh_row_half {
    typedef typename E::item item;
    static constexpr int items = 4;
    static constexpr uint32_t lowest = E::lowest;
    template <bool NT> static __device__ __forceinline__ nbh_u32x4 load(const item *p)
    {
        const nbh_u32x2_any *q = reinterpret_cast<const nbh_u32x2_any *>(p);
        const nbh_u32x2 v = NT ? __builtin_nontemporal_load(q) : *q;
        return nbh_u32x4{v[0], v[1], 0, 0};
    }
    static __device__ __forceinline__ uint32_t bits(item x) { return E::bits(x); }
    static __device__ __forceinline__ void unpack(nbh_u32x4 v, float (&f)[4])
    {
        float all[8];
        E::unpack(v, all);
        for (int i = 0; i < 4; ++i)
            f[i] = all[i];
    }
};

// Elements from the last multiple of 16 bytes before a row to its beginning.  Vectors counted from there are
// aligned: a wavefront's load then covers 8 cache lines, not 9 (10 % of a row's reading time).
template <typename E> __device__ __forceinline__ int nbh_row_before(const typename E::item *row)
{
    return (int)((uintptr_t)row / sizeof(typename E::item) % E::items);
}
// The most that can be for the rows of an array.
static inline int nbh_row_spare(const void *address, int64_t stride, int dtype)
{
    return ((uintptr_t)address | (uintptr_t)stride) & 15 ? (dtype == NBH_ROW_F32 ? 3 : 7) : 0;
}
// The 16 bytes at element `at` of a row of `n` elements; elements before the row and behind its end read as
// `fill`, the raw one as its bits.
template <typename E, bool NT>
__device__ __forceinline__ nbh_u32x4 nbh_row_load_raw(const typename E::item *row, int64_t at, int64_t n, uint32_t fill)
{
    if (at >= 0 && at + E::items <= n)
        return E::template load<NT>(row + at);
    nbh_u32x4 v = {};
    for (int i = 0; i < E::items; ++i) {
        const uint32_t bits = at + i >= 0 && at + i < n ? E::bits(row[at + i]) : fill;
        if (sizeof(typename E::item) == 4)
            v[i] = bits;
        else
            v[i / 2] |= bits << (i % 2 * 16);
    }
    return v;
}
template <typename E, bool NT>
__device__ __forceinline__ void nbh_row_load(const typename E::item *row, int64_t at, int64_t n, float fill,
                                             float (&f)[E::items])
{
    if (at >= 0 && at + E::items <= n) {
        E::unpack(nbh_load16<sizeof(typename E::item), NT>(row + at), f);
    } else {
        for (int i = 0; i < E::items; ++i)
            f[i] = at + i >= 0 && at + i < n ? E::get(row[at + i]) : fill;
    }
}
template <typename E, bool NT>
__device__ __forceinline__ void nbh_row_store(typename E::item *row, int64_t at, int64_t n, const float (&f)[E::items])
{
    if (at >= 0 && at + E::items <= n) {
        nbh_store16<sizeof(typename E::item), NT>(row + at, E::pack(f));
    } else {
        for (int i = 0; i < E::items; ++i)
            if (at + i >= 0 && at + i < n)
                row[at + i] = E::put(f[i]);
    }
}

// Running softmax statistics of values x, with scale = log2(e) / temperature: `sum` is the sum of
// 2^(x scale - origin) for a reference `peak` (-inf before the first value above -inf), which is at
// most 32 powers of two below the largest value: it is raised only when a value would exceed that, so that
// nearly all values cost one fused multiply-add, one exponential and one addition.
// The origin is peak scale.  Below 2^22 it is that product rounded once, which the rounding moves by at most a
// quarter: used so everywhere, that is harmless.  Beyond, the rounding would take whole powers of two off
// (masked rows, tiny temperatures), so the origin is the exact product there and the terms are
// 2^((x - peak) scale).  Where a step of float32 at the peak is as large as the 32 powers of two, rounding may let
// a value of up to 64 pass: 2^31 of them still add up to a finite sum.
// A NaN stays in `sum`; a row of -inf has peak -inf and sum 0; +inf makes `sum` inf.
struct nbh_softmax {
    float peak, sum;
};
__device__ __forceinline__ nbh_softmax nbh_softmax_empty() { return {-INFINITY, 0.0f}; }
__device__ __forceinline__ float nbh_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ bool nbh_softmax_near(float product) { return fabsf(product) < 0x1p22f; }
// 2^(x scale - origin of peak - shift); `shift` counts only where that product is not near.
__device__ __forceinline__ float nbh_softmax_term(float x, float peak, float scale, float shift = 0.0f)
{
    const float product = peak * scale;
    return nbh_exp2(nbh_softmax_near(product) ? fmaf(x, scale, -product) : (x - peak) * scale - shift);
}
// What rounding took off the product that is the origin.
__device__ __forceinline__ float nbh_softmax_rest(float peak, float scale)
{
    const float product = peak * scale;
    return nbh_softmax_near(product) ? fmaf(peak, scale, -product) : 0.0f;
}
// 2^(origin of one peak - origin of another)
__device__ __forceinline__ float nbh_softmax_factor(float from, float to, float scale)
{
    const float a = from * scale, b = to * scale;
    return nbh_exp2(nbh_softmax_near(a) && nbh_softmax_near(b)
                        ? a - b
                        : (from - to) * scale - nbh_softmax_rest(from, scale) + nbh_softmax_rest(to, scale));
}
// Values f, the largest of which is `most` (or NaN).
template <int N>
__device__ __forceinline__ void nbh_softmax_add(nbh_softmax &s, const float (&f)[N], float most, float scale)
{
    // 32 powers of two above the reference
    if (__any(!(most <= fmaf(32.0f, __builtin_amdgcn_rcpf(scale), s.peak)))) {
        const float peak = fmaxf(s.peak, fminf(most, FLT_MAX));
        if (peak != s.peak) {
            s.sum *= nbh_exp2((s.peak - peak) * scale - nbh_softmax_rest(s.peak, scale) + nbh_softmax_rest(peak, scale));
            s.peak = peak;
        }
    }
    const float product = s.peak == -INFINITY ? 0.0f : s.peak * scale;
    float sum[2] = {0.0f, 0.0f};
    if (__any(!nbh_softmax_near(product))) {
        // for all lanes of the wavefront, those of which the product is near too
        const float peak = s.peak == -INFINITY ? 0.0f : s.peak, rest = nbh_softmax_rest(peak, scale);
        for (int i = 0; i < N; ++i)
            sum[i & 1] += nbh_exp2((f[i] - peak) * scale + rest);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            sum[i & 1] += nbh_exp2(fmaf(f[i], scale, -product));
    }
    s.sum += sum[0] + sum[1];
}
template <int N> __device__ __forceinline__ float nbh_row_most(const float (&f)[N])
{
    float most = f[0];
#pragma unroll
    for (int i = 1; i < N; ++i)
        most = __builtin_elementwise_maximum(most, f[i]);
    return most;
}
__device__ __forceinline__ nbh_softmax nbh_softmax_join(nbh_softmax a, nbh_softmax b, float scale)
{
    const float peak = fmaxf(a.peak, b.peak);
    if (peak == -INFINITY)
        return {peak, a.sum + b.sum};
    return {peak, a.sum * nbh_softmax_factor(a.peak, peak, scale) + b.sum * nbh_softmax_factor(b.peak, peak, scale)};
}
// log sum exp(x / temperature)
__device__ __forceinline__ float nbh_softmax_lse(nbh_softmax s, float temperature, float scale)
{
    const float product = s.peak * scale;
    return nbh_softmax_near(product) ? (product + log2f(s.sum)) * 0.693147180559945309f
                                     : s.peak / temperature + logf(s.sum);
}
// The sum for the reference `peak`, which is not below its own.
__device__ __forceinline__ float nbh_softmax_raised(nbh_softmax s, float peak, float scale)
{
    return peak == -INFINITY ? s.sum : s.sum * nbh_softmax_factor(s.peak, peak, scale);
}
// Over a wavefront, whose lanes' sums are brought to one reference first; every lane gets the result.
__device__ __forceinline__ nbh_softmax nbh_softmax_wave(nbh_softmax s, float scale)
{
    float peak = s.peak;
    for (int step = 32; step; step >>= 1)
        peak = fmaxf(peak, __shfl_xor(peak, step));
    float sum = nbh_softmax_raised(s, peak, scale);
    for (int step = 32; step; step >>= 1)
        sum += __shfl_xor(sum, step);
    return {peak, sum};
}
// Over a workgroup of `T` lanes; `room` holds T / 64 entries.  Every lane gets the result.
template <int T>
__device__ __forceinline__ nbh_softmax nbh_softmax_group(nbh_softmax s, float scale, nbh_softmax *room)
{
    s = nbh_softmax_wave(s, scale);
    if ((threadIdx.x & 63) == 0)
        room[threadIdx.x >> 6] = s;
    __syncthreads();
    if (T == 64)
        return s;
    float peak = room[0].peak, sum = 0.0f;
    for (int w = 1; w < T / 64; ++w)
        peak = fmaxf(peak, room[w].peak);
    for (int w = 0; w < T / 64; ++w)
        sum += nbh_softmax_raised(room[w], peak, scale);
    return {peak, sum};
}

// A workgroup of T lanes goes through elements begin .. end of a row in chunks of `kNbhAhead` 16-byte
// vectors per lane, the next chunk on its way while the last is looked at: chunk(at, raw), where vector j
// of a lane starts at element at + (j T + lane) items.  What lies behind the end reads as -inf.
// Whole chunks take turns in two sets of registers, and no load in that loop is conditional: a copy from
// one set to the other, or a load on one path only, would make the compiler wait for all of them.
// BACK: from the end to the beginning, for a second reading of the row that finds the end of the first in
// the caches.
constexpr int kNbhAhead = 4;
template <typename E, int T, bool NT, bool BACK = false, typename F>
__device__ __forceinline__ void nbh_row_stream(const typename E::item *in, int64_t begin, int64_t end, F chunk)
{
    constexpr int64_t kChunk = kNbhAhead * T * E::items, kStep = BACK ? -kChunk : kChunk;
    auto ask = [&](nbh_u32x4(&to)[kNbhAhead], int64_t at) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kNbhAhead; ++j)
            to[j] = E::template load<NT>(in + at + (j * T + threadIdx.x) * E::items);
    };
    nbh_u32x4 a[kNbhAhead], b[kNbhAhead], tail[kNbhAhead];
    int64_t left = (end - begin) / kChunk;
    const int64_t rest = begin + left * kChunk;
    auto ask_tail = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < kNbhAhead; ++j)
            tail[j] = nbh_row_load_raw<E, NT>(in, rest + (j * T + threadIdx.x) * E::items, end, E::lowest);
    };
    int64_t at = BACK ? rest - kChunk : begin;
    if (BACK && rest < end)
        ask_tail();
    if (left)
        ask(a, at);
    if (BACK && rest < end)
        chunk(rest, tail);
#pragma unroll 1
    for (; left > 2; left -= 2, at += 2 * kStep) {
        ask(b, at + kStep);
        chunk(at, a);
        ask(a, at + 2 * kStep);
        chunk(at + kStep, b);
    }
    if (left == 2)
        ask(b, at + kStep);
    if (!BACK && rest < end)
        ask_tail();
    if (left)
        chunk(at, a);
    if (left == 2)
        chunk(at + kStep, b);
    if (!BACK && rest < end)
        chunk(rest, tail);
}
// N vectors of a row's statistics.
template <typename E, int N>
__device__ __forceinline__ void nbh_row_stats(nbh_softmax &stats, const nbh_u32x4 (&raw)[N], float scale)
{
#pragma unroll
    for (int j = 0; j < N; ++j) {
        float f[E::items];
        E::unpack(raw[j], f);
        nbh_softmax_add(stats, f, nbh_row_most(f), scale);
    }
}

// Temperatures whose reciprocal is an ordinary float32 number.
static inline bool nbh_row_temperature(double t) { return t >= 1e-30 && t <= 1e30; }

// 4- or 8-byte integers, as the caller's arrays hold them.
__device__ __forceinline__ int64_t nbh_row_int(const void *p, int bytes, int64_t at)
{
    return bytes == 8 ? static_cast<const int64_t *>(p)[at] : static_cast<const int32_t *>(p)[at];
}
__device__ __forceinline__ int64_t nbh_row_clamp(int64_t x, int64_t low, int64_t high)
{
    return x < low ? low : x > high ? high : x;
}
