// nbh_logits_adjust: penalties for repeated tokens, biases and grammar masks on rows of logits.
//
//   seen(v)  = token v occurs in the row's history;  c(v) = how often behind the history's prompt
//   x' = seen(v) ? (x > 0 ? x / repetition : x * repetition) : x
//   x' = (x' - frequency * c(v)) - presence * [c(v) > 0]
//   x' = x' + bias(v)                      the last pair of the row that names v
//   out = v allowed by the mask ? x' : -inf
//
// A workgroup owns a tile of one row's vocabulary.  It asks for the tile's logits and mask first and
// counts the row's history into one LDS word per entry (below) while they are on their way; every tile of
// a row reads the whole history, from L2.  The bias pairs leave the largest of their numbers in the same words
// afterwards (in words of their own, 256 x 131072 with 64 pairs took 60 us instead of 45, as half as many
// workgroups fit a compute unit).  Integer LDS atomics only: the order in which lanes arrive changes nothing.
//
// Bound by memory where rows are many, by the start of a launch and the walk through the history where they are
// few.  256 x 131072 bfloat16 to float32 with masks, 64 biases and histories of 4096 a row: 42 us, its 208 MB at
// 4.9 TB/s (72 us while results of four bytes left a lane in two stores 16 bytes apart, hence the half vectors; 98
// us with inputs read past the caches).  8 x 131072 float32 with histories of 131071: 15.5 us, each tile's walk.
#include "rows.h"

namespace {

// The word of an entry: bit 31 it occurs in the history, below it how often it occurs behind the prompt; then
// again, one more than the number of the last pair that names it.
constexpr uint32_t kSeen = 0x80000000u, kCount = 0x7fffffffu;

struct Adjust {
    const char *in;
    char *out;
    int64_t in_stride, out_stride, vocab, row0;
    int tiles;
    const void *tokens, *offsets, *prompts;
    int token_bytes, offset_bytes, prompt_bytes;
    int64_t n_tokens;
    const float *repetition, *presence, *frequency;
    float repetition_value, presence_value, frequency_value;
    const void *bias_tokens, *bias_offsets;
    const float *bias_values;
    int bias_token_bytes, bias_offset_bytes;
    int64_t n_bias;
    const uint8_t *mask;
    int64_t mask_stride;
};

// The integers p[0 .. count), 16 bytes per lane and load, four loads on their way at a time:
// visit(v - first, number) for every v in [first, first + n).
template <int T, typename I, typename F>
__device__ __forceinline__ void visit_tokens(const I *p, int count, int64_t first, uint32_t n, F visit)
{
    constexpr int kEach = 16 / sizeof(I), kAhead = 4;
    auto use = [&](nbh_u32x4 v, int at) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if constexpr (sizeof(I) == 4) {
                const uint32_t t = v[i] - (uint32_t)first;
                if (t < n)
                    visit(t, at + i);
            } else {
                const uint64_t t = ((uint64_t)v[2 * i + 1] << 32 | v[2 * i]) - (uint64_t)first;
                if (t < n)
                    visit((uint32_t)t, at + i);
            }
        }
    };
    int base = 0;                        // of the workgroup
    for (; base + kAhead * T * kEach <= count; base += kAhead * T * kEach) {
        nbh_u32x4 v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            v[j] = nbh_load16<sizeof(I), false>(p + base + (j * T + threadIdx.x) * kEach);
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            use(v[j], base + (j * T + threadIdx.x) * kEach);
    }
    for (int at = base + threadIdx.x * kEach; at < count; at += T * kEach) {
        if (at + kEach <= count) {
            use(nbh_load16<sizeof(I), false>(p + at), at);
        } else {
            for (int i = at; i < count; ++i) {
                const uint64_t t = (uint64_t)((int64_t)p[i] - first);
                if (t < n)
                    visit((uint32_t)t, i);
            }
        }
    }
}
template <int T, typename F>
__device__ __forceinline__ void visit_tokens(const void *p, int bytes, int64_t begin, int64_t end, int64_t first,
                                             uint32_t n, F visit)
{
    if (bytes == 4)
        visit_tokens<T>(static_cast<const int32_t *>(p) + begin, (int)(end - begin), first, n, visit);
    else
        visit_tokens<T>(static_cast<const int64_t *>(p) + begin, (int)(end - begin), first, n, visit);
}

template <typename In, typename Out, int T, int TILE, bool BIASES>
__global__ __launch_bounds__(T) void adjust_rows(Adjust a)
{
    constexpr int kItems = In::items, kVecs = TILE / (T * kItems);
    static_assert(Out::items == kItems, "as many entries per vector on both sides");
    __shared__ uint32_t words[TILE];
    // Rows first (8 x 131072 float32, histories of 131071: 15.5 us, tiles first 16.8; 64 x 50021 float16 7.9 and
    // 8.7; 256 x 131072 42 either way).
    const uint32_t now = gridDim.x / a.tiles;
    const int64_t row = a.row0 + blockIdx.x % now;
    const int tile = blockIdx.x / now;
    const int64_t first = (int64_t)tile * TILE;
    const int n = (int)(a.vocab - first < TILE ? a.vocab - first : TILE);

    const typename In::item *in = reinterpret_cast<const typename In::item *>(a.in + row * a.in_stride) + first;
    const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride + first / 8 : nullptr;
    nbh_u32x4 raw[kVecs];
    uint32_t bits[kVecs];
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
        const int at = (j * T + threadIdx.x) * kItems;
        raw[j] = nbh_row_load_raw<In, false>(in, at, n, 0);
        // bits of these entries, the first the lowest; a mask row ends with its last entry's word
        bits[j] = mask && at < n ? (uint32_t)mask[at / 8] >> (at & 7) : 0xffu;
    }

    // everything about the row, asked for at once
    const bool history = a.tokens != nullptr;
    int64_t begin = 0, end = 0, prompt_length = 0, pair0 = 0, pair1 = 0;
    if (history) {
        begin = nbh_row_int(a.offsets, a.offset_bytes, row);
        end = nbh_row_int(a.offsets, a.offset_bytes, row + 1);
        prompt_length = a.prompts ? nbh_row_int(a.prompts, a.prompt_bytes, row) : 0;
    }
    if (BIASES) {
        pair0 = nbh_row_int(a.bias_offsets, a.bias_offset_bytes, row);
        pair1 = nbh_row_int(a.bias_offsets, a.bias_offset_bytes, row + 1);
    }
    const float repetition = a.repetition ? a.repetition[row] : a.repetition_value;
    const float presence = a.presence ? a.presence[row] : a.presence_value;
    const float frequency = a.frequency ? a.frequency[row] : a.frequency_value;
    auto clear = [&]() {
        for (int i = threadIdx.x * 4; i < TILE; i += T * 4)
            *reinterpret_cast<uint4 *>(words + i) = uint4{0, 0, 0, 0};
        __syncthreads();
    };
    float f[kVecs][kItems];
    if (history) {
        clear();
        begin = nbh_row_clamp(begin, 0, a.n_tokens);
        end = nbh_row_clamp(end, begin, a.n_tokens);
        const int prompt = (int)nbh_row_clamp(prompt_length, 0, end - begin);
        visit_tokens<T>(a.tokens, a.token_bytes, begin, end, first, n, [&](uint32_t t, int i) {
            if (i < prompt)
                atomicOr(&words[t], kSeen);
            else
                atomicAdd(&words[t], 1u);
        });
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
        const int at = (j * T + threadIdx.x) * kItems;
        In::unpack(raw[j], f[j]);
        if (!history || at >= n)
            continue;
        uint32_t word[kItems], any = 0;
        for (int i = 0; i < kItems; ++i) {
            word[i] = words[at + i];
            any |= word[i];
        }
        if (any)
            for (int i = 0; i < kItems; ++i) {
                if (!word[i])
                    continue;
                const uint32_t count = word[i] & kCount;
                float x = f[j][i];
                x = x > 0.0f ? x / repetition : x * repetition;
                if (count) {
                    x = x - frequency * (float)count;
                    x = x - presence;
                }
                f[j][i] = x;
            }
    }
    if (BIASES) {
        if (history)
            __syncthreads();             // the words have been read
        clear();
        pair0 = nbh_row_clamp(pair0, 0, a.n_bias);
        pair1 = nbh_row_clamp(pair1, pair0, a.n_bias);
        visit_tokens<T>(a.bias_tokens, a.bias_token_bytes, pair0, pair1, first, n,
                        [&](uint32_t t, int i) { atomicMax(&words[t], (uint32_t)i + 1); });
        __syncthreads();
    }

    typename Out::item *out = reinterpret_cast<typename Out::item *>(a.out + row * a.out_stride) + first;
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
        const int at = (j * T + threadIdx.x) * kItems;
        if (at >= n)
            break;
        if (BIASES) {
            uint32_t pair[kItems], any = 0;
            for (int i = 0; i < kItems; ++i) {
                pair[i] = words[at + i];
                any |= pair[i];
            }
            if (any) {
                float bias[kItems];      // all on their way at once; there is at least one pair
                for (int i = 0; i < kItems; ++i)
                    bias[i] = a.bias_values[pair[i] ? pair0 + pair[i] - 1 : 0];
                for (int i = 0; i < kItems; ++i)
                    f[j][i] = pair[i] ? f[j][i] + bias[i] : f[j][i];
            }
        }
        for (int i = 0; i < kItems; ++i)
            f[j][i] = bits[j] >> i & 1u ? f[j][i] : -INFINITY;
        nbh_row_store<Out, true>(out, at, n, f[j]);
    }
}

template <typename In, typename Out, int T, int TILE>
int launch_adjust(Adjust a, int64_t rows, hipStream_t stream)
{
    a.tiles = (int)((a.vocab + TILE - 1) / TILE);
    // a launch holds less than 2^32 lanes
    const int64_t most = NBH_ROW_MOST_GROUPS / a.tiles;
    for (a.row0 = 0; a.row0 < rows; a.row0 += most) {
        const int64_t groups = (rows - a.row0 < most ? rows - a.row0 : most) * a.tiles;
        if (a.bias_tokens)
            adjust_rows<In, Out, T, TILE, true><<<dim3((unsigned)groups), dim3(T), 0, stream>>>(a);
        else
            adjust_rows<In, Out, T, TILE, false><<<dim3((unsigned)groups), dim3(T), 0, stream>>>(a);
        if (const int status = nbh_launch_status())
            return status;
    }
    return 0;
}
template <typename In, typename Out>
int launch_adjust(const Adjust &a, int64_t rows, hipStream_t stream)
{
    // Every tile of a row reads the whole history, so long ones are read by fewer, larger workgroups; they start
    // and end less evenly.  256 x 4096 against 1024 x 8192 on rows of 131072 bfloat16, mean history 8192: 64 rows
    // 17.4 and 18.9 us, 256 rows 48 and 55; 16384: 64 rows 22.8 and 20.6, 256 rows 62 and 64; 65536: 1 row 34 and
    // 16, 64 rows 64 and 40, 256 rows 164 and 125.  (8 rows of 131072 float32, 65536: tiles of 16384 18.8 us, of
    // 8192 16.7, of 32768 21.9.)
    // Only the mean is known here, the lengths are on the device.  One history of 131071 among rows of 100 tokens
    // waits for its 32 workgroups: 16 rows 32 and 14.5 us, 64 rows 67 and 31, 256 rows 69 and 47; of 16384 64 rows
    // 14.5 and 12.9, 256 rows 24 and 30.
    if (a.n_tokens / rows > 12288)
        return launch_adjust<In, Out, 1024, 8192>(a, rows, stream);
    return launch_adjust<In, Out, 256, 4096>(a, rows, stream);
}

}  // namespace

extern "C" int nbh_logits_adjust(const struct nbh_logits_adjust_args *p, nbh_stream_t stream)
{
    if (!p || p->struct_bytes != (int64_t)sizeof(*p) || p->rows < 0 || p->vocab < 0)
        return (int)hipErrorInvalidValue;
    if (p->rows == 0 || p->vocab == 0)
        return 0;
    const bool same = p->out_dtype == p->dtype;
    if (!p->logits || !p->out || p->dtype < 0 || p->dtype > NBH_ROW_BF16 || !(same || p->out_dtype == NBH_ROW_F32) ||
        p->vocab > INT32_MAX || p->n_tokens < 0 || p->n_tokens >= (1 << 30) || p->n_bias < 0 || p->n_bias >= (1 << 30))
        return (int)hipErrorInvalidValue;
    auto width = [](int64_t b) { return b == 4 || b == 8; };
    const bool history = p->tokens && p->n_tokens, biases = p->bias_tokens && p->n_bias;
    if (history && (!p->offsets || !width(p->token_bytes) || !width(p->offset_bytes) ||
                    (p->prompts && !width(p->prompt_bytes))))
        return (int)hipErrorInvalidValue;
    if (biases && (!p->bias_offsets || !p->bias_values || !width(p->bias_token_bytes) || !width(p->bias_offset_bytes)))
        return (int)hipErrorInvalidValue;
    Adjust a = {};
    a.in = (const char *)p->logits;
    a.out = (char *)p->out;
    a.in_stride = p->in_stride;
    a.out_stride = p->out_stride;
    a.vocab = p->vocab;
    if (history) {
        a.tokens = p->tokens;
        a.offsets = p->offsets;
        a.prompts = p->prompts;
        a.token_bytes = (int)p->token_bytes;
        a.offset_bytes = (int)p->offset_bytes;
        a.prompt_bytes = (int)p->prompt_bytes;
        a.n_tokens = p->n_tokens;
    }
    a.repetition = p->repetition;
    a.presence = p->presence;
    a.frequency = p->frequency;
    a.repetition_value = (float)p->repetition_value;
    a.presence_value = (float)p->presence_value;
    a.frequency_value = (float)p->frequency_value;
    if (biases) {
        a.bias_tokens = p->bias_tokens;
        a.bias_offsets = p->bias_offsets;
        a.bias_values = p->bias_values;
        a.bias_token_bytes = (int)p->bias_token_bytes;
        a.bias_offset_bytes = (int)p->bias_offset_bytes;
        a.n_bias = p->n_bias;
    }
    a.mask = (const uint8_t *)p->mask;
    a.mask_stride = p->mask_stride;

    const hipStream_t s = nbh_hip_stream(stream);
    nbh_stream_report report(s);
    switch (p->dtype) {
    case NBH_ROW_F32:
        return launch_adjust<nbh_row_f32, nbh_row_f32>(a, p->rows, s);
    case NBH_ROW_F16:
        return same ? launch_adjust<nbh_row_f16, nbh_row_f16>(a, p->rows, s)
                    : launch_adjust<nbh_row_half<nbh_row_f16>, nbh_row_f32>(a, p->rows, s);
    default:
        return same ? launch_adjust<nbh_row_bf16, nbh_row_bf16>(a, p->rows, s)
                    : launch_adjust<nbh_row_half<nbh_row_bf16>, nbh_row_f32>(a, p->rows, s);
    }
}
