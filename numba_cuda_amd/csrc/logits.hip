// nbh_logits_adjust: penalties for repeated tokens, biases and grammar masks on rows of logits.
//
//   seen(v)  = token v occurs in the row's history;  c(v) = how often behind the history's prompt
//   x' = seen(v) ? (x > 0 ? x / repetition : x * repetition) : x
//   x' = (x' - frequency * c(v)) - presence * [c(v) > 0]
//   x' = x' + bias(v)                      the last pair of the row that names v
//   out = v allowed by the mask ? x' : -inf
//
// A workgroup owns a tile of one row's vocabulary.  It counts the row's history into one LDS word per
// entry (bit 31: seen, below it the count) and notes the bias pairs that fall into the tile, each token
// of the history read by every tile of the row (from L2), then streams the tile once: 16 bytes per lane,
// one or two LDS reads for what the tile knows about them.  Integer LDS atomics only: the order in which
// lanes arrive changes nothing.
#include "rows.h"

namespace {

constexpr uint32_t kSeen = 0x80000000u;
constexpr int kTile = 4096;

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

// One entry, everything but the mask.
__device__ __forceinline__ float adjusted(float x, uint32_t word, float bias, bool biased, float repetition,
                                          float presence, float frequency)
{
    if (word) {
        x = x > 0.0f ? x / repetition : x * repetition;
        const uint32_t count = word & ~kSeen;
        if (count) {
            x = x - frequency * (float)count;
            x = x - presence;
        }
    }
    return biased ? x + bias : x;
}

template <typename In, typename Out, int T>
__global__ __launch_bounds__(T) void adjust_rows(Adjust a)
{
    extern __shared__ uint32_t words[];              // kTile words, then kTile pair numbers if there are biases
    constexpr int kItems = In::items;
    const int64_t row = a.row0 + blockIdx.x / a.tiles;
    const int tile = blockIdx.x % a.tiles;
    const int64_t first = (int64_t)tile * kTile;
    const int n = (int)(a.vocab - first < kTile ? a.vocab - first : kTile);
    uint32_t *const pairs = words + kTile;

    const bool history = a.tokens != nullptr, biases = a.bias_tokens != nullptr;
    if (history)
        for (int i = threadIdx.x * 4; i < kTile; i += T * 4)
            *reinterpret_cast<uint4 *>(words + i) = uint4{0, 0, 0, 0};
    if (biases)
        for (int i = threadIdx.x * 4; i < kTile; i += T * 4)
            *reinterpret_cast<uint4 *>(pairs + i) = uint4{0, 0, 0, 0};
    if (history || biases)
        __syncthreads();
    if (history) {
        const int64_t begin = nbh_row_clamp(nbh_row_int(a.offsets, a.offset_bytes, row), 0, a.n_tokens);
        const int64_t end = nbh_row_clamp(nbh_row_int(a.offsets, a.offset_bytes, row + 1), begin, a.n_tokens);
        const int64_t made =
            a.prompts ? begin + nbh_row_clamp(nbh_row_int(a.prompts, a.prompt_bytes, row), 0, end - begin) : begin;
        for (int64_t i = begin + threadIdx.x; i < end; i += T) {
            const int64_t at = nbh_row_int(a.tokens, a.token_bytes, i) - first;
            if (at >= 0 && at < n) {
                if (i >= made)
                    atomicAdd(&words[at], 1u);
                else
                    atomicOr(&words[at], kSeen);
            }
        }
    }
    int64_t pair0 = 0;
    if (biases) {
        pair0 = nbh_row_clamp(nbh_row_int(a.bias_offsets, a.bias_offset_bytes, row), 0, a.n_bias);
        const int64_t end = nbh_row_clamp(nbh_row_int(a.bias_offsets, a.bias_offset_bytes, row + 1), pair0, a.n_bias);
        for (int64_t i = pair0 + threadIdx.x; i < end; i += T) {
            const int64_t at = nbh_row_int(a.bias_tokens, a.bias_token_bytes, i) - first;
            if (at >= 0 && at < n)
                atomicMax(&pairs[at], (uint32_t)(i - pair0 + 1));
        }
    }
    if (history || biases)
        __syncthreads();

    const float repetition = a.repetition ? a.repetition[row] : a.repetition_value;
    const float presence = a.presence ? a.presence[row] : a.presence_value;
    const float frequency = a.frequency ? a.frequency[row] : a.frequency_value;
    const typename In::item *in = reinterpret_cast<const typename In::item *>(a.in + row * a.in_stride) + first;
    typename Out::item *out = reinterpret_cast<typename Out::item *>(a.out + row * a.out_stride) + first;
    const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride + first / 8 : nullptr;

    for (int at = threadIdx.x * kItems; at < n; at += T * kItems) {
        float f[kItems];
        nbh_row_load<In, true>(in, at, n, 0.0f, f);
        // bits of these entries, the first the lowest; a mask row ends with its last entry's word
        const uint32_t bits = mask ? (uint32_t)mask[at / 8] >> (at & 7) : 0xffu;
        uint32_t word[kItems], pair[kItems], any = 0;
        for (int i = 0; i < kItems; ++i) {
            word[i] = history ? words[at + i] : 0u;
            pair[i] = biases ? pairs[at + i] : 0u;
            any |= word[i] | pair[i];
        }
        if (any)
            for (int i = 0; i < kItems; ++i)
                f[i] = adjusted(f[i], word[i], pair[i] ? a.bias_values[pair0 + pair[i] - 1] : 0.0f, pair[i] != 0,
                                repetition, presence, frequency);
        for (int i = 0; i < kItems; ++i)
            f[i] = bits >> i & 1u ? f[i] : -INFINITY;
        if constexpr (Out::items == kItems) {
            nbh_row_store<Out, true>(out, at, n, f);
        } else {
            for (int h = 0; h < kItems; h += Out::items) {
                float part[Out::items];
                for (int i = 0; i < Out::items; ++i)
                    part[i] = f[h + i];
                nbh_row_store<Out, true>(out, at + h, n, part);
            }
        }
    }
}

template <typename In, typename Out>
int launch_adjust(Adjust a, int64_t rows, hipStream_t stream)
{
    const size_t lds = (size_t)kTile * 4 * ((a.tokens ? 1 : 0) + (a.bias_tokens ? 1 : 0));
    // the pair numbers follow the words in any case
    const size_t bytes = a.bias_tokens ? (size_t)kTile * 8 : lds;
    // a launch holds less than 2^32 lanes
    const int64_t most = NBH_ROW_MOST_GROUPS / a.tiles;
    for (a.row0 = 0; a.row0 < rows; a.row0 += most) {
        const int64_t groups = (rows - a.row0 < most ? rows - a.row0 : most) * a.tiles;
        adjust_rows<In, Out, 256><<<dim3((unsigned)groups), dim3(256), bytes, stream>>>(a);
        if (const int status = nbh_launch_status())
            return status;
    }
    return 0;
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
        p->vocab > INT32_MAX || p->n_tokens < 0 || p->n_tokens > INT32_MAX || p->n_bias < 0 || p->n_bias > INT32_MAX)
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
    a.tiles = (int)((p->vocab + kTile - 1) / kTile);
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
                    : launch_adjust<nbh_row_f16, nbh_row_f32>(a, p->rows, s);
    default:
        return same ? launch_adjust<nbh_row_bf16, nbh_row_bf16>(a, p->rows, s)
                    : launch_adjust<nbh_row_bf16, nbh_row_f32>(a, p->rows, s);
    }
}
