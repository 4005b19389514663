// Rules on the logits of a batch before its tokens are picked: for row b and token v, with c the
// times v stands in the row's history,
//   z = x + bias[v];  z = z > 0 ? z / repetition : z * repetition  where v is in the history or the prompt;
//   z -= c * frequency + (c > 0) * presence;  z = -inf where v's mask bit is 0.
//
// A workgroup takes one segment of one row's vocabulary: it counts the segment's tokens of the
// history and the prompt in LDS (whole-number additions, so their order does not matter), while its
// logits are on their way, and stores the segment. One launch, nothing kept between calls. Bound by
// reading and writing the logits once (from memory: 256 rows of 151643 fp16 31.4 us, 5.0 TB/s, of 151936 fp32 57,
// 5.4), by latency for a row or two (3.5 us), and where the ids are many by looking through them: every segment
// of a row reads all of them (from L2), a few 32-bit instructions each (24 rows of 152064 with 4000 + 770
// ids: 9.9 us, 4.8 without; 8 rows with 30000: 11). Compared as 64-bit integers the ids cost twice as much;
// counters looked at one by one where the vector's were all zero cost 256 rows 4 us more.
#include "pe_common.h"

namespace pe {

constexpr uint32_t kInPrompt = 0x80000000u;  // the counter's top bit; counts stay below it

struct LogitArgs {
    const void* x;
    int64_t x_row;
    void* y;
    int64_t y_row;
    int64_t vocab;
    const void* history;  // row b at b * history_row ids
    int64_t history_row, history_len;
    const void* lengths;  // NULL: history_len ids in every row
    const void* prompt;
    int64_t prompt_row, prompt_len;
    int ids_wide, lengths_wide, prompt_wide;
    const float* rules[3];  // repetition, frequency, presence of each row, or NULL
    float rule[3];
    const float* bias;
    int64_t bias_row;
    const uint32_t* mask;
    int64_t mask_row;
};

// Loads and stores of whole vectors at the element's own alignment (rows of an odd vocabulary).
template <typename T, int V>
struct Loose {
    typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};

PE_DEV int64_t id_at(const void* ids, int wide, int64_t i) {
    return wide ? static_cast<const int64_t*>(ids)[i] : (int64_t) static_cast<const int*>(ids)[i];
}

// Adds to, or marks, the counters of the ids in [v0, v0 + seg): two ids a load, four of them in flight.
// An id under 0 has a high word, or is over every segment.
template <bool MARK, typename I>
PE_DEV void count_ids(uint32_t* count, const I* ids, int64_t n, uint32_t v0, uint32_t seg) {
    constexpr int U = 4;
    typedef typename Loose<I, 2>::type pair;
    const auto one = [&](I id) {
        const uint32_t o = (uint32_t)id - v0;
        if (o >= seg || (sizeof(I) == 8 && (uint64_t)id >> 32)) return;
        if constexpr (MARK)
            atomicOr(&count[o], kInPrompt);
        else
            atomicAdd(&count[o], 1u);
    };
    int64_t i = 2 * threadIdx.x;
    for (; i + 512 * (U - 1) + 2 <= n; i += 512 * U) {
        pair id[U];
#pragma unroll
        for (int u = 0; u < U; ++u) id[u] = *reinterpret_cast<const pair*>(ids + i + 512 * u);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            one(id[u].x);
            one(id[u].y);
        }
    }
    // under 512 U left: all of a thread's in flight again
    pair id[U - 1];
#pragma unroll
    for (int u = 0; u < U - 1; ++u) {
        const int64_t at = i + 512 * u;
        id[u] = pair{(I)-1, (I)-1};
        if (at + 2 <= n)
            id[u] = *reinterpret_cast<const pair*>(ids + at);
        else if (at < n)
            id[u].x = ids[at];
    }
#pragma unroll
    for (int u = 0; u < U - 1; ++u) {
        one(id[u].x);
        one(id[u].y);
    }
    for (i += 512 * (U - 1); i < n; i += 512) one(ids[i]);  // at most one id
}
template <bool MARK>
PE_DEV void count_ids(uint32_t* count, const void* ids, int wide, int64_t at, int64_t n, uint32_t v0, uint32_t seg) {
    if (wide)
        count_ids<MARK>(count, static_cast<const int64_t*>(ids) + at, n, v0, seg);
    else
        count_ids<MARK>(count, static_cast<const int*>(ids) + at, n, v0, seg);
}

template <typename T, int STEPS>
__global__ __launch_bounds__(256) void k_adjust_logits(LogitArgs p) {
    constexpr int V = 16 / sizeof(T), SEG = 256 * V * STEPS;
    typedef typename Loose<T, V>::type vec;
    typedef typename Loose<float, 4>::type vec4;
    __shared__ __attribute__((aligned(16))) uint32_t count[SEG];
    const int t = threadIdx.x;
    const int64_t b = blockIdx.y, v0 = (int64_t)blockIdx.x * SEG;
    const T* x = static_cast<const T*>(p.x) + b * p.x_row;
    T* y = static_cast<T*>(p.y) + b * p.y_row;
    const bool ids = p.history || p.prompt;
    // everything the segment needs is on its way before the ids are counted
    vec r[STEPS];
    float bias[STEPS][V];
    uint32_t mask[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int64_t v = v0 + (int64_t)(s * 256 + t) * V;
        if (v + V <= p.vocab) {
            r[s] = *reinterpret_cast<const vec*>(x + v);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) r[s][i] = v + i < p.vocab ? x[v + i] : (T)0.f;
        }
        if (p.bias) {
            const float* from = p.bias + b * p.bias_row + v;
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                vec4 w = {0.f, 0.f, 0.f, 0.f};
                if (v + V <= p.vocab) {
                    w = *reinterpret_cast<const vec4*>(from + i);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[k] = v + i + k < p.vocab ? from[i + k] : 0.f;
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) bias[s][i + k] = w[k];
            }
        }
        // V divides 32: the elements of a vector share a word
        mask[s] = p.mask && v < p.vocab ? p.mask[b * p.mask_row + (v >> 5)] >> (v & 31) : 0xFFFFFFFFu;
    }
    const float rep = p.rules[0] ? p.rules[0][b] : p.rule[0];
    const float freq = p.rules[1] ? p.rules[1][b] : p.rule[1];
    const float pres = p.rules[2] ? p.rules[2][b] : p.rule[2];
    if (ids) {
#pragma unroll
        for (int i = 0; i < SEG; i += 1024) *reinterpret_cast<uint4*>(count + i + 4 * t) = make_uint4(0, 0, 0, 0);
        __syncthreads();
        if (p.prompt)
            count_ids<true>(count, p.prompt, p.prompt_wide, b * p.prompt_row, p.prompt_len, (uint32_t)v0, SEG);
        if (p.history) {
            int64_t n = p.history_len;
            if (p.lengths) {
                const int64_t l = id_at(p.lengths, p.lengths_wide, b);
                n = l < 0 ? 0 : l < n ? l : n;
            }
            count_ids<false>(count, p.history, p.ids_wide, b * p.history_row, n, (uint32_t)v0, SEG);
        }
        __syncthreads();
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int o = (s * 256 + t) * V;
        const int64_t v = v0 + o;
        if (v >= p.vocab) break;
        const bool whole = v + V <= p.vocab;
        float z[V];
#pragma unroll
        for (int i = 0; i < V; ++i) z[i] = (float)r[s][i];
        if (p.bias) {
#pragma unroll
            for (int i = 0; i < V; ++i) z[i] += bias[s][i];
        }
        if (ids) {
            uint32_t c[V], any = 0;
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                const uint4 x = *reinterpret_cast<const uint4*>(count + o + i);
                c[i] = x.x, c[i + 1] = x.y, c[i + 2] = x.z, c[i + 3] = x.w;
                any |= x.x | x.y | x.z | x.w;
            }
            if (any) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (!c[i]) continue;
                    z[i] = z[i] > 0.f ? z[i] / rep : z[i] * rep;
                    const uint32_t n = c[i] & ~kInPrompt;
                    if (n) z[i] = (z[i] - freq * (float)n) - pres;
                }
            }
        }
        if (p.mask) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (!(mask[s] >> i & 1)) z[i] = -__builtin_huge_valf();
        }
        if (whole) {
            vec h;
#pragma unroll
            for (int i = 0; i < V; ++i) h[i] = (T)z[i];
            *reinterpret_cast<vec*>(y + v) = h;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (v + i < p.vocab) y[v + i] = (T)z[i];
        }
    }
}

template <typename T>
static int launch_logits(const LogitArgs& p, int64_t batch, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    // Segments of 8 KB, or of a vector a thread where those leave fewer than two workgroups per CU. Longer
    // ones read the ids less often but wait longer for them, shorter ones have too few bytes on their way (us
    // at 4 | 8 | 16 KB, from memory: 256 rows of 151643 fp16 and 300 ids 38 | 34 | 43; at 8 | 16 | 32 KB, 256 rows of 151936
    // fp32 and 300 ids 57 | 63 | 69, 24 rows of 152064 and 4770 ids 9.9 | 9.3 | 12.5, 8 rows and 30000 ids 11 | 14 | 14).
    constexpr int kLong = 2;
    const auto blocks = [&](int steps) { return (p.vocab + 256 * V * steps - 1) / (256 * V * steps); };
    const bool many = batch * blocks(kLong) >= 512;
    // rows per launch: grid.y's limit, and 2^32 threads in a grid
    int64_t most = (1 << 23) / blocks(many ? kLong : 1);
    most = most < 1 ? 1 : most > 65535 ? 65535 : most;
    for (int64_t b0 = 0; b0 < batch; b0 += most) {
        LogitArgs a = p;
        const int64_t n = batch - b0 < most ? batch - b0 : most;
        a.x = static_cast<const T*>(p.x) + b0 * p.x_row;
        a.y = static_cast<T*>(p.y) + b0 * p.y_row;
        if (p.history) a.history = static_cast<const char*>(p.history) + b0 * p.history_row * (p.ids_wide ? 8 : 4);
        if (p.lengths) a.lengths = static_cast<const char*>(p.lengths) + b0 * (p.lengths_wide ? 8 : 4);
        if (p.prompt) a.prompt = static_cast<const char*>(p.prompt) + b0 * p.prompt_row * (p.prompt_wide ? 8 : 4);
        for (int i = 0; i < 3; ++i)
            if (p.rules[i]) a.rules[i] = p.rules[i] + b0;
        if (p.bias) a.bias = p.bias + b0 * p.bias_row;
        if (p.mask) a.mask = p.mask + b0 * p.mask_row;
        if (many)
            hipLaunchKernelGGL((k_adjust_logits<T, kLong>), dim3((unsigned)blocks(kLong), (unsigned)n), dim3(256), 0, s, a);
        else
            hipLaunchKernelGGL((k_adjust_logits<T, 1>), dim3((unsigned)blocks(1), (unsigned)n), dim3(256), 0, s, a);
    }
    return launch_status();
}

}  // namespace pe

using namespace pe;

extern "C" int pe_adjust_logits(const pe_logit_args* a, pe_stream_t stream) {
    if (!a) return PE_ERR_NULL;
    if (a->type != PE_TYPE_F32 && a->type != PE_TYPE_F16) return PE_ERR_TYPE;
    const auto ids_ok = [](const void* ids, int dtype) { return !ids || dtype == 1 || dtype == 2; };
    if (!ids_ok(a->history, a->history_dtype) || !ids_ok(a->lengths, a->lengths_dtype) ||
        !ids_ok(a->prompt, a->prompt_dtype))
        return PE_ERR_TYPE;
    if (a->batch < 0 || a->vocab <= 0 || a->vocab > 0x7FFFFFFF || (a->batch > 1 && a->y_stride < a->vocab) ||
        a->x_stride < 0 || a->history_len < 0 || a->history_len > 0x7FFFFFFF || a->prompt_len < 0 ||
        a->prompt_len > 0x7FFFFFFF || a->history_stride < 0 || a->prompt_stride < 0 || a->bias_stride < 0 ||
        a->mask_stride < 0)
        return PE_ERR_SHAPE;
    if (a->batch == 0) return PE_OK;
    if (!a->x || !a->y) return PE_ERR_NULL;
    if (a->x == a->y && a->batch > 1 && a->x_stride != a->y_stride) return PE_ERR_SHAPE;  // in place: the rows stay
    const size_t e = a->type == PE_TYPE_F16 ? 2 : 4;
    const auto wide = [](int dtype) { return dtype == 2; };
    if (!aligned(a->x, e) || !aligned(a->y, e) || !aligned(a->history, wide(a->history_dtype) ? 8 : 4) ||
        !aligned(a->lengths, wide(a->lengths_dtype) ? 8 : 4) || !aligned(a->prompt, wide(a->prompt_dtype) ? 8 : 4) ||
        !aligned(a->repetition_rows, 4) || !aligned(a->frequency_rows, 4) || !aligned(a->presence_rows, 4) ||
        !aligned(a->bias, 4) || !aligned(a->mask, 4))
        return PE_ERR_ALIGN;
    LogitArgs p{a->x, a->x_stride, a->y, a->y_stride, a->vocab,
                a->history_len ? a->history : nullptr, a->history_stride, a->history_len, a->lengths,
                a->prompt_len ? a->prompt : nullptr, a->prompt_stride, a->prompt_len,
                wide(a->history_dtype), wide(a->lengths_dtype), wide(a->prompt_dtype),
                {a->repetition_rows, a->frequency_rows, a->presence_rows},
                {a->repetition, a->frequency, a->presence},
                a->bias, a->bias_stride, static_cast<const uint32_t*>(a->mask), a->mask_stride};
    hipStream_t s = (hipStream_t)stream;
    return a->type == PE_TYPE_F16 ? launch_logits<_Float16>(p, a->batch, s) : launch_logits<float>(p, a->batch, s);
}
