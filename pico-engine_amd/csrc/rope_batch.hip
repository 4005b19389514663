// Rotary positions of any rows at any positions, and the decode step of several sequences:
//   rope_positions  the heads of token t rotated by positions[t]
//   rope_append     the fused QKV rows of B sequences: q rotated, k rotated and v copied into row
//                   positions[b] + slot_offset of sequence b's own cache
// The pair j of a head turns by the angle t = position * f_j and grows by amp:
//   (x, y) -> (amp (x cos t - y sin t), amp (x sin t + y cos t)),
// pairs (j, j + r/2) or, interleaved, (2j, 2j + 1) of the first r elements of a head; the others stay.
//
// The angles are made here, not read: a table row costs as many bytes as half a head, and the angle
// of a far position needs more than 32 bits (at position 10^6 an fp32 product is off by 0.06).
// position * f_j / (pi/2) in 64 bits, the product's own rounding error added back, leaves the
// quarter turn and a rest in [-1/2, 1/2] whose error is that of f_j alone; sine and cosine of the
// rest are their Taylor series in 32 bits (the first terms left out are under 3e-9).
#include "rope_common.h"

namespace pe {

struct RopeArgs {
    const void* x;
    int64_t x_token, x_head;
    void* y;
    int64_t y_token, y_head;
    const void* positions;
    int wide;
    const double* freqs;
    int half, hd;  // pairs, elements of a head
    float amp;
    int n_head, groups;  // heads; a thread takes every groups-th head
    int heads_inside;    // the heads of a token lie closer together than the tokens of a head
    int64_t tokens;
};

// Item = (token, V pairs or 2 V elements that stay, group of heads), the sine and cosine for all heads of
// the group; neighbouring lanes take what is next to each other in memory. Bound by the loads and
// stores: 8191 x 16 x 64 fp32 in 12.5 us (5.4 TB/s), 65537 x 4 x 128 fp16 in
// 25.5 (5.3); with a launch's groups of heads one after the other in memory 15 and 26.
template <typename T, int V, bool IL>
__global__ __launch_bounds__(256) void k_rope_positions(RopeArgs p) {
    const int turn = (p.half + V - 1) / V, rest = (p.hd - 2 * p.half + 2 * V - 1) / (2 * V), per = turn + rest;
    const uint32_t idx = blockIdx.x * 256 + threadIdx.x;  // the launch keeps it under 2^31
    if (idx >= (uint32_t)p.tokens * (uint32_t)(per * p.groups)) return;
    const uint32_t rest1 = idx / (uint32_t)per;
    const int c = (int)(idx - rest1 * (uint32_t)per);
    const uint32_t inner = p.heads_inside ? (uint32_t)p.groups : (uint32_t)p.tokens, o = rest1 / inner, i = rest1 - o * inner;
    const int64_t t = p.heads_inside ? o : i;
    const int h0 = (int)(p.heads_inside ? i : o);
    const bool turns = c < turn;
    // first element, and how far the second V lie behind it
    const int at = turns ? (IL ? 2 * V * c : V * c) : 2 * p.half + 2 * V * (c - turn);
    const int far = turns && !IL ? p.half : V;
    const bool two = turns || at + far < p.hd;  // a last element alone
    const T* x = static_cast<const T*>(p.x) + t * p.x_token + (int64_t)h0 * p.x_head + at;
    T* y = static_cast<T*>(p.y) + t * p.y_token + (int64_t)h0 * p.y_head + at;
    SinCos w[V];
    if (turns) {
        const double pos = (double)position_of(p.positions, p.wide, t);
#pragma unroll
        for (int i = 0; i < V; ++i)
            w[i] = sincos_quarters(pos, p.freqs[V * c + i] * 0.63661977236758134, p.amp);
    }
    for (int h = h0; h < p.n_head; h += p.groups, x += p.groups * p.x_head, y += p.groups * p.y_head) {
        float a[V], b[V];
        load_vec<T, V>(x, a);
        if (two) load_vec<T, V>(x + far, b);
        if (turns) rotate<V, IL>(a, b, w);
        store_vec<T, V>(y, a);
        if (two) store_vec<T, V>(y + far, b);
    }
}

struct AppendArgs {
    const float* qkv;
    int64_t qkv_row;
    const void* positions;
    int wide;
    const double* freqs;  // or, NULL, the table rows
    const float* cos_tab;
    const float* sin_tab;
    int64_t tab_rows;
    int half, hd;
    float amp;
    int n_head, n_kv;
    float* q;
    void* k;
    void* v;
    int64_t capacity, slot_offset;
    int batch;
};

// Item = (sequence, head of q, k or v, V pairs or 2 V elements); few enough that each makes its own
// sines. Bound by latency: one chain of position, angle and store (1 sequence of 14/2 heads of 64
// 2.4 us, 96 of 28/4 heads of 128 3.3).
template <typename C, int V, bool IL>
__global__ __launch_bounds__(256) void k_rope_append(AppendArgs p) {
    const int turn = (p.half + V - 1) / V, rest = (p.hd - 2 * p.half + 2 * V - 1) / (2 * V);
    const int per = turn + rest, heads = p.n_head + 2 * p.n_kv;
    const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (idx >= (int64_t)p.batch * heads * per) return;
    const uint32_t bh = (uint32_t)idx / (uint32_t)per;
    const int c = (int)((uint32_t)idx - bh * (uint32_t)per);
    const int b = (int)(bh / (uint32_t)heads), h = (int)(bh - (uint32_t)b * heads);
    const bool turns = c < turn;
    const int at = turns ? (IL ? 2 * V * c : V * c) : 2 * p.half + 2 * V * (c - turn);
    const int far = turns && !IL ? p.half : V;
    const bool two = turns || at + far < p.hd;
    const float* x = p.qkv + (int64_t)b * p.qkv_row + (int64_t)h * p.hd + at;
    float u[V], w[V];
    load_vec<float, V>(x, u);
    if (two) load_vec<float, V>(x + far, w);
    const int64_t pos = position_of(p.positions, p.wide, b);
    if (turns && h < p.n_head + p.n_kv) {
        SinCos sc[V];
        if (p.freqs) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                sc[i] = sincos_quarters((double)pos, p.freqs[V * c + i] * 0.63661977236758134, p.amp);
        } else {
            const int64_t row = pos < 0 ? 0 : pos < p.tab_rows ? pos : p.tab_rows - 1;
#pragma unroll
            for (int i = 0; i < V; ++i)
                sc[i] = {p.sin_tab[row * p.half + V * c + i] * p.amp, p.cos_tab[row * p.half + V * c + i] * p.amp};
        }
        rotate<V, IL>(u, w, sc);
    }
    if (h < p.n_head) {
        float* y = p.q + ((int64_t)b * p.n_head + h) * p.hd + at;
        store_vec<float, V>(y, u);
        if (two) store_vec<float, V>(y + far, w);
        return;
    }
    const int64_t slot = pos + p.slot_offset;
    if (slot < 0 || slot >= p.capacity) return;  // a sequence that takes no part
    const bool isv = h >= p.n_head + p.n_kv;
    const int hh = h - p.n_head - (isv ? p.n_kv : 0);
    C* y = static_cast<C*>(isv ? p.v : p.k) + (((int64_t)b * p.n_kv + hh) * p.capacity + slot) * p.hd + at;
    store_vec<C, V>(y, u);
    if (two) store_vec<C, V>(y + far, w);
}

template <typename T>
static int launch_positions(RopeArgs p, bool vec, bool il, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int v = vec ? V : 1;
    const int64_t per = (p.half + v - 1) / v + (p.hd - 2 * p.half + 2 * v - 1) / (2 * v);
    // Heads a thread takes with one sine and cosine: as many as leave the chip about 8 waves per SIMD.
    const int64_t threads = p.tokens * per, want = (524288 + threads - 1) / threads;
    p.groups = (int)(want < p.n_head ? want : p.n_head);
    p.heads_inside = p.n_head > 1 && (p.tokens == 1 || p.x_head < p.x_token);
    const int64_t most = (1LL << 30) / (per * (int64_t)p.groups);  // tokens per launch: item numbers of 32 bits
    if (most == 0) return PE_ERR_SHAPE;
    for (int64_t t0 = 0; t0 < p.tokens; t0 += most) {
        RopeArgs a = p;
        a.tokens = p.tokens - t0 < most ? p.tokens - t0 : most;
        a.x = static_cast<const T*>(p.x) + t0 * p.x_token;
        a.y = static_cast<T*>(p.y) + t0 * p.y_token;
        a.positions = static_cast<const char*>(p.positions) + t0 * (p.wide ? 8 : 4);
        const dim3 g((unsigned)((a.tokens * per * p.groups + 255) / 256));
        if (vec && il)
            hipLaunchKernelGGL((k_rope_positions<T, V, true>), g, dim3(256), 0, s, a);
        else if (vec)
            hipLaunchKernelGGL((k_rope_positions<T, V, false>), g, dim3(256), 0, s, a);
        else if (il)
            hipLaunchKernelGGL((k_rope_positions<T, 1, true>), g, dim3(256), 0, s, a);
        else
            hipLaunchKernelGGL((k_rope_positions<T, 1, false>), g, dim3(256), 0, s, a);
    }
    return launch_status();
}

template <typename C>
static int launch_append(const AppendArgs& p, bool vec, bool il, hipStream_t s) {
    const int v = vec ? 4 : 1;
    const int64_t per = (p.half + v - 1) / v + (p.hd - 2 * p.half + 2 * v - 1) / (2 * v);
    const int64_t items = (int64_t)p.batch * (p.n_head + 2 * p.n_kv) * per;
    if (items > 0x7FFFFFFF) return PE_ERR_SHAPE;
    const dim3 g((unsigned)((items + 255) / 256));
    if (vec && il)
        hipLaunchKernelGGL((k_rope_append<C, 4, true>), g, dim3(256), 0, s, p);
    else if (vec)
        hipLaunchKernelGGL((k_rope_append<C, 4, false>), g, dim3(256), 0, s, p);
    else if (il)
        hipLaunchKernelGGL((k_rope_append<C, 1, true>), g, dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((k_rope_append<C, 1, false>), g, dim3(256), 0, s, p);
    return launch_status();
}

static size_t elem_size(int type) { return type == PE_TYPE_F16 ? 2 : 4; }

}  // namespace pe

using namespace pe;

extern "C" int pe_rope_positions(int type, const void* x, int64_t x_token, int64_t x_head, const void* positions,
                                 int pos_dtype, const double* freqs, int rot_dim, float amp, int interleaved, void* y,
                                 int64_t y_token, int64_t y_head, int64_t tokens, int n_head, int head_dim,
                                 pe_stream_t stream) {
    if ((type != PE_TYPE_F32 && type != PE_TYPE_F16) || (pos_dtype != 1 && pos_dtype != 2)) return PE_ERR_TYPE;
    if (tokens < 0 || n_head <= 0 || n_head > 4096 || head_dim <= 0 || head_dim > 65536 || rot_dim <= 0 ||
        rot_dim % 2 || rot_dim > head_dim || x_token < 0 || x_head < 0 || y_token < 0 || y_head < 0 ||
        (n_head > 1 && y_head < head_dim) || (tokens > 1 && y_token < head_dim))
        return PE_ERR_SHAPE;
    // rows of y that share memory: heads inside a token row, or tokens inside a head's rows
    if (tokens > 1 && n_head > 1 && y_token < y_head * (n_head - 1) + head_dim &&
        y_head < y_token * (tokens - 1) + head_dim)
        return PE_ERR_SHAPE;
    if (tokens == 0) return PE_OK;
    if (!x || !positions || !freqs || !y) return PE_ERR_NULL;
    // in place, every element has to stay where it is
    if (x == y && ((tokens > 1 && x_token != y_token) || (n_head > 1 && x_head != y_head))) return PE_ERR_SHAPE;
    const size_t e = elem_size(type);
    if (!aligned(x, e) || !aligned(y, e) || !aligned(positions, pos_dtype == 2 ? 8 : 4) || !aligned(freqs, 8))
        return PE_ERR_ALIGN;
    RopeArgs p{x, x_token, x_head, y, y_token, y_head, positions, pos_dtype == 2, freqs, rot_dim / 2, head_dim, amp,
               n_head, 1, 0, tokens};
    // 16 bytes at a time where every piece of a row is whole and aligned, else single elements (65536 x 4 heads of 80:
    // 20 rotated 39 to 41 us in fp32, 4.2 TB/s, 28 to 29 in fp16, 2.9; all 80 rotated 16.5 to 17 in fp16, 5.0)
    const int v = (int)(16 / e);
    const int64_t strides = x_token | x_head | y_token | y_head;
    const bool vec = (interleaved ? rot_dim % (2 * v) == 0 : rot_dim / 2 % v == 0) && head_dim % v == 0 &&
                     strides % v == 0 && aligned(x, 16) && aligned(y, 16);
    hipStream_t s = (hipStream_t)stream;
    return type == PE_TYPE_F16 ? launch_positions<_Float16>(p, vec, interleaved, s)
                               : launch_positions<float>(p, vec, interleaved, s);
}

extern "C" int pe_rope_append(const float* qkv, int64_t qkv_stride, const void* positions, int pos_dtype,
                              const double* freqs, const float* cos_tab, const float* sin_tab, int64_t tab_rows,
                              int rot_dim, float amp, int interleaved, int n_head, int n_kv, int head_dim,
                              int64_t batch, float* q_out, int cache_type, void* k_cache, void* v_cache,
                              int64_t capacity, int64_t slot_offset, pe_stream_t stream) {
    if ((cache_type != PE_TYPE_F32 && cache_type != PE_TYPE_F16) || (pos_dtype != 1 && pos_dtype != 2))
        return PE_ERR_TYPE;
    if (batch < 0 || batch > 0x7FFFFFFF || n_head <= 0 || n_kv <= 0 || n_head > 65535 || n_kv > 65535 ||
        head_dim <= 0 || head_dim > 65536 || rot_dim <= 0 || rot_dim % 2 || rot_dim > head_dim || capacity <= 0 ||
        capacity > (1LL << 40) || qkv_stride < (int64_t)(n_head + 2 * n_kv) * head_dim ||
        (!freqs && tab_rows <= 0))
        return PE_ERR_SHAPE;
    if (batch == 0) return PE_OK;
    if (!qkv || !positions || (!freqs && (!cos_tab || !sin_tab)) || !q_out || !k_cache || !v_cache)
        return PE_ERR_NULL;
    const size_t e = elem_size(cache_type);
    if (!aligned(qkv, 4) || !aligned(q_out, 4) || !aligned(k_cache, e) || !aligned(v_cache, e) ||
        !aligned(positions, pos_dtype == 2 ? 8 : 4) || !aligned(freqs, 8) || !aligned(cos_tab, 4) || !aligned(sin_tab, 4))
        return PE_ERR_ALIGN;
    AppendArgs p{qkv, qkv_stride, positions, pos_dtype == 2, freqs, cos_tab, sin_tab, tab_rows, rot_dim / 2, head_dim,
                 amp, n_head, n_kv, q_out, k_cache, v_cache, capacity, slot_offset, (int)batch};
    const bool vec = (interleaved ? rot_dim % 8 == 0 : rot_dim / 2 % 4 == 0) && head_dim % 4 == 0 &&
                     qkv_stride % 4 == 0 && aligned(qkv, 16) && aligned(q_out, 16) && aligned(k_cache, 4 * e) &&
                     aligned(v_cache, 4 * e);
    hipStream_t s = (hipStream_t)stream;
    return cache_type == PE_TYPE_F16 ? launch_append<_Float16>(p, vec, interleaved, s)
                                     : launch_append<float>(p, vec, interleaved, s);
}
