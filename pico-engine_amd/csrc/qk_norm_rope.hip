// Norms of the query and key heads with their rotary positions in one pass: head x of token t
//   y = turn(x * w / sqrt(mean(x^2) + eps), positions[t])
// with the rotation of rope_positions (angles made in 64 bits) and one weight an element, or per head and
// element. The mean is a sum over the lanes of a group that holds the head in registers, so a head is read
// and written once.
#include "rope_common.h"

namespace pe {

struct NormSide {
    const void* x;
    int64_t x_token, x_head;
    void* y;
    int64_t y_token, y_head;
    const float* w;  // NULL: no norm
    int64_t w_head;
};

struct QkNormArgs {
    NormSide q, k;
    const void* positions;
    int wide;
    const double* freqs;
    int half, hd;
    float amp, eps;
    int n_head, heads;  // query heads, all heads
    int groups;         // a group of lanes takes every groups-th head of its token
    int64_t tokens;
};

template <int W>
PE_DEV float lanes_sum(float v) {
    if constexpr (W >= 16) {
        v = wave_sum<W>(v);
    } else {
        v += dpp_mov<0xB1>(v);                         // quad_perm [1,0,3,2]
        v += dpp_mov<0x4E>(v);                         // quad_perm [2,3,0,1]
        if constexpr (W == 8) v += dpp_mov<0x141>(v);  // row_half_mirror
    }
    return v;
}

// V weights, 16 bytes at a time where the rows go so (the caller sees to the alignment then).
template <int V>
PE_DEV void load_weights(const float* w, float* v) {
    if constexpr (V == 1) {
        v[0] = w[0];
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4) load_vec<float, 4>(w + i, v + i);
    }
}

// A group of W lanes holds a head, a lane NI pieces of V pairs or of 2 V elements that stay. Bound by memory: 8191 x 40 heads
// of 128, fp16, 168 MB, 38 us, 4.4 TB/s (45.8 us without the next head under way); one token 3.1 us, the launch and its loads.
template <typename T, int V, bool IL, int W, int NI>
__global__ __launch_bounds__(256) void k_qk_norm_rope(QkNormArgs p) {
    const int turn = (p.half + V - 1) / V, per = turn + (p.hd - 2 * p.half + 2 * V - 1) / (2 * V);
    const int64_t item = (int64_t)blockIdx.x * (256 / W) + threadIdx.x / W;
    const int lane = threadIdx.x % W;
    const int64_t t = item / p.groups;
    const int h0 = (int)(item - t * p.groups);
    if (t >= p.tokens) return;
    const double pos = (double)position_of(p.positions, p.wide, t);
    int at[NI], far[NI];
    bool one[NI], two[NI], turns[NI];
    SinCos sc[NI][V];
#pragma unroll
    for (int n = 0; n < NI; ++n) {
        const int c = lane + W * n;
        turns[n] = c < turn;
        at[n] = turns[n] ? (IL ? 2 * V * c : V * c) : 2 * p.half + 2 * V * (c - turn);
        far[n] = turns[n] && !IL ? p.half : V;
        one[n] = c < per;
        two[n] = one[n] && (turns[n] || at[n] + far[n] < p.hd);
        if (turns[n]) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                sc[n][i] = sincos_quarters(pos, p.freqs[V * c + i] * 0.63661977236758134, p.amp);
        }
    }
    const float inv_hd = 1.0f / (float)p.hd;
    const auto side = [&](int h) -> const NormSide& { return h < p.n_head ? p.q : p.k; };
    const auto load = [&](int h, float (&a)[NI][V], float (&b)[NI][V]) {
        const NormSide& s = side(h);
        const T* x = static_cast<const T*>(s.x) + t * s.x_token + (h < p.n_head ? h : h - p.n_head) * s.x_head;
#pragma unroll
        for (int n = 0; n < NI; ++n) {
#pragma unroll
            for (int i = 0; i < V; ++i) a[n][i] = b[n][i] = 0.f;
            if (one[n]) load_vec<T, V>(x + at[n], a[n]);
            if (two[n]) load_vec<T, V>(x + at[n] + far[n], b[n]);
        }
    };
    float a[NI][V], b[NI][V], wa[NI][V], wb[NI][V];
    const float* held = nullptr;  // the weights in wa, wb
    load(h0, a, b);
    for (int h = h0; h < p.heads; h += p.groups) {
        // the next head is under way while this one is summed up and turned
        float na[NI][V], nb[NI][V];
        if (h + p.groups < p.heads) load(h + p.groups, na, nb);
        const NormSide& s = side(h);
        const int hh = h < p.n_head ? h : h - p.n_head;
        if (s.w) {
            const float* w = s.w + hh * s.w_head;
            if (w != held) {
                held = w;
#pragma unroll
                for (int n = 0; n < NI; ++n) {
                    if (one[n]) load_weights<V>(w + at[n], wa[n]);
                    if (two[n]) load_weights<V>(w + at[n] + far[n], wb[n]);
                }
            }
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < NI; ++n)
#pragma unroll
                for (int i = 0; i < V; ++i) sum = fmaf(a[n][i], a[n][i], fmaf(b[n][i], b[n][i], sum));
            const float r = 1.0f / sqrtf(lanes_sum<W>(sum) * inv_hd + p.eps);
#pragma unroll
            for (int n = 0; n < NI; ++n)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    a[n][i] = a[n][i] * r * (one[n] ? wa[n][i] : 0.f);
                    b[n][i] = b[n][i] * r * (two[n] ? wb[n][i] : 0.f);
                }
        }
        T* y = static_cast<T*>(s.y) + t * s.y_token + hh * s.y_head;
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            if (turns[n]) rotate<V, IL>(a[n], b[n], sc[n]);
            if (one[n]) store_vec<T, V>(y + at[n], a[n]);
            if (two[n]) store_vec<T, V>(y + at[n] + far[n], b[n]);
        }
#pragma unroll
        for (int n = 0; n < NI; ++n)
#pragma unroll
            for (int i = 0; i < V; ++i) a[n][i] = na[n][i], b[n][i] = nb[n][i];
    }
}

template <typename T, int V, bool IL, int W, int NI>
static int launch_qk_norm(QkNormArgs p, hipStream_t s) {
    // heads a group takes with one sine and cosine: as many as leave the chip about 8 waves per SIMD
    const int64_t lanes = p.tokens * W, want = (524288 + lanes - 1) / lanes;
    p.groups = (int)(want < p.heads ? want : p.heads);
    const int64_t blocks = (p.tokens * p.groups + 256 / W - 1) / (256 / W);
    if (blocks >= (1 << 24)) return PE_ERR_SHAPE;  // a grid holds 2^32 threads
    hipLaunchKernelGGL((k_qk_norm_rope<T, V, IL, W, NI>), dim3((unsigned)blocks), dim3(256), 0, s, p);
    return launch_status();
}

template <typename T, bool IL>
static int launch_qk_norm(const QkNormArgs& p, bool vec, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    if (!vec) return p.hd <= 128 ? launch_qk_norm<T, 1, IL, 64, 1>(p, s) : launch_qk_norm<T, 1, IL, 64, 4>(p, s);
    const int per = (p.half + V - 1) / V + (p.hd - 2 * p.half + 2 * V - 1) / (2 * V);
    if (per <= 4) return launch_qk_norm<T, V, IL, 4, 1>(p, s);
    if (per <= 8) return launch_qk_norm<T, V, IL, 8, 1>(p, s);
    if (per <= 16) return launch_qk_norm<T, V, IL, 16, 1>(p, s);
    if (per <= 32) return launch_qk_norm<T, V, IL, 32, 1>(p, s);
    return launch_qk_norm<T, V, IL, 64, 1>(p, s);
}

// The heads of one side; PE_OK or what is wrong with them.
static int side_ok(const NormSide& s, int64_t tokens, int n, int hd, size_t e) {
    if (s.x_token < 0 || s.x_head < 0 || s.y_token < 0 || s.y_head < 0 || (n > 1 && s.y_head < hd) ||
        (tokens > 1 && s.y_token < hd) || (s.w_head != 0 && s.w_head < hd))
        return PE_ERR_SHAPE;
    // rows of y that share memory: heads inside a token row, or tokens inside a head's rows
    if (tokens > 1 && n > 1 && s.y_token < s.y_head * (n - 1) + hd && s.y_head < s.y_token * (tokens - 1) + hd)
        return PE_ERR_SHAPE;
    if (!s.x || !s.y) return PE_ERR_NULL;
    if (s.x == s.y && ((tokens > 1 && s.x_token != s.y_token) || (n > 1 && s.x_head != s.y_head)))
        return PE_ERR_SHAPE;
    if (!aligned(s.x, e) || !aligned(s.y, e) || !aligned(s.w, 4)) return PE_ERR_ALIGN;
    return PE_OK;
}

}  // namespace pe

using namespace pe;

extern "C" int pe_qk_norm_rope(const pe_qk_norm_args* a, pe_stream_t stream) {
    if (!a) return PE_ERR_NULL;
    if ((a->type != PE_TYPE_F32 && a->type != PE_TYPE_F16) || (a->pos_dtype != 1 && a->pos_dtype != 2))
        return PE_ERR_TYPE;
    const int64_t T = a->tokens;
    if (T < 0 || T > (1LL << 40) || a->n_head < 0 || a->n_kv < 0 || a->n_head > 4096 || a->n_kv > 4096 ||
        a->n_head + a->n_kv == 0 || a->head_dim <= 0 || a->head_dim > 512 || a->rot_dim <= 0 || a->rot_dim % 2 ||
        a->rot_dim > a->head_dim)
        return PE_ERR_SHAPE;
    if (T == 0) return PE_OK;
    const size_t e = a->type == PE_TYPE_F16 ? 2 : 4;
    const NormSide q{a->q, a->q_token, a->q_head, a->q_out, a->q_out_token, a->q_out_head, a->q_weight, a->q_weight_head};
    const NormSide k{a->k, a->k_token, a->k_head, a->k_out, a->k_out_token, a->k_out_head, a->k_weight, a->k_weight_head};
    if (const int st = a->n_head ? side_ok(q, T, a->n_head, a->head_dim, e) : 0) return st;
    if (const int st = a->n_kv ? side_ok(k, T, a->n_kv, a->head_dim, e) : 0) return st;
    if (!a->positions || !a->freqs) return PE_ERR_NULL;
    if (!aligned(a->positions, a->pos_dtype == 2 ? 8 : 4) || !aligned(a->freqs, 8)) return PE_ERR_ALIGN;
    QkNormArgs p{q, k, a->positions, a->pos_dtype == 2, a->freqs, a->rot_dim / 2, a->head_dim, a->amp, a->eps,
                 a->n_head, a->n_head + a->n_kv, 1, T};
    // 16 bytes at a time where every piece of every row is whole and aligned, else single elements
    const int v = (int)(16 / e);
    bool vec = (a->interleaved ? a->rot_dim % (2 * v) == 0 : a->rot_dim / 2 % v == 0) && a->head_dim % v == 0;
    for (const NormSide* s : {&q, &k})
        if (s == &q ? a->n_head : a->n_kv)
            vec = vec && (s->x_token | s->x_head | s->y_token | s->y_head) % v == 0 && aligned(s->x, 16) &&
                  aligned(s->y, 16) && aligned(s->w, 16) && s->w_head % 4 == 0;
    hipStream_t s = (hipStream_t)stream;
    if (a->type == PE_TYPE_F16)
        return a->interleaved ? launch_qk_norm<_Float16, true>(p, vec, s) : launch_qk_norm<_Float16, false>(p, vec, s);
    return a->interleaved ? launch_qk_norm<float, true>(p, vec, s) : launch_qk_norm<float, false>(p, vec, s);
}
