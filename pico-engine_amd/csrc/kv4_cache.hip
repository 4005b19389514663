// Writing and reading the paged 4-bit cache (kv4.h):
//   kv4_append  new rows of several sequences: q and k normed and rotated, k and v rounded to 4 bits and written to
//               the slots behind what their sequence holds
//   kv4_read    the values a cache stands for
#include "kv4.h"
#include "rope_common.h"

namespace pe {

// ---- append ---------------------------------------------------------------------------------
// Keys, their norm and their rotation are computed in 64 bits: a key next to a rounding border would
// otherwise fall to one side or the other with the last bits of a sine, and differ by a whole step.

// (sin, cos) of pos * f quarter turns: as sincos_quarters, the series up to x^17 (what is left out is under 2e-18).
struct SinCos64 {
    double s, c;
};
PE_DEV SinCos64 sincos_quarters64(double pos, double f) {
    const double p = pos * f, e = fma(pos, f, -p), n = rint(p);
    const double x = ((p - n) + e) * 1.5707963267948966;
    const int q = (int)(int64_t)(n - 4.0 * floor(n * 0.25));
    const double z = x * x;
    double s = fma(z, 2.8114572543455206e-15, -7.6471637318198164e-13);
    s = fma(z, s, 1.6059043836821613e-10);
    s = fma(z, s, -2.5052108385441720e-8);
    s = fma(z, s, 2.7557319223985893e-6);
    s = fma(z, s, -1.9841269841269841e-4);
    s = fma(z, s, 8.3333333333333333e-3);
    s = fma(z, s, -1.6666666666666667e-1);
    s = fma(x * z, s, x);
    double c = fma(z, 4.7794773323873853e-14, -1.1470745597729725e-11);
    c = fma(z, c, 2.0876756987868099e-9);
    c = fma(z, c, -2.7557319223985888e-7);
    c = fma(z, c, 2.4801587301587302e-5);
    c = fma(z, c, -1.3888888888888889e-3);
    c = fma(z, c, 4.1666666666666667e-2);
    c = fma(z, c, -0.5);
    c = fma(z, c, 1.0);
    const double a = q & 1 ? c : s, b = q & 1 ? s : c;
    return {q & 2 ? -a : a, (q + 1) & 2 ? -b : b};
}

struct Kv4AppendArgs {
    const void* q;
    int64_t q_token, q_head;
    void* q_out;
    int64_t out_token, out_head;
    const void* k;
    int64_t k_token, k_head;
    const void* v;
    int64_t v_token, v_head;
    uint8_t* pages;
    int64_t page_stride, n_pages;
    int tiles;  // of a page
    const int* table;
    int64_t table_row;
    int table_cols;
    const void* lengths;
    int len_wide;
    const void* starts;
    int starts_wide;
    const double* freqs;  // NULL: no rotation
    int half;
    float amp;
    int interleaved;
    const float* q_weight;
    const float* k_weight;
    float eps;
    int64_t tokens, batch;
    int n_head, n_kv, q_parts;  // q_parts: workgroups for a token's query heads
};

// A lane's run, 16 bytes at a time (8 where it has no more).
template <typename T, int E>
PE_DEV void load_run(const T* p, float* v) {
    constexpr int N = E * sizeof(T) > 16 ? 16 / sizeof(T) : E;
#pragma unroll
    for (int i = 0; i < E; i += N) load_vec<T, N>(p + i, v + i);
}
template <typename T, int E>
PE_DEV void store_run(T* p, const float* v) {
    constexpr int N = E * sizeof(T) > 16 ? 16 / sizeof(T) : E;
#pragma unroll
    for (int i = 0; i < E; i += N) store_vec<T, N>(p + i, v + i);
}

// Codes of the E elements of a lane, the scale shared with the 32 / E lanes of its block.
template <int E>
PE_DEV uint32_t encode(const double* y, uint32_t& scale) {
    uint64_t top = 0;  // the bits of magnitudes order as they do, infinities and NaN above all
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const uint64_t m = (uint64_t)__double_as_longlong(y[i]) & 0x7FFFFFFFFFFFFFFFull;
        top = m > top ? m : top;
    }
#pragma unroll
    for (int o = 16 / E; o > 0; o >>= 1) {
        const uint64_t m = (uint64_t)__shfl_xor((unsigned long long)top, o, kWave);
        top = m > top ? m : top;
    }
    if (top >= 0x7FF0000000000000ull) {
        scale = 255;
        return 0;
    }
    int e = (int)(top >> 52) - 1023 - 2 + ((top & 0xFFFFFFFFFFFFFull) > 0xC000000000000ull);
    e = e < kKv4MinExp ? kKv4MinExp : e > kKv4MaxExp ? kKv4MaxExp : e;
    scale = e + 127;
    const double f = __longlong_as_double((long long)(1023 - e) << 52);  // 2^-e
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const double z = y[i] * f, a = fabs(z);
        // halfway values go to the even code
        const uint32_t c = (a > 0.25) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0);
        codes |= (c | (z < 0 ? 8u : 0u)) << (4 * i);
    }
    return codes;
}

// A lane's run of E elements from channel `at` on (own), and of what each is turned with (other).
template <typename T, int E, bool VEC>
PE_DEV void load_pairs(const T* x, int at, int rot, int half, float* own, float* other) {
    const auto partner = [&](int c) { return c < half ? c + half : c - half; };
    if constexpr (VEC) {
        load_run<T, E>(x + at, own);
        if (at < rot) load_run<T, E>(x + partner(at), other);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) own[i] = (float)x[at + i];
#pragma unroll
        for (int i = 0; i < E; ++i) other[i] = at + i < rot ? (float)x[partner(at + i)] : 0.f;
    }
}

// The norm's 1 / root of a head held by 16 lanes.
template <int HD, typename F>
PE_DEV F inverse_root(const F* y, float eps) {
    F sum = 0;
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) sum = fma(y[i], y[i], sum);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
    return (F)1 / sqrt(sum * (F)(1.0 / HD) + (F)eps);
}

// The run normed and rotated, in F.
template <int HD, typename F, typename SC>
PE_DEV void turn_run(const Kv4AppendArgs& p, const float* own, const float* other, int at, const float* w, const SC* turn, F* y) {
    constexpr int E = HD / 16;
#pragma unroll
    for (int i = 0; i < E; ++i) y[i] = own[i];
    F r = 1;
    if (w) {
        r = inverse_root<HD, F>(y, p.eps);
#pragma unroll
        for (int i = 0; i < E; ++i) y[i] = y[i] * r * (F)w[at + i];
    }
    if (!p.freqs) return;
    if (p.interleaved) {
#pragma unroll
        for (int i = 0; i < E; i += 2)
            if (at + i < 2 * p.half) {
                const SC sc = turn[(at + i) / 2];
                const F u = y[i], z = y[i + 1];
                y[i] = (u * sc.c - z * sc.s) * p.amp;
                y[i + 1] = (u * sc.s + z * sc.c) * p.amp;
            }
        return;
    }
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int c = at + i;
        if (c < 2 * p.half) {
            const bool low = c < p.half;
            const int d = low ? c + p.half : c - p.half;
            const SC sc = turn[low ? c : d];
            F z = other[i];
            if (w) z = z * r * (F)w[d];
            y[i] = (low ? y[i] * sc.c - z * sc.s : z * sc.s + y[i] * sc.c) * p.amp;
        }
    }
}

// A workgroup takes 16 heads of a token, of q or of k and v, 16 lanes each, a lane a run of HD / 16 elements. The
// elements that a rotated one is made with are loaded beside it (they are in the same cache lines), so that a
// lane holds a whole run of codes whatever the pairs are. The token's sines are made once, in LDS. VEC: the lanes'
// runs are aligned in q, k, v and q_out, and so are their partners'.
template <typename T, int HD, bool VEC>
__global__ __launch_bounds__(256) void k_kv4_append(Kv4AppendArgs p) {
    constexpr int E = HD / 16;
    __shared__ SinCos64 turn[HD / 2];
    const int64_t t = blockIdx.x;
    const int lane = threadIdx.x % 16, at = lane * E, group = threadIdx.x / 16;
    const bool isq = (int)blockIdx.y < p.q_parts;
    const int h = (isq ? blockIdx.y : blockIdx.y - p.q_parts) * 16 + group;
    const bool isv = !isq && h >= p.n_kv, active = h < (isq ? p.n_head : 2 * p.n_kv);
    const int hh = isv ? h - p.n_kv : h, rot = p.freqs && !p.interleaved && !isv ? 2 * p.half : 0;
    float own[E] = {}, other[E] = {};
    if (active) {
        const T* x = static_cast<const T*>(isq ? p.q : isv ? p.v : p.k) + t * (isq ? p.q_token : isv ? p.v_token : p.k_token) +
                     hh * (isq ? p.q_head : isv ? p.v_head : p.k_head);
        load_pairs<T, E, VEC>(x, at, rot, p.half, own, other);
    }
    const int64_t b = sequence_of(p.starts, p.starts_wide, p.batch, t);
    if (b < 0) return;
    int64_t len = int_at(p.lengths, p.len_wide, b);
    len = len > (1LL << 40) ? 1LL << 40 : len;
    const int64_t slot = len + (p.starts ? t - int_at(p.starts, p.starts_wide, b) : 0);
    if (isq) {
        SinCos* turn32 = reinterpret_cast<SinCos*>(turn);
        if (p.freqs) {
            if ((int)threadIdx.x < p.half)
                turn32[threadIdx.x] = sincos_quarters((double)slot, p.freqs[threadIdx.x] * 0.63661977236758134, 1.f);
            __syncthreads();
        }
        float y[E];
        turn_run<HD, float>(p, own, other, at, p.q_weight, turn32, y);
        if (!active) return;
        T* o = static_cast<T*>(p.q_out) + t * p.out_token + hh * p.out_head + at;
        if constexpr (VEC) {
            store_run<T, E>(o, y);
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) o[i] = (T)y[i];
        }
        return;
    }
    if (p.freqs) {
        if ((int)threadIdx.x < p.half)
            turn[threadIdx.x] = sincos_quarters64((double)slot, p.freqs[threadIdx.x] * 0.63661977236758134);
        __syncthreads();
    }
    double y[E];
    if (isv) {
#pragma unroll
        for (int i = 0; i < E; ++i) y[i] = own[i];
    } else {
        turn_run<HD, double>(p, own, other, at, p.k_weight, turn, y);
    }
    uint32_t scale;
    const uint32_t codes = encode<E>(y, scale);
    // a negative length takes no part; a slot behind the table's end or on a page that there is not is not written
    const int page_tokens = p.tiles * kKv4Tile;
    if (!active || len < 0 || slot >= (int64_t)p.table_cols * page_tokens) return;
    const int col = (int)slot / page_tokens, off = (int)slot - col * page_tokens, tok = off % kKv4Tile;
    const int page = p.table[b * p.table_row + col];
    if (page < 0 || page >= p.n_pages) return;
    uint8_t* z = p.pages + page * p.page_stride + ((int64_t)hh * p.tiles + off / kKv4Tile) * (17 * HD);
    uint8_t* c = isv ? z + 8 * HD + tok / 4 * (2 * HD) + lane * (2 * E) + tok % 4 * (E / 2)
                     : z + tok * (HD / 2) + lane * (E / 2);
    if constexpr (E == 8)
        *reinterpret_cast<uint32_t*>(c) = codes;
    else
        *reinterpret_cast<uint16_t*>(c) = (uint16_t)codes;
    const int block = at / 32;
    if (lane % (32 / E) == 0)
        z[16 * HD + (isv ? HD / 2 + (tok / 4 * (HD / 32) + block) * 4 + tok % 4 : tok * (HD / 32) + block)] = (uint8_t)scale;
}

// ---- read -----------------------------------------------------------------------------------
struct Kv4ReadArgs {
    const uint8_t* pages;
    int64_t page_stride, n_pages;
    int tiles;
    const int* table;
    int64_t table_row;
    int table_cols;
    const void* lengths;
    int len_wide;
    int n_kv;
    int64_t rows;
    int row_tiles;
    void* k;
    void* v;
};

template <int E>
PE_DEV void decode(uint32_t codes, uint32_t scale, float* y) {
    const float f = scale == 255 ? __uint_as_float(0x7FC00000u) : __uint_as_float(scale << 23);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const uint32_t c = codes >> (4 * i), m = c & 7;
        // magnitudes m / 2 up to 2 (m = 4), then 3, 4, 6
        const float a = m < 4 ? 0.5f * (float)m : (float)((2 + (m & 1)) << ((m >> 1) - 2));
        y[i] = (c & 8 ? -a : a) * f;
    }
}

// A workgroup takes a tile of a sequence and kv head, 16 lanes a token.
template <typename T, int HD>
__global__ __launch_bounds__(256) void k_kv4_read(Kv4ReadArgs p) {
    constexpr int E = HD / 16;
    const int lane = threadIdx.x % 16, tok = threadIdx.x / 16;
    const uint32_t pair = blockIdx.x / (uint32_t)p.row_tiles;
    const int rt = (int)(blockIdx.x - pair * (uint32_t)p.row_tiles);
    const int64_t b = pair / (uint32_t)p.n_kv;
    const int h = (int)(pair - (uint32_t)b * (uint32_t)p.n_kv);
    const int64_t row = (int64_t)rt * kKv4Tile + tok;
    if (row >= p.rows) return;
    float k[E] = {}, v[E] = {};
    const int col = rt / p.tiles;
    if (row < int_at(p.lengths, p.len_wide, b) && col < p.table_cols) {
        const int page = p.table[b * p.table_row + col];
        if (page >= 0 && page < p.n_pages) {
            const uint8_t* z = p.pages + page * p.page_stride + ((int64_t)h * p.tiles + rt % p.tiles) * (17 * HD);
            const uint8_t* kc = z + tok * (HD / 2) + lane * (E / 2);
            const uint8_t* vc = z + 8 * HD + tok / 4 * (2 * HD) + lane * (2 * E) + tok % 4 * (E / 2);
            const int block = lane * E / 32;
            const uint32_t ks = z[16 * HD + tok * (HD / 32) + block];
            const uint32_t vs = z[16 * HD + HD / 2 + (tok / 4 * (HD / 32) + block) * 4 + tok % 4];
            if constexpr (E == 8) {
                decode<E>(*reinterpret_cast<const uint32_t*>(kc), ks, k);
                decode<E>(*reinterpret_cast<const uint32_t*>(vc), vs, v);
            } else {
                decode<E>(*reinterpret_cast<const uint16_t*>(kc), ks, k);
                decode<E>(*reinterpret_cast<const uint16_t*>(vc), vs, v);
            }
        }
    }
    const int64_t at = ((int64_t)pair * p.rows + row) * HD + lane * E;
    store_run<T, E>(static_cast<T*>(p.k) + at, k);
    store_run<T, E>(static_cast<T*>(p.v) + at, v);
}

template <typename T>
static int launch_append(const Kv4AppendArgs& p, int hd, bool vec, hipStream_t s) {
    const dim3 g((unsigned)p.tokens, (unsigned)(p.q_parts + (2 * p.n_kv + 15) / 16));
    if (hd == 64 && vec)
        hipLaunchKernelGGL((k_kv4_append<T, 64, true>), g, dim3(256), 0, s, p);
    else if (hd == 64)
        hipLaunchKernelGGL((k_kv4_append<T, 64, false>), g, dim3(256), 0, s, p);
    else if (vec)
        hipLaunchKernelGGL((k_kv4_append<T, 128, true>), g, dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((k_kv4_append<T, 128, false>), g, dim3(256), 0, s, p);
    return launch_status();
}

static bool int_dtype(int d) { return d == 1 || d == 2; }
static bool int_aligned(const void* p, int d) { return aligned(p, d == 2 ? 8 : 4); }

}  // namespace pe

using namespace pe;

extern "C" int pe_kv4_append(const pe_kv4_append_args* a, pe_stream_t stream) {
    if (!a) return PE_ERR_NULL;
    if ((a->type != PE_TYPE_F32 && a->type != PE_TYPE_F16) || !int_dtype(a->lengths_dtype) ||
        (a->starts && !int_dtype(a->starts_dtype)))
        return PE_ERR_TYPE;
    const int64_t T = a->tokens;
    const int nq = a->q ? a->n_head : 0;
    const int64_t strides[] = {a->q_token, a->q_head, a->q_out_token, a->q_out_head, a->k_token, a->k_head, a->v_token, a->v_head};
    for (const int64_t st : strides)
        if (st < 0) return PE_ERR_SHAPE;
    if (T < 0 || T >= (1 << 23) || a->batch < 0 || a->batch > (1 << 20) || (!a->starts && a->batch != T) ||
        nq < 0 || nq > 4096 || (a->q && nq == 0) || T * ((nq + 15) / 16 + (2 * (int64_t)a->n_kv + 15) / 16) >= (1 << 24) ||
        (a->freqs && (a->rot_dim <= 0 || a->rot_dim % 2 || a->rot_dim > a->head_dim)))
        return PE_ERR_SHAPE;
    if (nq && ((nq > 1 && a->q_out_head < a->head_dim) || (T > 1 && a->q_out_token < a->head_dim) ||
               (T > 1 && nq > 1 && a->q_out_token < a->q_out_head * (nq - 1) + a->head_dim &&
                a->q_out_head < a->q_out_token * (T - 1) + a->head_dim)))
        return PE_ERR_SHAPE;  // rows of q_out that share memory
    if (const int st = kv4_pool_ok(&a->pool, a->n_kv, a->head_dim)) return st;
    if (T == 0 || a->batch == 0) return PE_OK;
    if (!a->k || !a->v || !a->lengths || (nq && !a->q_out)) return PE_ERR_NULL;
    if (nq && a->q == a->q_out &&
        ((T > 1 && a->q_token != a->q_out_token) || (nq > 1 && a->q_head != a->q_out_head)))
        return PE_ERR_SHAPE;
    const size_t e = a->type == PE_TYPE_F16 ? 2 : 4;
    if (!aligned(a->q, e) || !aligned(a->q_out, e) || !aligned(a->k, e) || !aligned(a->v, e) ||
        !int_aligned(a->lengths, a->lengths_dtype) || (a->starts && !int_aligned(a->starts, a->starts_dtype)) ||
        !aligned(a->freqs, 8) || !aligned(a->q_weight, 4) || !aligned(a->k_weight, 4))
        return PE_ERR_ALIGN;
    const int run = a->head_dim / 16;
    int64_t all = (a->freqs && !a->interleaved ? a->rot_dim / 2 : 0) | a->k_token | a->k_head | a->v_token | a->v_head;
    if (nq) all |= a->q_token | a->q_head | a->q_out_token | a->q_out_head;
    const size_t r = run * e < 16 ? run * e : 16;  // a run's loads: 8, 16 or twice 16 bytes
    const bool vec = all % run == 0 && aligned(a->k, r) && aligned(a->v, r) && (!nq || (aligned(a->q, r) && aligned(a->q_out, r)));
    Kv4AppendArgs p{a->q, a->q_token, a->q_head, a->q_out, a->q_out_token, a->q_out_head, a->k, a->k_token, a->k_head,
                    a->v, a->v_token, a->v_head, static_cast<uint8_t*>(a->pool.pages), a->pool.page_stride, a->pool.n_pages,
                    (int)(a->pool.page_tokens / kKv4Tile), a->pool.table, a->pool.table_stride, (int)a->pool.table_cols,
                    a->lengths, a->lengths_dtype == 2, a->starts, a->starts_dtype == 2, a->freqs, a->freqs ? a->rot_dim / 2 : 0,
                    a->amp, a->interleaved, a->q_weight, a->k_weight, a->eps, T, a->batch, nq, a->n_kv, (nq + 15) / 16};
    return a->type == PE_TYPE_F16 ? launch_append<_Float16>(p, a->head_dim, vec, (hipStream_t)stream)
                                  : launch_append<float>(p, a->head_dim, vec, (hipStream_t)stream);
}

extern "C" int pe_kv4_read(int type, const pe_kv4_pool* pool, const void* lengths, int lengths_dtype, int64_t batch, int n_kv,
                           int head_dim, int64_t rows, void* k, void* v, pe_stream_t stream) {
    if (!pool) return PE_ERR_NULL;
    if ((type != PE_TYPE_F32 && type != PE_TYPE_F16) || !int_dtype(lengths_dtype)) return PE_ERR_TYPE;
    if (batch < 0 || batch > (1 << 20) || rows < 0 || rows > (1LL << 30)) return PE_ERR_SHAPE;
    if (const int st = kv4_pool_ok(pool, n_kv, head_dim)) return st;
    if (batch == 0 || rows == 0) return PE_OK;
    const int64_t row_tiles = (rows + kKv4Tile - 1) / kKv4Tile;
    if (row_tiles * n_kv * batch >= (1 << 24)) return PE_ERR_SHAPE;  // a grid holds 2^32 threads
    if (!lengths || !k || !v) return PE_ERR_NULL;
    if (!aligned(k, 16) || !aligned(v, 16) || !int_aligned(lengths, lengths_dtype)) return PE_ERR_ALIGN;
    Kv4ReadArgs p{static_cast<const uint8_t*>(pool->pages), pool->page_stride, pool->n_pages,
                  (int)(pool->page_tokens / kKv4Tile), pool->table, pool->table_stride, (int)pool->table_cols, lengths,
                  lengths_dtype == 2, n_kv, rows, (int)row_tiles, k, v};
    const dim3 g((unsigned)(row_tiles * n_kv * batch));
    hipStream_t s = (hipStream_t)stream;
    if (type == PE_TYPE_F16 && head_dim == 64)
        hipLaunchKernelGGL((k_kv4_read<_Float16, 64>), g, dim3(256), 0, s, p);
    else if (type == PE_TYPE_F16)
        hipLaunchKernelGGL((k_kv4_read<_Float16, 128>), g, dim3(256), 0, s, p);
    else if (head_dim == 64)
        hipLaunchKernelGGL((k_kv4_read<float, 64>), g, dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((k_kv4_read<float, 128>), g, dim3(256), 0, s, p);
    return launch_status();
}
