// Writing and reading the paged 4-bit cache (kv4.h):
//   kv4_append  new rows of several sequences: q and k normed and rotated, k and v rounded to 4 bits and written to
//               the slots behind what their sequence holds
//   kv4_read    the values a cache stands for
#include <type_traits>

#include "kv4.h"
#include "rope_common.h"

namespace pe {

// ---- append ---------------------------------------------------------------------------------
// Keys, their norm and their rotation are computed in 64 bits: a key next to a rounding border would
// otherwise fall to one side or the other with the last bits of a sine, and differ by a whole step.

// (sin, cos) of pos * f quarter turns: as sincos_quarters, the series up to x^17 and x^16 (what is left out is under 2.1e-18).
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

// A 64-bit number in 32 bits, cut off, its last bit set if anything was: comparisons with short numbers, and rounding to
// far fewer bits, come out as they would in 64. Beyond 2^128 the largest number, below 2^-126 zero; infinities and NaN stay so.
PE_DEV uint32_t cut_short(double y) {
    const uint64_t w = (uint64_t)__double_as_longlong(y);
    const uint32_t hi = (uint32_t)(w >> 32), lo = (uint32_t)w, m = hi & 0x7FFFFFFFu;
    uint32_t f = ((m - 0x38000000u) << 3 | lo >> 29) | (lo << 3 ? 1u : 0u);
    f = m >= 0x47F00000u ? (m >= 0x7FF00000u ? 0x7FC00000u : 0x7F7FFFFFu) : m < 0x38100000u ? 0u : f;
    return f | (hi & 0x80000000u);
}

// Codes of the E elements of a lane (bits of floats), the scale shared with the 32 / E lanes of its block.
template <int E>
PE_DEV uint32_t encode(const uint32_t* y, uint32_t& scale) {
    uint32_t top = 0;  // the bits of magnitudes order as they do, infinities and NaN above all
#pragma unroll
    for (int i = 0; i < E; ++i) top = max(top, y[i] & 0x7FFFFFFFu);
    const auto other = [](uint32_t v, auto ctrl) { return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, decltype(ctrl)::value, 0xF, 0xF, false); };
    top = max(top, other(top, std::integral_constant<int, 0xB1>{}));                        // quad_perm [1,0,3,2]
    top = max(top, other(top, std::integral_constant<int, 0x4E>{}));                        // quad_perm [2,3,0,1]
    if constexpr (E == 4) top = max(top, other(top, std::integral_constant<int, 0x141>{}));  // row_half_mirror
    if (top >= 0x7F800000u) {
        scale = 255;
        return 0;
    }
    // the mantissa beyond 1.75: 7 times a quarter of the power of two
    int e = (int)(top >> 23) - 2 + ((top & 0x7FFFFFu) > 0x600000u);
    e = e < kKv4MinExp + 127 ? kKv4MinExp + 127 : e > kKv4MaxExp + 127 ? kKv4MaxExp + 127 : e;
    scale = e;
    // to the nearest code, halfway to the even one, 6 beyond 6: what the conversion does
    const float f = __uint_as_float((uint32_t)e << 23);
    uint32_t codes = 0;
#define PE_TWO(i) codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, __uint_as_float(y[2 * i]), __uint_as_float(y[2 * i + 1]), f, i)
    PE_TWO(0);
    PE_TWO(1);
    if constexpr (E == 8) {
        PE_TWO(2);
        PE_TWO(3);
    }
#undef PE_TWO
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
// runs are aligned in q, k, v and q_out, and so are their partners'. 4101 rows of 32 + 2 x 8 heads of 128, fp16, take 24.4 us,
// 17 at the copy rate: 12300 workgroups of about 4 us each, loads one behind the other (sequence, page), eight a CU.
template <typename T, int HD, bool VEC>
__global__ __launch_bounds__(256) void k_kv4_append(Kv4AppendArgs p) {
    constexpr int E = HD / 16;
    __shared__ SinCos64 turn[HD / 2];
    // Workgroups go to the eight XCDs in turn: of each 128, sixteen neighbours go to one, whose L2 then gathers the pieces
    // of a tile's lines.
    int t = blockIdx.x;
    if ((t | 127) < (int)p.tokens) t = (t & ~127) + (t & 7) * 16 + (t >> 3 & 15);
    if (t >= (int)p.tokens) return;
    const int lane = threadIdx.x % 16, at = lane * E, group = threadIdx.x / 16;
    const bool isq = (int)blockIdx.y < p.q_parts;
    const int h = (isq ? blockIdx.y : blockIdx.y - p.q_parts) * 16 + group;
    const bool isv = !isq && h >= p.n_kv, active = h < (isq ? p.n_head : 2 * p.n_kv);
    const int hh = isv ? h - p.n_kv : h, rot = p.freqs && !p.interleaved && !isv ? 2 * p.half : 0;
    // first what the rest waits for: where every sequence begins and what it holds, one a lane, if there are few (26.4 ->
    // 24.4 us against looking for the sequence, then for its length, behind the rows' loads)
    const int wl = threadIdx.x & 63;
    const bool few = p.starts && p.batch < kWave;
    int64_t start = 0, held = 0;
    if (few && wl <= p.batch) {
        start = int_at(p.starts, p.starts_wide, wl);
        held = int_at(p.lengths, p.len_wide, wl < p.batch ? wl : 0);
    }
    const double freq = p.freqs && (int)threadIdx.x < p.half ? p.freqs[threadIdx.x] * 0.63661977236758134 : 0;
    float own[E] = {}, other[E] = {};
    if (active) {
        const T* x = static_cast<const T*>(isq ? p.q : isv ? p.v : p.k) + t * (isq ? p.q_token : isv ? p.v_token : p.k_token) +
                     hh * (isq ? p.q_head : isv ? p.v_head : p.k_head);
        load_pairs<T, E, VEC>(x, at, rot, p.half, own, other);
    }
    int64_t b, len, lo;
    if (few) {
        b = __popcll(__ballot(wl <= p.batch && start <= t)) - 1;
        if (b < 0 || b >= p.batch) return;
        len = lane_of(held, (int)b);
        lo = lane_of(start, (int)b);
    } else {
        b = sequence_of(p.starts, p.starts_wide, p.batch, t);
        if (b < 0) return;
        len = uniform(int_at(p.lengths, p.len_wide, b));
        lo = p.starts ? uniform(int_at(p.starts, p.starts_wide, b)) : t;
    }
    len = len > (1LL << 40) ? 1LL << 40 : len;
    lo = lo < 0 ? 0 : lo;
    if (t < lo) return;  // starts that are out of order
    const int64_t slot = len + (t - lo);
    if (isq) {
        SinCos* turn32 = reinterpret_cast<SinCos*>(turn);
        if (p.freqs) {
            if ((int)threadIdx.x < p.half)
                turn32[threadIdx.x] = sincos_quarters((double)slot, freq, 1.f);
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
            turn[threadIdx.x] = sincos_quarters64((double)slot, freq);
        __syncthreads();
    }
    uint32_t bits[E];
    if (isv) {
#pragma unroll
        for (int i = 0; i < E; ++i) bits[i] = __float_as_uint(own[i]);
    } else {
        double y[E];
        turn_run<HD, double>(p, own, other, at, p.k_weight, turn, y);
#pragma unroll
        for (int i = 0; i < E; ++i) bits[i] = cut_short(y[i]);
    }
    uint32_t scale;
    const uint32_t codes = encode<E>(bits, scale);
    // a negative length takes no part; a slot behind the table's end or on a page that there is not is not written
    const int page_tokens = p.tiles * kKv4Tile;
    if (len < 0 || slot >= (int64_t)p.table_cols * page_tokens) return;
    const int col = (int)slot / page_tokens, off = (int)slot - col * page_tokens, tok = off % kKv4Tile;
    const int page = __builtin_amdgcn_readfirstlane(p.table[b * p.table_row + col]);
    if (!active || page < 0 || page >= p.n_pages) return;
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
    int row_blocks;  // workgroups of a sequence and kv head
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

// A run to memory, past the caches where STREAM.
template <typename T, int E, bool STREAM>
PE_DEV void write_run(T* p, const float* v) {
    if constexpr (!STREAM) {
        store_run<T, E>(p, v);
    } else {
        constexpr int N = E * sizeof(T) > 16 ? 16 / sizeof(T) : E;
#pragma unroll
        for (int i = 0; i < E; i += N) {
            typename Vec<T, N>::type x;
#pragma unroll
            for (int j = 0; j < N; ++j) x[j] = (T)v[i + j];
            __builtin_nontemporal_store(x, reinterpret_cast<typename Vec<T, N>::type*>(p + i));
        }
    }
}

// A workgroup takes NT tiles of a sequence and kv head, 16 lanes a token; the tiles' pages, then their codes, are under
// way together. Bound by memory: 5 x 20000 rows of 4 heads of 128, fp16, 237 MB, 43 us, 5.5 TB/s.
template <typename T, int HD, int NT, bool STREAM>
__global__ __launch_bounds__(256) void k_kv4_read(Kv4ReadArgs p) {
    constexpr int E = HD / 16;
    typedef typename std::conditional<E == 8, uint32_t, uint16_t>::type run;
    const int lane = threadIdx.x % 16, tok = threadIdx.x / 16;
    const uint32_t pair = blockIdx.x / (uint32_t)p.row_blocks;
    const int rt = (int)(blockIdx.x - pair * (uint32_t)p.row_blocks) * NT;
    const int64_t b = pair / (uint32_t)p.n_kv;
    const int h = (int)(pair - (uint32_t)b * (uint32_t)p.n_kv);
    const int64_t len = int_at(p.lengths, p.len_wide, b);
    int page[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int col = (rt + i) / p.tiles;
        page[i] = col < p.table_cols ? p.table[b * p.table_row + col] : -1;
    }
    uint32_t kc[NT], vc[NT], ks[NT], vs[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        kc[i] = vc[i] = ks[i] = vs[i] = 0;
        if ((int64_t)(rt + i) * kKv4Tile + tok < len && (uint32_t)page[i] < (uint32_t)p.n_pages) {
            const uint8_t* z = p.pages + page[i] * p.page_stride + ((int64_t)h * p.tiles + (rt + i) % p.tiles) * (17 * HD);
            const int block = lane * E / 32;
            kc[i] = *reinterpret_cast<const run*>(z + tok * (HD / 2) + lane * (E / 2));
            vc[i] = *reinterpret_cast<const run*>(z + 8 * HD + tok / 4 * (2 * HD) + lane * (2 * E) + tok % 4 * (E / 2));
            ks[i] = z[16 * HD + tok * (HD / 32) + block];
            vs[i] = z[16 * HD + HD / 2 + (tok / 4 * (HD / 32) + block) * 4 + tok % 4];
        }
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int64_t row = (int64_t)(rt + i) * kKv4Tile + tok;
        if (row >= p.rows) return;
        const int64_t at = ((int64_t)pair * p.rows + row) * HD + lane * E;
        float y[E];
        decode<E>(kc[i], ks[i], y);
        write_run<T, E, STREAM>(static_cast<T*>(p.k) + at, y);
        decode<E>(vc[i], vs[i], y);
        write_run<T, E, STREAM>(static_cast<T*>(p.v) + at, y);
    }
}

template <typename T, int HD>
static int launch_read(Kv4ReadArgs p, int64_t pairs, hipStream_t s) {
    const int64_t tiles = (p.rows + kKv4Tile - 1) / kKv4Tile;
    // Two tiles a workgroup where that leaves 20 of one tile and more to each CU (3 x 3833 rows of 8 heads of 128, fp16, 13.4 us
    // against 16; 48 x 397 of 4, fp32, 16.5 against 15.5; four tiles are slower at both). Outputs that the last-level
    // cache would not hold go past it (5 x 20000 of 4, fp16, 205 MB, 50 -> 42 us; 78 MB 16 -> 23).
    const int nt = tiles * pairs >= 20 * 256 ? 2 : 1;
    const bool stream = 2 * pairs * p.rows * HD * (int64_t)sizeof(T) > (128 << 20);
    p.row_blocks = (int)((tiles + nt - 1) / nt);
    if (p.row_blocks * pairs >= (1 << 24)) return PE_ERR_SHAPE;  // a grid holds 2^32 threads
    const dim3 g((unsigned)(p.row_blocks * pairs));
    if (stream)
        hipLaunchKernelGGL((k_kv4_read<T, HD, 2, true>), g, dim3(256), 0, s, p);
    else if (nt == 2)
        hipLaunchKernelGGL((k_kv4_read<T, HD, 2, false>), g, dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((k_kv4_read<T, HD, 1, false>), g, dim3(256), 0, s, p);
    return launch_status();
}

template <typename T>
static int launch_append(const Kv4AppendArgs& p, int hd, bool vec, hipStream_t s) {
    const dim3 g((unsigned)(p.tokens + 7) / 8 * 8, (unsigned)(p.q_parts + (2 * p.n_kv + 15) / 16));
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
    if ((rows + 2 * kKv4Tile - 1) / (2 * kKv4Tile) * n_kv * batch >= (1 << 24)) return PE_ERR_SHAPE;
    if (!lengths || !k || !v) return PE_ERR_NULL;
    if (!aligned(k, 16) || !aligned(v, 16) || !int_aligned(lengths, lengths_dtype)) return PE_ERR_ALIGN;
    Kv4ReadArgs p{static_cast<const uint8_t*>(pool->pages), pool->page_stride, pool->n_pages,
                  (int)(pool->page_tokens / kKv4Tile), pool->table, pool->table_stride, (int)pool->table_cols, lengths,
                  lengths_dtype == 2, n_kv, rows, 0, k, v};
    hipStream_t s = (hipStream_t)stream;
    const int64_t pairs = batch * n_kv;
    if (type == PE_TYPE_F16)
        return head_dim == 64 ? launch_read<_Float16, 64>(p, pairs, s) : launch_read<_Float16, 128>(p, pairs, s);
    return head_dim == 64 ? launch_read<float, 64>(p, pairs, s) : launch_read<float, 128>(p, pairs, s);
}
