// Decode attention of a batch whose sequences share a prefix: for sequence b and query head h (kv
// head j = h / group), with the keys of the prefix and then the sequence's own,
//   out[b][h] = sum_s softmax_s(scale q[b][h] . K_s) V_s.
// softmax over two sets of keys is the merge of the softmaxes over each (running maximum, sum and
// unnormalised row), so the prefix is taken once for all: the batch x group queries of a kv head are
// the rows of one matrix product with its keys, on the matrix cores, and only the own keys are taken
// per sequence. The records (row, maximum, sum) of key chunks are merged by a second launch.
//
// A wave forms 32 x 32 tiles: scores transposed (keys x queries), so that a query's scores sit in a
// lane pair and P^T is the second product's operand as it stands. Scores, maxima, sums and rows are
// fp32. Two ways over the keys, by the rows of a kv head:
//   shared: a workgroup's eight waves take four row tiles of 32 and two halves of every 64-key
//     block, staged once for all of them in LDS (two buffers, one barrier a block);
//   solo: a wave takes 32 rows and its own key tiles in its own LDS without barriers, up to eight
//     waves of an item merged at the end. The own keys, a group's rows each, always go this way.
// Products: fp32 caches that are taken solo run on the fp32 matrix instructions (bound by memory at
// these row counts). All others run on v_mfma_f32_32x32x16_f16 with the fp32 factors as the sum of
// two fp16 values, 22 bits (one would cost 2^-12 of each): the query, scaled by a power of two to at
// most 2^14; the probability times 2^14; and an fp32 cache's keys and values, every 8 keys scaled by a
// power of two of their largest element. Products of two low parts are left out (2^-22). That is 2
// instructions for 16-bit caches and 3 for fp32 ones in place of 16 fp32 instructions of twice the
// time each.
#include "pe_common.h"

namespace pe {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef _Float16 h4v __attribute__((ext_vector_type(4)));
typedef short s4v __attribute__((ext_vector_type(4)));

constexpr int kSpWaves = 8;
constexpr int kSpBlock = 64;       // keys of a shared block
constexpr float kLift = 14.f;      // log2 of the factor of the probabilities
constexpr float kLog2e = 1.4426950408889634f;

struct SpArgs {
    const float* q;
    const void* kp;
    const void* vp;
    int64_t p_cap;
    const void* ko;
    const void* vo;
    int64_t o_cap;
    const void* p_len;
    int p_dtype;
    int64_t p_add;
    const void* o_len;
    int o_dtype;
    int64_t o_add;
    int batch, n_head, n_kv, group;
    float scale;
    // how the work is cut (sp_plan): chunks that the capacities have and keys of each; row tiles of a
    // kv head (of 128 rows shared, 32 solo) and of a group; waves that share an item's own keys
    int shared, p_chunks, p_keys, p_tiles, o_chunks, o_keys, o_tiles, o_split;
    int p_blocks, o_items;
    float* rec;  // (batch, n_head, chunks, hd)
    float* ml;   // (batch, n_head, chunks, 2)
    int round_fp16;
    float* out;
};

PE_DEV int64_t sp_length(const void* len, int dtype, int64_t i, int64_t add, int64_t cap) {
    int64_t n = add;
    if (dtype == 1) n += static_cast<const int*>(len)[i];
    if (dtype == 2) n += static_cast<const int64_t*>(len)[i];
    return n < cap ? n : cap;
}

PE_DEV uint32_t lds_address(const uint8_t* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p;
}
// 16 bytes per lane from global g into LDS at m0 + 16 lane (one wave instruction: 1 KB)
PE_DEV void sp_load16(const void* g, uint32_t m0) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(m0) : "memory", "m0");
}
template <int N>
PE_DEV void sp_wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
PE_DEV void sp_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

PE_DEV float exp2_int(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
PE_DEV int exponent_of(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }

// LDS image of a key tile: row r's 16-byte chunk c at chunk position c ^ swizzle(r), so that the
// rows that one read takes cover the banks. 16-bit values are read by rows of four (transposing
// reads), everything else by rows of eight.
template <int SIZE, bool VALUES>
PE_DEV int sp_swizzle(int r) {
    return VALUES && SIZE == 2 ? 2 * (r & 3) : r & 7;
}

// Pieces f0 .. f0 + N - 1 (1 KB each) of the tile of rows row0 .. of base; rows past `last` are
// the last one again (their scores are masked and their values cleared).
template <typename T, int HD, bool VALUES, int N>
PE_DEV void sp_stage(const T* base, int64_t row0, int64_t last, uint32_t lds, int lane, int f0) {
    constexpr int E = 16 / sizeof(T), C = HD / E;
#pragma unroll
    for (int f = 0; f < N; ++f) {
        const int slot = (f0 + f) * 64 + lane, r = slot / C, c = (slot % C) ^ sp_swizzle<sizeof(T), VALUES>(r);
        const int64_t row = row0 + r < last ? row0 + r : last;
        sp_load16(base + row * HD + E * c, __builtin_amdgcn_readfirstlane(lds + (f0 + f) * 1024));
    }
}

// Clears rows [n, 32) of a tile of values (copies of the last one, which may be infinite).
template <int ROW>
PE_DEV void sp_clear_rows(uint8_t* vt, int n, int rows, int first, int step) {
    for (int i = n * (ROW / 16) + first; i < rows * (ROW / 16); i += step)
        *reinterpret_cast<float4*>(vt + 16 * i) = make_float4(0.f, 0.f, 0.f, 0.f);
}

// A wave's 32 queries as matrix operands and the products with a tile of 32 keys. One lane: query
// (or key, or dim) li = lane & 31, half g = lane >> 5. Register r of the scores is key
// 8 (r / 4) + 4 g + r % 4; they have to be multiplied by `unscale`.
template <int HD>
struct RowsF32 {
    static constexpr float kUp = 0.f, unscale = 1.f;
    float4 q[HD / 8];
    PE_DEV void load(const float* row, float scale, int g) {
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) {
            q[j] = row ? *reinterpret_cast<const float4*>(row + 8 * j + 4 * g) : make_float4(0.f, 0.f, 0.f, 0.f);
            q[j].x *= scale;
            q[j].y *= scale;
            q[j].z *= scale;
            q[j].w *= scale;
        }
    }
    PE_DEV f16v scores(const uint8_t* kt, int li, int g) const {
        f16v s = {};
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) {
            const float4 k = *reinterpret_cast<const float4*>(kt + li * (HD * 4) + (((2 * j + g) ^ (li & 7)) * 16));
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(k.x, q[j].x, s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(k.y, q[j].y, s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(k.z, q[j].z, s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(k.w, q[j].w, s, 0, 0, 0);
        }
        return s;
    }
    // o += V^T P^T
    static PE_DEV void accumulate(const uint8_t* vt, const f16v& p, f16v* o, int li, int g) {
        int col[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) col[i] = (((li >> 2) ^ (4 * g + i)) & 7) * 16 + (li & 3) * 4;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const uint8_t* vr = vt + (8 * (r >> 2) + 4 * g + (r & 3)) * (HD * 4) + col[r & 3];
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
                o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(*reinterpret_cast<const float*>(vr + 128 * d), p[r], o[d], 0, 0, 0);
        }
    }
};

template <int HD>
struct RowsF16 {
    static constexpr float kUp = kLift;
    h8v hi[HD / 16], lo[HD / 16];
    float unscale;
    PE_DEV void load(const float* row, float scale, int g) {
        float v[HD / 2], top = 0.f;
#pragma unroll
        for (int j = 0; j < HD / 16; ++j)
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                const float4 x = row ? *reinterpret_cast<const float4*>(row + 16 * j + 8 * g + i) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[8 * j + i] = x.x * scale;
                v[8 * j + i + 1] = x.y * scale;
                v[8 * j + i + 2] = x.z * scale;
                v[8 * j + i + 3] = x.w * scale;
            }
#pragma unroll
        for (int i = 0; i < HD / 2; ++i) top = fmaxf(top, fabsf(v[i]));
        top = swap32_max(top);
        // 2^(13 - exponent of the largest), within what fp32 holds with its inverse
        int e = exponent_of(top);
        e = e < -100 ? -100 : e > 120 ? 120 : e;
        const float f = exp2_int(13 - e);
        unscale = exp2_int(e - 13);
#pragma unroll
        for (int j = 0; j < HD / 16; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = v[8 * j + i] * f;
                hi[j][i] = (_Float16)x;
                lo[j][i] = (_Float16)(x - (float)hi[j][i]);
            }
    }
    // `low`: bytes from a tile to its low parts, 0: it has none
    template <int LOW>
    PE_DEV f16v scores(const uint8_t* kt, int li, int g) const {
        f16v s = {};
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) {
            const uint8_t* at = kt + li * (HD * 2) + (((2 * j + g) ^ (li & 7)) * 16);
            const h8v k = *reinterpret_cast<const h8v*>(at);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, hi[j], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, lo[j], s, 0, 0, 0);
            if constexpr (LOW) {
                const h8v l = *reinterpret_cast<const h8v*>(at + LOW);
                s = __builtin_amdgcn_mfma_f32_32x32x16_f16(l, hi[j], s, 0, 0, 0);
            }
        }
        return s;
    }
    // a dim's 8 keys of the lane's half, from two transposing reads: 16 lanes read 4 keys of 16 dims,
    // 8 bytes each, and get one dim's 4 keys each
    static PE_DEV h8v values(uint32_t a) {
        typedef __attribute__((address_space(3))) s4v lds_s4;
        typedef short s8v __attribute__((ext_vector_type(8)));
        const s4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)a);
        const s4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)(a + 8 * (HD * 2)));
        const s8v v = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_bit_cast(h8v, v);
    }
    template <int LOW>
    static PE_DEV void accumulate(const uint8_t* vt, const f16v& p, f16v* o, int li, int g) {
        const int i16 = li & 15, key = 4 * g + (i16 >> 2), half = li >> 4;
        const uint32_t base = lds_address(vt) + key * (HD * 2) + (i16 & 1) * 8;
        const int c0 = (2 * half + ((i16 >> 1) & 1)) ^ (2 * (key & 3));  // chunk of dims 0 .. 31
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            h8v ph, pl;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                ph[i] = (_Float16)p[8 * b + i];
                pl[i] = (_Float16)(p[8 * b + i] - (float)ph[i]);
            }
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) {
                const uint32_t a = base + b * 16 * (HD * 2) + (((4 * (d & 1)) ^ c0) + 8 * (d >> 1)) * 16;
                const h8v v = values(a);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph, o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl, o[d], 0, 0, 0);
                if constexpr (LOW) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(values(a + LOW), ph, o[d], 0, 0, 0);
            }
        }
    }
};

// The softmax of a wave's rows so far: o = sum p V, l = sum p (a lane's half) of the probabilities
// p = exp2(s - r), r the running maximum less `up`.
template <int HD>
struct SpState {
    f16v o[HD / 32];
    float r, l;
    PE_DEV void clear() {
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) o[d] = f16v{};
        r = -__builtin_huge_valf();
        l = 0.f;
    }
    PE_DEV void scale(float f) {
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) o[d] *= f;
    }
    // scores of a tile, to be multiplied by c[r / 4] (positive) -> its probabilities; keys from n on
    // are masked
    PE_DEV void softmax(f16v& s, const float* c, float up, int n, int g) {
        const float NEG_INF = -__builtin_huge_valf();
        if (n < 32) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (8 * (i >> 2) + 4 * g + (i & 3) >= n) s[i] = NEG_INF;
        }
        float mx = NEG_INF;
#pragma unroll
        for (int i = 0; i < 16; i += 4) mx = fmaxf(mx, fmaxf(fmaxf(s[i], s[i + 1]), fmaxf(s[i + 2], s[i + 3])) * c[i >> 2]);
        mx = swap32_max(mx);
        const float rn = fmaxf(r, mx - up);
        const float rs = rn == NEG_INF ? 0.f : rn;  // a row none of whose keys came yet
        const float alpha = __builtin_amdgcn_exp2f(r - rs);
        if (__any(alpha != 1.f)) {
            l *= alpha;
            scale(alpha);
        }
        r = rn;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c[i >> 2], -rs));
            l += s[i];
        }
    }
};

// An fp32 cache's share of a 64-key block on its way through a wave's registers: 8 keys and their
// values, split into two fp16 parts each.
template <int HD>
struct SpSplit {
    static constexpr int N = HD / 32, R = 256 / HD, kPlane = kSpBlock * HD * 2;
    float4 k[N], v[N];
    PE_DEV void load(const float* kb, const float* vb, int64_t row0, int64_t last, int w, int lane) {
#pragma unroll
        for (int f = 0; f < N; ++f) {
            int64_t row = row0 + 8 * w + R * f + lane / (HD / 4);
            row = row < last ? row : last;
            k[f] = *reinterpret_cast<const float4*>(kb + row * HD + 4 * (lane % (HD / 4)));
            v[f] = *reinterpret_cast<const float4*>(vb + row * HD + 4 * (lane % (HD / 4)));
        }
    }
    // E, a multiple of 8, with the largest finite element under 2^(15 + E)
    static PE_DEV int exponent(const float4* x) {
        float top = 0.f;
#pragma unroll
        for (int f = 0; f < N; ++f)
            top = fmaxf(fmaxf(fmaxf(top, fabsf(x[f].x)), fmaxf(fabsf(x[f].y), fabsf(x[f].z))), fabsf(x[f].w));
        top = wave_max<64>(top);
        if (__float_as_uint(top) >= 0x7F800000u) {  // uniform: the same among the finite ones
            top = 0.f;
#pragma unroll
            for (int f = 0; f < N; ++f) {
                const float e[4] = {fabsf(x[f].x), fabsf(x[f].y), fabsf(x[f].z), fabsf(x[f].w)};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (__float_as_uint(e[i]) < 0x7F800000u) top = fmaxf(top, e[i]);
            }
            top = wave_max<64>(top);
        }
        const int e = exponent_of(top);
        return ((e < -100 ? -100 : e) - 14 + 7) >> 3 << 3;
    }
    template <bool VALUES>
    static PE_DEV void store(const float4* x, float f, uint8_t* plane, int w, int lane) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = 8 * w + R * i + lane / (HD / 4), c4 = lane % (HD / 4);
            const float y[4] = {x[i].x * f, x[i].y * f, x[i].z * f, x[i].w * f};
            h4v hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                hi[e] = (_Float16)y[e];
                lo[e] = (_Float16)(y[e] - (float)hi[e]);
            }
            uint8_t* at = plane + row * (HD * 2) + ((c4 >> 1) ^ sp_swizzle<2, VALUES>(row)) * 16 + (c4 & 1) * 8;
            *reinterpret_cast<h4v*>(at) = hi;
            *reinterpret_cast<h4v*>(at + kPlane) = lo;
        }
    }
    // planes: K high, K low, V high, V low; e: exponents of the block's 8 key groups, then of their
    // values. n: keys of the block, the values behind them are cleared.
    PE_DEV void convert(uint8_t* planes, int* e, int n, int w, int lane) {
        if (n < kSpBlock) {
#pragma unroll
            for (int f = 0; f < N; ++f)
                if (8 * w + R * f + lane / (HD / 4) >= n) v[f] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        const int ek = exponent(k), ev = exponent(v);
        store<false>(k, exp2_int(-ek), planes, w, lane);
        store<true>(v, exp2_int(-ev), planes + 2 * kPlane, w, lane);
        if (lane == 0) {
            e[w] = ek;
            e[8 + w] = ev;
        }
    }
};

// The rows of a solo item: fp32 caches on the fp32 matrix instructions.
template <typename T, int HD>
struct SpPick {
    typedef RowsF16<HD> type;
};
template <int HD>
struct SpPick<float, HD> {
    typedef RowsF32<HD> type;
};
template <int HD>
PE_DEV f16v sp_scores(const RowsF32<HD>& q, const uint8_t* kt, int li, int g) {
    return q.scores(kt, li, g);
}
template <int HD>
PE_DEV f16v sp_scores(const RowsF16<HD>& q, const uint8_t* kt, int li, int g) {
    return q.template scores<0>(kt, li, g);
}
template <int HD>
PE_DEV void sp_accumulate(const RowsF32<HD>&, const uint8_t* vt, const f16v& s, f16v* o, int li, int g) {
    RowsF32<HD>::accumulate(vt, s, o, li, g);
}
template <int HD>
PE_DEV void sp_accumulate(const RowsF16<HD>&, const uint8_t* vt, const f16v& s, f16v* o, int li, int g) {
    RowsF16<HD>::template accumulate<0>(vt, s, o, li, g);
}

template <typename T, int HD>
__global__ __launch_bounds__(64 * kSpWaves, 2) void k_shared_prefix(SpArgs p) {
    constexpr bool kHalf = sizeof(T) == 2;
    constexpr int kTile = 32 * HD * (int)sizeof(T), kPieces = kTile / 1024, D = HD / 32, OS = HD + 4;
    // solo: a K and a V tile per wave, or one buffer for both in turn where two are over 16 KB
    constexpr bool kOne = kTile > 8192;
    constexpr int kWaveLds = kOne ? kTile : 2 * kTile;
    // shared: two buffers of a block's planes
    constexpr int kPlane = kSpBlock * HD * 2, kPlanes = (kHalf ? 2 : 4) * kPlane, kLow = kHalf ? 0 : kPlane;
    constexpr int kMerge = kSpWaves * 32 * OS * 4;
    constexpr int kSolo = kSpWaves * kWaveLds, kMost = kSolo > 2 * kPlanes ? kSolo : 2 * kPlanes;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kMost > kMerge ? kMost : kMerge];
    __shared__ float part[kSpWaves][2][32];
    __shared__ int exps[2][16];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 5, li = lane & 31;

    // The wave's item: which rows, which keys [k0, k1) of which cache.
    const bool prefix = (int)blockIdx.x < p.p_blocks, shared = prefix && p.shared;
    const int split = prefix ? (shared ? 2 : kSpWaves) : p.o_split;  // waves that share an item
    const int item = shared ? w & 3 : w / split, sub = shared ? w >> 2 : w % split;
    const T *kb = nullptr, *vb = nullptr;
    int64_t k0 = 0, k1 = 0, row_base;  // output row of r: row_base + r, or by sequence
    int chunk, row0, rows;
    if (prefix) {
        const int kc = p.n_kv * p.p_chunks, tile = blockIdx.x / kc, at = blockIdx.x - tile * kc, j = at % p.n_kv;
        chunk = at / p.n_kv;
        const int64_t len = sp_length(p.p_len, p.p_dtype, 0, p.p_add, p.p_cap);
        k0 = (int64_t)chunk * p.p_keys;
        k1 = k0 + p.p_keys < len ? k0 + p.p_keys : len;
        kb = static_cast<const T*>(p.kp) + (int64_t)j * p.p_cap * HD;
        vb = static_cast<const T*>(p.vp) + (int64_t)j * p.p_cap * HD;
        row0 = shared ? 128 * tile + 32 * item : 32 * tile;
        rows = p.batch * p.group;
        row_base = (int64_t)j * p.group;
        if (k1 <= k0) return;  // the whole workgroup: a chunk past the length
    } else {
        int at = (blockIdx.x - p.p_blocks) * (kSpWaves / split) + item;
        const bool live = at < p.o_items;
        at = live ? at : 0;
        const int per = p.batch * p.n_kv * p.o_tiles;
        chunk = at / per;
        at -= chunk * per;
        const int tile = at % p.o_tiles, j = at / p.o_tiles % p.n_kv, b = at / p.o_tiles / p.n_kv;
        const int64_t len = live ? sp_length(p.o_len, p.o_dtype, b, p.o_add, p.o_cap) : 0;
        k0 = (int64_t)chunk * p.o_keys;
        k1 = k0 + p.o_keys < len ? k0 + p.o_keys : len;
        kb = static_cast<const T*>(p.ko) + ((int64_t)b * p.n_kv + j) * p.o_cap * HD;
        vb = static_cast<const T*>(p.vo) + ((int64_t)b * p.n_kv + j) * p.o_cap * HD;
        row0 = 32 * tile;
        rows = p.group;
        row_base = (int64_t)b * p.n_head + j * p.group;
        chunk += p.p_chunks;
    }
    const auto out_row = [&](int64_t base, int r) {
        if (!prefix) return base + r;
        const int b = r / p.group;
        return base + (int64_t)b * p.n_head + (r - b * p.group);
    };
    const int keys = k1 > k0 ? (int)(k1 - k0) : 0;
    const int64_t last = k1 - 1;
    const int chunks = p.p_chunks + p.o_chunks;
    const bool works = keys > 0 && row0 < rows;
    const float* qrow = works && row0 + li < rows ? p.q + out_row(row_base, row0 + li) * HD : nullptr;
    SpState<HD> st;
    st.clear();
    float up = kLift;
    int top = 0;  // exponent of the values that o holds

    if (shared) {
        RowsF16<HD> q;
        q.load(qrow, p.scale, g);
        const int blocks = (keys + kSpBlock - 1) / kSpBlock;
        const auto take = [&](int t) {
            const uint8_t* kt = lds + (t & 1) * kPlanes + 32 * sub * (HD * 2);
            const int left = keys - kSpBlock * t - 32 * sub, n = left < 32 ? left : 32;
            if (!works || n <= 0) return;
            f16v s = q.template scores<kLow>(kt, li, g);
            float c[4] = {q.unscale, q.unscale, q.unscale, q.unscale};
            float vs[4] = {1.f, 1.f, 1.f, 1.f};
            bool same = true;
            if constexpr (!kHalf) {
                const int* e = exps[t & 1] + 4 * sub;
                int ev[4], t2 = t ? top : -128;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // no smaller than fp32's least: a masked score times c stays -inf
                    c[i] = fminf(fmaxf(ldexpf(c[i], e[i]), 1.1754943508222875e-38f), 1.7014118346046923e38f);
                    ev[i] = e[8 + i];
                    t2 = ev[i] > t2 ? ev[i] : t2;
                }
                t2 = __builtin_amdgcn_readfirstlane(t2);
                if (t && t2 != top) st.scale(ldexpf(1.f, top - t2));
                top = t2;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    vs[i] = ldexpf(1.f, ev[i] - top);
                    same = same && ev[i] == top;
                }
            }
            st.softmax(s, c, kLift, n, g);
            if constexpr (!kHalf) {
                if (!same) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] *= vs[i >> 2];
                }
            }
            RowsF16<HD>::template accumulate<kLow>(kt + (kHalf ? 1 : 2) * kPlane, s, st.o, li, g);
        };
        if constexpr (kHalf) {
            constexpr int N = kPlane / 1024 / kSpWaves;
            const auto stage = [&](int t) {
                const uint32_t at = lds_address(lds) + (t & 1) * kPlanes;
                sp_stage<T, HD, false, N>(kb, k0 + kSpBlock * t, last, at, lane, w * N);
                sp_stage<T, HD, true, N>(vb, k0 + kSpBlock * t, last, at + kPlane, lane, w * N);
            };
            sp_wait_loads<0>();
            stage(0);
            for (int t = 0; t < blocks; ++t) {
                sp_wait_loads<0>();
                __syncthreads();  // the block is there, and nobody reads the other buffer any more
                if (t + 1 < blocks) stage(t + 1);
                const int n = keys - kSpBlock * t;
                if (n < kSpBlock) {
                    sp_clear_rows<HD * 2>(lds + (t & 1) * kPlanes + kPlane, n, kSpBlock, threadIdx.x, 64 * kSpWaves);
                    __syncthreads();
                }
                take(t);
            }
        } else {
            SpSplit<HD> x;
            const auto convert = [&](int t) {
                const int n = keys - kSpBlock * t;
                x.convert(lds + (t & 1) * kPlanes, exps[t & 1], n < kSpBlock ? n : kSpBlock, w, lane);
                if (t + 1 < blocks) x.load(kb, vb, k0 + kSpBlock * (t + 1), last, w, lane);
            };
            x.load(kb, vb, k0, last, w, lane);
            convert(0);
            for (int t = 0; t < blocks; ++t) {
                __syncthreads();  // the block is there, and nobody reads the other buffer any more
                // half of the waves split the next block while the others are at their products
                if (sub == 0 && t + 1 < blocks) convert(t + 1);
                take(t);
                if (sub == 1 && t + 1 < blocks) convert(t + 1);
            }
        }
    } else {
        typename SpPick<T, HD>::type q;
        up = q.kUp;
        q.load(qrow, p.scale, g);
        const int tiles = works ? (keys + 31) / 32 : 0;
        uint8_t* const kt = lds + w * kWaveLds;
        uint8_t* const vt = kOne ? kt : kt + kTile;
        const uint32_t kt_a = lds_address(kt), vt_a = lds_address(vt);
        const float c[4] = {q.unscale, q.unscale, q.unscale, q.unscale};
        sp_wait_loads<0>();
        if (sub < tiles) {
            sp_stage<T, HD, false, kPieces>(kb, k0 + 32 * sub, last, kt_a, lane, 0);
            if (!kOne) sp_stage<T, HD, true, kPieces>(vb, k0 + 32 * sub, last, vt_a, lane, 0);
        }
        for (int t = sub; t < tiles; t += split) {
            const bool more = t + split < tiles;
            const int64_t next = k0 + 32 * (t + split);
            sp_wait_loads<kOne ? 0 : kPieces>();  // K is there, V may be in flight
            f16v s = sp_scores(q, kt, li, g);
            sp_wait_lds();
            if (kOne)
                sp_stage<T, HD, true, kPieces>(vb, k0 + 32 * t, last, vt_a, lane, 0);
            else if (more)
                sp_stage<T, HD, false, kPieces>(kb, next, last, kt_a, lane, 0);
            const int n = keys - 32 * t < 32 ? keys - 32 * t : 32;
            st.softmax(s, c, q.kUp, n, g);
            if (!kOne && more)
                sp_wait_loads<kPieces>();  // V is there, the next K may be in flight
            else
                sp_wait_loads<0>();
            if (n < 32) {
                sp_clear_rows<HD * (int)sizeof(T)>(vt, n, 32, lane, 64);
                sp_wait_lds();
            }
            sp_accumulate(q, vt, s, st.o, li, g);
            sp_wait_lds();
            if (more) {
                if (kOne)
                    sp_stage<T, HD, false, kPieces>(kb, next, last, kt_a, lane, 0);
                else
                    sp_stage<T, HD, true, kPieces>(vb, next, last, vt_a, lane, 0);
            }
        }
    }

    // The records, probabilities and values without their factors. Waves that share an item leave
    // theirs in LDS ([query][dim]) and merge.
    const float down = exp2_int(-(int)up), vscale = ldexpf(down, top);
    const float l = swap32_sum(st.l) * down, r = st.r + up;
    st.scale(vscale);
    if (split == 1) {  // uniform
        if (works && row0 + li < rows) {
            const int64_t at = out_row(row_base, row0 + li) * chunks + chunk;
#pragma unroll
            for (int d = 0; d < D; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    *reinterpret_cast<float4*>(p.rec + at * HD + 32 * d + 8 * (i >> 2) + 4 * g) =
                        make_float4(st.o[d][i], st.o[d][i + 1], st.o[d][i + 2], st.o[d][i + 3]);
            if (g == 0) *reinterpret_cast<float2*>(p.ml + at * 2) = make_float2(r, l);
        }
        return;
    }
    __syncthreads();  // the tiles are no longer read
    float* const po = reinterpret_cast<float*>(lds) + w * 32 * OS;
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<float4*>(po + li * OS + 32 * d + 8 * (i >> 2) + 4 * g) =
                make_float4(st.o[d][i], st.o[d][i + 1], st.o[d][i + 2], st.o[d][i + 3]);
    if (g == 0) {
        part[w][0][li] = r;
        part[w][1][li] = l;
    }
    __syncthreads();
    // the item's waves take its rows; wave `first + step s` holds part s
    const int first = shared ? item : item * split, step = shared ? 4 : 1;
    if (!works) return;
    const int live = rows - row0 < 32 ? rows - row0 : 32;
    for (int it = 64 * sub + lane; it < live * (HD / 4); it += 64 * split) {
        const int qi = it / (HD / 4), c = it % (HD / 4);
        float most = -__builtin_huge_valf();
        for (int s = 0; s < split; ++s) most = fmaxf(most, part[first + step * s][0][qi]);
        const float rs = most == -__builtin_huge_valf() ? 0.f : most;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
        for (int s = 0; s < split; ++s) {
            const int ws = first + step * s;
            const float f = __builtin_amdgcn_exp2f(part[ws][0][qi] - rs);
            sum = fmaf(f, part[ws][1][qi], sum);
            const float4 o = *reinterpret_cast<const float4*>(reinterpret_cast<float*>(lds) + (ws * 32 + qi) * OS + 4 * c);
            v = make_float4(fmaf(f, o.x, v.x), fmaf(f, o.y, v.y), fmaf(f, o.z, v.z), fmaf(f, o.w, v.w));
        }
        const int64_t at = out_row(row_base, row0 + qi) * chunks + chunk;
        *reinterpret_cast<float4*>(p.rec + at * HD + 4 * c) = v;
        if (c == 0) *reinterpret_cast<float2*>(p.ml + at * 2) = make_float2(most, sum);
    }
}

// W waves per (sequence, head): the records of the prefix's chunks and then of the own keys'. HD / 4
// lanes hold a row, the lane groups take every so-many-th record, four loads in flight each.
template <int HD, int W>
__global__ __launch_bounds__(256) void k_shared_prefix_merge(SpArgs p) {
    constexpr int L = HD / 4, N = 64 / L * W, U = 4;
    __shared__ float4 rows[4][L];
    __shared__ float sums[4];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t row = W == 1 ? (int64_t)blockIdx.x * 4 + w : blockIdx.x;
    if (row >= (int64_t)p.batch * p.n_head) return;  // W == 1 only, uniform per wave
    const int64_t b = row / p.n_head;
    const int64_t pl = sp_length(p.p_len, p.p_dtype, 0, p.p_add, p.p_cap);
    const int64_t ol = sp_length(p.o_len, p.o_dtype, b, p.o_add, p.o_cap);
    const int np = pl > 0 ? (int)((pl + p.p_keys - 1) / p.p_keys) : 0;
    const int no = ol > 0 ? (int)((ol + p.o_keys - 1) / p.o_keys) : 0;
    const int n = ol < 0 ? 0 : np + no;  // a sequence that takes no part: zeros
    const int64_t at = row * (p.p_chunks + p.o_chunks);
    const auto record = [&](int i) { return at + (i < np ? i : p.p_chunks + i - np); };
    const float NEG_INF = -__builtin_huge_valf();
    float top = NEG_INF;
    for (int i = lane; i < n; i += 64) top = fmaxf(top, p.ml[record(i) * 2]);
    top = wave_max<64>(top);
    const float rs = top == NEG_INF ? 0.f : top;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    for (int i0 = (W == 1 ? 0 : w * (64 / L)) + lane / L; i0 < n; i0 += N * U) {
        float2 ml[U];
        float4 o[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + N * u;
            const int64_t rec = record(i < n ? i : i0);
            ml[u] = *reinterpret_cast<const float2*>(p.ml + rec * 2);
            o[u] = *reinterpret_cast<const float4*>(p.rec + rec * HD + 4 * (lane % L));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + N * u >= n) break;
            const float f = __builtin_amdgcn_exp2f(ml[u].x - rs);
            sum = fmaf(f, ml[u].y, sum);
            v = make_float4(fmaf(f, o[u].x, v.x), fmaf(f, o[u].y, v.y), fmaf(f, o[u].z, v.z), fmaf(f, o[u].w, v.w));
        }
    }
#pragma unroll
    for (int o = 32; o >= L; o >>= 1) {
        sum += __shfl_xor(sum, o, kWave);
        v.x += __shfl_xor(v.x, o, kWave);
        v.y += __shfl_xor(v.y, o, kWave);
        v.z += __shfl_xor(v.z, o, kWave);
        v.w += __shfl_xor(v.w, o, kWave);
    }
    if constexpr (W > 1) {
        if (lane < L) rows[w][lane] = v;
        if (lane == 0) sums[w] = sum;
        __syncthreads();
        if (w) return;
#pragma unroll
        for (int s = 1; s < W; ++s) {
            if (lane < L) {
                const float4 o = rows[s][lane];
                v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
            }
            sum += sums[s];
        }
    }
    if (lane >= L) return;
    float4 y = n ? make_float4(v.x / sum, v.y / sum, v.z / sum, v.w / sum) : v;
    if (p.round_fp16) y = make_float4(round_to_f16(y.x), round_to_f16(y.y), round_to_f16(y.z), round_to_f16(y.w));
    *reinterpret_cast<float4*>(p.out + row * HD + 4 * lane) = y;
}

struct SpPlan {
    int shared, p_chunks, p_keys, p_tiles, o_chunks, o_keys, o_tiles, o_split;
};

// How the work is cut. Rows of a kv head over 64 go the shared way. The chip holds about 256
// workgroups of eight waves: the prefix is cut into as many chunks as that takes, the own keys into
// items of one to eight waves.
static SpPlan sp_plan(int64_t batch, int n_head, int n_kv, int64_t p_keys, int64_t o_cap) {
    SpPlan s;
    const int64_t group = n_head / n_kv, rows = batch * group;
    s.shared = rows > 64;
    s.p_tiles = (int)(s.shared ? (rows + 127) / 128 : (rows + 31) / 32);
    s.o_tiles = (int)((group + 31) / 32);
    const auto cut = [](int64_t keys, int64_t want, int64_t step, int& chunks, int& per) {
        int64_t k = (keys + want - 1) / want;
        k = (k + step - 1) / step * step;
        k = k < step ? step : k;
        per = (int)k;
        chunks = (int)((keys + k - 1) / k);
    };
    int64_t want = 256 / (n_kv * (int64_t)s.p_tiles);
    cut(p_keys, want < 1 ? 1 : want, s.shared ? kSpBlock : 32 * kSpWaves, s.p_chunks, s.p_keys);
    const int64_t pairs = batch * n_kv * s.o_tiles, tiles = (o_cap + 31) / 32;
    s.o_split = 1;
    while (s.o_split < kSpWaves && s.o_split < tiles && pairs * s.o_split < 2048) s.o_split *= 2;
    want = 2048 / (pairs * s.o_split);
    cut(o_cap, want < 1 ? 1 : want, 32 * s.o_split, s.o_chunks, s.o_keys);
    return s;
}

static bool sp_shape_ok(int64_t batch, int n_head, int n_kv, int head_dim, int64_t p_cap, int64_t o_cap) {
    return batch > 0 && n_head > 0 && n_kv > 0 && n_head % n_kv == 0 && (head_dim == 64 || head_dim == 128) &&
           p_cap >= 0 && o_cap >= 0 && p_cap <= (1LL << 30) && o_cap <= (1LL << 30) && batch <= (1 << 20) &&
           n_head <= (1 << 16) && batch * n_head <= (1 << 24);
}

static int64_t sp_bytes(const SpPlan& s, int64_t batch, int n_head, int head_dim) {
    return batch * n_head * (int64_t)(s.p_chunks + s.o_chunks) * (head_dim + 2) * 4;
}

template <typename T, int HD>
static void launch_shared_prefix(const SpArgs& p, int64_t blocks, hipStream_t s) {
    if (blocks > 0) hipLaunchKernelGGL((k_shared_prefix<T, HD>), dim3((unsigned)blocks), dim3(64 * kSpWaves), 0, s, p);
    const int64_t rows = (int64_t)p.batch * p.n_head;
    // few rows of many records: four waves a row
    if (rows < 2048 && p.p_chunks + p.o_chunks > 8)
        hipLaunchKernelGGL((k_shared_prefix_merge<HD, 4>), dim3((unsigned)rows), dim3(256), 0, s, p);
    else
        hipLaunchKernelGGL((k_shared_prefix_merge<HD, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, p);
}

}  // namespace pe

using namespace pe;

extern "C" int64_t pe_shared_prefix_attn_workspace_bytes(int64_t batch, int n_head, int n_kv, int head_dim,
                                                         int64_t prefix_keys, int64_t own_capacity) {
    if (!sp_shape_ok(batch, n_head, n_kv, head_dim, prefix_keys, own_capacity)) return -PE_ERR_SHAPE;
    return sp_bytes(sp_plan(batch, n_head, n_kv, prefix_keys, own_capacity), batch, n_head, head_dim);
}

extern "C" int pe_shared_prefix_attn(const pe_shared_prefix_args* a, pe_stream_t stream) {
    if (!a) return PE_ERR_NULL;
    if (a->cache_type != PE_TYPE_F32 && a->cache_type != PE_TYPE_F16) return PE_ERR_TYPE;
    if (a->prefix_len_dtype < 0 || a->prefix_len_dtype > 2 || a->own_len_dtype < 0 || a->own_len_dtype > 2)
        return PE_ERR_TYPE;
    if (a->batch == 0) return PE_OK;
    if (!sp_shape_ok(a->batch, a->n_head, a->n_kv, a->head_dim, a->prefix_capacity, a->own_capacity))
        return PE_ERR_SHAPE;
    // the prefix's keys that the launch is cut for: its length where the host knows it
    int64_t keys = a->prefix_capacity;
    if (!a->prefix_len_dtype) {
        keys = a->prefix_len_add < keys ? a->prefix_len_add : keys;
        if (keys < 0) keys = 0;
    }
    const SpPlan s = sp_plan(a->batch, a->n_head, a->n_kv, keys, a->own_capacity);
    const int64_t need = sp_bytes(s, a->batch, a->n_head, a->head_dim);
    if (!a->q || !a->out || (keys && (!a->k_prefix || !a->v_prefix)) ||
        (a->own_capacity && (!a->k_own || !a->v_own)) || (a->prefix_len_dtype && !a->prefix_len) ||
        (a->own_len_dtype && !a->own_len) || (need && !a->workspace))
        return PE_ERR_NULL;
    if (!aligned(a->q, 16) || !aligned(a->out, 16) || !aligned(a->k_prefix, 16) || !aligned(a->v_prefix, 16) ||
        !aligned(a->k_own, 16) || !aligned(a->v_own, 16) || !aligned(a->workspace, 16) ||
        (a->prefix_len_dtype && !aligned(a->prefix_len, a->prefix_len_dtype == 2 ? 8 : 4)) ||
        (a->own_len_dtype && !aligned(a->own_len, a->own_len_dtype == 2 ? 8 : 4)))
        return PE_ERR_ALIGN;
    if (a->workspace_bytes < need) return PE_ERR_SPACE;
    const int64_t p_blocks = (int64_t)a->n_kv * s.p_chunks * s.p_tiles;
    const int64_t items = a->batch * a->n_kv * s.o_tiles * s.o_chunks, per = kSpWaves / s.o_split;
    const int64_t blocks = p_blocks + (items + per - 1) / per;
    if (blocks >= (1 << 23) || items > 0x7FFFFFFF) return PE_ERR_SHAPE;  // a grid holds 2^32 threads
    const int64_t records = a->batch * a->n_head * (int64_t)(s.p_chunks + s.o_chunks);
    SpArgs p{a->q, a->k_prefix, a->v_prefix, a->prefix_capacity, a->k_own, a->v_own, a->own_capacity,
             a->prefix_len, a->prefix_len_dtype, a->prefix_len_add, a->own_len, a->own_len_dtype, a->own_len_add,
             (int)a->batch, a->n_head, a->n_kv, a->n_head / a->n_kv, a->scale * kLog2e,
             s.shared, s.p_chunks, s.p_keys, s.p_tiles, s.o_chunks, s.o_keys, s.o_tiles, s.o_split, (int)p_blocks, (int)items,
             static_cast<float*>(a->workspace), static_cast<float*>(a->workspace) + records * a->head_dim,
             a->round_fp16, a->out};
    hipStream_t st = (hipStream_t)stream;
    if (a->cache_type == PE_TYPE_F16)
        a->head_dim == 64 ? launch_shared_prefix<_Float16, 64>(p, blocks, st)
                          : launch_shared_prefix<_Float16, 128>(p, blocks, st);
    else
        a->head_dim == 64 ? launch_shared_prefix<float, 64>(p, blocks, st)
                          : launch_shared_prefix<float, 128>(p, blocks, st);
    return launch_status();
}
