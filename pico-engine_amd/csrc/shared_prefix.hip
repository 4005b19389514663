// Decode attention of a batch whose sequences share a prefix: for sequence b and query head h (kv
// head j = h / group), with the keys of the prefix and then the sequence's own,
//   out[b][h] = sum_s softmax_s(scale q[b][h] . K_s) V_s.
// softmax over two sets of keys is the merge of the softmaxes over each (running maximum, sum and
// unnormalised row), so the prefix is taken once for all: the batch x group queries of a kv head are
// the rows of one matrix product with its keys, on the matrix cores, and only the own keys are taken
// per sequence. The records (row, maximum, sum) of key chunks are merged by a second launch.
//
// A wave forms 32 x 32 tiles: scores transposed (keys x queries), so that a query's scores sit in a
// lane pair and P^T is the second product's operand as it stands. fp32 caches: the fp32 matrix
// instructions. fp16 caches: v_mfma_f32_32x32x16_f16 on the keys and values as they are, with the
// query (scaled by a power of two to at most 2^14) and the probability (times 2^14) each as the sum of
// two fp16 values, 22 bits: a single fp16 value would cost 2^-12 of each. Scores, maxima, sums and
// rows are fp32.
//
// Two ways over the keys, by the rows of a kv head:
//   shared: four waves of 32 rows each on the same tiles, staged once per workgroup (two buffers, one
//     barrier a tile);
//   solo: 32 rows, the four waves on every fourth tile each, in their own LDS without barriers,
//     merged at the end. The own keys, a group's rows each, always go this way.
#include "pe_common.h"

namespace pe {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef short s4v __attribute__((ext_vector_type(4)));

constexpr int kSpWaves = 4;
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
    int p_chunks, p_keys, o_chunks, o_keys;  // chunks the capacities have, keys of each
    int p_rows, p_tiles, o_tiles;  // rows of a kv head, its row tiles (of 128 or 32), a group's
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

// 16 bytes per lane from global g into LDS at m0 + 16 lane (one wave instruction: 1 KB)
PE_DEV void sp_load16(const void* g, uint32_t m0) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(m0) : "memory", "m0");
}
template <int N>
PE_DEV void sp_wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
PE_DEV void sp_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// LDS image of a 32-key tile: row r's 16-byte chunk c at chunk position c ^ swizzle(r), so that the
// rows that one read takes cover the banks. Values in fp16 are read by rows of four (transposing
// reads), everything else by rows of eight.
template <typename T, bool VALUES>
PE_DEV int sp_swizzle(int r) {
    return VALUES && sizeof(T) == 2 ? 2 * (r & 3) : r & 7;
}

// Pieces [f0, f1) (1 KB each) of the tile of rows row0 .. row0 + 31 of base; rows past `last` are
// the last one again (their scores are masked and their values cleared).
template <typename T, int HD, bool VALUES>
PE_DEV void sp_stage(const T* base, int64_t row0, int64_t last, uint32_t lds, int lane, int f0, int f1) {
    constexpr int E = 16 / sizeof(T), C = HD / E;
#pragma unroll
    for (int f = f0; f < f1; ++f) {
        const int slot = f * 64 + lane, r = slot / C, c = (slot % C) ^ sp_swizzle<T, VALUES>(r);
        const int64_t row = row0 + r < last ? row0 + r : last;
        sp_load16(base + row * HD + E * c, __builtin_amdgcn_readfirstlane(lds + f * 1024));
    }
}

// The rows of a wave's tile: its queries as matrix operands, and the softmax so far.
template <typename T, int HD>
struct SpRows;

// One lane: query li = lane & 31, half g = lane >> 5.
template <int HD>
struct SpRows<float, HD> {
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
        f16v s = {}, s2 = {};  // two chains of half the head's dims: fewer roundings in a row
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) {
            const float4 k = *reinterpret_cast<const float4*>(kt + li * (HD * 4) + (((2 * j + g) ^ (li & 7)) * 16));
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(k.x, q[j].x, s, 0, 0, 0);
            s2 = __builtin_amdgcn_mfma_f32_32x32x2f32(k.y, q[j].y, s2, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(k.z, q[j].z, s, 0, 0, 0);
            s2 = __builtin_amdgcn_mfma_f32_32x32x2f32(k.w, q[j].w, s2, 0, 0, 0);
        }
        return s + s2;
    }
    static constexpr float kLift = 0.f;
    // o += V^T P^T, register r of p the probability of key 8 (r / 4) + 4 g + r % 4
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
struct SpRows<_Float16, HD> {
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
        int e = (int)(__float_as_uint(top) >> 23) - 127;
        e = e < -100 ? -100 : e > 120 ? 120 : e;
        const float f = __uint_as_float((uint32_t)(127 + 13 - e) << 23);
        unscale = __uint_as_float((uint32_t)(127 + e - 13) << 23);
#pragma unroll
        for (int j = 0; j < HD / 16; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = v[8 * j + i] * f;
                hi[j][i] = (_Float16)x;
                lo[j][i] = (_Float16)(x - (float)hi[j][i]);
            }
    }
    PE_DEV f16v scores(const uint8_t* kt, int li, int g) const {
        f16v s = {}, s2 = {};
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) {
            const h8v k = *reinterpret_cast<const h8v*>(kt + li * (HD * 2) + (((2 * j + g) ^ (li & 7)) * 16));
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, hi[j], s, 0, 0, 0);
            s2 = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, lo[j], s2, 0, 0, 0);
        }
        return (s + s2) * unscale;
    }
    static constexpr float kLift = 14.f;
    static PE_DEV void accumulate(const uint8_t* vt, const f16v& p, f16v* o, int li, int g) {
        // 16 lanes read 4 keys of 16 dims, 8 bytes each, and get one dim's 4 keys each
        const int i16 = li & 15, key = 4 * g + (i16 >> 2), half = li >> 4;
        typedef __attribute__((address_space(3))) s4v lds_s4;
        const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)vt + key * (HD * 2) + (i16 & 1) * 8;
        const int c0 = (2 * half + ((i16 >> 1) & 1)) ^ (2 * (key & 3));  // chunk within 8, of dims 0 .. 31
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
                const s4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)a);
                const s4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)(a + 8 * (HD * 2)));
                typedef short s8v __attribute__((ext_vector_type(8)));
                const h8v v = __builtin_bit_cast(h8v, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, ph, o[d], 0, 0, 0);
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pl, o[d], 0, 0, 0);
            }
        }
    }
};

// The softmax of a wave's rows so far: o = sum exp2(s - r) V, l = sum exp2(s - r) (a lane's half).
template <typename T, int HD>
struct SpState {
    f16v o[HD / 32];
    float r, l;
    PE_DEV void clear() {
#pragma unroll
        for (int d = 0; d < HD / 32; ++d) o[d] = f16v{};
        r = -__builtin_huge_valf();
        l = 0.f;
    }
    // scores of a tile -> its probabilities; keys from `n` on are masked
    PE_DEV void softmax(f16v& s, int n, int g) {
        const float NEG_INF = -__builtin_huge_valf();
        if (n < 32) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (8 * (i >> 2) + 4 * g + (i & 3) >= n) s[i] = NEG_INF;
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
        mx = swap32_max(mx);
        const float rn = fmaxf(r, mx - SpRows<T, HD>::kLift);
        const float rs = rn == NEG_INF ? 0.f : rn;  // a row none of whose keys came yet
        const float alpha = __builtin_amdgcn_exp2f(r - rs);
        if (__any(alpha != 1.f)) {
            l *= alpha;
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) o[d] *= alpha;
        }
        r = rn;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(s[i] - rs);
            l += s[i];
        }
    }
};

// Clears the values of a tile's rows from n on (copies of the last one, which may be infinite).
template <typename T, int HD>
PE_DEV void sp_clear_rows(uint8_t* vt, int n, int first, int step) {
    for (int i = n * (HD * (int)sizeof(T) / 16) + first; i < 32 * (HD * (int)sizeof(T) / 16); i += step)
        *reinterpret_cast<float4*>(vt + 16 * i) = make_float4(0.f, 0.f, 0.f, 0.f);
}

template <typename T, int HD>
__global__ __launch_bounds__(64 * kSpWaves, 2) void k_shared_prefix(SpArgs p, int shared, int p_blocks) {
    constexpr int kTile = 32 * HD * (int)sizeof(T), D = HD / 32, kPieces = kTile / 1024, OS = HD + 4;
    // solo: a K and a V tile per wave, or, where that is too much to have two workgroups on a CU, one
    // buffer for both in turn; shared: two buffers of both
    constexpr bool kOne = kTile > 8192;
    constexpr int kWaveLds = kOne ? kTile : 2 * kTile;
    constexpr int kMerge = kSpWaves * 32 * OS * 4;
    constexpr int kLds = kSpWaves * kWaveLds > kMerge ? kSpWaves * kWaveLds : kMerge;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kLds];
    __shared__ float part[kSpWaves][2][32];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, g = lane >> 5, li = lane & 31;
    const uint32_t lds_a = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;

    // which keys, which rows
    int blk = blockIdx.x;
    const bool prefix = blk < p_blocks;
    const T *kb, *vb;
    int64_t k0, k1;  // keys [k0, k1)
    int j, chunk, row0, rows, b = 0;
    if (prefix) {
        const int kc = p.n_kv * p.p_chunks;
        const int tile = blk / kc;
        blk -= tile * kc;
        j = blk % p.n_kv;
        chunk = blk / p.n_kv;
        const int64_t len = sp_length(p.p_len, p.p_dtype, 0, p.p_add, p.p_cap);
        k0 = (int64_t)chunk * p.p_keys;
        k1 = k0 + p.p_keys < len ? k0 + p.p_keys : len;
        kb = static_cast<const T*>(p.kp) + (int64_t)j * p.p_cap * HD;
        vb = static_cast<const T*>(p.vp) + (int64_t)j * p.p_cap * HD;
        row0 = tile * (shared ? 32 * kSpWaves : 32) + (shared ? 32 * w : 0);
        rows = p.p_rows;
    } else {
        blk -= p_blocks;
        const int per = p.batch * p.n_kv * p.o_tiles;
        chunk = blk / per;
        blk -= chunk * per;
        const int tile = blk % p.o_tiles;
        blk /= p.o_tiles;
        j = blk % p.n_kv;
        b = blk / p.n_kv;
        const int64_t len = sp_length(p.o_len, p.o_dtype, b, p.o_add, p.o_cap);
        k0 = (int64_t)chunk * p.o_keys;
        k1 = k0 + p.o_keys < len ? k0 + p.o_keys : len;
        kb = static_cast<const T*>(p.ko) + ((int64_t)b * p.n_kv + j) * p.o_cap * HD;
        vb = static_cast<const T*>(p.vo) + ((int64_t)b * p.n_kv + j) * p.o_cap * HD;
        row0 = 32 * tile;
        rows = p.group;
        chunk += p.p_chunks;
    }
    if (k1 <= k0) return;  // uniform: a chunk past the length
    // row r of the kv head: sequence r / group (the prefix; b for own keys), head j group + r % group
    const auto out_row = [&](int r) {
        const int bb = prefix ? r / p.group : b;
        return (int64_t)bb * p.n_head + j * p.group + (prefix ? r - bb * p.group : r);
    };
    SpRows<T, HD> q;
    q.load(row0 + li < rows ? p.q + out_row(row0 + li) * HD : nullptr, p.scale, g);
    SpState<T, HD> st;
    st.clear();
    const int tiles = (int)((k1 - k0 + 31) / 32);
    const int64_t last = k1 - 1;
    const int chunks = p.p_chunks + p.o_chunks;
    sp_wait_loads<0>();

    if (prefix && shared) {
        const int f0 = w * (kPieces / kSpWaves), f1 = f0 + kPieces / kSpWaves;
        const bool works = row0 < rows;
        const auto stage = [&](int t) {
            const uint32_t at = lds_a + (t & 1) * 2 * kTile;
            sp_stage<T, HD, false>(kb, k0 + 32 * t, last, at, lane, f0, f1);
            sp_stage<T, HD, true>(vb, k0 + 32 * t, last, at + kTile, lane, f0, f1);
        };
        stage(0);
        for (int t = 0; t < tiles; ++t) {
            sp_wait_loads<0>();
            __syncthreads();  // the tile is there, and nobody reads the other buffer any more
            if (t + 1 < tiles) stage(t + 1);
            uint8_t* kt = lds + (t & 1) * 2 * kTile;
            const int n = (int)(k1 - k0 - 32 * t < 32 ? k1 - k0 - 32 * t : 32);
            if (n < 32) {
                sp_clear_rows<T, HD>(kt + kTile, n, threadIdx.x, 64 * kSpWaves);
                __syncthreads();
            }
            if (works) {
                f16v s = q.scores(kt, li, g);
                st.softmax(s, n, g);
                SpRows<T, HD>::accumulate(kt + kTile, s, st.o, li, g);
            }
        }
        if (!works) return;  // no barrier follows
        const float l = swap32_sum(st.l);
        if (row0 + li < rows) {
            const int64_t at = out_row(row0 + li) * chunks + chunk;
            float* o = p.rec + at * HD;
#pragma unroll
            for (int d = 0; d < D; ++d)
#pragma unroll
                for (int r = 0; r < 16; r += 4)
                    *reinterpret_cast<float4*>(o + 32 * d + 8 * (r >> 2) + 4 * g) =
                        make_float4(st.o[d][r], st.o[d][r + 1], st.o[d][r + 2], st.o[d][r + 3]);
            if (g == 0) *reinterpret_cast<float2*>(p.ml + at * 2) = make_float2(st.r, l);
        }
        return;
    }

    uint8_t* const kt = lds + w * kWaveLds;
    uint8_t* const vt = kOne ? kt : kt + kTile;
    const uint32_t kt_a = lds_a + w * kWaveLds, vt_a = kOne ? kt_a : kt_a + kTile;
    if (w < tiles) {
        sp_stage<T, HD, false>(kb, k0 + 32 * w, last, kt_a, lane, 0, kPieces);
        if (!kOne) sp_stage<T, HD, true>(vb, k0 + 32 * w, last, vt_a, lane, 0, kPieces);
    }
    for (int t = w; t < tiles; t += kSpWaves) {
        const bool more = t + kSpWaves < tiles;
        sp_wait_loads<kOne ? 0 : kPieces>();  // K is there, V may be in flight
        f16v s = q.scores(kt, li, g);
        sp_wait_lds();
        if (kOne)
            sp_stage<T, HD, true>(vb, k0 + 32 * t, last, vt_a, lane, 0, kPieces);
        else if (more)
            sp_stage<T, HD, false>(kb, k0 + 32 * (t + kSpWaves), last, kt_a, lane, 0, kPieces);
        const int n = (int)(k1 - k0 - 32 * t < 32 ? k1 - k0 - 32 * t : 32);
        st.softmax(s, n, g);
        if (!kOne && more)
            sp_wait_loads<kPieces>();  // V is there, the next K may be in flight
        else
            sp_wait_loads<0>();
        if (n < 32) {
            sp_clear_rows<T, HD>(vt, n, lane, 64);
            sp_wait_lds();
        }
        SpRows<T, HD>::accumulate(vt, s, st.o, li, g);
        sp_wait_lds();
        if (more) {
            if (kOne)
                sp_stage<T, HD, false>(kb, k0 + 32 * (t + kSpWaves), last, kt_a, lane, 0, kPieces);
            else
                sp_stage<T, HD, true>(vb, k0 + 32 * (t + kSpWaves), last, vt_a, lane, 0, kPieces);
        }
    }
    // the waves' partials: unnormalised rows [query][dim], reference and sum
    const float l = swap32_sum(st.l);
    __syncthreads();  // the partials' rows may lie on another wave's tiles
    float* const po = reinterpret_cast<float*>(lds) + w * 32 * OS;
#pragma unroll
    for (int d = 0; d < D; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<float4*>(po + li * OS + 32 * d + 8 * (r >> 2) + 4 * g) =
                make_float4(st.o[d][r], st.o[d][r + 1], st.o[d][r + 2], st.o[d][r + 3]);
    if (g == 0) {
        part[w][0][li] = st.r;
        part[w][1][li] = l;
    }
    __syncthreads();
    const int live = rows - row0 < 32 ? rows - row0 : 32;
    for (int it = threadIdx.x; it < live * (HD / 4); it += 64 * kSpWaves) {
        const int qi = it / (HD / 4), c = it % (HD / 4);
        float top = part[0][0][qi];
#pragma unroll
        for (int s = 1; s < kSpWaves; ++s) top = fmaxf(top, part[s][0][qi]);
        const float rs = top == -__builtin_huge_valf() ? 0.f : top;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.f;
#pragma unroll
        for (int s = 0; s < kSpWaves; ++s) {
            const float f = __builtin_amdgcn_exp2f(part[s][0][qi] - rs);
            sum = fmaf(f, part[s][1][qi], sum);
            const float4 o = *reinterpret_cast<const float4*>(reinterpret_cast<float*>(lds) + (s * 32 + qi) * OS + 4 * c);
            v = make_float4(fmaf(f, o.x, v.x), fmaf(f, o.y, v.y), fmaf(f, o.z, v.z), fmaf(f, o.w, v.w));
        }
        const int64_t at = out_row(row0 + qi) * chunks + chunk;
        *reinterpret_cast<float4*>(p.rec + at * HD + 4 * c) = v;
        if (c == 0) *reinterpret_cast<float2*>(p.ml + at * 2) = make_float2(top, sum);
    }
}

// One wave per (sequence, head): the records of the prefix's chunks, then of the own keys', in that
// order; HD / 4 lanes hold a row, the lane groups take every 64 / (HD / 4)-th record.
template <int HD>
__global__ __launch_bounds__(256) void k_shared_prefix_merge(SpArgs p) {
    constexpr int L = HD / 4, N = 64 / L;
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= (int64_t)p.batch * p.n_head) return;  // uniform per wave
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
    for (int i = lane / L; i < n; i += N) {
        const int64_t rec = record(i);
        const float2 ml = *reinterpret_cast<const float2*>(p.ml + rec * 2);
        const float f = __builtin_amdgcn_exp2f(ml.x - rs);
        sum = fmaf(f, ml.y, sum);
        const float4 o = *reinterpret_cast<const float4*>(p.rec + rec * HD + 4 * (lane % L));
        v = make_float4(fmaf(f, o.x, v.x), fmaf(f, o.y, v.y), fmaf(f, o.z, v.z), fmaf(f, o.w, v.w));
    }
#pragma unroll
    for (int o = 32; o >= L; o >>= 1) {
        sum += __shfl_xor(sum, o, kWave);
        v.x += __shfl_xor(v.x, o, kWave);
        v.y += __shfl_xor(v.y, o, kWave);
        v.z += __shfl_xor(v.z, o, kWave);
        v.w += __shfl_xor(v.w, o, kWave);
    }
    if (lane >= L) return;
    float4 y = n ? make_float4(v.x / sum, v.y / sum, v.z / sum, v.w / sum) : v;
    if (p.round_fp16) y = make_float4(round_to_f16(y.x), round_to_f16(y.y), round_to_f16(y.z), round_to_f16(y.w));
    *reinterpret_cast<float4*>(p.out + row * HD + 4 * lane) = y;
}

struct SpPlan {
    bool shared;
    int p_chunks, p_keys, p_tiles, o_chunks, o_keys, o_tiles;
};

// How the work is cut: the keys of each workgroup, so that the launch holds about two workgroups per
// CU, and at least the 128 keys that the four waves of one take at a time.
static SpPlan sp_plan(int64_t batch, int n_head, int n_kv, int64_t p_keys, int64_t o_cap) {
    SpPlan s;
    const int64_t group = n_head / n_kv, rows = batch * group;
    s.shared = rows > 64;
    s.p_tiles = (int)(s.shared ? (rows + 127) / 128 : (rows + 31) / 32);
    s.o_tiles = (int)((group + 31) / 32);
    const auto cut = [](int64_t keys, int64_t items, int64_t blocks, int& chunks, int& per) {
        int64_t want = (blocks + items - 1) / items;
        int64_t k = (keys + want - 1) / want;
        k = (k + 127) / 128 * 128;
        if (k < 128) k = 128;
        per = (int)k;
        chunks = (int)((keys + k - 1) / k);
    };
    cut(p_keys, (int64_t)n_kv * s.p_tiles, 512, s.p_chunks, s.p_keys);
    cut(o_cap, batch * n_kv * s.o_tiles, 512, s.o_chunks, s.o_keys);
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
static void launch_shared_prefix(const SpArgs& p, bool shared, hipStream_t s) {
    const int64_t pb = (int64_t)p.n_kv * p.p_chunks * p.p_tiles;
    const int64_t ob = (int64_t)p.batch * p.n_kv * p.o_tiles * p.o_chunks;
    if (pb + ob > 0)
        hipLaunchKernelGGL((k_shared_prefix<T, HD>), dim3((unsigned)(pb + ob)), dim3(64 * kSpWaves), 0, s, p,
                           shared ? 1 : 0, (int)pb);
    hipLaunchKernelGGL(k_shared_prefix_merge<HD>, dim3((unsigned)(((int64_t)p.batch * p.n_head + 3) / 4)), dim3(256), 0,
                       s, p);
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
    const int64_t blocks = (int64_t)a->n_kv * s.p_chunks * s.p_tiles + a->batch * a->n_kv * s.o_tiles * s.o_chunks;
    if (blocks >= (1 << 24)) return PE_ERR_SHAPE;  // a grid holds 2^32 threads
    const int64_t records = a->batch * a->n_head * (int64_t)(s.p_chunks + s.o_chunks);
    SpArgs p{a->q, a->k_prefix, a->v_prefix, a->prefix_capacity, a->k_own, a->v_own, a->own_capacity,
             a->prefix_len, a->prefix_len_dtype, a->prefix_len_add, a->own_len, a->own_len_dtype, a->own_len_add,
             (int)a->batch, a->n_head, a->n_kv, a->n_head / a->n_kv, a->scale * kLog2e,
             s.p_chunks, s.p_keys, s.o_chunks, s.o_keys, (int)(a->batch * (a->n_head / a->n_kv)), s.p_tiles, s.o_tiles,
             static_cast<float*>(a->workspace), static_cast<float*>(a->workspace) + records * a->head_dim,
             a->round_fp16, a->out};
    hipStream_t st = (hipStream_t)stream;
    if (a->cache_type == PE_TYPE_F16)
        a->head_dim == 64 ? launch_shared_prefix<_Float16, 64>(p, s.shared, st)
                          : launch_shared_prefix<_Float16, 128>(p, s.shared, st);
    else
        a->head_dim == 64 ? launch_shared_prefix<float, 64>(p, s.shared, st)
                          : launch_shared_prefix<float, 128>(p, s.shared, st);
    return launch_status();
}
