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
//   solo: the eight waves take 32 rows and every eighth key tile each, in their own LDS without
//     barriers, merged at the end. The own keys go the same way by groups of 16 rows, one to eight
//     waves an item.
// Products: fp32 caches that are taken solo run on the fp32 matrix instructions (bound by memory at
// these row counts). All others run on v_mfma_f32_32x32x16_f16 with the fp32 factors as the sum of
// two fp16 values, 22 bits (one would cost 2^-12 of each): the query, scaled by a power of two to at
// most 2^14; the probability; and an fp32 cache's keys and values, every 8 keys scaled by a
// power of two of their largest element. Products of two low parts are left out (2^-22). A chunk whose keys,
// values or queries lie too far apart for their two parts (SpSplit::find) is taken again by its workgroup on the fp32
// instructions (33 x 8001 with such a key: 36 us to 124, with one in every block 149). Per 16 elements of
// a dot product that is 2 instructions for 16-bit caches and 3 for fp32 ones in place of 8 fp32 instructions
// of twice the time each.
//
// Bounds and times (heads 28/4 of 128, then 14/2 of 64; us, the merge after the +):
//   64 sequences, 32768 fp16 keys, up to 1000 own: 77 + 5.6. The matrix cores; a shared block in steady state
//     keeps them at 1.22 PFLOP/s (a large library product reaches 1.18); the own keys stream at 4.7 to
//     5.5 TB/s, about 9 us are a workgroup's start and end;
//   33 sequences, 8001 fp32 keys, up to 515 own: 31 + 4.4. A shared block takes 6800 cycles, the matrix
//     instructions of a SIMD's two waves 3100 of them; the rest is the vector work that does not fit
//     beside them (split, softmax) and the skew of the two waves at the barrier;
//   3 sequences, 32768 fp16 keys: 8.6 + 4.2; 16 sequences, 1500 fp32 keys: 8.6 + 3.8; 4 sequences, 277 fp32
//     keys: 9.0 in one launch. Latency: lengths, queries, first tiles, a block or two, records.
// Both run at about 1.8 GHz (busy cycles over time), as long matrix work here does. Tried without gain: key
// rows swizzled over all 64 banks; the barrier of a block between softmax and values, so that values and
// the next scores run back to back (30.3 for 28.9 us, fp16 85 for 75); half the waves half a block behind
// the others, with a barrier every half block (30.5 for 29.5, fp16 83 for 78); low parts by one instruction
// that rounds to a half register (30.9 for 29.5).
#include "pe_common.h"

#include <cmath>

namespace pe {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef _Float16 h4v __attribute__((ext_vector_type(4)));
typedef short s4v __attribute__((ext_vector_type(4)));

constexpr int kSpWaves = 8;
constexpr int kSpBlock = 64;       // keys of a shared block
// The probabilities are exp2(s - r) for a reference r that starts kUp under a row's maximum and
// moves when a score comes to lie more than kRoom over it: up to 2^15 they fit fp16, and the rows are
// rescaled a few times instead of in most tiles.
constexpr float kUp = 8.f, kRoom = 15.f;
constexpr float kLog2e = 1.4426950408889634f;
// Exponents of the values of fp32 caches in the shared way: of a group of zeros, and how far apart those that a
// wave takes may lie, so that its sums stay within fp32.
constexpr int kZeros = -114, kFar = 64;

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
// 16 bytes per lane from global g (uniform) + off into LDS at m0 + 16 lane (one wave instruction: 1 KB). The
// address goes through a scalar copy: read back from a spill, which is a vector instruction's work, it would have to
// be five wait states old, and the compiler does not see the load.
PE_DEV void sp_load16(const void* g, uint32_t off, uint32_t m0) {
    const void* at;
    asm volatile("s_mov_b32 m0, %3\n\ts_mov_b64 %0, %2\n\tglobal_load_lds_dwordx4 %1, %0"
                 : "=&s"(at)
                 : "v"(off), "s"(g), "s"(m0)
                 : "memory", "m0");
}
// the same from an address per lane
PE_DEV void sp_load16(const float* g, uint32_t m0) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(g), "s"(m0) : "memory", "m0");
}
template <int N>
PE_DEV void sp_wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
PE_DEV void sp_wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The largest of a wave's whole numbers.
template <int CTRL>
PE_DEV uint32_t dpp_max(uint32_t v) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xF, 0xF, false);
    return v > o ? v : o;
}

// Records go past the L2, whose dirty lines the launch's end would have to write back. A store of 16 bytes reads its
// data after it has issued, and the compiler does not see this one: the wait keeps the registers from the next
// instruction.
PE_DEV void store_record(float* p, const float4& v) {
    typedef float f4v __attribute__((ext_vector_type(4)));
    const f4v x = {v.x, v.y, v.z, v.w};
    asm volatile("global_store_dwordx4 %0, %1, off sc0 sc1\n\ts_nop 1" ::"v"(p), "v"(x) : "memory");
}

PE_DEV float exp2_int(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
PE_DEV int exponent_of(float x) { return (int)(__float_as_uint(x) >> 23) - 127; }

// 8 fp32 values as the sums of two fp16 values, each rounded to nearest: within 2^-23 of the value from
// 2^-3 on, 2^-25 below. The low part's difference is one instruction that reads the high part's half.
typedef float f2v __attribute__((ext_vector_type(2)));
typedef _Float16 h2v __attribute__((ext_vector_type(2)));
PE_DEV void split2(float a, float b, h2v& hi, h2v& lo) {
    const f2v x = {a, b};
    hi = __builtin_convertvector(x, h2v);
    f2v d;
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]" : "=v"(d.x) : "v"(hi), "v"(a));
    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(d.y) : "v"(hi), "v"(b));
    lo = __builtin_convertvector(d, h2v);
}

// A positive factor of scores: no smaller than fp32's least (a masked score times it stays -inf).
PE_DEV float sp_positive(float c) { return fminf(fmaxf(c, 1.1754943508222875e-38f), 1.7014118346046923e38f); }

// LDS image of a key tile: row r's 16-byte chunk c at chunk position c ^ swizzle(r), so that the
// rows that one read takes cover the banks. 16-bit values are read by rows of four (transposing
// reads), everything else by rows of eight.
template <int SIZE, bool VALUES>
PE_DEV int sp_swizzle(int r) {
    return VALUES && SIZE == 2 ? 2 * (r & 3) : r & 7;
}

// Pieces f0 .. f0 + N - 1 (1 KB each) of the tile that starts at base, whose rows behind `last` are that
// one again (their scores are masked and their values cleared). A piece is contiguous in memory;
// the lanes take its chunks in the image's order.
template <typename T, int HD, bool VALUES, int N>
PE_DEV void sp_stage(const T* base, int64_t last, uint32_t lds, int lane, int f0) {
    constexpr int E = 16 / sizeof(T), C = HD / E, ROWS = 64 / C;
    const bool whole = last >= ROWS * (f0 + N) - 1;
#pragma unroll
    for (int f = 0; f < N; ++f) {
        const int r = ROWS * (f0 + f) + lane / C, x = lane ^ sp_swizzle<sizeof(T), VALUES>(r);
        const uint32_t at = __builtin_amdgcn_readfirstlane(lds + (f0 + f) * 1024);
        if (whole)
            sp_load16(reinterpret_cast<const uint8_t*>(base) + 1024 * (f0 + f), 16 * x, at);
        else
            sp_load16(base, (uint32_t)((r < (int)last ? r : (int)last) * C + x % C) * 16, at);
    }
}

// Clears rows [n, 32) of a tile of values (copies of the last one, which may be infinite).
template <int ROW>
PE_DEV void sp_clear_rows(uint8_t* vt, int n, int rows, int first, int step) {
    for (int i = n * (ROW / 16) + first; i < rows * (ROW / 16); i += step)
        *reinterpret_cast<float4*>(vt + 16 * i) = make_float4(0.f, 0.f, 0.f, 0.f);
}

// A dim's 4 keys from a and 4 from a + STEP, by transposing reads: 16 lanes read 4 keys of 16 dims, 8
// bytes each, and get one dim's 4 keys each.
template <int STEP>
PE_DEV h8v transposed(uint32_t a) {
    typedef __attribute__((address_space(3))) s4v lds_s4;
    typedef short s8v __attribute__((ext_vector_type(8)));
    const s4v x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)a);
    const s4v y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)(a + STEP));
    const s8v v = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(h8v, v);
}

// A wave's share, ROWS, of a workgroup's queries into an LDS image of rows of HD floats, chunk c of row r
// at c ^ (r & 7): rows [first, first + ROWS) of the kv head, of which `rows` are there (the last one
// stands in for the others). Read by each lane for itself, 32 rows an instruction, they took 3 of a
// workgroup's first 6 us.
template <int HD, int ROWS>
PE_DEV void sp_stage_queries(const SpArgs& p, int j, int first, int rows, uint32_t lds, int lane) {
    constexpr int C = HD / 4, R = 64 / C;
    int r = first + lane / C;
    int seq = r / p.group, head = r - seq * p.group;
#pragma unroll
    for (int f = 0; f < ROWS / R; ++f) {
        const bool there = r < rows;
        const int64_t row = there ? (int64_t)seq * p.n_head + j * p.group + head : (int64_t)p.batch * p.n_head - p.n_head + (j + 1) * p.group - 1;
        const uint32_t at = __builtin_amdgcn_readfirstlane(lds + f * 1024);
        sp_load16(p.q + row * HD + ((lane % C) ^ (r & 7)) * 4, at);
        r += R;
        for (head += R; head >= p.group; head -= p.group) ++seq;
    }
}

// A wave's 32 queries as matrix operands and the products with a tile of 32 keys. One lane: query
// (or key, or dim) li = lane & 31, half g = lane >> 5. Register r of the scores is key
// 8 (r / 4) + 4 g + r % 4; they have to be multiplied by `unscale`.
template <int HD>
struct RowsF32 {
    static constexpr float unscale = 1.f;
    float4 q[HD / 8];
    // row r of an image of queries (sp_stage_queries)
    PE_DEV void load(const uint8_t* image, int r, float scale, int g) {
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) {
            q[j] = *reinterpret_cast<const float4*>(image + r * (HD * 4) + ((2 * j + g) ^ (r & 7)) * 16);
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
    h8v hi[HD / 16], lo[HD / 16];
    float unscale;
    int down;     // unscale is 2^down times the scale's magnitude
    bool uneven;  // eight neighbouring elements lie 2^-16 under the row's largest, or that one is tiny or infinite (SpSplit)
    PE_DEV void load(const uint8_t* image, int r, float scale, int g) {
        float v[HD / 2], top = 0.f;
#pragma unroll
        for (int j = 0; j < HD / 16; ++j)
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                const float4 x = *reinterpret_cast<const float4*>(image + r * (HD * 4) + ((4 * j + 2 * g + i / 4) ^ (r & 7)) * 16);
                v[8 * j + i] = x.x;
                v[8 * j + i + 1] = x.y;
                v[8 * j + i + 2] = x.z;
                v[8 * j + i + 3] = x.w;
            }
        uint32_t least = 0xFFFFFFFFu;
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) {
            float m = 0.f;
#pragma unroll
            for (int i = 8 * j; i < 8 * j + 8; ++i) m = fmaxf(m, fabsf(v[i]));
            top = fmaxf(top, m);
            const uint32_t b = __float_as_uint(m) - 1;  // zeros are no small values
            least = b < least ? b : least;
        }
        top = swap32_max(top);
        uneven = top > 0.f && (!(top >= 0x1p-99f && top < __builtin_huge_valf()) || least < __float_as_uint(top) - (16u << 23));
        // the row's largest element to 2^13 .. 2^14, by factors that fp32 holds with their inverses (under
        // 2^-113 it stays smaller); the scale of the scores comes after the products
        int e = exponent_of(top);
        e = e < -113 ? -113 : e > 127 ? 127 : e;
        const float f = copysignf(exp2_int(13 - e), scale);
        down = e - 13;
        unscale = sp_positive(exp2_int(down) * fabsf(scale));
#pragma unroll
        for (int j = 0; j < HD / 16; ++j)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                h2v h, l;
                split2(v[8 * j + i] * f, v[8 * j + i + 1] * f, h, l);
                hi[j][i] = h.x, hi[j][i + 1] = h.y;
                lo[j][i] = l.x, lo[j][i + 1] = l.y;
            }
    }
    // LOW: bytes from a tile to its low parts, 0: it has none. Four operands are in flight: each one's
    // registers take the fourth next as soon as its products have read them. beside(i): work for the
    // vector units while the i-th operand's products run.
    template <int LOW, typename F>
    PE_DEV f16v scores(const uint8_t* kt, int li, int g, const F& beside) const {
        constexpr int J = HD / 16, N = LOW ? 2 * J : J;
        const uint8_t* at = kt + li * (HD * 2);
        const int x = (g ^ (li & 7)) * 16;  // chunk 2 j + g: j flips bits above g's
        const auto operand = [&](int i) { return *reinterpret_cast<const h8v*>(at + (i < J ? 0 : LOW) + (x ^ (32 * (i % J)))); };
        h8v k[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) k[i] = operand(i);
        f16v s = {};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[i & 3], hi[i % J], s, 0, 0, 0);
            if (i < J) s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[i & 3], lo[i % J], s, 0, 0, 0);
            if (i + 4 < N) k[i & 3] = operand(i + 4);
            beside(i);
            __builtin_amdgcn_sched_barrier(0);
        }
        return s;
    }
    // operand i of a tile's values: keys 16 (i / D) .., dims 32 (i % D) ..
    static PE_DEV uint32_t values_at(const uint8_t* vt, int li, int g) {
        const int i16 = li & 15, key = 4 * g + (i16 >> 2), half = li >> 4;
        const int c0 = (2 * half + ((i16 >> 1) & 1)) ^ (2 * (key & 3));  // chunk of dims 0 .. 31
        return lds_address(vt) + key * (HD * 2) + (i16 & 1) * 8 + c0 * 16;
    }
    // in the order of use: the dims of the first 16 keys, high and low parts, then of the others
    template <int LOW>
    static PE_DEV h8v values_of(uint32_t at, int i) {
        constexpr int D = HD / 32, P = LOW ? 2 : 1;
        const int d = i % D, low = i / D % P, b = i / (D * P);
        return transposed<8 * HD * 2>((at ^ (64 * (d & 1))) + 128 * (d >> 1) + b * 16 * (HD * 2) + low * LOW);
    }
    template <int LOW>
    static PE_DEV void load_values(uint32_t at, h8v* v) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = values_of<LOW>(at, i);
    }
    template <int LOW, typename F>
    static PE_DEV void accumulate(uint32_t at, h8v* v, const f16v& p, f16v* o, const F& beside) {
        constexpr int D = HD / 32, P = LOW ? 2 : 1, N = 2 * D * P;
        h8v ph[2], pl[2];
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
            h2v h, l;
            split2(p[i], p[i + 1], h, l);
            ph[i >> 3][i & 7] = h.x, ph[i >> 3][(i & 7) + 1] = h.y;
            pl[i >> 3][i & 7] = l.x, pl[i >> 3][(i & 7) + 1] = l.y;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int d = i % D, low = i / D % P, b = i / (D * P);
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i & 3], ph[b], o[d], 0, 0, 0);
            if (!low) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i & 3], pl[b], o[d], 0, 0, 0);
            if (i + 4 < N) v[i & 3] = values_of<LOW>(at, i + 4);
            beside(i);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
};

// The softmax of a wave's rows so far: o = sum p V, l = sum p (a lane's half) of the probabilities
// p = exp2(s - r). With weighted values V = 2^w V' the tiles hold V': p = exp2(s + w - r) for the row, without 2^w
// for the sum.
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
    // are masked. WEIGHTED: probabilities times 2^w[r / 4] (uniform, at most 128 apart in all), the exponents of the
    // keys' values: the largest product sets the reference, so that fp16's bits go to the keys that make the
    // result and not to those with the largest values.
    template <bool WEIGHTED>
    PE_DEV void softmax(f16v& s, const float* c, const int* w, int n, int g) {
        const float NEG_INF = -__builtin_huge_valf();
        if (n < 32) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (8 * (i >> 2) + 4 * g + (i & 3) >= n) s[i] = NEG_INF;
        }
        float mx = NEG_INF;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const float m = fmaxf(fmaxf(fmaxf(fmaxf(NEG_INF, s[i]), s[i + 1]), s[i + 2]), s[i + 3]);
            mx = fmaxf(mx, WEIGHTED ? fmaf(m, c[i >> 2], (float)w[i >> 2]) : m * c[i >> 2]);
        }
        mx = swap32_max(mx);
        const bool moves = mx > r + kRoom;  // the first finite score does
        if (__any(moves)) {
            const float rn = moves ? mx - kUp : r, alpha = moves ? __builtin_amdgcn_exp2f(r - rn) : 1.f;
            r = rn;
            l *= alpha;
            scale(alpha);
        }
        const float rs = r == NEG_INF ? 0.f : r;  // a row none of whose keys came yet
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const float from = WEIGHTED ? (float)w[i >> 2] - rs : -rs;
            float sum = 0.f;
#pragma unroll
            for (int k = i; k < i + 4; ++k) {
                s[k] = __builtin_amdgcn_exp2f(fmaf(s[k], c[i >> 2], from));
                if constexpr (WEIGHTED)
                    sum = k > i ? sum + s[k] : s[k];
                else
                    l += s[k];
            }
            if constexpr (WEIGHTED) l += ldexpf(sum, -w[i >> 2]);
        }
    }
};

// The own keys of a group: 16 queries and tiles of TK keys, on the 16 x 16 instructions. One lane:
// query (or key, or dim) qi = lane & 15, quarter h = lane >> 4. Score 4 u + r is key 16 u + 4 h + r.
typedef float f4v __attribute__((ext_vector_type(4)));

template <typename T, int HD>
struct OwnRows;

template <int HD>
struct OwnRows<float, HD> {
    static constexpr int TK = HD == 64 ? 32 : 16, U = TK / 16;
    float4 q[HD / 16];
    static constexpr float unscale = 1.f;
    PE_DEV void load(const float* row, float scale, int h) {
#pragma unroll
        for (int j = 0; j < HD / 16; ++j) {
            q[j] = row ? *reinterpret_cast<const float4*>(row + 16 * j + 4 * h) : make_float4(0.f, 0.f, 0.f, 0.f);
            q[j].x *= scale;
            q[j].y *= scale;
            q[j].z *= scale;
            q[j].w *= scale;
        }
    }
    PE_DEV void scores(const uint8_t* kt, float* out, int qi, int h) const {
        f4v s[U] = {};
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) {
                const float4 k = *reinterpret_cast<const float4*>(kt + (16 * u + qi) * (HD * 4) + (((4 * j + h) ^ (qi & 7)) * 16));
                s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(k.x, q[j].x, s[u], 0, 0, 0);
                s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(k.y, q[j].y, s[u], 0, 0, 0);
                s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(k.z, q[j].z, s[u], 0, 0, 0);
                s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(k.w, q[j].w, s[u], 0, 0, 0);
            }
#pragma unroll
        for (int i = 0; i < 4 * U; ++i) out[i] = s[i >> 2][i & 3];
    }
    static PE_DEV void accumulate(const uint8_t* vt, const float* p, f4v* o, int qi, int h) {
#pragma unroll
        for (int i = 0; i < 4 * U; ++i) {
            const int row = 16 * (i >> 2) + 4 * h + (i & 3), x = (4 * h + (i & 3)) & 7;
            const uint8_t* at = vt + row * (HD * 4) + (qi & 3) * 4;
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) {
                const int c = ((4 * (d & 1) + (qi >> 2)) ^ x) + 8 * (d >> 1);
                o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(*reinterpret_cast<const float*>(at + 16 * c), p[i], o[d], 0, 0, 0);
            }
        }
    }
};

template <int HD>
struct OwnRows<_Float16, HD> {
    static constexpr int TK = 32, U = 2;
    h8v hi[HD / 32], lo[HD / 32];
    float unscale;
    PE_DEV void load(const float* row, float scale, int h) {
        float v[HD / 4], top = 0.f;
#pragma unroll
        for (int i = 0; i < HD / 4; i += 4) {
            const float4 x = row ? *reinterpret_cast<const float4*>(row + 32 * (i / 8) + 8 * h + i % 8) : make_float4(0.f, 0.f, 0.f, 0.f);
            v[i] = x.x;
            v[i + 1] = x.y;
            v[i + 2] = x.z;
            v[i + 3] = x.w;
        }
#pragma unroll
        for (int i = 0; i < HD / 4; ++i) top = fmaxf(top, fabsf(v[i]));
        top = swap32_max(swap16_max(top));
        int e = exponent_of(top);
        e = e < -113 ? -113 : e > 127 ? 127 : e;
        const float f = copysignf(exp2_int(13 - e), scale);
        unscale = sp_positive(exp2_int(e - 13) * fabsf(scale));
#pragma unroll
        for (int i = 0; i < HD / 4; i += 2) {
            h2v a, b;
            split2(v[i] * f, v[i + 1] * f, a, b);
            hi[i / 8][i % 8] = a.x, hi[i / 8][i % 8 + 1] = a.y;
            lo[i / 8][i % 8] = b.x, lo[i / 8][i % 8 + 1] = b.y;
        }
    }
    PE_DEV void scores(const uint8_t* kt, float* out, int qi, int h) const {
        f4v s[U] = {};
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < HD / 32; ++j) {
                const h8v k = *reinterpret_cast<const h8v*>(kt + (16 * u + qi) * (HD * 2) + (((4 * j + h) ^ (qi & 7)) * 16));
                s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, hi[j], s[u], 0, 0, 0);
                s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, lo[j], s[u], 0, 0, 0);
            }
#pragma unroll
        for (int i = 0; i < 4 * U; ++i) out[i] = s[i >> 2][i & 3];
    }
    static PE_DEV void accumulate(const uint8_t* vt, const float* p, f4v* o, int qi, int h) {
        h8v ph, pl;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            h2v a, b;
            split2(p[i], p[i + 1], a, b);
            ph[i] = a.x, ph[i + 1] = a.y;
            pl[i] = b.x, pl[i + 1] = b.y;
        }
        const int row = 4 * h + (qi >> 2);  // and 16 on
        const uint32_t base = lds_address(vt) + row * (HD * 2) + (qi & 1) * 8;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) {
            const int c = ((2 * (d & 3) + ((qi >> 1) & 1)) ^ (2 * (row & 3))) + 8 * (d >> 2);
            const h8v v = transposed<16 * HD * 2>(base + 16 * c);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, ph, o[d], 0, 0, 0);
            o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pl, o[d], 0, 0, 0);
        }
    }
};

// A wave's 8 keys, or their values, of a 64-key block of an fp32 cache on their way through its registers
// into two fp16 parts each, in kSteps steps that go beside the products with the block before.
template <int HD, bool VALUES>
struct SpSplit {
    static constexpr int N = HD / 32, R = 256 / HD, kPlane = kSpBlock * HD * 2, kSteps = HD / 8;
    float4 x[N];
    uint32_t top, least;
    float f;
    uint64_t uneven = 0;  // not 0: see find
    h2v h0, l0;
    // the wave's 8 rows of the block at base, which holds n keys; the rows behind them are zeros
    PE_DEV void load(const float* base, int n, int w, int lane) {
        typedef unsigned int u4v __attribute__((ext_vector_type(4)));
        const auto all = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(base), 0, n * (HD * 4), 0x00020000);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const u4v y = __builtin_amdgcn_raw_buffer_load_b128(all, 8 * w * (HD * 4) + 16 * lane + 1024 * i, 0, 0);
            x[i] = __builtin_bit_cast(float4, y);
        }
    }
    // The exponent E with the largest element in [2^(14 + E), 2^(15 + E)): the two parts hold every element to
    // 2^-23 of itself or 2^-39 of the largest. `uneven` says where that is not enough: where four neighbouring
    // dims of a key lie kUneven under the largest (zeros are exact), so that a value keeps 2^-25 of its neighbours and a
    // key's element 2^-23, and where the largest is infinite or under 2^-99. Four normal values lie 2^-14 under the
    // largest of 1024 once in 10^11 blocks, and a key whose values are all 2^8 smaller than the others' stays even. Eight
    // stages.
    static constexpr uint32_t kUneven = (VALUES ? 14u : 16u) << 23;
    // from 0 on, two instructions: maxima of two unknown values quieten both first
    static PE_DEV float largest(const float4& a) { return fmaxf(fmaxf(fmaxf(fmaxf(0.f, fabsf(a.x)), fabsf(a.y)), fabsf(a.z)), fabsf(a.w)); }
    // the smaller, a zero being no small value: the bits less one
    static PE_DEV uint32_t smaller(uint32_t least, float a) {
        const uint32_t b = __float_as_uint(a) - 1;
        return b < least ? b : least;
    }
    PE_DEV void find(int stage, int* e) {
        if (stage == 0) {
            least = 0xFFFFFFFFu;
            float m = 0.f;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float r = largest(x[i]);
                m = fmaxf(m, r);
                least = smaller(least, r);
            }
            top = __float_as_uint(m);
        }
        if (stage == 1) top = dpp_max<0xB1>(top);   // quad_perm [1,0,3,2]
        if (stage == 2) top = dpp_max<0x4E>(top);   // quad_perm [2,3,0,1]
        if (stage == 3) top = dpp_max<0x141>(top);  // row_half_mirror
        if (stage == 4) top = dpp_max<0x140>(top);  // row_mirror
        if (stage == 5) {
            const auto a = __builtin_amdgcn_permlane16_swap(top, top, false, false);
            top = a[0] > a[1] ? a[0] : a[1];
        }
        if (stage == 6) {
            const auto a = __builtin_amdgcn_permlane32_swap(top, top, false, false);
            top = __builtin_amdgcn_readfirstlane(a[0] > a[1] ? a[0] : a[1]);
        }
        if (stage == 7) {
            int k = (int)(top >> 23) - 127;
            k = (k < -100 ? -100 : k) - 14;
            f = exp2_int(-k);
            if ((threadIdx.x & 63) == 0) *e = k;
            // zeros alone are even, all that comes with a tiny or infinite largest element is not
            const bool odd = top - (28u << 23) >= 0x7F800000u - (28u << 23);
            uneven |= __ballot(least < (!top ? 0 : odd ? 0xFFFFFFFEu : top - kUneven));
        }
    }
    // Where a lane's half chunk of the wave's first rows goes in a plane; those of piece i lie i R rows on, at
    // the chunk with other bits flipped (sp_swizzle).
    static PE_DEV uint32_t place(int w, int lane) {
        const int row = 8 * w + lane / (HD / 4), c4 = lane % (HD / 4);
        return row * (HD * 2) + ((c4 >> 1) ^ sp_swizzle<2, VALUES>(row)) * 16 + (c4 & 1) * 8;
    }
    // step i: planes: LDS address of the high parts, the low ones behind them; e: the group's exponent
    PE_DEV void step(int i, uint32_t planes, uint32_t place, int* e) {
        constexpr int H = kSteps / 2;
        if (i < H) {
#pragma unroll
            for (int k = 8 / H * i; k < 8 / H * (i + 1); ++k) find(k, e);
        } else if (const int n = (i - H) >> 1; (i - H) & 1) {
            h2v h1, l1;
            split2(x[n].z * f, x[n].w * f, h1, l1);
            const h4v hi = {h0.x, h0.y, h1.x, h1.y}, lo = {l0.x, l0.y, l1.x, l1.y};
            typedef __attribute__((address_space(3))) h4v lds_h4;
            const uint32_t at = planes + (place ^ (16 * sp_swizzle<2, VALUES>(R * n))) + R * n * (HD * 2);
            *(lds_h4*)(uintptr_t)at = hi;
            *(lds_h4*)(uintptr_t)(at + kPlane) = lo;
        } else {
            split2(x[n].x * f, x[n].y * f, h0, l0);
        }
    }
};

// What a workgroup's waves exchange at the end: the rows of their items ([query][dim]) over the tiles,
// and per query its reference, sum and output row.
struct SpShared {
    uint8_t* lds;
    float (*ref)[32];
    float (*sum)[32];
    int (*row)[32];
};

PE_DEV float4 sp_rounded(const float4& y, int round_fp16) {
    return round_fp16 ? make_float4(round_to_f16(y.x), round_to_f16(y.y), round_to_f16(y.z), round_to_f16(y.w)) : y;
}

// The record of a wave's Q queries (lane = query + Q part; v[i]: dims 256 / Q i + 4 part ..): stored, or
// merged with those of the item's other waves (sub of split; the waves first, first + step, ..) in LDS.
// ALL: the waves had all of the queries' keys, so the merge is the output.
template <int HD, int Q, bool ALL>
PE_DEV void sp_finish(const SpArgs& p, const SpShared& m, float4* v, float r, float l, int my_row, bool works, int live, int chunk,
                      int item, int sub, int split, int step) {
    constexpr int W = 256 / Q, N = HD / W, OS = HD + 4;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), qi = lane % Q, at = 4 * (lane / Q);
    const int chunks = p.p_chunks + p.o_chunks;
    live = live < Q ? live : Q;
    if (!ALL && split == 1) {  // uniform
        if (works && qi < live) {
            const int64_t rec = (int64_t)my_row * chunks + chunk;
#pragma unroll
            for (int i = 0; i < N; ++i) store_record(p.rec + rec * HD + W * i + at, v[i]);
            if (at == 0) *reinterpret_cast<float2*>(p.ml + rec * 2) = make_float2(r, l);
        }
        return;
    }
    if (at == 0) m.ref[w][qi] = r;
    __syncthreads();  // and the tiles are no longer read
    const int first = step > 1 ? item : item * split;
    float most = m.ref[first][qi];
    for (int s = 1; s < split; ++s) most = fmaxf(most, m.ref[first + step * s][qi]);
    const float f = __builtin_amdgcn_exp2f(r - (most == -__builtin_huge_valf() ? 0.f : most));
    float* const po = reinterpret_cast<float*>(m.lds) + (w * Q + qi) * OS + at;
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<float4*>(po + W * i) = make_float4(v[i].x * f, v[i].y * f, v[i].z * f, v[i].w * f);
    if (at == 0) {
        m.sum[w][qi] = l * f;
        m.row[w][qi] = my_row;
    }
    __syncthreads();
    if (!ALL && !works) return;
    // every wave of the item takes its share of the rows
    if (!ALL && sub == 0 && lane < live) {
        float sum = m.sum[first][lane];
        for (int s = 1; s < split; ++s) sum += m.sum[first + step * s][lane];
        *reinterpret_cast<float2*>(p.ml + ((int64_t)my_row * chunks + chunk) * 2) = make_float2(most, sum);
    }
    const float* const p0 = reinterpret_cast<float*>(m.lds) + first * Q * OS;
#pragma unroll 2
    for (int it = 64 * sub + lane; it < live * (HD / 4); it += 64 * split) {
        const int row = it / (HD / 4), c = it % (HD / 4);
        const float* o = p0 + row * OS + 4 * c;
        float4 x = *reinterpret_cast<const float4*>(o);
        for (int s = 1; s < split; ++s) {
            const float4 y = *reinterpret_cast<const float4*>(o + s * step * Q * OS);
            x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
        }
        if constexpr (ALL) {
            float sum = m.sum[first][row];
            for (int s = 1; s < split; ++s) sum += m.sum[first + step * s][row];
            // a sequence without keys: zeros
            x = works ? make_float4(x.x / sum, x.y / sum, x.z / sum, x.w / sum) : make_float4(0.f, 0.f, 0.f, 0.f);
            *reinterpret_cast<float4*>(p.out + (int64_t)m.row[first][row] * HD + 4 * c) = sp_rounded(x, p.round_fp16);
        } else {
            store_record(p.rec + ((int64_t)m.row[first][row] * chunks + chunk) * HD + 4 * c, x);
        }
    }
}

// 16 queries of a group on the keys of one sequence, by waves of their own: the own keys' items of split
// waves each, or, ALL, the prefix's keys and then the own ones by a whole workgroup.
template <typename T, int HD, bool ALL>
PE_DEV void sp_own(const SpArgs& p, const SpShared& m, int block) {
    typedef OwnRows<T, HD> Rows;
    constexpr int TK = Rows::TK, N = 4 * Rows::U, kTile = TK * HD * (int)sizeof(T), kPieces = kTile / 1024;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), qi = lane & 15, h = lane >> 4;
    const int split = ALL ? kSpWaves : p.o_split, item = ALL ? 0 : w / split, sub = ALL ? w : w % split;
    int at = block * (kSpWaves / split) + item;
    const bool live = at < p.o_items;
    at = live ? at : 0;
    const int per = p.batch * p.n_kv * p.o_tiles, chunk = ALL ? 0 : at / per;
    at -= chunk * per;
    const int tile = at % p.o_tiles, j = at / p.o_tiles % p.n_kv, b = at / p.o_tiles / p.n_kv;
    const int64_t len = live ? sp_length(p.o_len, p.o_dtype, b, p.o_add, p.o_cap) : 0, k0 = ALL ? 0 : (int64_t)chunk * p.o_keys;
    const int keys = len <= k0 ? 0 : ALL || len - k0 < p.o_keys ? (int)(len - k0) : p.o_keys;
    const int64_t first = (((int64_t)b * p.n_kv + j) * p.o_cap + k0) * HD;
    const T *kb = static_cast<const T*>(p.ko) + first, *vb = static_cast<const T*>(p.vo) + first;
    // the prefix's keys and tiles in front of them
    int p_keys = 0, p_tiles = 0;
    const T *kp = nullptr, *vp = nullptr;
    if constexpr (ALL) {
        const int64_t n = len < 0 ? 0 : sp_length(p.p_len, p.p_dtype, 0, p.p_add, p.p_cap);
        p_keys = n > 0 ? (int)n : 0;
        p_tiles = (p_keys + TK - 1) / TK;
        kp = static_cast<const T*>(p.kp) + (int64_t)j * p.p_cap * HD;
        vp = static_cast<const T*>(p.vp) + (int64_t)j * p.p_cap * HD;
    }
    const int row0 = 16 * tile, my_row = b * p.n_head + j * p.group + row0 + qi, tiles = p_tiles + (keys + TK - 1) / TK;
    uint8_t *const kt = m.lds + w * 2 * kTile, *const vt = kt + kTile;
    const uint32_t kt_a = lds_address(kt), vt_a = lds_address(vt);
    // keys left from tile t on, in its set
    const auto left = [&](int t) { return t < p_tiles ? p_keys - t * TK : keys - (t - p_tiles) * TK; };
    const auto stage_k = [&](int t) {
        const T* from = t < p_tiles ? kp + (int64_t)t * TK * HD : kb + (int64_t)(t - p_tiles) * TK * HD;
        sp_stage<T, HD, false, kPieces>(from, left(t) - 1, kt_a, lane, 0);
    };
    const auto stage_v = [&](int t) {
        const T* from = t < p_tiles ? vp + (int64_t)t * TK * HD : vb + (int64_t)(t - p_tiles) * TK * HD;
        sp_stage<T, HD, true, kPieces>(from, left(t) - 1, vt_a, lane, 0);
    };
    if (sub < tiles) {
        stage_k(sub);
        stage_v(sub);
    }
    Rows q;
    q.load(tiles > 0 && row0 + qi < p.group ? p.q + (int64_t)my_row * HD : nullptr, p.scale, h);
    const float NEG_INF = -__builtin_huge_valf();
    float r = NEG_INF, l = 0.f;
    f4v o[HD / 16] = {};
    for (int t = sub; t < tiles; t += split) {
        const bool more = t + split < tiles;
        // K is there, V may be in flight (the first time the queries' loads are behind both)
        if (t == sub)
            sp_wait_loads<0>();
        else
            sp_wait_loads<kPieces>();
        float s[N];
        q.scores(kt, s, qi, h);
        sp_wait_lds();
        if (more) stage_k(t + split);
        const int n = left(t);
        if (n < TK) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (16 * (i >> 2) + 4 * h + (i & 3) >= n) s[i] = NEG_INF;
        }
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < N; ++i) mx = fmaxf(mx, s[i]);
        mx = swap32_max(swap16_max(mx)) * q.unscale;
        const bool moves = mx > r + kRoom;
        if (__any(moves)) {
            const float rn = moves ? mx - kUp : r, alpha = moves ? __builtin_amdgcn_exp2f(r - rn) : 1.f;
            r = rn;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < HD / 16; ++d) o[d] *= alpha;
        }
        const float rs = r == NEG_INF ? 0.f : r;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], q.unscale, -rs));
            l += s[i];
        }
        if (more)
            sp_wait_loads<kPieces>();  // V is there, the next K may be in flight
        else
            sp_wait_loads<0>();
        if (n < TK) {
            sp_clear_rows<HD * (int)sizeof(T)>(vt, n, TK, lane, 64);
            sp_wait_lds();
        }
        Rows::accumulate(vt, s, o, qi, h);
        sp_wait_lds();
        if (more) stage_v(t + split);
    }
    const float down = exp2_int(-(int)kUp);
    float4 v[HD / 16];
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) v[d] = make_float4(o[d][0] * down, o[d][1] * down, o[d][2] * down, o[d][3] * down);
    l = swap32_sum(swap16_sum(l)) * down;
    sp_finish<HD, 16, ALL>(p, m, v, r + kUp, l, my_row, tiles > 0, p.group - row0, p.p_chunks + chunk, item, sub, split, 1);
}

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
    return q.template scores<0>(kt, li, g, [](int) {});
}
template <int HD>
PE_DEV void sp_accumulate(const RowsF32<HD>&, const uint8_t* vt, const f16v& s, f16v* o, int li, int g) {
    RowsF32<HD>::accumulate(vt, s, o, li, g);
}
template <int HD>
PE_DEV void sp_accumulate(const RowsF16<HD>&, const uint8_t* vt, const f16v& s, f16v* o, int li, int g) {
    const uint32_t va = RowsF16<HD>::values_at(vt, li, g);
    h8v v[4];
    RowsF16<HD>::template load_values<0>(va, v);
    RowsF16<HD>::template accumulate<0>(va, v, s, o, [](int) {});
}

template <typename T, int HD>
__global__ __launch_bounds__(64 * kSpWaves, 2) void k_shared_prefix(SpArgs p) {
    constexpr bool kHalf = sizeof(T) == 2;
    constexpr int kTile = 32 * HD * (int)sizeof(T), kPieces = kTile / 1024;
    // solo: a K and a V tile per wave, or one buffer for both in turn where two are over 16 KB
    constexpr bool kOne = kTile > 8192;
    constexpr int kWaveLds = kOne ? kTile : 2 * kTile;
    // shared: two buffers of a block's planes
    constexpr int kPlane = kSpBlock * HD * 2, kPlanes = (kHalf ? 2 : 4) * kPlane, kLow = kHalf ? 0 : kPlane;
    constexpr int kMerge = kSpWaves * 32 * (HD + 4) * 4;
    // the queries' image, read before the loops: shared, fp32: the second buffer, else behind the tiles
    constexpr int kQueries = kHalf ? 2 * kPlanes : kPlanes, kSolo = kSpWaves * kWaveLds;
    constexpr int kShared = kHalf ? kQueries + 128 * HD * 4 : 2 * kPlanes, kAlone = kSolo + 32 * HD * 4;
    constexpr int kMost = kAlone > kShared ? kAlone : kShared;
    static_assert(kQueries + 128 * HD * 4 <= kMost, "the queries' image");
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kMost > kMerge ? kMost : kMerge];
    __shared__ float ref[kSpWaves][32], sums[kSpWaves][32];
    __shared__ int exps[2][16], row_of[kSpWaves][32], uneven;
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 5, li = lane & 31;

    const SpShared m{lds, ref, sums, row_of};
    if ((int)blockIdx.x >= p.p_blocks) return sp_own<T, HD, false>(p, m, blockIdx.x - p.p_blocks);

    // The workgroup's rows of a kv head, by tiles of 32, and its keys [k0, k1).
    const bool shared = p.shared;
    // The row tiles of a chunk read the same keys: workgroups a multiple of 8 apart, which share an L2.
    const int kc = p.n_kv * p.p_chunks, even = kc & ~7, b = blockIdx.x;
    const int unit = b < even * p.p_tiles ? 8 : kc - even, first = b < even * p.p_tiles ? 0 : even;
    const int turn = (b - first * p.p_tiles) / unit, tile = turn % p.p_tiles;
    const int at = first + turn / p.p_tiles * unit + (b - first * p.p_tiles) % unit, j = at % p.n_kv, chunk = at / p.n_kv;
    const int64_t len = sp_length(p.p_len, p.p_dtype, 0, p.p_add, p.p_cap);
    const int64_t k0 = (int64_t)chunk * p.p_keys, k1 = k0 + p.p_keys < len ? k0 + p.p_keys : len;
    if (k1 <= k0) return;  // the whole workgroup: a chunk past the length
    const T* kb = static_cast<const T*>(p.kp) + (int64_t)j * p.p_cap * HD;
    const T* vb = static_cast<const T*>(p.vp) + (int64_t)j * p.p_cap * HD;
    const int rows = p.batch * p.group, keys = (int)(k1 - k0);
    const int64_t last = k1 - 1;
    // the record of a wave's rows from row0 on, by split waves step apart of which it is the sub-th
    const auto finish = [&](SpState<HD>& st, int base, int row0, int item, int sub, int split, int step) {
        // row r of the kv head is (sequence r / group, head r % group of the kv head's)
        const int seq = (row0 + li) / p.group, my_row = seq * p.n_head + j * p.group + (row0 + li - seq * p.group);
        const float down = exp2_int(-(int)kUp);  // probabilities and values without their factors
        st.scale(ldexpf(down, base));
        float4 v[HD / 8];
#pragma unroll
        for (int i = 0; i < HD / 8; ++i)
            v[i] = make_float4(st.o[i >> 2][4 * (i & 3)], st.o[i >> 2][4 * (i & 3) + 1], st.o[i >> 2][4 * (i & 3) + 2], st.o[i >> 2][4 * (i & 3) + 3]);
        sp_finish<HD, 32, false>(p, m, v, st.r + kUp, swap32_sum(st.l) * down, my_row, row0 < rows, rows - row0, chunk, item, sub, split, step);
    };

    // the wave's share of rows [row0, row0 + 32) and all of the chunk's keys, every eighth tile of them
    const auto solo = [&](int row0, int lane) {
        const int li = lane & 31, g = lane >> 5;
        SpState<HD> st;
        st.clear();
        typename SpPick<T, HD>::type q;
        const uint8_t* const image = lds + kSolo;
        sp_stage_queries<HD, 4>(p, j, row0 + 4 * w, rows, lds_address(image) + 4 * w * (HD * 4), lane);
        const int tiles = (keys + 31) / 32;
        uint8_t* const kt = lds + w * kWaveLds;
        uint8_t* const vt = kOne ? kt : kt + kTile;
        const uint32_t kt_a = lds_address(kt), vt_a = lds_address(vt);
        const auto stage_k = [&](int t) {
            const int64_t row = k0 + 32 * t;
            sp_stage<T, HD, false, kPieces>(kb + row * HD, last - row, kt_a, lane, 0);
        };
        const auto stage_v = [&](int t) {
            const int64_t row = k0 + 32 * t;
            sp_stage<T, HD, true, kPieces>(vb + row * HD, last - row, vt_a, lane, 0);
        };
        if (w < tiles) {
            stage_k(w);
            if (!kOne) stage_v(w);
        }
        sp_wait_loads<0>();
        __syncthreads();
        q.load(image, li, p.scale, g);
        const float c[4] = {q.unscale, q.unscale, q.unscale, q.unscale};
        for (int t = w; t < tiles; t += kSpWaves) {
            const bool more = t + kSpWaves < tiles;
            sp_wait_loads<kOne ? 0 : kPieces>();  // K is there, V may be in flight
            f16v s = sp_scores(q, kt, li, g);
            sp_wait_lds();
            if (kOne)
                stage_v(t);
            else if (more)
                stage_k(t + kSpWaves);
            const int n = keys - 32 * t < 32 ? keys - 32 * t : 32;
            st.template softmax<false>(s, c, nullptr, n, g);
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
                    stage_k(t + kSpWaves);
                else
                    stage_v(t + kSpWaves);
            }
        }
        finish(st, 0, row0, 0, w, kSpWaves, 1);
    };

    if (shared) {
        const int item = w & 3, sub = w >> 2, row0 = 128 * tile + 32 * item;
        SpState<HD> st;
        st.clear();
        int base = kHalf ? 0 : kZeros, most = kZeros, least = 127;  // exponents of the values: what o holds, and their range
        RowsF16<HD> q;
        const uint8_t* const image = lds + kQueries;
        sp_stage_queries<HD, 16>(p, j, 128 * tile + 16 * w, rows, lds_address(image) + 16 * w * (HD * 4), lane);
        const int blocks = (keys + kSpBlock - 1) / kSpBlock;
        // the products with block t; kbeside, vbeside: work beside them
        const auto take = [&](int t, const auto& kbeside, const auto& vbeside) {
            const uint8_t* kt = lds + (t & 1) * kPlanes + 32 * sub * (HD * 2);
            // no branch round waves without rows or keys: o would be copied on every way
            const int n = keys - kSpBlock * t - 32 * sub;
            f16v s = q.template scores<kLow>(kt, li, g, kbeside);
            float c[4] = {q.unscale, q.unscale, q.unscale, q.unscale};
            int ev[4];
            if constexpr (!kHalf) {
                const int* e = exps[t & 1] + 4 * sub;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    c[i] = sp_positive(ldexpf(fabsf(p.scale), q.down + e[i]));  // together: one of them may leave fp32's range
                    ev[i] = __builtin_amdgcn_readfirstlane(e[8 + i]);
                    most = ev[i] > most ? ev[i] : most;
                    least = ev[i] > kZeros && ev[i] < least ? ev[i] : least;
                }
                base = base == kZeros ? most : base;
                // groups of zeros, which no weight makes larger, count as far under the others
#pragma unroll
                for (int i = 0; i < 4; ++i) ev[i] = (ev[i] == kZeros ? most - kFar : ev[i]) - base;
            }
            const uint32_t va = RowsF16<HD>::values_at(kt + (kHalf ? 1 : 2) * kPlane, li, g);
            h8v v[4];
            RowsF16<HD>::template load_values<kLow>(va, v);
            __builtin_amdgcn_sched_barrier(0);
            st.template softmax<!kHalf>(s, c, ev, n, g);
            RowsF16<HD>::template accumulate<kLow>(va, v, s, st.o, vbeside);
        };
        if constexpr (kHalf) {
            constexpr int N = kPlane / 1024 / kSpWaves;
            const auto stage = [&](int t) {
                const uint32_t at = lds_address(lds) + (t & 1) * kPlanes;
                const int64_t row = k0 + kSpBlock * t;
                sp_stage<T, HD, false, N>(kb + row * HD, last - row, at, lane, w * N);
                sp_stage<T, HD, true, N>(vb + row * HD, last - row, at + kPlane, lane, w * N);
            };
            stage(0);
            sp_wait_loads<0>();
            __syncthreads();
            q.load(image, 32 * item + li, p.scale, g);
            for (int t = 0; t < blocks; ++t) {
                sp_wait_loads<0>();
                __syncthreads();  // the block is there, and nobody reads the other buffer any more
                if (t + 1 < blocks) stage(t + 1);
                const int n = keys - kSpBlock * t;
                if (n < kSpBlock) {
                    sp_clear_rows<HD * 2>(lds + (t & 1) * kPlanes + kPlane, n, kSpBlock, threadIdx.x, 64 * kSpWaves);
                    __syncthreads();
                }
                take(t, [](int) {}, [](int) {});
            }
        } else {
            SpSplit<HD, false> xk;
            SpSplit<HD, true> xv;
            const uint32_t k_place = xk.place(w, lane), v_place = xv.place(w, lane) + 2 * kPlane;
            const auto planes = [&](int t) { return lds_address(lds) + (t & 1) * kPlanes; };
            const auto left = [&](int t) { return keys - kSpBlock * t < kSpBlock ? keys - kSpBlock * t : kSpBlock; };
            const auto k_step = [&](int t, int i) { xk.step(i, planes(t), k_place, &exps[t & 1][w]); };
            const auto v_step = [&](int t, int i) { xv.step(i, planes(t), v_place, &exps[t & 1][8 + w]); };
            const auto k_load = [&](int t) {
                if (t < blocks) xk.load(kb + (k0 + kSpBlock * t) * HD, left(t), w, lane);
            };
            const auto v_load = [&](int t) {
                if (t < blocks) xv.load(vb + (k0 + kSpBlock * t) * HD, left(t), w, lane);
            };
            k_load(0);
            v_load(0);
            if (threadIdx.x == 0) uneven = 0;
            sp_wait_loads<0>();
            __syncthreads();
            q.load(image, 32 * item + li, p.scale, g);
            if (q.uneven) uneven = 1;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                k_step(0, i);
                v_step(0, i);
            }
            k_load(1);
            v_load(1);
            for (int t = 0; t < blocks; ++t) {
                __syncthreads();  // block t is there, and nobody reads the other buffer any more
                // beside its products the next block is split (behind the last one, that one again)
                take(
                    t,
                    [&](int i) {
                        k_step(t + 1, i);
                        if (i == HD / 8 - 1) k_load(t + 2);
                    },
                    [&](int i) {
                        v_step(t + 1, i);
                        if (i == HD / 8 - 1) v_load(t + 2);
                    });
            }
            if (lane == 0 && ((xk.uneven | xv.uneven) || (least <= most && most - least > kFar))) uneven = 1;
        }
        // keys, values or queries too far apart for their two parts: the chunk again on the fp32 instructions, by
        // 32 rows
        bool again = false;
        if constexpr (!kHalf) {
            __syncthreads();
            again = __builtin_amdgcn_readfirstlane(uneven);
        }
        if (__builtin_expect(again, 0)) {
            for (int row1 = 128 * tile;;) {
                int l = lane;
                asm volatile("" : "+v"(l));  // nothing is kept from one tile to the next, for want of registers
                solo(row1, l);
                row1 += 32;
                // ends here, so that the other way's rows need not outlive this
                if (row1 >= 128 * tile + 128 || row1 >= rows) __builtin_amdgcn_endpgm();
                __syncthreads();
            }
        }
        return finish(st, base, row0, item, sub, 2, 4);
    }
    solo(32 * tile, lane);
}

// Few keys: all of them by one workgroup per sequence, kv head and 16 queries of its group, in one launch.
template <typename T, int HD>
__global__ __launch_bounds__(64 * kSpWaves, 2) void k_shared_prefix_few(SpArgs p) {
    constexpr int kTiles = kSpWaves * 2 * OwnRows<T, HD>::TK * HD * (int)sizeof(T), kMerge = kSpWaves * 16 * (HD + 4) * 4;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kTiles > kMerge ? kTiles : kMerge];
    __shared__ float ref[kSpWaves][32], sums[kSpWaves][32];
    __shared__ int row_of[kSpWaves][32];
    sp_own<T, HD, true>(p, SpShared{lds, ref, sums, row_of}, blockIdx.x);
}

// W waves per (sequence, head): the records of the prefix's chunks and then of the own keys'. HD / 4
// lanes hold a row, the lane groups take every so-many-th record, four loads in flight each, with a
// running maximum of their own; bound by the latency of a launch and the records (14 heads x 16 sequences x
// 25 records of 64: 3.8 us; 28 x 64 x 15 of 128: 5.9, 14 x 3 x 65 of 64: 4.6).
template <int HD, int W>
__global__ __launch_bounds__(256) void k_shared_prefix_merge(SpArgs p) {
    constexpr int L = HD / 4, N = 64 / L * W, U = 4;
    __shared__ float4 rows[4][L];
    __shared__ float refs[4], sums[4];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int row = __builtin_amdgcn_readfirstlane(W == 1 ? blockIdx.x * 4 + w : blockIdx.x);
    if (row >= p.batch * p.n_head) return;  // W == 1 only, uniform per wave
    const int64_t at = (int64_t)row * (p.p_chunks + p.o_chunks);
    const int total = p.p_chunks + p.o_chunks;
    int i0 = (W == 1 ? 0 : w * (64 / L)) + lane / L;
    float2 ml[U];
    float4 o[U];
    // the first records come while the lengths do, there or not
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t rec = at + (i0 + N * u < total ? i0 + N * u : 0);
        ml[u] = *reinterpret_cast<const float2*>(p.ml + rec * 2);
        o[u] = *reinterpret_cast<const float4*>(p.rec + rec * HD + 4 * (lane % L));
    }
    // lengths are at most 2^30
    const int64_t pl = sp_length(p.p_len, p.p_dtype, 0, p.p_add, p.p_cap);
    const int64_t ol = sp_length(p.o_len, p.o_dtype, row / p.n_head, p.o_add, p.o_cap);
    // a sequence that takes no part has no records: zeros
    const int np = pl > 0 && ol >= 0 ? (int)((uint32_t)(pl + p.p_keys - 1) / (uint32_t)p.p_keys) : 0;
    const int no = ol > 0 ? (int)((uint32_t)(ol + p.o_keys - 1) / (uint32_t)p.o_keys) : 0;
    const int n = np + no;
    const auto there = [&](int i) { return i < np || (i >= p.p_chunks && i - p.p_chunks < no); };
    const float NEG_INF = -__builtin_huge_valf();
    float top = NEG_INF, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    // takes (x, y): a row over the reference r with the sum l
    const auto take = [&](float r, float l, const float4& o) {
        const float most = fmaxf(top, r), rs = most == NEG_INF ? 0.f : most;
        const float a = __builtin_amdgcn_exp2f(top - rs), f = __builtin_amdgcn_exp2f(r - rs);
        top = most;
        sum = fmaf(f, l, a * sum);
        v = make_float4(fmaf(f, o.x, a * v.x), fmaf(f, o.y, a * v.y), fmaf(f, o.z, a * v.z), fmaf(f, o.w, a * v.w));
    };
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (there(i0 + N * u)) take(ml[u].x, ml[u].y, o[u]);
    for (i0 += N * U; i0 < total; i0 += N * U) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (there(i0 + N * u)) {
                const int64_t rec = at + i0 + N * u;
                ml[u] = *reinterpret_cast<const float2*>(p.ml + rec * 2);
                o[u] = *reinterpret_cast<const float4*>(p.rec + rec * HD + 4 * (lane % L));
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (there(i0 + N * u)) take(ml[u].x, ml[u].y, o[u]);
    }
#pragma unroll
    for (int o = 32; o >= L; o >>= 1) {
        const float r = __shfl_xor(top, o, kWave), l = __shfl_xor(sum, o, kWave);
        const float4 x = make_float4(__shfl_xor(v.x, o, kWave), __shfl_xor(v.y, o, kWave), __shfl_xor(v.z, o, kWave),
                                     __shfl_xor(v.w, o, kWave));
        take(r, l, x);
    }
    if constexpr (W > 1) {
        if (lane < L) rows[w][lane] = v;
        if (lane == 0) refs[w] = top, sums[w] = sum;
        __syncthreads();
        if (w) return;
#pragma unroll
        for (int s = 1; s < W; ++s) take(refs[s], sums[s], rows[s][lane % L]);
    }
    if (lane >= L) return;
    const float4 y = n ? make_float4(v.x / sum, v.y / sum, v.z / sum, v.w / sum) : v;
    *reinterpret_cast<float4*>(p.out + (int64_t)row * HD + 4 * lane) = sp_rounded(y, p.round_fp16);
}

struct SpPlan {
    int few, shared, p_chunks, p_keys, p_tiles, o_chunks, o_keys, o_tiles, o_split;
};

// How the work is cut. Rows of a kv head over 64 go the shared way: up to there an fp32 prefix keeps fp32 products. Solo | shared
// (us, 2000 and 30000 keys at head size 64, then at 128):
//   fp16, 64 rows  9.7 | 10.3, 13 | 17, 12.6 | 14.2, 22 | 33    fp32, 33 rows  13.0 | 11.6, 21 | 21, 19 | 17, 56 | 48
//         96 rows  9.7 | 10.3, 15 | 17, 12.9 | 15.2, 27 | 29          64 rows  13.4 | 11.8, 21 | 22, 19 | 17, 60 | 49
//        128 rows  9.7 | 10.4, 16 | 18, 13.3 | 15.8, 31 | 30          96 rows  13.1 | 12.0, 32 | 22, 20 | 18, 77 | 51
// so by time alone the line would lie near 128 rows for fp16 and 33 for fp32. A CU holds one workgroup (by its LDS; 16-bit
// caches at head size 64 by its registers); those of the
// prefix come first, the own keys' fill the other CUs and follow where one ends. Of a few numbers of waves and
// chunks for an item's own keys, and of two or three lengths of the prefix's chunks for each, the plan is the one
// whose longest workgroup, or whose work spread over 256 CUs, and whose records take least, by the times
// measured at head size 128 (us): 9.5 for a prefix workgroup's start and end, 1.85 (16-bit caches) and 3.1
// (fp32) for a shared block of 64 keys, 1.5 and 7 for eight solo tiles; 9 and 12 for an own workgroup's, 1.5 and
// 5.3 for a wave's 32 keys (at 64 the steps count half). The own keys' work counts three quarters (their lengths are on the device). Best
// of 56 cuts | this one (us, caches two thirds full): 33 x 8001 fp32 with 515 own keys (28/4 heads) 36 | 37, 64 x
// 32768 with 1000 142 | 147 and fp16 80 | 82, 16 x 4096 fp16 with 2000 20 | 20, 24 x 2000 fp32 with 1000 25 | 25,
// 8 x 30000 fp32 with 4000 56 | 63; with the own waves chosen first and the rest filled with chunks 39, 165, 82, 23, 25, 63.
// An item's own keys are cut into six chunks at most, so a few sequences with tens of thousands of them leave most
// CUs idle: one of 30000 fp32 own keys at head size 64 takes 65 us, 6 at the copy rate.
static SpPlan sp_plan(int64_t batch, int n_head, int n_kv, int hd, bool half, int64_t p_keys, int64_t o_cap) {
    SpPlan s;
    const int64_t group = n_head / n_kv, rows = batch * group;
    s.shared = rows > 64;
    s.p_tiles = (int)(s.shared ? (rows + 127) / 128 : (rows + 31) / 32);
    s.o_tiles = (int)((group + 15) / 16);
    const auto cut = [](int64_t keys, int want, int step, int& chunks, int& per) {
        int64_t k = (keys + want - 1) / want;
        k = (k + step - 1) / step * step;
        k = k < step ? step : k;
        per = (int)k;
        chunks = (int)((keys + k - 1) / k);
    };
    const int64_t pairs = batch * n_kv * s.o_tiles, tiles = (o_cap + 31) / 32;
    // Few keys: the prefix is read again for every sequence (from L2), but there is one launch and
    // nothing to merge. Measured, few | two launches (us, 4 sequences, own capacity 64, prefix of 256, 512,
    // 1024; heads 14/2 of 64 and 28/4 of 128): fp32 8.1 | 13.4, 10.5 | 13.3, 15.9 | 14.0 and 11 | 20,
    // 16 | 21, 27 | 21; fp16 5.5 | 9.8, 6.4 | 9.9, 8.2 | 10.4 and 7.5 | 13, 8.9 | 13.5, 12 | 14; the same
    // for up to 256 workgroups.
    s.few = (pairs + 255) / 256 * (p_keys + o_cap) <= (half ? 1280 : 640);
    if (s.few) {
        s.p_chunks = s.o_chunks = 0;
        s.p_keys = s.o_keys = 0;
        s.o_split = kSpWaves;
        return s;
    }
    const double each = hd / 128.0, t_step = (s.shared ? (half ? 1.85 : 3.1) : (half ? 1.5 : 7.0)) * each;
    const double a_own = half ? 9 : 12, t_own = (half ? 1.5 : 5.3) * each, t_record = (double)batch * n_head * hd * 8 / 5e6;
    const int per_chunk = n_kv * s.p_tiles, step = s.shared ? kSpBlock : 32 * kSpWaves, steps = (int)((p_keys + step - 1) / step);
    double best = 1e30;
    for (int o_split = 1, chunks = 1; o_split <= kSpWaves;) {
        SpPlan c = s;
        c.o_split = o_split;
        cut(o_cap, chunks, 32 * o_split, c.o_chunks, c.o_keys);
        const int per = kSpWaves / o_split, o_tiles = c.o_keys / (32 * o_split);
        const int o_blocks = (int)((pairs * c.o_chunks + per - 1) / per);
        const double own = o_blocks ? a_own + t_own * o_tiles : 0, own_work = o_blocks * (a_own + 0.75 * t_own * o_tiles);
        // steps of a chunk: those of one round, and those where the chunks end with all the work spread evenly
        const auto consider = [&](double want) {
            SpPlan n = c;
            const int k = want < 1 ? 1 : want > steps ? steps : (int)want;
            n.p_chunks = (steps + k - 1) / k;
            n.p_keys = (steps + n.p_chunks - 1) / n.p_chunks * step;
            const int p_blocks = per_chunk * n.p_chunks;
            const double prefix = 9.5 + t_step * (n.p_keys / step);
            double time = (p_blocks * prefix + own_work) / 256;
            if (p_blocks > 256) time += prefix / 2;
            else if (p_blocks + o_blocks > 256) time += own / 6;
            time = (time > prefix ? time : prefix);
            time = (time > own ? time : own) + t_record * (n.p_chunks + n.o_chunks);
            if (time < best) best = time, s = n;
        };
        if (!steps) {
            const double time = (own > own_work / 256 ? own : own_work / 256) + t_record * c.o_chunks;
            if (time < best) best = time, s = c;
        } else {
            const int room = 256 - o_blocks;
            if (room >= per_chunk) consider((steps + room / per_chunk - 1) / (room / per_chunk));
            const double all = (double)per_chunk * steps * t_step, a = 9.5 * per_chunk / 256, k = (all + own_work) / 256 - 9.5;
            const double even = steps * 2 * a / (sqrt(k * k + 4 * a * steps * t_step) - k);
            consider(even);
            consider(even + 1);
        }
        if (!o_cap || tiles <= o_split) break;
        if (o_split < kSpWaves)
            o_split *= 2;
        else if (++chunks > 6 || c.o_keys <= 32 * kSpWaves)
            break;
    }
    if (!steps) s.p_chunks = 0, s.p_keys = step;
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
static void launch_shared_prefix(const SpArgs& p, bool few, int64_t blocks, hipStream_t s) {
    if (few) {
        hipLaunchKernelGGL((k_shared_prefix_few<T, HD>), dim3((unsigned)p.o_items), dim3(64 * kSpWaves), 0, s, p);
        return;
    }
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

extern "C" int64_t pe_shared_prefix_attn_workspace_bytes(int cache_type, int64_t batch, int n_head, int n_kv,
                                                         int head_dim, int64_t prefix_keys, int64_t own_capacity) {
    if (cache_type != PE_TYPE_F32 && cache_type != PE_TYPE_F16) return -PE_ERR_TYPE;
    if (!sp_shape_ok(batch, n_head, n_kv, head_dim, prefix_keys, own_capacity)) return -PE_ERR_SHAPE;
    const bool half = cache_type == PE_TYPE_F16;
    return sp_bytes(sp_plan(batch, n_head, n_kv, head_dim, half, prefix_keys, own_capacity), batch, n_head, head_dim);
}

extern "C" int pe_shared_prefix_attn(const pe_shared_prefix_args* a, pe_stream_t stream) {
    if (!a) return PE_ERR_NULL;
    if (a->cache_type != PE_TYPE_F32 && a->cache_type != PE_TYPE_F16) return PE_ERR_TYPE;
    if (a->prefix_len_dtype < 0 || a->prefix_len_dtype > 2 || a->own_len_dtype < 0 || a->own_len_dtype > 2)
        return PE_ERR_TYPE;
    if (a->batch == 0) return PE_OK;
    if (!sp_shape_ok(a->batch, a->n_head, a->n_kv, a->head_dim, a->prefix_capacity, a->own_capacity) ||
        !std::isfinite(a->scale))
        return PE_ERR_SHAPE;
    // the prefix's keys that the launch is cut for: its length where the host knows it
    int64_t keys = a->prefix_capacity;
    if (!a->prefix_len_dtype) {
        keys = a->prefix_len_add < keys ? a->prefix_len_add : keys;
        if (keys < 0) keys = 0;
    }
    const SpPlan s = sp_plan(a->batch, a->n_head, a->n_kv, a->head_dim, a->cache_type == PE_TYPE_F16, keys,
                             a->own_capacity);
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
    const int64_t items = a->batch * a->n_kv * s.o_tiles * (s.few ? 1 : s.o_chunks), per = kSpWaves / s.o_split;
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
        a->head_dim == 64 ? launch_shared_prefix<_Float16, 64>(p, s.few, blocks, st)
                          : launch_shared_prefix<_Float16, 128>(p, s.few, blocks, st);
    else
        a->head_dim == 64 ? launch_shared_prefix<float, 64>(p, s.few, blocks, st)
                          : launch_shared_prefix<float, 128>(p, s.few, blocks, st);
    return launch_status();
}
