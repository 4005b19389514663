// Attention of new rows of several sequences over their pages of the 4-bit cache (kv4.h):
//   out[t][h] = softmax_j(scale q[t][h] . k[j]) v[j],  j < keys that row t sees
// where row i of sequence b sees its first lengths[b] + first + i keys (causal among the new rows).
//
// Codes times a power of two are exact in bf16 (two bits of mantissa), one conversion instruction for two of
// them, so both products run on the bf16 matrix cores with the cache's side exact; the other side is a sum of bf16
// parts that are each the rest of the one before: two for an fp16 query (its 11 bits fit 2 x 8 exactly),
// three for an fp32 one (24 bits); two parts of the probabilities for fp16 outputs (2^-17 of each), three for fp32.
//
// A wave computes S^T = K Q^T: a lane then holds, for the query row lane % 16, the scores of keys 4 (lane / 16) ..
// + 3 of every 16 keys, which is how the second product O^T = V^T P^T takes its keys when its 32 are numbered
// (8 g + i: key 4 g + i of the first 16 for i < 4, of the second for i >= 4). So probabilities go from one product to
// the other in their lane, and the running maximum and sum belong to the lane's own row.
#include <cmath>

#include "kv4.h"

namespace pe {

constexpr int kKv4Step = 64;    // keys a wave takes at a time
constexpr int kKv4Waves = 4;    // of a workgroup
constexpr float kKv4Log2e = 1.4426950408889634f;

typedef __bf16 bf8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf2v __attribute__((ext_vector_type(2)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));

struct Kv4AttnArgs {
    const void* q;
    int64_t q_token, q_head;
    void* out;
    int64_t out_token, out_head;
    const uint8_t* pages;
    int64_t page_stride;
    int n_pages, tiles;
    const int* table;
    int64_t table_row;
    int table_cols;
    const void* lengths;
    int len_wide;
    int64_t first;
    const void* starts;
    int starts_wide;
    int64_t tokens;
    int batch, n_head, n_kv, group;
    float scale;  // times log2 e
    int items, blocks;  // workgroups a kv head, row blocks at most
    int min_chunk;
    int4* plan;         // of every sequence: first item, chunks, row blocks
    float* record;      // [kv head][item][row][HD]
    float* stat;        // [kv head][item][row] (maximum, sum)
};

// Work of a sequence.
struct Kv4Seq {
    int64_t lo;      // first row
    int rows;        // rows times the heads of a group
    int64_t keys;    // keys that its first row sees (0: it takes no part)
};

PE_DEV Kv4Seq kv4_seq(const Kv4AttnArgs& p, int b) {
    int64_t lo, hi;
    rows_of(p.starts, p.starts_wide, b, p.tokens, lo, hi);
    const int64_t len = int_at(p.lengths, p.len_wide, b);
    return {lo, (int)(hi - lo) * p.group, len < 0 ? -(1LL << 42) : (len > (1LL << 41) ? 1LL << 41 : len) + p.first};
}

// Keys that row i (of a token) sees.
PE_DEV int kv4_keys(const Kv4AttnArgs& p, int64_t first_keys, int i) {
    const int64_t cap = (int64_t)p.table_cols * p.tiles * kKv4Tile, k = first_keys + i;
    return (int)(k < 0 ? 0 : k > cap ? cap : k);
}

PE_DEV int64_t wave_sum64(int64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((long long)v, o, kWave);
    return v;
}

struct Kv4Item {
    int b, block, chunk, chunks, blocks, base, span;  // span: keys of a chunk
};

// Which work the item is: a (sequence, row block, chunk of keys). All sequences' keys times row blocks are cut by
// one length, the least (in steps) that makes no more items than the launch has. Every wave finds it for itself.
template <int RB>
PE_DEV bool kv4_find(const Kv4AttnArgs& p, int item, Kv4Item& w) {
    const int lane = threadIdx.x & 63;
    int span = 1 << 30;
    if (p.items > p.blocks) {
        int64_t cost = 0;
        for (int b = lane; b < p.batch; b += 64) {
            const Kv4Seq s = kv4_seq(p, b);
            const int nb = (s.rows + RB - 1) / RB;
            if (nb) cost += (int64_t)nb * kv4_keys(p, s.keys, s.rows / p.group - 1);
        }
        cost = wave_sum64(cost);
        const int64_t room = p.items - p.blocks, even = ((cost + room - 1) / room + kKv4Step - 1) / kKv4Step * kKv4Step;
        span = (int)(even < p.min_chunk ? p.min_chunk : even > (1 << 30) ? 1 << 30 : even);
    }
    int base = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
        int nb = 0, chunks = 1;
        if (b0 + lane < p.batch) {
            const Kv4Seq s = kv4_seq(p, b0 + lane);
            nb = (s.rows + RB - 1) / RB;
            if (nb) {
                const int keys = kv4_keys(p, s.keys, s.rows / p.group - 1);
                chunks = keys > span ? (keys + span - 1) / span : 1;
            }
        }
        int upto = nb * chunks;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(upto, o, kWave);
            if (lane >= o) upto += v;
        }
        const uint64_t beyond = __ballot(base + upto > item);
        if (beyond) {
            const int at = __builtin_ctzll(beyond);
            w.b = b0 + at;
            w.blocks = __builtin_amdgcn_readlane(nb, at);
            w.chunks = __builtin_amdgcn_readlane(chunks, at);
            w.base = base + __builtin_amdgcn_readlane(upto, at) - w.blocks * w.chunks;
            w.span = span;
            // blocks of the same keys one after the other
            w.chunk = (item - w.base) / w.blocks;
            w.block = item - w.base - w.chunk * w.blocks;
            return true;
        }
        base += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// Two values as N words of bf16 pairs that sum up to them.
template <int N>
PE_DEV void split_pair(float a, float b, uint32_t* w) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bf2v z = {(__bf16)a, (__bf16)b};
        w[i] = __builtin_bit_cast(uint32_t, z);
        a -= __uint_as_float(w[i] << 16);
        b -= __uint_as_float(w[i] & 0xFFFF0000u);
    }
}

// The two codes of byte SEL of w as a pair of bf16 (low half: the low four bits), times scale.
PE_DEV uint32_t two_codes(uint32_t w, float scale, int sel) {
    bf2v z;
    if (sel == 0)
        z = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0);
    else if (sel == 1)
        z = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1);
    else if (sel == 2)
        z = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2);
    else
        z = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
    return __builtin_bit_cast(uint32_t, z);
}

// A lane's part of 64 keys: codes, scale bytes, and the number of each 16 keys' first one (scalar).
template <int HD>
struct Kv4Raw {
    static constexpr int N = HD / 32;  // words of codes per 16 keys
    uint32_t k[4][N], v[4][N], ks[4], vs[4];
    int key[4];
};

// Where a wave's next 64 keys lie.
struct Kv4Walk {
    int col, tile;   // page of the table, tile in it, of the next step's first 16 keys
    int key, end;    // the first key, the item's last
    int step_cols, step_tiles;
};

constexpr int kNoKeys = 0x7FFFFF00;  // number of the first key of 16 that are not there

template <int HD>
PE_DEV void kv4_load(const Kv4AttnArgs& p, const int* table, const uint8_t* head, Kv4Walk& w, int lane, Kv4Raw<HD>& r) {
    constexpr int N = HD / 32;
    const int n = lane & 15, g = lane >> 4;
    int col = w.col, tile = w.tile;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        int page = -1;
        if (w.key + 16 * i < w.end) page = table[col];
        page = __builtin_amdgcn_readfirstlane(page);
        const bool there = page >= 0 && page < p.n_pages;
        r.key[i] = there ? w.key + 16 * i : kNoKeys;
        // keys that are not there are loaded from the pool's first page, and masked
        const uint8_t* z = head + (there ? page * p.page_stride + (int64_t)tile * (17 * HD) : 0);
        const uint8_t* kc = z + n * (HD / 2) + g * (HD / 8);
        const uint8_t* vc = z + 8 * HD + g * (2 * HD) + n * (HD / 8);
        if constexpr (N == 4) {
            const u4v a = *reinterpret_cast<const u4v*>(kc), b = *reinterpret_cast<const u4v*>(vc);
#pragma unroll
            for (int j = 0; j < 4; ++j) r.k[i][j] = a[j], r.v[i][j] = b[j];
        } else {
            const u2v a = *reinterpret_cast<const u2v*>(kc), b = *reinterpret_cast<const u2v*>(vc);
#pragma unroll
            for (int j = 0; j < 2; ++j) r.k[i][j] = a[j], r.v[i][j] = b[j];
        }
        r.ks[i] = z[16 * HD + n * (HD / 32) + g * (HD / 32) / 4];
        r.vs[i] = *reinterpret_cast<const uint32_t*>(z + 16 * HD + HD / 2 + (g * (HD / 32) + n * (HD / 16) / 32) * 4);
        if (++tile == p.tiles) tile = 0, ++col;
    }
    w.key += (w.step_cols * p.tiles + w.step_tiles) * kKv4Tile;
    w.col += w.step_cols;
    w.tile += w.step_tiles;
    if (w.tile >= p.tiles) w.tile -= p.tiles, ++w.col;
}

// The state of RT x 16 query rows.
template <int HD, int RT, int NP>
struct Kv4State {
    uint32_t q[RT][NP][HD / 32][4];  // parts of the queries, in the operand's order
    f4v o[RT][HD / 16];              // O^T: channel (4 g + i) HD/16 + j of row lane % 16 in o[j][i]
    float m[RT], l[RT];              // maximum (of the row), sum (of the lane's keys), base 2
    int lim[RT];                     // keys that the lane's row sees
};

PE_DEV bf8v operand(const uint32_t* w) {
    const u4v z = {w[0], w[1], w[2], w[3]};
    return __builtin_bit_cast(bf8v, z);
}

template <int HD, int RT, int NP>
PE_DEV void kv4_step(const Kv4AttnArgs& p, Kv4Raw<HD>& r, Kv4State<HD, RT, NP>& st, int least, int most, int lane) {
    constexpr int N = HD / 32, E = HD / 16;
    const int g = lane >> 4;
    // scores: [rows][16 keys][4 keys of the lane]
    float s[RT][4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float scale = __uint_as_float(r.ks[i] << 23);
        f4v acc[RT] = {};
#pragma unroll
        for (int j = 0; j < N; ++j) {
            uint32_t w[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) w[c] = two_codes(r.k[i][j], scale, c);
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int n = 0; n < NP; ++n)
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(w), operand(st.q[t][n][j]), acc[t], 0, 0, 0);
        }
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[t][i][c] = acc[t][c] * p.scale;
    }
    // keys that some row does not see, or that are not there
    const bool masked = r.key[0] + 16 > least || r.key[1] + 16 > least || r.key[2] + 16 > least || r.key[3] + 16 > least;
    uint32_t bad[2] = {0, 0};  // 16 keys: the lane's value scales (bit c: key c) that are no number
    if (masked) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // a key scale that is no number: the byte's 2^128 made infinities of the codes, and NaN of zeros only
            uint64_t nan = __ballot(r.ks[i] == 255);
            nan |= nan >> 32;
            const uint32_t rows = (uint32_t)(nan | nan >> 16) >> (4 * g);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int key = r.key[i] + 4 * g + c;
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    if (rows >> c & 1) s[t][i][c] = __uint_as_float(0x7FC00000u);
                    if (key >= st.lim[t]) s[t][i][c] = -INFINITY;
                }
                const bool none = key >= most;
                const uint32_t byte = r.vs[i] >> (8 * c) & 255;
                if (!none && byte == 255) bad[i >> 1] |= 1u << ((i & 1) * 4 + c);
                // what no row sees may hold anything, and a value that is no number must not reach rows that do not
                // see it: zero codes, and scale 1
                if (none || byte == 255) {
                    r.vs[i] = (r.vs[i] & ~(255u << (8 * c))) | 127u << (8 * c);
                    if constexpr (HD == 128)
                        r.v[i][c] = 0;
                    else
                        r.v[i][c >> 1] &= c & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint64_t nan = __ballot(r.ks[i] == 255);
            if (nan) {
                nan |= nan >> 32;
                const uint32_t rows = (uint32_t)(nan | nan >> 16) >> (4 * g);
#pragma unroll
                for (int t = 0; t < RT; ++t)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        if (rows >> c & 1) s[t][i][c] = __uint_as_float(0x7FC00000u);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if ((r.vs[i] >> (8 * c) & 255) == 255) {
                    bad[i >> 1] |= 1u << ((i & 1) * 4 + c);
                    r.vs[i] = (r.vs[i] & ~(255u << (8 * c))) | 127u << (8 * c);
                    if constexpr (HD == 128)
                        r.v[i][c] = 0;
                    else
                        r.v[i][c >> 1] &= c & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                }
        }
    }
    // running maximum and sum
    uint32_t pr[RT][2][NP][4];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) top = fmaxf(top, s[t][i][c]);
        top = swap32_max(swap16_max(top));
        const float m = fmaxf(st.m[t], top), base = m == -INFINITY ? 0.f : m;
        const float shrink = __builtin_amdgcn_exp2f(st.m[t] - base);
        st.m[t] = m;
        st.l[t] *= shrink;
#pragma unroll
        for (int j = 0; j < E; ++j) st.o[t][j] *= shrink;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float e[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                e[c] = __builtin_amdgcn_exp2f(s[t][i][c] - base);
                st.l[t] += e[c];
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t w[NP];
                split_pair<NP>(e[2 * c], e[2 * c + 1], w);
#pragma unroll
                for (int n = 0; n < NP; ++n) pr[t][i >> 1][n][2 * (i & 1) + c] = w[n];
            }
        }
    }
    // values: 32 keys at a time, two channels of a run at a time
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float scale[8];
#pragma unroll
        for (int c = 0; c < 8; ++c)
            scale[c] = __uint_as_float((r.vs[2 * h + (c >> 2)] >> (8 * (c & 3)) & 255u) << 23);
#pragma unroll
        for (int j = 0; j < E; j += 2) {
            uint32_t two[8], lo[4], hi[4];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const int i = 2 * h + (c >> 2), k = c & 3;
                two[c] = HD == 128 ? two_codes(r.v[i][k], scale[c], j >> 1) : two_codes(r.v[i][k >> 1], scale[c], (k & 1) * 2 + (j >> 1));
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                lo[c] = __builtin_amdgcn_perm(two[2 * c + 1], two[2 * c], 0x05040100u);
                hi[c] = __builtin_amdgcn_perm(two[2 * c + 1], two[2 * c], 0x07060302u);
            }
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    st.o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(lo), operand(pr[t][h][n]), st.o[t][j], 0, 0, 0);
                    st.o[t][j + 1] =
                        __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(hi), operand(pr[t][h][n]), st.o[t][j + 1], 0, 0, 0);
                }
        }
        // values that are no number: how many of them a row sees, in every run (all its channels share the scale)
        if (__ballot(bad[h] != 0)) {
            uint32_t w[4];
#pragma unroll
            for (int c = 0; c < 4; ++c)
                w[c] = (bad[h] >> (2 * c) & 1 ? 0x3F80u : 0u) | (bad[h] >> (2 * c + 1) & 1 ? 0x3F800000u : 0u);
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                uint32_t sees[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int key = r.key[2 * h + (c >> 1)] + 4 * g + 2 * (c & 1);
                    sees[c] = (key < st.lim[t] ? 0x3F80u : 0u) | (key + 1 < st.lim[t] ? 0x3F800000u : 0u);
                }
                f4v count = {};
                count = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(w), operand(sees), count, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (count[i] > 0.f)
#pragma unroll
                        for (int j = 0; j < E; ++j) st.o[t][j][i] = __uint_as_float(0x7FC00000u);
            }
        }
    }
}

template <typename T>
constexpr int kKv4Parts = sizeof(T) == 2 ? 2 : 3;

// SPLIT: the workgroup's rows are RT x 16, its waves take steps in turn and are merged in LDS. Otherwise every wave has
// RT x 16 rows of its own and takes all the item's keys.
template <typename T, int HD, int RT, bool SPLIT>
__global__ __launch_bounds__(64 * kKv4Waves) void k_kv4_attn(Kv4AttnArgs p) {
    constexpr int NP = kKv4Parts<T>, E = HD / 16, R = 16 * RT, RB = SPLIT ? R : R * kKv4Waves;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int item = blockIdx.x, kvh = blockIdx.y;
    Kv4Item w;
    if (!kv4_find<RB>(p, item, w)) return;
    const Kv4Seq seq = kv4_seq(p, w.b);
    if (w.chunk == 0 && w.block == 0 && kvh == 0 && threadIdx.x == 0 && p.plan)
        p.plan[w.b] = make_int4(w.base, w.chunks, w.blocks, 0);

    // the wave's rows: r0 + 16 t + n
    const int r0 = w.block * RB + (SPLIT ? 0 : wave * R), last = (r0 + R < seq.rows ? r0 + R : seq.rows) - 1;
    Kv4State<HD, RT, NP> st;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int row = r0 + 16 * t + n, i = row / p.group;
        const bool there = row < seq.rows;
        st.lim[t] = there ? kv4_keys(p, seq.keys, i) : 0;
        st.m[t] = -INFINITY;
        st.l[t] = 0.f;
#pragma unroll
        for (int j = 0; j < E; ++j) st.o[t][j] = f4v{};
        const T* q = static_cast<const T*>(p.q) + (seq.lo + i) * p.q_token + (int64_t)(kvh * p.group + row - i * p.group) * p.q_head +
                     g * (HD / 4);
#pragma unroll
        for (int j = 0; j < HD / 32; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t z[NP];
                split_pair<NP>(there ? (float)q[8 * j + 2 * c] : 0.f, there ? (float)q[8 * j + 2 * c + 1] : 0.f, z);
#pragma unroll
                for (int k = 0; k < NP; ++k) st.q[t][k][j][c] = z[k];
            }
    }
    const bool rows = r0 < seq.rows;
    const int least = rows ? kv4_keys(p, seq.keys, r0 / p.group) : 0, most = rows ? kv4_keys(p, seq.keys, last / p.group) : 0;
    const int64_t begin = (int64_t)w.chunk * w.span, stop = begin + w.span;
    Kv4Walk walk;
    walk.end = (int)(stop < most ? stop : most);
    walk.key = (int)begin + (SPLIT ? wave * kKv4Step : 0);
    const int stride = SPLIT ? 4 * kKv4Waves : 4;  // tiles from step to step
    walk.step_cols = stride / p.tiles;
    walk.step_tiles = stride - walk.step_cols * p.tiles;
    walk.col = walk.key / kKv4Tile / p.tiles;
    walk.tile = walk.key / kKv4Tile - walk.col * p.tiles;
    const int* table = p.table + w.b * p.table_row;
    const uint8_t* head = p.pages + (int64_t)kvh * p.tiles * (17 * HD);
    while (walk.key < walk.end) {
        Kv4Raw<HD> raw;
        kv4_load<HD>(p, table, head, walk, lane, raw);
        kv4_step<HD, RT, NP>(p, raw, st, least, most, lane);
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) st.l[t] = swap32_sum(swap16_sum(st.l[t]));

    const int64_t rec = ((int64_t)kvh * p.items + item) * RB;
    if constexpr (SPLIT) {
        __shared__ float part[kKv4Waves][R][HD + 4];
        __shared__ float pm[kKv4Waves][R], pl[kKv4Waves][R];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int row = 16 * t + n;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < E; ++j) part[wave][row][(4 * g + i) * E + j] = st.o[t][j][i];
            if (g == 0) pm[wave][row] = st.m[t], pl[wave][row] = st.l[t];
        }
        __syncthreads();
        for (int x = threadIdx.x; x < R * 16; x += 64 * kKv4Waves) {
            const int row = x / 16, c = x % 16 * E, r = r0 + row;
            if (r >= seq.rows) break;
            float m = -INFINITY;
#pragma unroll
            for (int k = 0; k < kKv4Waves; ++k) m = fmaxf(m, pm[k][row]);
            const float base = m == -INFINITY ? 0.f : m;
            float l = 0.f, o[E] = {};
#pragma unroll
            for (int k = 0; k < kKv4Waves; ++k) {
                const float f = __builtin_amdgcn_exp2f(pm[k][row] - base);
                l = fmaf(pl[k][row], f, l);
#pragma unroll
                for (int j = 0; j < E; ++j) o[j] = fmaf(part[k][row][c + j], f, o[j]);
            }
            if (w.chunks == 1) {
                const int i = r / p.group;
                const float f = l == 0.f ? 0.f : 1.f / l;
                T* y = static_cast<T*>(p.out) + (seq.lo + i) * p.out_token + (int64_t)(kvh * p.group + r - i * p.group) * p.out_head + c;
#pragma unroll
                for (int j = 0; j < E; ++j) y[j] = (T)(o[j] * f);
            } else {
                float* y = p.record + (rec + row) * HD + c;
#pragma unroll
                for (int j = 0; j < E; ++j) y[j] = o[j];
                if (c == 0) p.stat[2 * (rec + row)] = m, p.stat[2 * (rec + row) + 1] = l;
            }
        }
    } else {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int row = wave * R + 16 * t + n, r = r0 + 16 * t + n;
            if (r >= seq.rows) continue;
            const int i = r / p.group;
            const float f = st.l[t] == 0.f ? 0.f : 1.f / st.l[t];
            if (w.chunks == 1) {
                T* y = static_cast<T*>(p.out) + (seq.lo + i) * p.out_token + (int64_t)(kvh * p.group + r - i * p.group) * p.out_head;
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int j = 0; j < E; ++j) y[(4 * g + k) * E + j] = (T)(st.o[t][j][k] * f);
            } else {
                float* y = p.record + (rec + row) * HD;
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int j = 0; j < E; ++j) y[(4 * g + k) * E + j] = st.o[t][j][k];
                if (g == 0) p.stat[2 * (rec + row)] = st.m[t], p.stat[2 * (rec + row) + 1] = st.l[t];
            }
        }
    }
}

// The chunks of a row: one wave per row of q, a lane HD / 64 channels.
template <typename T, int HD, int RB>
__global__ __launch_bounds__(256) void k_kv4_merge(Kv4AttnArgs p) {
    constexpr int C = HD / 64;
    const int lane = threadIdx.x & 63;
    const int64_t x = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), t = x / p.n_head;
    const int h = (int)(x - t * p.n_head);
    if (t >= p.tokens) return;
    const int64_t b = sequence_of(p.starts, p.starts_wide, p.batch, t);
    if (b < 0) return;
    const Kv4Seq seq = kv4_seq(p, (int)b);
    const int kvh = h / p.group, r = (int)(t - seq.lo) * p.group + h - kvh * p.group;
    const int4 plan = p.plan[b];
    // (a plan that no workgroup wrote, of starts that are out of order, holds anything)
    if (plan.y <= 1 || plan.z <= 0 || plan.x < 0 || r < 0 || r / RB >= plan.z || (int64_t)plan.x + (int64_t)plan.y * plan.z > p.items) return;
    float m = -INFINITY, l = 0.f, o[C] = {};
    for (int c = 0; c < plan.y; ++c) {
        const int64_t rec = ((int64_t)kvh * p.items + plan.x + c * plan.z + r / RB) * RB + r % RB;
        const float mc = p.stat[2 * rec], lc = p.stat[2 * rec + 1];
        const float top = fmaxf(m, mc), base = top == -INFINITY ? 0.f : top;
        const float f = __builtin_amdgcn_exp2f(m - base), e = __builtin_amdgcn_exp2f(mc - base);
        l = l * f + lc * e;
#pragma unroll
        for (int j = 0; j < C; ++j) o[j] = o[j] * f + p.record[rec * HD + lane * C + j] * e;
        m = top;
    }
    const float f = l == 0.f ? 0.f : 1.f / l;
    T* y = static_cast<T*>(p.out) + t * p.out_token + (int64_t)h * p.out_head + lane * C;
#pragma unroll
    for (int j = 0; j < C; ++j) y[j] = (T)(o[j] * f);
}

// How a call is cut: rows of a workgroup and workgroups of a kv head, from what the host knows (the lengths are on the device).
struct Kv4Plan {
    int rt, split;   // 16-row tiles of a wave; the waves share the rows and split the keys
    int rb;          // rows of a workgroup
    int64_t blocks, items;
    int min_chunk;
};

static Kv4Plan kv4_plan(int64_t tokens, int64_t batch, bool ragged, int n_head, int n_kv, int64_t capacity) {
    Kv4Plan s;
    const int group = n_head / n_kv;
    const int64_t rows = ragged ? (tokens + batch - 1) / batch * group : group;  // of a sequence, on average
    s.rt = rows <= 16 ? 1 : 2;
    s.split = rows <= 32;
    s.rb = 16 * s.rt * (s.split ? 1 : kKv4Waves);
    s.blocks = ragged ? tokens * group / s.rb + batch : batch * ((group + s.rb - 1) / s.rb);
    s.min_chunk = kKv4Step * (s.split ? kKv4Waves : 4);
    // as many workgroups more as fill the chip, three on each CU, and let uneven sequences be cut evenly
    const int64_t want = (768 + n_kv - 1) / n_kv, chunks = (capacity + s.min_chunk - 1) / s.min_chunk;
    int64_t extra = s.blocks < want ? want - s.blocks : 0;
    if (extra < want / 4) extra = want / 4;
    if (chunks <= 1)
        extra = 0;
    else if (extra > s.blocks * (chunks - 1))
        extra = s.blocks * (chunks - 1);
    s.items = s.blocks + extra;
    return s;
}

static bool kv4_shape_ok(int64_t tokens, int64_t batch, bool ragged, int n_head, int n_kv, int hd, int64_t capacity) {
    return tokens >= 0 && tokens <= (1 << 22) && batch > 0 && batch <= (1 << 20) && (ragged || tokens == batch) && n_head > 0 &&
           n_head <= 4096 && n_kv > 0 && n_head % n_kv == 0 && (hd == 64 || hd == 128) && capacity >= 0 && capacity <= (1LL << 30) &&
           tokens * (n_head / n_kv) < (1LL << 30);
}

static int64_t kv4_bytes(const Kv4Plan& s, int64_t batch, int n_kv, int hd) {
    return s.items > s.blocks ? (batch * 16 + s.items * n_kv * s.rb * (int64_t)(hd + 2) * 4 + 15) / 16 * 16 : 0;
}

template <typename T, int HD>
static void launch_kv4(const Kv4AttnArgs& p, const Kv4Plan& s, hipStream_t st) {
    const dim3 g((unsigned)s.items, (unsigned)p.n_kv), m((unsigned)((p.tokens * p.n_head + 3) / 4));
    if (!s.split) {
        hipLaunchKernelGGL((k_kv4_attn<T, HD, 2, false>), g, dim3(64 * kKv4Waves), 0, st, p);
        if (p.plan) hipLaunchKernelGGL((k_kv4_merge<T, HD, 32 * kKv4Waves>), m, dim3(256), 0, st, p);
    } else if (s.rt == 2) {
        hipLaunchKernelGGL((k_kv4_attn<T, HD, 2, true>), g, dim3(64 * kKv4Waves), 0, st, p);
        if (p.plan) hipLaunchKernelGGL((k_kv4_merge<T, HD, 32>), m, dim3(256), 0, st, p);
    } else {
        hipLaunchKernelGGL((k_kv4_attn<T, HD, 1, true>), g, dim3(64 * kKv4Waves), 0, st, p);
        if (p.plan) hipLaunchKernelGGL((k_kv4_merge<T, HD, 16>), m, dim3(256), 0, st, p);
    }
}

}  // namespace pe

using namespace pe;

extern "C" int64_t pe_kv4_attn_workspace_bytes(int64_t tokens, int64_t batch, int ragged, int n_head, int n_kv, int head_dim,
                                               int64_t capacity) {
    if (!kv4_shape_ok(tokens, batch, ragged, n_head, n_kv, head_dim, capacity)) return -PE_ERR_SHAPE;
    return kv4_bytes(kv4_plan(tokens, batch, ragged, n_head, n_kv, capacity), batch, n_kv, head_dim);
}

extern "C" int pe_kv4_attn(const pe_kv4_attn_args* a, pe_stream_t stream) {
    if (!a) return PE_ERR_NULL;
    if ((a->type != PE_TYPE_F32 && a->type != PE_TYPE_F16) || (a->lengths_dtype != 1 && a->lengths_dtype != 2) ||
        (a->starts && a->starts_dtype != 1 && a->starts_dtype != 2))
        return PE_ERR_TYPE;
    if (a->tokens == 0 || a->batch == 0) return PE_OK;
    if (const int st = kv4_pool_ok(&a->pool, a->n_kv, a->head_dim)) return st;
    const int64_t T = a->tokens, capacity = a->pool.table_cols * a->pool.page_tokens;
    const bool ragged = a->starts != nullptr;
    if (!kv4_shape_ok(T, a->batch, ragged, a->n_head, a->n_kv, a->head_dim, capacity) || !std::isfinite(a->scale) ||
        a->first < -(1LL << 40) || a->first > (1LL << 40) || a->q_token < 0 || a->q_head < 0 || a->out_token < 0 || a->out_head < 0 ||
        (a->n_head > 1 && a->out_head < a->head_dim) || (T > 1 && a->out_token < a->head_dim) ||
        (T > 1 && a->n_head > 1 && a->out_token < a->out_head * (a->n_head - 1) + a->head_dim &&
         a->out_head < a->out_token * (T - 1) + a->head_dim))
        return PE_ERR_SHAPE;
    const Kv4Plan s = kv4_plan(T, a->batch, ragged, a->n_head, a->n_kv, capacity);
    const int64_t need = kv4_bytes(s, a->batch, a->n_kv, a->head_dim);
    if (!a->q || !a->out || !a->lengths || (need && !a->workspace)) return PE_ERR_NULL;
    const size_t e = a->type == PE_TYPE_F16 ? 2 : 4;
    if (!aligned(a->q, e) || !aligned(a->out, e) || !aligned(a->lengths, a->lengths_dtype == 2 ? 8 : 4) ||
        (ragged && !aligned(a->starts, a->starts_dtype == 2 ? 8 : 4)) || !aligned(a->workspace, 16))
        return PE_ERR_ALIGN;
    if (a->workspace_bytes < need) return PE_ERR_SPACE;
    if (s.items * a->n_kv >= (1 << 24) || T * a->n_head >= (1LL << 26)) return PE_ERR_SHAPE;  // a grid holds 2^32 threads
    int4* plan = need ? static_cast<int4*>(a->workspace) : nullptr;
    float* record = need ? reinterpret_cast<float*>(plan + a->batch) : nullptr;
    Kv4AttnArgs p{a->q, a->q_token, a->q_head, a->out, a->out_token, a->out_head, static_cast<const uint8_t*>(a->pool.pages),
                  a->pool.page_stride, (int)a->pool.n_pages, (int)(a->pool.page_tokens / kKv4Tile), a->pool.table,
                  a->pool.table_stride, (int)a->pool.table_cols, a->lengths, a->lengths_dtype == 2, a->first, a->starts,
                  a->starts_dtype == 2, T, (int)a->batch, a->n_head, a->n_kv, a->n_head / a->n_kv, a->scale * kKv4Log2e,
                  (int)s.items, (int)s.blocks, s.min_chunk, plan, record,
                  need ? record + s.items * a->n_kv * s.rb * a->head_dim : nullptr};
    hipStream_t st = (hipStream_t)stream;
    if (a->type == PE_TYPE_F16)
        a->head_dim == 64 ? launch_kv4<_Float16, 64>(p, s, st) : launch_kv4<_Float16, 128>(p, s, st);
    else
        a->head_dim == 64 ? launch_kv4<float, 64>(p, s, st) : launch_kv4<float, 128>(p, s, st);
    return launch_status();
}
