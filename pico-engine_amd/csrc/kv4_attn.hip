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

constexpr int kKv4Waves = 4;   // of a workgroup
constexpr int kKv4Span = 64;   // chunks are whole multiples of it
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
    float scale;        // of fp16 queries' scores, above 0
    double q_scale;     // of queries: with the scores' factor the scale times log2 e
    int64_t capacity;   // slots of a sequence
    int vec;            // q's rows are whole pieces of 16 bytes
    int items, blocks;  // workgroups a kv head, row blocks at most
    int records;        // chunks that there is room for, a kv head
    int min_chunk;      // least keys of a chunk
    float weight;       // of all keys in the square of a chunk's length
    int rec_rows;       // rows of a record
    float round;        // workgroups of a kv head that are resident at once
    int4* plan;         // of every sequence: first record (if it is cut), chunks, row blocks
    float* record;      // [kv head][records][row][HD], a row block's chunks one after the other
    float* stat;        // [kv head][records][row] (maximum, sum)
};

// Work of a sequence.
struct Kv4Seq {
    int64_t lo;   // first row
    int rows;     // rows times the heads of a group
    int64_t keys; // keys that its first row sees (far below 0: it takes no part)
};

PE_DEV Kv4Seq kv4_seq(const Kv4AttnArgs& p, int b) {
    int64_t lo, hi;
    rows_of(p.starts, p.starts_wide, b, p.tokens, lo, hi);
    const int64_t len = int_at(p.lengths, p.len_wide, b);
    return {lo, (int)(hi - lo) * p.group, len < 0 ? -(1LL << 42) : (len > (1LL << 41) ? 1LL << 41 : len) + p.first};
}

// Keys that row i (of a token) sees.
PE_DEV int kv4_keys(const Kv4AttnArgs& p, int64_t first_keys, int i) {
    const int64_t k = first_keys + i;
    return (int)(k < 0 ? 0 : k > p.capacity ? p.capacity : k);
}

// Sum over the lanes up to and including each (six steps of DPP: rows of 16, then the rows below).
PE_DEV int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);  // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, true);  // row_bcast 15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, true);  // row_bcast 31 into rows 2 and 3
    return v;
}

struct Kv4Item {
    int b, block, chunk, chunks, blocks, record, span;  // record: the sequence's first, if it is cut; span: keys of a chunk
    Kv4Seq seq;
};

// Which work the item is: a (sequence, row block, chunk of keys). Every wave finds it for itself, from all lengths.
// A chunk's length S weighs what workgroups cost beside their keys against the time that the last one takes
// alone: all keys' time + S a + (all keys / S) F / (256 c), with a of a key, F of a workgroup, c of them on a CU
// at once, is least at S = sqrt(all keys F / (256 c a)). Keys of all kv heads times row blocks, and a weight for the rest,
// 0.75, for a few fp32 queries of 128 channels, which take longer over a key, 0.5. In us with 0.25, 0.5, 0.75 and 2.5 (28 heads
// of 128, fp32) one new row on 33 x 4001 keys 23.4, 22.9, 24.4 and 24.6, on 8 x 8000 18.3, 16.7, 18.6 and 19.6, on 64 x 4096
// 53, 49.6, 49 and 55, 2 x 1021 rows on 8000 keys 537, 516, 508 and 522; fp16: 64 x 16384 (32 heads) 146, 145, 142 and 150, 2 x
// 1021 rows 404, 378, 368 and 369.
//
// Records are numbered as items are, in blocks of 128 rows cut sequences' alone: a second scan of all sequences, which costs a call of
// few rows more than the room is worth (one row on 700 keys 9.6 -> 10.0 us).
template <int RB>
PE_DEV bool kv4_find(const Kv4AttnArgs& p, int item, Kv4Item& w) {
    const int lane = threadIdx.x & 63;
    const auto look = [&](int b, Kv4Seq& s, int& nb, int& keys) {  // the sequence, its row blocks, keys of the last row
        nb = keys = 0;
        if (b >= p.batch) return;
        s = kv4_seq(p, b);
        nb = (s.rows + RB - 1) / RB;
        if (nb) keys = kv4_keys(p, s.keys, s.rows / p.group - 1);
    };
    constexpr bool CUT_ALONE = RB > 16;
    const auto chunks_of = [](int keys, int span) { return keys > span ? (int)((uint32_t)(keys + span - 1) / (uint32_t)span) : 1; };
    Kv4Seq seq0{}, seq;
    int nb0, keys0;
    look(lane, seq0, nb0, keys0);
    int span = 1 << 30;
    if (p.items > p.blocks) {
        int64_t cost = (int64_t)nb0 * keys0;
        for (int b = lane + 64; b < p.batch; b += 64) {
            int nb, keys;
            look(b, seq, nb, keys);
            cost += (int64_t)nb * keys;
        }
        const float all = wave_sum<64>((float)cost);
        span = ((int)fmaxf(sqrtf(all * p.weight), (float)p.min_chunk) + kKv4Span - 1) / kKv4Span * kKv4Span;
        float count = (float)nb0 * (float)chunks_of(keys0, span), cut = CUT_ALONE && keys0 > span ? count : 0.f;
        for (int b = lane + 64; b < p.batch; b += 64) {
            int nb, keys;
            look(b, seq, nb, keys);
            const float c = (float)nb * (float)chunks_of(keys, span);
            count += c;
            if (CUT_ALONE && keys > span) cut += c;
        }
        // Up to 1.6 rounds of what is resident at once are made one, of longer chunks (5 rows on 80000 keys, 32 heads of
        // 128, fp16: 47.9 -> 43.7 us, on 120000 63.5 -> 59.3; 128 x 8000, 14 heads of 64: 36.4 -> 34.4; 2 x 700 rows on
        // 3000 keys, fp32 81 -> 75; 3 x 300 on 6000, 28 heads of 128, 116 -> 118).
        count = wave_sum<64>(count);
        if (count > p.round && count < 1.6f * p.round)
            span = ((int)((float)span * count / p.round) + kKv4Span - 1) / kKv4Span * kKv4Span;
        // more than the launch has (both are whole numbers, exact below 2^24, and there are fewer items): keys times blocks
        // shared out evenly, in 32-bit floats, and a 4096th more, which is beyond what their rounding takes off
        if (count > (float)p.items || (CUT_ALONE && wave_sum<64>(cut) > (float)p.records)) {
            const float safe = all / (float)(p.items - p.blocks) * (1.f + 1.f / 4096) + kKv4Span;
            span = safe < (float)(1 << 30) ? (int)safe / kKv4Span * kKv4Span : 1 << 30;
            span = span < p.min_chunk ? p.min_chunk : span;
        }
    }
    int base = 0, records = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
        int nb = nb0, keys = keys0;
        seq = seq0;
        if (b0) look(b0 + lane, seq, nb, keys);
        const int chunks = chunks_of(keys, span);
        const int upto = wave_scan(nb * chunks), recorded = CUT_ALONE ? wave_scan(chunks > 1 ? nb * chunks : 0) : upto;
        const uint64_t beyond = __ballot(base + upto > item);
        if (beyond) {
            const int at = __builtin_ctzll(beyond);
            w.b = b0 + at;
            w.seq = {lane_of(seq.lo, at), __builtin_amdgcn_readlane(seq.rows, at), lane_of(seq.keys, at)};
            w.blocks = __builtin_amdgcn_readlane(nb, at);
            w.chunks = __builtin_amdgcn_readlane(chunks, at);
            const int first = base + __builtin_amdgcn_readlane(upto, at) - w.blocks * w.chunks;
            w.record = CUT_ALONE ? records + __builtin_amdgcn_readlane(recorded, at) - w.blocks * w.chunks : first;
            w.span = span;
            // starts that are out of order can ask for more than there is room for
            if (first < 0 || first + (int64_t)w.blocks * w.chunks > p.items) return false;
            if (CUT_ALONE && w.chunks > 1 && (w.record < 0 || w.record + (int64_t)w.blocks * w.chunks > p.records)) return false;
            const int local = item - first;
            if (w.blocks == 1) {
                w.chunk = local, w.block = 0;
            } else if (RB == 16) {
                // Few blocks: eight chunks side by side, the blocks of each eight items apart. Workgroups go to the eight
                // XCDs in turn, so blocks that read the same keys find them in one L2 (two blocks on 65536 keys: 43 -> 41.5 us).
                const int eight = local / (8 * w.blocks), rest = local - eight * 8 * w.blocks;
                const int side = w.chunks - 8 * eight < 8 ? w.chunks - 8 * eight : 8;
                w.block = rest / side;
                w.chunk = 8 * eight + rest - w.block * side;
            } else {  // many blocks: those of the same keys one after the other (2 x 1021 rows: 379 us, as above 390)
                w.chunk = local / w.blocks;
                w.block = local - w.chunk * w.blocks;
            }
            return true;
        }
        base += __builtin_amdgcn_readlane(upto, 63);
        if (CUT_ALONE) records += __builtin_amdgcn_readlane(recorded, 63);
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

// The two codes of byte sel of w as a pair of bf16 (low half: the low four bits), times scale, of which the exponent's
// bits alone count; all of them set makes NaN.
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

// Which keys a wave takes next, and where they lie: all scalar.
template <int TS>
struct Kv4Walk {
    const uint8_t* at[TS];  // the 16 keys' tiles
    int key[TS];            // numbers of their first keys
    int id[TS];             // pages of the step behind
    int col, tile;          // page of the table, tile in it, of that step's first 16 keys
    int next, end;          // its first key, the item's last
    int cols, tiles;        // from step to step
};

constexpr int kNoKeys = 0x7FFFFF00;  // number of the first key of 16 that are not there

// The table's pages of the next step: read a step ahead of the loads that go there.
template <int TS>
PE_DEV void kv4_pages(const Kv4AttnArgs& p, const int* table, Kv4Walk<TS>& w) {
    typedef const __attribute__((address_space(4))) int* scalar_ints;
    const scalar_ints ids = (scalar_ints)(uintptr_t)table;
    int col = w.col, tile = w.tile;
#pragma unroll
    for (int i = 0; i < TS; ++i) {
        w.id[i] = -1;
        if (w.next + 16 * i < w.end) w.id[i] = ids[col];
        if (++tile == p.tiles) tile = 0, ++col;
    }
}

template <int HD, int TS>
PE_DEV void kv4_advance(const Kv4AttnArgs& p, const int* table, const uint8_t* head, Kv4Walk<TS>& w) {
    int tile = w.tile;
#pragma unroll
    for (int i = 0; i < TS; ++i) {
        const bool there = (uint32_t)w.id[i] < (uint32_t)p.n_pages;
        w.key[i] = there ? w.next + 16 * i : kNoKeys;
        // keys that are not there are loaded from the pool's first page, and masked
        w.at[i] = head + (there ? w.id[i] * p.page_stride + (int64_t)tile * (17 * HD) : 0);
        if (++tile == p.tiles) tile = 0;
    }
    w.next += (w.cols * p.tiles + w.tiles) * kKv4Tile;
    w.col += w.cols;
    w.tile += w.tiles;
    if (w.tile >= p.tiles) w.tile -= p.tiles, ++w.col;
    kv4_pages<TS>(p, table, w);
}

// A lane's part of a step's keys: codes and scale bytes.
template <int HD, int TS>
struct Kv4Raw {
    static constexpr int N = HD / 32;  // words of codes per 16 keys
    uint32_t c[TS][N], s[TS];
};
template <int N>
PE_DEV void kv4_words(const uint8_t* at, uint32_t* w) {
    if constexpr (N == 4) {
        const u4v a = *reinterpret_cast<const u4v*>(at);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = a[j];
    } else {
        const u2v a = *reinterpret_cast<const u2v*>(at);
        w[0] = a[0], w[1] = a[1];
    }
}
template <int HD, int TS>
PE_DEV void kv4_load_keys(const Kv4Walk<TS>& w, int lane, Kv4Raw<HD, TS>& r) {
    const uint32_t n = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < TS; ++i) {
        kv4_words<HD / 32>(w.at[i] + (n * (HD / 2) + g * (HD / 8)), r.c[i]);
        r.s[i] = w.at[i][16 * HD + (n * (HD / 32) + g * (HD / 32) / 4)];
    }
}
template <int HD, int TS>
PE_DEV void kv4_load_values(const Kv4Walk<TS>& w, int lane, Kv4Raw<HD, TS>& r) {
    const uint32_t n = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < TS; ++i) {
        kv4_words<HD / 32>(w.at[i] + 8 * HD + (g * (2 * HD) + n * (HD / 8)), r.c[i]);
        r.s[i] = *reinterpret_cast<const uint32_t*>(w.at[i] + 16 * HD + HD / 2 + (g * (HD / 32) + n * (HD / 16) / 32) * 4);
    }
}

// The state of RT x 16 query rows.
template <int HD, int RT>
struct Kv4State {
    f4v o[RT][HD / 16];  // O^T: channel (4 g + i) HD/16 + j of row lane % 16 in o[j][i]
    float m[RT], l[RT];  // what exponents are taken from (of the row), sum (of the lane's keys), base 2
    float scale[RT];     // of the row's scores
    int lim[RT];         // keys that the lane's row sees
};

PE_DEV bf8v operand(const uint32_t* w) {
    const u4v z = {w[0], w[1], w[2], w[3]};
    return __builtin_bit_cast(bf8v, z);
}

// Scores of a step's keys for 16 rows: s[16 keys][4 keys of the lane]. q: the lane's operands in LDS, parts of the queries
// [NP][HD / 32][64 lanes]. A scale byte of 255 converts every code to NaN.
template <int HD, int NP, int TS>
PE_DEV void kv4_scores(const Kv4Raw<HD, TS>& r, const u4v* q, f4v (&s)[TS]) {
#pragma unroll
    for (int i = 0; i < TS; ++i) s[i] = f4v{};
    // products of different scores one after the other: one that adds to the last one's would wait for it
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) {
        uint32_t w[TS][4];
#pragma unroll
        for (int i = 0; i < TS; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) w[i][c] = two_codes(r.c[i][j], __uint_as_float(r.s[i] << 23), c);
#pragma unroll
        for (int n = 0; n < NP; ++n) {
            const bf8v z = __builtin_bit_cast(bf8v, q[(n * (HD / 32) + j) * 64]);
#pragma unroll
            for (int i = 0; i < TS; ++i) s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(w[i]), z, s[i], 0, 0, 0);
        }
    }
}

// Values that no row sees (from key `most` on) may hold anything, and one that is no number must not reach rows that do not
// see it: their codes become 0 and their scale 1. bad tells of the latter that some row sees (bit 4 (i % 2) + c of bad[i /
// 2]: key c of the lane's in the 16 keys i).
template <int HD, int TS>
PE_DEV void kv4_mask_value(int key, int i, int c, int most, Kv4Raw<HD, TS>& v, uint32_t* bad) {
    const bool none = key >= most, nan = (v.s[i] >> (8 * c) & 255) == 255;
    if (!none && nan) bad[i >> 1] |= 1u << ((i & 1) * 4 + c);
    if (none || nan) {
        v.s[i] = (v.s[i] & ~(255u << (8 * c))) | 127u << (8 * c);
        if constexpr (HD == 128)
            v.c[i][c] = 0;
        else
            v.c[i][c >> 1] &= c & 1 ? 0x0000FFFFu : 0xFFFF0000u;
    }
}
template <int HD, int TS>
PE_DEV void kv4_mask_values(const int* keys, int most, int g, Kv4Raw<HD, TS>& v, uint32_t* bad) {
#pragma unroll
    for (int i = 0; i < TS; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) kv4_mask_value<HD, TS>(keys[i] + 4 * g + c, i, c, most, v, bad);
}
// Scores of keys that a row does not see become -inf; the values too are masked, if the wave holds them.
template <int HD, int RT, int TS>
PE_DEV void kv4_mask_scores(const int* keys, int g, const Kv4State<HD, RT>& st, f4v (&s)[RT][TS], int most = 0,
                            Kv4Raw<HD, TS>* v = nullptr, uint32_t* bad = nullptr) {
#pragma unroll
    for (int i = 0; i < TS; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int key = keys[i] + 4 * g + c;
#pragma unroll
            for (int t = 0; t < RT; ++t)
                if (key >= st.lim[t]) s[t][i][c] = -INFINITY;
            if (v) kv4_mask_value<HD, TS>(key, i, c, most, *v, bad);
        }
}

// NaN into the channels of the runs whose values are no numbers, of the rows that see them: counted by a product of both.
template <int HD, int RT, int TS>
PE_DEV void kv4_no_numbers(const int* keys, int g, const uint32_t* bad, Kv4State<HD, RT>& st) {
#pragma unroll
    for (int h = 0; h < TS / 2; ++h) {
        if (!__ballot(bad[h] != 0)) continue;
        uint32_t w[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
            w[c] = (bad[h] >> (2 * c) & 1 ? 0x3F80u : 0u) | (bad[h] >> (2 * c + 1) & 1 ? 0x3F800000u : 0u);
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            uint32_t sees[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int key = keys[2 * h + (c >> 1)] + 4 * g + 2 * (c & 1);
                sees[c] = (key < st.lim[t] ? 0x3F80u : 0u) | (key + 1 < st.lim[t] ? 0x3F800000u : 0u);
            }
            f4v count = {};
            count = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(w), operand(sees), count, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (count[i] > 0.f)
#pragma unroll
                    for (int j = 0; j < HD / 16; ++j) st.o[t][j][i] = __uint_as_float(0x7FC00000u);
        }
    }
}

// How far above the number that exponents are taken from a score may lie before the state is rescaled (base 2):
// probabilities up to 2^6 cost no accuracy, and after a sequence's first keys hardly a step rescales.
constexpr float kKv4Slack = 6.f;

template <int HD, int RT, int NP, int TS>
PE_DEV void kv4_softmax(Kv4State<HD, RT>& st, const f4v (&s)[RT][TS], uint32_t (&pr)[RT][TS / 2][NP][4]) {
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < TS; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) top = fmaxf(top, s[t][i][c]);
        top *= st.scale[t];
        if (__ballot(top > st.m[t] + kKv4Slack)) {
            const float m = fmaxf(st.m[t], swap32_max(swap16_max(top)));
            const float shrink = __builtin_amdgcn_exp2f(st.m[t] - (m == -INFINITY ? 0.f : m));
            st.m[t] = m;
            st.l[t] *= shrink;
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) st.o[t][j] *= shrink;
        }
        const float base = st.m[t] == -INFINITY ? 0.f : -st.m[t];
#pragma unroll
        for (int i = 0; i < TS; ++i) {
            float e[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                e[c] = __builtin_amdgcn_exp2f(fmaf(s[t][i][c], st.scale[t], base));
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
}

// The scales of the lane's 8 keys of tiles i and i + 1; the conversion looks at the exponent's bits alone.
template <int HD, int TS>
PE_DEV void kv4_value_scales(const Kv4Raw<HD, TS>& r, int i, float (&scale)[8]) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        const uint32_t w = r.s[i + (c >> 2)];
        scale[c] = __uint_as_float((c & 3) < 3 ? w << (23 - 8 * (c & 3)) : w >> 1);
    }
}

// The operands of channels j and j + 1 of the lane's run (j even), for the 32 keys of tiles i and i + 1: a conversion
// gives two channels of one key, a permutation two keys of one channel.
template <int HD, int TS>
PE_DEV void kv4_value_operands(const Kv4Raw<HD, TS>& r, int i, int j, const float* scale, uint32_t (&lo)[4], uint32_t (&hi)[4]) {
    uint32_t two[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        const int k = c & 3, at = i + (c >> 2);
        two[c] = HD == 128 ? two_codes(r.c[at][k], scale[c], j >> 1) : two_codes(r.c[at][k >> 1], scale[c], (k & 1) * 2 + (j >> 1));
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        lo[c] = __builtin_amdgcn_perm(two[2 * c + 1], two[2 * c], 0x05040100u);
        hi[c] = __builtin_amdgcn_perm(two[2 * c + 1], two[2 * c], 0x07060302u);
    }
}

// O^T += V^T P^T, 32 keys at a time, two channels of a run at a time.
template <int HD, int NP, int TS>
PE_DEV void kv4_values(const Kv4Raw<HD, TS>& r, Kv4State<HD, 1>& st, const uint32_t (&pr)[1][TS / 2][NP][4]) {
#pragma unroll
    for (int h = 0; h < TS / 2; ++h) {
        float scale[8];
        kv4_value_scales<HD, TS>(r, 2 * h, scale);
#pragma unroll
        for (int j = 0; j < HD / 16; j += 2) {
            uint32_t lo[4], hi[4];
            kv4_value_operands<HD, TS>(r, 2 * h, j, scale, lo, hi);
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                st.o[0][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(lo), operand(pr[0][h][n]), st.o[0][j], 0, 0, 0);
                st.o[0][j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(operand(hi), operand(pr[0][h][n]), st.o[0][j + 1], 0, 0, 0);
            }
        }
    }
}

template <typename T>
constexpr int kKv4Parts = sizeof(T) == 2 ? 2 : 3;

// A lane's HD / 4 elements of query row `row` (of the sequence's rows times heads) as operands: to(j, z) gets the NP
// parts z[four words][NP] of the j-th 32 channels; zeros where the row is not there. Returns the factor of the row's scores.
//
// An fp32 row times its scale is moved by a power of two 2^e, which its scores get back: its largest element then lies in
// [2^-9, 2^-8), so that no sum of products with keys (under 2^127.6 each) leaves fp32 and the parts of elements down to
// 2^-94 of the largest are normal numbers, wherever queries, scale and keys lie. Up to e = 64: what falls under fp32's
// normal numbers is then less than 2^-55 of a score, and beyond it the scores themselves leave 2^64 of room.
template <typename T, int HD, int NP, typename F>
PE_DEV float kv4_query(const Kv4AttnArgs& p, const Kv4Seq& seq, int kvh, int row, int last, int g, const F& to) {
    const bool there = row < seq.rows;
    row = there ? row : last;
    const int i = row / p.group;
    const T* x = static_cast<const T*>(p.q) + (seq.lo + i) * p.q_token + (int64_t)(kvh * p.group + row - i * p.group) * p.q_head +
                 g * (HD / 4);
    float q[HD / 4];
    if (p.vec) {
        typedef T piece __attribute__((ext_vector_type(16 / sizeof(T))));
#pragma unroll
        for (int j = 0; j < HD / 4; j += 16 / (int)sizeof(T)) {
            const piece z = *reinterpret_cast<const piece*>(x + j);
#pragma unroll
            for (int c = 0; c < 16 / (int)sizeof(T); ++c) q[j + c] = (float)z[c];
        }
    } else {
#pragma unroll
        for (int j = 0; j < HD / 4; ++j) q[j] = (float)x[j];
    }
    double q_scale = p.q_scale;
    float scale = p.scale;
    if constexpr (sizeof(T) == 4) {
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < HD / 4; ++j) top = fmaxf(top, fabsf(q[j]));
        top = swap32_max(swap16_max(top));
        int e = __builtin_amdgcn_frexp_exp(top * q_scale) + 8;  // (0, infinite, no number: 8)
        e = e < -126 ? -126 : e <= 64 ? e : e <= 64 + 8 + 126 ? 64 : e <= 126 + 8 + 126 ? e - 8 - 126 : 126;
        q_scale = __builtin_amdgcn_ldexp(q_scale, -e);
        scale = __uint_as_float((uint32_t)(e + 127) << 23);
    }
#pragma unroll
    for (int j = 0; j < HD / 32; ++j) {
        uint32_t z[4][NP];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float a = (float)(q[8 * j + 2 * c] * q_scale), b = (float)(q[8 * j + 2 * c + 1] * q_scale);
            split_pair<NP>(there ? a : 0.f, there ? b : 0.f, z[c]);
        }
        to(j, z);
    }
    return scale;
}

template <int TS>
PE_DEV void kv4_begin(const Kv4AttnArgs& p, Kv4Walk<TS>& w, int first, int end, int stride) {
    w.next = first;
    w.end = end;
    w.cols = stride / p.tiles;
    w.tiles = stride - w.cols * p.tiles;
    w.col = first / kKv4Tile / p.tiles;
    w.tile = first / kKv4Tile - w.col * p.tiles;
}

// Records of a kv head (as in kv4_find).
template <int RB>
PE_DEV int64_t kv4_room(const Kv4AttnArgs& p) {
    return RB > 16 ? p.records : p.items;
}

PE_DEV void kv4_tell(const Kv4AttnArgs& p, const Kv4Item& w, int kvh) {
    if (w.chunk == 0 && w.block == 0 && kvh == 0 && threadIdx.x == 0 && p.plan)
        p.plan[w.b] = make_int4(w.record, w.chunks, w.blocks, 0);
}

// Few rows (one new token, drafted ones, up to short pieces of prompts): 16 rows a workgroup, its waves take steps of 32
// keys in turn, each with a state of its own, and are merged in LDS. What bounds it: memory once the caches are long (64 x
// 16384 keys of 8 heads of 128, fp16: 127 us a call, 4.6 TB/s, and 136 to 145 replayed back to back, when the clock is lower;
// with the join), else the start's chain of loads (lengths, queries, table, keys), about 4 us of a workgroup's time (28 heads of
// 128 on 33 x 4001 keys, fp32: 21 to 22 us with the join, 8.0 at the copy rate). Four waves a SIMD, 128 registers each, are what
// keeps enough keys under way: with the queries in registers and steps of 64 keys, two waves, 145 us where this was 135; with a
// second step in registers 150.
template <typename T, int HD>
__global__ __launch_bounds__(64 * kKv4Waves, 4) void k_kv4_attn(Kv4AttnArgs p) {
    constexpr int NP = kKv4Parts<T>, E = HD / 16, R = 16, TS = 2;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.y;
    Kv4Item w;
    if (!kv4_find<R>(p, blockIdx.x, w)) return;
    const Kv4Seq& seq = w.seq;
    kv4_tell(p, w, kvh);
    const int r0 = w.block * R, last = (r0 + R < seq.rows ? r0 + R : seq.rows) - 1;
    const int least = kv4_keys(p, seq.keys, r0 / p.group), most = kv4_keys(p, seq.keys, last / p.group);
    const int64_t begin = (int64_t)w.chunk * w.span, stop = begin + w.span;
    constexpr int QUERIES = NP * (HD / 32) * 64, PART = kKv4Waves * R * (HD + 4 + 2) * 4;
    static_assert(PART >= QUERIES * 16, "queries lie in the merge's room");
    __shared__ __attribute__((aligned(16))) char lds[PART];
    __shared__ float scales[R];  // of fp32 rows' scores
    u4v* queries = reinterpret_cast<u4v*>(lds) + lane;
    if (wave == 0) {
        const float scale = kv4_query<T, HD, NP>(p, seq, kvh, r0 + n, last, g, [&](int j, const uint32_t (&z)[4][NP]) {
#pragma unroll
            for (int k = 0; k < NP; ++k) queries[(k * (HD / 32) + j) * 64] = u4v{z[0][k], z[1][k], z[2][k], z[3][k]};
        });
        if (sizeof(T) == 4 && g == 0) scales[n] = scale;
    }
    Kv4State<HD, 1> st;
    st.lim[0] = r0 + n < seq.rows ? kv4_keys(p, seq.keys, (r0 + n) / p.group) : 0;
    st.m[0] = -INFINITY;
    st.l[0] = 0.f;
#pragma unroll
    for (int j = 0; j < E; ++j) st.o[0][j] = f4v{};
    __syncthreads();
    st.scale[0] = sizeof(T) == 4 ? scales[n] : p.scale;
    Kv4Walk<TS> walk;
    kv4_begin(p, walk, (int)begin + wave * TS * kKv4Tile, (int)(stop < most ? stop : most), TS * kKv4Waves);
    if (walk.next < walk.end) {
        const int* table = p.table + w.b * p.table_row;
        const uint8_t* head = p.pages + (int64_t)kvh * p.tiles * (17 * HD);
        Kv4Raw<HD, TS> keys, values;
        kv4_pages<TS>(p, table, walk);
        kv4_advance<HD, TS>(p, table, head, walk);
        kv4_load_keys<HD, TS>(walk, lane, keys);
        kv4_load_values<HD, TS>(walk, lane, values);
        // the next step's keys are under way during softmax and values, its values during the next scores
        for (;;) {
            asm volatile("" ::: "memory");  // the queries stay in LDS: registers for more waves are worth more
            int at[TS];
            bool masked = false;
#pragma unroll
            for (int i = 0; i < TS; ++i) {
                at[i] = walk.key[i];
                masked |= at[i] + kKv4Tile > least;
            }
            const bool more = walk.next < walk.end;
            f4v s[1][TS];
            kv4_scores<HD, NP, TS>(keys, queries, s[0]);
            if (more) {
                kv4_advance<HD, TS>(p, table, head, walk);
                kv4_load_keys<HD, TS>(walk, lane, keys);
            }
            uint32_t bad[TS / 2] = {}, pr[1][TS / 2][NP][4];
            if (masked) kv4_mask_scores<HD, 1, TS>(at, g, st, s, most, &values, bad);
            kv4_softmax<HD, 1, NP, TS>(st, s, pr);
            kv4_values<HD, NP, TS>(values, st, pr);
            if (masked) kv4_no_numbers<HD, 1, TS>(at, g, bad, st);
            if (!more) break;
            kv4_load_values<HD, TS>(walk, lane, values);
        }
    }
    st.l[0] = swap32_sum(swap16_sum(st.l[0]));

    const int64_t rec = (kvh * kv4_room<R>(p) + w.record + (int64_t)w.block * w.chunks + w.chunk) * p.rec_rows;  // (if cut)
    float(*part)[R][HD + 4] = reinterpret_cast<float(*)[R][HD + 4]>(lds);
    float(*pm)[R] = reinterpret_cast<float(*)[R]>(lds + kKv4Waves * R * (HD + 4) * 4), (*pl)[R] = pm + kKv4Waves;
    __syncthreads();  // the queries have been read
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < E; ++j) part[wave][n][(4 * g + i) * E + j] = st.o[0][j][i];
    if (g == 0) pm[wave][n] = st.m[0], pl[wave][n] = st.l[0];
    __syncthreads();
    const int row = threadIdx.x / 16, c = threadIdx.x % 16 * E, r = r0 + row;
    if (r >= seq.rows) return;
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

// Many rows (pieces of prompts): 32 rows a wave, 128 a workgroup, all on the same keys. The waves convert a step's codes
// for one another, into LDS in the order of the products' operands, two steps deep; the queries are in registers. Bound by
// the matrix cores and the vector instructions, which add up with two waves a SIMD (2 x 1021 rows of 28 heads of 128
// on 8000 keys, fp16: 45 % and 54 % of the cycles, 290 to 365 us by the card's clock, the join of the chunks 30; the two parts of
// each factor alone are 265 at the rate of a large product). With every wave converting for itself 367 and, fp32, 588 us; so 360 and 493.
template <typename T, int HD>
constexpr int kKv4RowTiles = sizeof(T) == 4 && HD == 128 ? 2 : 4;  // 16 keys a step; fp32's queries take half the registers

template <typename T, int HD>
__global__ __launch_bounds__(64 * kKv4Waves, 2) void k_kv4_attn_rows(Kv4AttnArgs p) {
    constexpr int NP = kKv4Parts<T>, E = HD / 16, RT = 2, R = 16 * RT, RB = R * kKv4Waves, TS = kKv4RowTiles<T, HD>, N = HD / 32;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.y;
    Kv4Item w;
    if (!kv4_find<RB>(p, blockIdx.x, w)) return;
    const Kv4Seq& seq = w.seq;
    kv4_tell(p, w, kvh);
    // the workgroup's rows, and the wave's (it has none: it converts alone)
    const int b0 = w.block * RB, b1 = (b0 + RB < seq.rows ? b0 + RB : seq.rows) - 1;
    const int least_all = kv4_keys(p, seq.keys, b0 / p.group), most_all = kv4_keys(p, seq.keys, b1 / p.group);
    const int r0 = b0 + wave * R, last = (r0 + R < seq.rows ? r0 + R : seq.rows) - 1;
    const bool rows = r0 < seq.rows;
    const int least = rows ? kv4_keys(p, seq.keys, r0 / p.group) : 0;
    const int64_t begin = (int64_t)w.chunk * w.span, stop = begin + w.span;
    const int end = (int)(stop < most_all ? stop : most_all);

    // Operands: keys [tile][32 channels][64 lanes], values [32 keys][channel of a run][64 lanes]. A wave converts a
    // quarter of each: KF of the keys' (of one tile), VF pairs of the values' (of 32 keys).
    constexpr int KF = TS * N / kKv4Waves, VF = TS / 2 * (E / 2) / kKv4Waves, PER = kKv4Waves / (TS / 2);
    __shared__ u4v k_ops[2][TS * N][64], v_ops[2][TS / 2 * E][64];
    __shared__ uint32_t no_number[2][TS / 2][64];
    __shared__ int first_key[2][TS];
    const int k_tile = wave * KF / N, k_part = wave * KF % N, v_half = wave / PER, v_pair = wave % PER * VF;

    Kv4State<HD, RT> st;
    uint32_t q[RT][NP][N][4] = {};
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        st.scale[t] = p.scale;
        if (rows)
            st.scale[t] = kv4_query<T, HD, NP>(p, seq, kvh, r0 + 16 * t + n, last, g, [&](int j, const uint32_t (&z)[4][NP]) {
#pragma unroll
                for (int k = 0; k < NP; ++k)
#pragma unroll
                    for (int c = 0; c < 4; ++c) q[t][k][j][c] = z[c][k];
            });
        const int row = r0 + 16 * t + n;
        st.lim[t] = row < seq.rows ? kv4_keys(p, seq.keys, row / p.group) : 0;
        st.m[t] = -INFINITY;
        st.l[t] = 0.f;
#pragma unroll
        for (int j = 0; j < E; ++j) st.o[t][j] = f4v{};
    }
    if (begin < end) {
        const int* table = p.table + w.b * p.table_row;
        const uint8_t* head = p.pages + (int64_t)kvh * p.tiles * (17 * HD);
        Kv4Walk<1> kw;
        Kv4Walk<2> vw;
        kv4_begin(p, kw, (int)begin + k_tile * kKv4Tile, end, TS);
        kv4_begin(p, vw, (int)begin + v_half * 2 * kKv4Tile, end, TS);
        kv4_pages<1>(p, table, kw);
        kv4_pages<2>(p, table, vw);
        Kv4Raw<HD, 1> keys;
        Kv4Raw<HD, 2> values;
        const auto load = [&] {
            kv4_advance<HD, 1>(p, table, head, kw);
            kv4_advance<HD, 2>(p, table, head, vw);
            kv4_load_keys<HD, 1>(kw, lane, keys);
            kv4_load_values<HD, 2>(vw, lane, values);
        };
        // a wave's pairs of channels are the lowest bytes of its words once they are shifted
        const auto mask = [&](int to) {
            uint32_t bad[1] = {0};
            if (vw.key[0] + kKv4Tile > least_all || vw.key[1] + kKv4Tile > least_all) kv4_mask_values<HD, 2>(vw.key, most_all, g, values, bad);
            no_number[to][v_half][lane] = bad[0];  // (several waves hold the same)
            first_key[to][k_tile] = kw.key[0];
        };
        const auto convert = [&](int to) {
            const float scale = __uint_as_float(keys.s[0] << 23);
#pragma unroll
            for (int f = 0; f < KF; ++f) {
                const uint32_t c = KF == N || k_part == 0 ? keys.c[0][f] : keys.c[0][f + N - KF];
                k_ops[to][k_tile * N + k_part + f][lane] = u4v{two_codes(c, scale, 0), two_codes(c, scale, 1), two_codes(c, scale, 2), two_codes(c, scale, 3)};
            }
            float scales[8];
            kv4_value_scales<HD, 2>(values, 0, scales);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < N; ++j) values.c[i][j] >>= 8 * v_pair;
#pragma unroll
            for (int f = 0; f < VF; ++f) {
                uint32_t lo[4], hi[4];
                kv4_value_operands<HD, 2>(values, 0, 2 * f, scales, lo, hi);
                v_ops[to][v_half * E + 2 * (v_pair + f)][lane] = u4v{lo[0], lo[1], lo[2], lo[3]};
                v_ops[to][v_half * E + 2 * (v_pair + f) + 1][lane] = u4v{hi[0], hi[1], hi[2], hi[3]};
            }
        };
        load();
        mask(0);
        convert(0);
        load();  // (past the end: keys that are not there, from the pool's first page)
        __syncthreads();
        int at = 0;
        for (int key = (int)begin; key < end; key += TS * kKv4Tile, at ^= 1) {
            int keys_at[TS];
            bool masked = false, masked_all = false;  // for the wave's rows, for the workgroup's (and in its conversions)
#pragma unroll
            for (int i = 0; i < TS; ++i) {
                keys_at[i] = __builtin_amdgcn_readfirstlane(first_key[at][i]);
                masked |= keys_at[i] + kKv4Tile > least;
                masked_all |= keys_at[i] + kKv4Tile > least_all;
            }
            f4v s[RT][TS];
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int i = 0; i < TS; ++i) s[t][i] = f4v{};
#pragma unroll
            for (int j = 0; j < N; ++j) {
                bf8v k[TS];
#pragma unroll
                for (int i = 0; i < TS; ++i) k[i] = __builtin_bit_cast(bf8v, k_ops[at][i * N + j][lane]);
#pragma unroll
                for (int c = 0; c < NP; ++c)
#pragma unroll
                    for (int t = 0; t < RT; ++t)
#pragma unroll
                        for (int i = 0; i < TS; ++i) s[t][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[i], operand(q[t][c][j]), s[t][i], 0, 0, 0);
            }
            if (masked) kv4_mask_scores<HD, RT, TS>(keys_at, g, st, s);
            mask(at ^ 1);
            uint32_t pr[RT][TS / 2][NP][4];
            kv4_softmax<HD, RT, NP, TS>(st, s, pr);
            // the next step's conversions beside this one's second product
            convert(at ^ 1);
#pragma unroll
            for (int h = 0; h < TS / 2; ++h)
#pragma unroll
                for (int j = 0; j < E; j += 2) {
                    const bf8v v0 = __builtin_bit_cast(bf8v, v_ops[at][h * E + j][lane]), v1 = __builtin_bit_cast(bf8v, v_ops[at][h * E + j + 1][lane]);
#pragma unroll
                    for (int c = 0; c < NP; ++c)
#pragma unroll
                        for (int t = 0; t < RT; ++t) {
                            st.o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, operand(pr[t][h][c]), st.o[t][j], 0, 0, 0);
                            st.o[t][j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, operand(pr[t][h][c]), st.o[t][j + 1], 0, 0, 0);
                        }
                }
            if (masked_all) {
                uint32_t bad[TS / 2];
#pragma unroll
                for (int h = 0; h < TS / 2; ++h) bad[h] = no_number[at][h][lane];
                kv4_no_numbers<HD, RT, TS>(keys_at, g, bad, st);
            }
            load();
            __syncthreads();  // the next step's operands are there, this one's have been read
        }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t) st.l[t] = swap32_sum(swap16_sum(st.l[t]));
    const int64_t rec = (kvh * kv4_room<RB>(p) + w.record + (int64_t)w.block * w.chunks + w.chunk) * p.rec_rows;  // (if cut)
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

// The chunks of a row of q, joined by WAVES waves: HD / 4 lanes take a chunk's record, so a wave has 256 / HD of them
// in flight beside each other, with the row's maximum known before the first.
template <typename T, int HD, int RB, int WAVES>
__global__ __launch_bounds__(256) void k_kv4_merge(Kv4AttnArgs p) {
    constexpr int L = HD / 4, SIDE = WAVES * 64 / L;
    __shared__ float4 part[4][64];
    __shared__ float parts[4][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, w = wave % WAVES;
    const int64_t x = (int64_t)blockIdx.x * (4 / WAVES) + wave / WAVES, t = x / p.n_head;
    const int h = (int)(x - t * p.n_head);
    int chunks = 0, r = 0;
    int64_t first = 0;
    if (t < p.tokens) {
        int64_t b, lo = t;
        int4 plan;
        if (p.starts && p.batch < kWave) {  // few sequences: all of them at once (2 x 1021 rows: 32.3 -> 29.9 us, 5 rows 5.4 -> 5.2)
            const int64_t start = lane <= p.batch ? int_at(p.starts, p.starts_wide, lane) : 0;
            const int4 all = p.plan[lane < p.batch ? lane : 0];
            b = __popcll(__ballot(lane <= p.batch && start <= t)) - 1;
            b = b < p.batch ? b : -1;
            const int at = b < 0 ? 0 : (int)b;
            lo = lane_of(start, at);
            plan = make_int4(__builtin_amdgcn_readlane(all.x, at), __builtin_amdgcn_readlane(all.y, at),
                             __builtin_amdgcn_readlane(all.z, at), 0);
        } else {
            b = sequence_of(p.starts, p.starts_wide, p.batch, t);
            plan = p.plan[b < 0 ? 0 : b];
            if (p.starts) lo = uniform(int_at(p.starts, p.starts_wide, b < 0 ? 0 : b));
        }
        lo = lo < 0 ? 0 : lo;
        if (b >= 0) {
            const int kvh = h / p.group;
            r = (int)(t - lo) * p.group + h - kvh * p.group;
            // (a plan that no workgroup wrote, of starts that are out of order, holds anything)
            if (plan.y > 1 && plan.z > 0 && plan.x >= 0 && r >= 0 && r / RB < plan.z && (int64_t)plan.x + (int64_t)plan.y * plan.z <= kv4_room<RB>(p)) {
                chunks = plan.y;
                first = (kvh * kv4_room<RB>(p) + plan.x + (int64_t)(r / RB) * plan.y) * p.rec_rows + r % RB;
            }
        }
    }
    float m = -INFINITY;
    for (int c = lane; c < chunks; c += 64) m = fmaxf(m, p.stat[2 * (first + (int64_t)c * p.rec_rows)]);
    m = wave_max<64>(m);
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f, o[4] = {};
    const int ch = lane % L * 4;
#pragma unroll 4
    for (int c = w * (64 / L) + lane / L; c < chunks; c += SIDE) {
        const int64_t rec = first + (int64_t)c * p.rec_rows;
        const float f = __builtin_amdgcn_exp2f(p.stat[2 * rec] - base);
        const float4 v = *reinterpret_cast<const float4*>(p.record + rec * HD + ch);
        l = fmaf(p.stat[2 * rec + 1], f, l);
        o[0] = fmaf(v.x, f, o[0]), o[1] = fmaf(v.y, f, o[1]), o[2] = fmaf(v.z, f, o[2]), o[3] = fmaf(v.w, f, o[3]);
    }
    const auto join = [&](float v) {
        if constexpr (L == 16) v = swap16_sum(v);
        return swap32_sum(v);
    };
    l = join(l);
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = join(o[j]);
    if constexpr (WAVES > 1) {
        part[wave][lane] = make_float4(o[0], o[1], o[2], o[3]);
        parts[wave][lane] = l;
        __syncthreads();
        if (w) return;
#pragma unroll
        for (int k = 1; k < WAVES; ++k) {
            const float4 v = part[wave + k][lane];
            o[0] += v.x, o[1] += v.y, o[2] += v.z, o[3] += v.w;
            l += parts[wave + k][lane];
        }
    }
    if (chunks == 0 || lane >= L) return;
    const float f = l == 0.f ? 0.f : 1.f / l;
    T* y = static_cast<T*>(p.out) + t * p.out_token + (int64_t)h * p.out_head + ch;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = (T)(o[j] * f);
}

// How a call is cut: rows of a workgroup and workgroups of a kv head, from what the host knows (the lengths are on the device).
struct Kv4Plan {
    int rt, split;   // 16-row tiles of a wave; the waves share the rows and split the keys
    int rb;          // rows of a workgroup
    int64_t blocks, items, records;  // (of a kv head)
    int min_chunk, rec_rows;
    float weight;  // of all keys in the square of a chunk's length
};

static Kv4Plan kv4_plan(int64_t tokens, int64_t batch, bool ragged, int n_head, int n_kv, int hd, int64_t capacity, bool half) {
    Kv4Plan s;
    const int group = n_head / n_kv;
    const int64_t rows = ragged ? (tokens + batch - 1) / batch * group : group;  // of a sequence, on average
    // Up to 512 rows in blocks of 16 (one sequence with 16000 keys, heads of 128, fp16, of 64 fp32; us in blocks of 16 | of
    // 128: 160 rows 47 | 70, 280 24 | 33; 320 73 | 85, 560 36 | 42; 600 122 | 115, 1050 55 | 64; 2400 384 | 318, 4200 158 | 145).
    s.split = rows <= 512;
    s.rt = s.split ? 1 : 2;
    s.rb = 16 * s.rt * (s.split ? 1 : kKv4Waves);
    s.blocks = ragged ? tokens * group / s.rb + batch : batch * ((group + s.rb - 1) / s.rb);
    s.min_chunk = 64 * (s.split ? kKv4Waves : 4);
    s.rec_rows = ragged || group > s.rb ? s.rb : group;
    s.weight = (s.split && !half && hd == 128 ? 0.5f : 0.75f) * (float)n_kv;
    // the most workgroups that a chunk's length makes of any lengths, within reason
    const int64_t chunks = (capacity + s.min_chunk - 1) / s.min_chunk;
    int64_t extra = (int64_t)sqrt((double)s.blocks * (double)capacity / s.weight) + 1;
    if (extra > 8192 / n_kv + 1) extra = 8192 / n_kv + 1;
    // up to four chunks (of heads of 64; three of 128) one workgroup takes them all: the second launch costs as much (14 heads, 500
    // keys: 7.6 us in one launch, 9.9 in two; 1000 keys 10.6 and 10.3, of 28 heads of 128 13.2 and 11.6)
    if (chunks <= (!s.split ? 1 : hd == 64 ? 4 : 3))
        extra = 0;
    else if (extra > s.blocks * (chunks - 1))
        extra = s.blocks * (chunks - 1);
    s.items = s.blocks + extra;
    // A record for every workgroup, in blocks of 128 rows for those of cut sequences alone: their chunks are two a row block at
    // least, so no more than twice those beyond the first of each row block; of these there are `extra`, and one a sequence where
    // the count of blocks above is over (65536 rows of 32 heads on 8 of 128 behind as many keys: 1.1 GB instead of 1.6; 2^20 rows
    // of 16 sequences 1.1 instead of 18). Rows of no sequence make that count larger still; the device then takes longer chunks.
    s.records = extra == 0 ? 0 : s.items;
    if (!s.split && extra + (ragged ? batch : 0) < s.records / 2) s.records = 2 * (extra + (ragged ? batch : 0));
    return s;
}

static bool kv4_shape_ok(int64_t tokens, int64_t batch, bool ragged, int n_head, int n_kv, int hd, int64_t capacity) {
    return tokens >= 0 && tokens <= (1 << 22) && batch > 0 && batch <= (1 << 20) && (ragged || tokens == batch) && n_head > 0 &&
           n_head <= 4096 && n_kv > 0 && n_head % n_kv == 0 && (hd == 64 || hd == 128) && capacity >= 0 && capacity <= (1LL << 30) &&
           tokens * (n_head / n_kv) < (1LL << 30);
}

static int64_t kv4_bytes(const Kv4Plan& s, int64_t batch, int n_kv, int hd) {
    return s.records ? (batch * 16 + s.records * n_kv * s.rec_rows * (int64_t)(hd + 2) * 4 + 15) / 16 * 16 : 0;
}

template <typename T, int HD, int RB>
static void launch_merge(const Kv4AttnArgs& p, hipStream_t st) {
    const int64_t rows = p.tokens * p.n_head;
    if (!p.plan) return;
    if (rows < 2048)  // few rows: four waves each
        hipLaunchKernelGGL((k_kv4_merge<T, HD, RB, 4>), dim3((unsigned)rows), dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL((k_kv4_merge<T, HD, RB, 1>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, p);
}

template <typename T, int HD>
static void launch_kv4(const Kv4AttnArgs& p, const Kv4Plan& s, hipStream_t st) {
    const dim3 g((unsigned)(s.items + 7) / 8 * 8, (unsigned)p.n_kv);
    if (!s.split) {
        hipLaunchKernelGGL((k_kv4_attn_rows<T, HD>), g, dim3(64 * kKv4Waves), 0, st, p);
        launch_merge<T, HD, 32 * kKv4Waves>(p, st);
    } else {
        hipLaunchKernelGGL((k_kv4_attn<T, HD>), g, dim3(64 * kKv4Waves), 0, st, p);
        launch_merge<T, HD, 16>(p, st);
    }
}

}  // namespace pe

using namespace pe;

extern "C" int64_t pe_kv4_attn_workspace_bytes(int64_t tokens, int64_t batch, int ragged, int n_head, int n_kv, int head_dim,
                                               int64_t capacity) {
    if (!kv4_shape_ok(tokens, batch, ragged, n_head, n_kv, head_dim, capacity)) return -PE_ERR_SHAPE;
    return kv4_bytes(kv4_plan(tokens, batch, ragged, n_head, n_kv, head_dim, capacity, false), batch, n_kv, head_dim);
}

extern "C" int pe_kv4_attn(const pe_kv4_attn_args* a, pe_stream_t stream) {
    if (!a) return PE_ERR_NULL;
    if ((a->type != PE_TYPE_F32 && a->type != PE_TYPE_F16) || (a->lengths_dtype != 1 && a->lengths_dtype != 2) ||
        (a->starts && a->starts_dtype != 1 && a->starts_dtype != 2))
        return PE_ERR_TYPE;
    if (a->tokens == 0 || a->batch == 0) return PE_OK;
    if (const int st = kv4_pool_ok(&a->pool, a->n_kv, a->head_dim)) return st;
    const int64_t T = a->tokens, capacity = a->pool.table_cols * a->pool.page_tokens;
    const bool ragged = a->starts != nullptr, half = a->type == PE_TYPE_F16;
    if (!kv4_shape_ok(T, a->batch, ragged, a->n_head, a->n_kv, a->head_dim, capacity) || !std::isfinite(a->scale * kKv4Log2e) ||
        a->first < -(1LL << 40) || a->first > (1LL << 40) || a->q_token < 0 || a->q_head < 0 || a->out_token < 0 || a->out_head < 0 ||
        (a->n_head > 1 && a->out_head < a->head_dim) || (T > 1 && a->out_token < a->head_dim) ||
        (T > 1 && a->n_head > 1 && a->out_token < a->out_head * (a->n_head - 1) + a->head_dim &&
         a->out_head < a->out_token * (T - 1) + a->head_dim))
        return PE_ERR_SHAPE;
    const Kv4Plan s = kv4_plan(T, a->batch, ragged, a->n_head, a->n_kv, a->head_dim, capacity, half);
    const int64_t need = kv4_bytes(s, a->batch, a->n_kv, a->head_dim);
    if (!a->q || !a->out || !a->lengths || (need && !a->workspace)) return PE_ERR_NULL;
    const size_t e = a->type == PE_TYPE_F16 ? 2 : 4;
    if (!aligned(a->q, e) || !aligned(a->out, e) || !aligned(a->lengths, a->lengths_dtype == 2 ? 8 : 4) ||
        (ragged && !aligned(a->starts, a->starts_dtype == 2 ? 8 : 4)) || !aligned(a->workspace, 16))
        return PE_ERR_ALIGN;
    if (a->workspace_bytes < need) return PE_ERR_SPACE;
    if ((s.items + 7) * a->n_kv >= (1 << 24) || T * a->n_head > (1LL << 26) - 4) return PE_ERR_SHAPE;  // a grid holds 2^32 threads
    const int piece = (int)(16 / e);
    const int vec = (a->q_token | a->q_head) % piece == 0 && aligned(a->q, 16);
    // fp32 queries are scaled in 64 bits before they are split, so that no rounding of the scale is left in the scores (what
    // power of two the scores get back is the row's own); fp16 ones only turned by its sign, so that their parts stay exact
    //
    // fp16 queries (2^-24 to 2^16, in parts down to 2^-24) go 2^24 down, where no sum of products with keys leaves fp32, and
    // their scores back up. Not with scales from 2^64 on: what falls under 2^-126 would show there (below, less than 2^-31 of
    // a score does), and sums that are too large are scores that are.
    const float up = half && std::fabs(a->scale) < 0x1p64f ? 0x1p24f : 1.f;
    const float scale = half && a->scale != 0 ? std::fabs(a->scale) * up * kKv4Log2e : 1.f;
    const double q_scale = half ? ((a->scale > 0) - (a->scale < 0)) / up : (double)a->scale * 1.4426950408889634;
    const float round = (s.split ? 4 : 2) * 256.f / (float)a->n_kv;
    int4* plan = need ? static_cast<int4*>(a->workspace) : nullptr;
    float* record = need ? reinterpret_cast<float*>(plan + a->batch) : nullptr;
    Kv4AttnArgs p{a->q, a->q_token, a->q_head, a->out, a->out_token, a->out_head, static_cast<const uint8_t*>(a->pool.pages),
                  a->pool.page_stride, (int)a->pool.n_pages, (int)(a->pool.page_tokens / kKv4Tile), a->pool.table,
                  a->pool.table_stride, (int)a->pool.table_cols, a->lengths, a->lengths_dtype == 2, a->first, a->starts,
                  a->starts_dtype == 2, T, (int)a->batch, a->n_head, a->n_kv, a->n_head / a->n_kv, scale, q_scale, capacity, vec,
                  (int)s.items, (int)s.blocks, (int)s.records, s.min_chunk, s.weight, s.rec_rows, round, plan, record,
                  need ? record + s.records * a->n_kv * s.rec_rows * a->head_dim : nullptr};
    hipStream_t st = (hipStream_t)stream;
    if (a->type == PE_TYPE_F16)
        a->head_dim == 64 ? launch_kv4<_Float16, 64>(p, s, st) : launch_kv4<_Float16, 128>(p, s, st);
    else
        a->head_dim == 64 ? launch_kv4<float, 64>(p, s, st) : launch_kv4<float, 128>(p, s, st);
    return launch_status();
}
