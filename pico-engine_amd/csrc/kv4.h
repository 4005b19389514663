// The paged 4-bit cache: where a token's codes and scales lie in a page, how 32 elements become codes.
//
// 32 neighbouring elements of a head share the scale 2^e, stored as the byte e + 127; a code is a sign (8)
// and one of eight magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6 (the block format of 32 four-bit floats that the
// matrix hardware converts by itself). e is the least in [-100, 125] that leaves the largest magnitude at
// 7 2^e or less: what lies in (6, 7] loses less as 6 than the other 31 elements would at twice the step
// (normal values keep 19.0 dB; 18.8 with scales that cut at 6 or at 8). Scales from 2^-100 up keep every value a normal bf16 number.
//
// A page holds whole tiles of 16 tokens for every kv head, so a tile's bytes lie together: 17 hd of them.
//   keys    [16 tokens][hd / 2]               a token's row of codes: a lane of the score product takes
//                                             16 (8) bytes of it, 16 tokens and 4 lane groups are one span
//   values  [4 groups][16 runs][4 tokens][hd / 32]   a run: hd / 16 elements of one token. A lane of the value
//                                             product takes 4 tokens of one run, 16 (8) bytes
//   key scales [16 tokens][hd / 32], value scales [4 groups][hd / 32][4 tokens]
#pragma once

#include "pe_common.h"

namespace pe {

constexpr int kKv4Tile = 16;   // tokens
constexpr int kKv4MinExp = -100, kKv4MaxExp = 125;

PE_DEV int64_t int_at(const void* p, int wide, int64_t i) {
    return wide ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int*>(p)[i];
}

// A value that all lanes hold, in scalar registers: what follows from it is then computed once a wave.
PE_DEV int64_t uniform(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// The value that lane `at` holds.
PE_DEV int64_t lane_of(int64_t v, int at) {
    const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, at), hi = __builtin_amdgcn_readlane((uint32_t)((uint64_t)v >> 32), at);
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// Rows [lo, hi) of sequence b: one each where starts is NULL; clamped to the rows there are.
PE_DEV void rows_of(const void* starts, int wide, int64_t b, int64_t tokens, int64_t& lo, int64_t& hi) {
    if (!starts) {
        lo = b;
        hi = b + 1;
        return;
    }
    lo = int_at(starts, wide, b);
    hi = int_at(starts, wide, b + 1);
    lo = lo < 0 ? 0 : lo > tokens ? tokens : lo;
    hi = hi < lo ? lo : hi > tokens ? tokens : hi;
}

// The sequence that row t belongs to, or -1: the last b with starts[b] <= t, if t lies before starts[b + 1]. All lanes of a
// wave look for the same row, 64 places at a time.
PE_DEV int64_t sequence_of(const void* starts, int wide, int64_t batch, int64_t t) {
    if (!starts) return t < batch ? t : -1;
    int64_t lo = 0, n = batch + 1;  // the first of starts that is beyond t lies in [lo, lo + n]
    while (n > 0) {
        const int64_t step = (n + 63) >> 6, at = (int64_t)(threadIdx.x & 63) * step;
        const int below = __popcll(__ballot(at < n && int_at(starts, wide, lo + (at < n ? at : 0)) <= t));
        if (below == 0) break;
        lo += (below - 1) * step + 1;
        n -= (below - 1) * step + 1;
        if (n > step - 1) n = step - 1;
    }
    return lo >= 1 && lo <= batch ? lo - 1 : -1;
}

// The pool and table that the entry points share: PE_OK or what is wrong with them.
inline int kv4_pool_ok(const pe_kv4_pool* c, int n_kv, int head_dim) {
    if (c->n_pages <= 0 || c->n_pages > 0x7FFFFFFF || c->page_tokens <= 0 || c->page_tokens % kKv4Tile ||
        c->page_tokens > (1 << 20) || c->table_cols < 0 || c->table_cols > (1 << 26) ||
        c->table_cols * c->page_tokens > (1LL << 30) || c->table_stride < 0 || n_kv <= 0 || n_kv > 4096 ||
        (head_dim != 64 && head_dim != 128) ||
        c->page_stride < (int64_t)n_kv * (c->page_tokens / kKv4Tile) * 17 * head_dim)
        return PE_ERR_SHAPE;
    if (!c->pages || (c->table_cols && !c->table)) return PE_ERR_NULL;
    if (!aligned(c->pages, 16) || c->page_stride % 16 || !aligned(c->table, 4)) return PE_ERR_ALIGN;
    return PE_OK;
}

}  // namespace pe
