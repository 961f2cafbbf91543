// Indexing of the paged K/V cache: the descriptors as the kernels get them, page layouts, and the reading
// of a batch with every number checked against the sizes.  Plain C++, so that it also compiles for
// the host.
#pragma once

#include <cstddef>
#include <cstdint>

#include "../../include/ronn_bitnet_hip.h"

#ifdef __HIPCC__
#include <hip/hip_fp16.h>
#define KV_FN __host__ __device__ __forceinline__
typedef __half KvHalf;
#else
#define KV_FN static inline
typedef uint16_t KvHalf;
#endif

constexpr int kKvBlock = RBN_KV_BLOCK;

struct KvTableArgs {
    int rows, max_blocks, pages;
    int32_t *table;
    const int32_t *len;
    int32_t *ring;
    const int32_t *ring_state;
};
struct KvBatchArgs {
    int max_tokens;
    int32_t *start, *row, *pos, *slot, *unit, *count;
};
struct KvLayerArgs {
    int kv_heads;
    uint8_t *k, *v;
    float *k_scale, *v_scale;
    KvHalf *k_open, *v_open;
};

// Byte of code (t, d) inside a page head, as the matrix instructions read them.
template <int HD>
KV_FN int kv_k_byte(int t, int d) {
    return (((t >> 4) * (HD / 64) + (d >> 6)) * 64 + ((d & 31) >> 3) * 16 + (t & 15)) * 16 + ((d >> 5) & 1) * 8 + (d & 7);
}
template <int HD>
KV_FN int kv_v_byte(int t, int d) {
    return ((d >> 5) * 64 + ((t & 15) >> 2) * 16 + (d & 15)) * 16 + ((d >> 4) & 1) * 8 + (t >> 4) * 4 + (t & 3);
}

// What a workgroup needs to know of unit u of a batch.
struct KvUnit {
    int row, first;  // first: the unit's first token
    int n;           // tokens of the unit; 0 if there is nothing (sound) to do
    int pos;         // position of its first token
    int row_first;   // the row's first token of the call
    int row_pos;     // ... and its position
    int row_n;       // tokens of the row in the call
};

// The unit whose first token is `i`, from what the batch says of that token (row, pos) and of its row (its first
// token and the first of the next row); .n = 0 if that does not fit the table and the batch's own sizes.
KV_FN KvUnit kv_make_unit(const KvTableArgs &t, int tokens, int i, int row, int pos, int row_first, int row_end) {
    KvUnit r;
    const int cap = t.max_blocks * kKvBlock;
    r.n = 0;
    r.first = i;
    r.row = row;
    r.pos = pos;
    r.row_first = row_first;
    if (i < 0 || i >= tokens || row < 0 || row >= t.rows || pos < 0 || pos >= cap) return r;
    if (row_first < 0 || row_first > i || row_end <= i || row_end > tokens) return r;
    r.row_n = row_end - row_first;
    r.row_pos = pos - (i - row_first);
    if (r.row_pos < 0 || r.row_pos + r.row_n > cap) return r;
    const int left = kKvBlock - (pos & (kKvBlock - 1));
    r.n = row_end - i < left ? row_end - i : left;
    return r;
}

// Unit u of a batch (u below kv_max_units); *bad is set if there is one but what the batch says of it is not sound.
// The loads do not wait for the counts; ahead(i) is called while those of the unit's first token `i` (-1: not one of the
// batch's places) are on their way.
template <typename Ahead>
KV_FN KvUnit kv_resolve_unit(const KvTableArgs &t, const KvBatchArgs &b, int u, bool *bad, Ahead ahead) {
    const int i = b.unit[u];
    const int tokens = b.count[0] < b.max_tokens ? b.count[0] : b.max_tokens;
    const int units = b.count[1] < b.max_tokens ? b.count[1] : b.max_tokens;
    const bool token = i >= 0 && i < b.max_tokens;  // (behind the count anything may stand there)
    const int row = token ? b.row[i] : -1, pos = token ? b.pos[i] : -1;
    ahead(token ? i : -1);
    const bool known = row >= 0 && row < t.rows;
    KvUnit r = kv_make_unit(t, tokens, i, row, pos, known ? b.start[row] : -1, known ? b.start[row + 1] : -1);
    *bad = u < units && r.n == 0;
    r.n = u < units ? r.n : 0;
    return r;
}

// Units a batch can have at most: a unit is a (row, block) pair, so no more than the tokens, and a
// row's n tokens touch at most n / 32 + 2 blocks.
KV_FN int kv_max_units(int max_tokens, int rows) {
    const int by_rows = max_tokens / RBN_KV_BLOCK + 2 * rows;
    return max_tokens < by_rows ? max_tokens : by_rows;
}

// Page of a row's block (both in range), or -1.
KV_FN int kv_page(const KvTableArgs &t, int row, int block) {
    const int page = t.table[(size_t)row * t.max_blocks + block];
    return page >= 0 && page < t.pages ? page : -1;
}

// Page of a slot, or -1.
KV_FN int kv_slot_page(const KvTableArgs &t, int slot) {
    const int page = slot / kKvBlock;
    return slot >= 0 && page < t.pages ? page : -1;
}
