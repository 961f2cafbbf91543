// What the kernels of the paged 8-bit K/V cache share: the checks of their host side and what
// device code needs besides kv_index.h (formats and layouts: include/ronn_bitnet_hip.h).
#pragma once

#include "common.hpp"
#include "kv_index.h"
#include "wave_ops.hpp"

static inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static inline int kv_check_table(const rbn_kv_table *t, KvTableArgs *out, const char *what) {
    RBN_REQUIRE(t && t->d_table && t->d_len, "null pointer in the table of %s", what);
    RBN_REQUIRE(t->rows > 0 && t->rows <= RBN_KV_MAX_ROWS && t->max_blocks > 0 &&
                    t->max_blocks <= RBN_KV_MAX_BLOCKS && t->pages > 0 && t->pages < (1ull << 31) / RBN_KV_BLOCK,
                "bad sizes in the table of %s (rows %llu, max_blocks %llu, pages %llu)", what,
                (unsigned long long)t->rows, (unsigned long long)t->max_blocks, (unsigned long long)t->pages);
    *out = KvTableArgs{(int)t->rows, (int)t->max_blocks, (int)t->pages, t->d_table, t->d_len, t->d_ring,
                       t->d_ring_state};
    return RBN_OK;
}

static inline int kv_check_batch(const rbn_kv_batch *b, KvBatchArgs *out, const char *what) {
    RBN_REQUIRE(b && b->d_start && b->d_row && b->d_pos && b->d_slot && b->d_unit && b->d_count,
                "null pointer in the batch of %s", what);
    RBN_REQUIRE(b->max_tokens > 0 && b->max_tokens <= RBN_KV_MAX_TOKENS, "bad max_tokens in the batch of %s", what);
    *out = KvBatchArgs{(int)b->max_tokens, b->d_start, b->d_row, b->d_pos, b->d_slot, b->d_unit, b->d_count};
    return RBN_OK;
}

static inline int kv_check_layer(const rbn_kv_layer *l, KvLayerArgs *out, const char *what) {
    RBN_REQUIRE(l && l->d_k && l->d_v && l->d_k_scale && l->d_v_scale && l->d_k_open && l->d_v_open,
                "null pointer in the layer of %s", what);
    RBN_REQUIRE(l->format == RBN_KV_I8 || l->format == RBN_KV_E4M3, "unknown K/V format %u in %s", l->format, what);
    RBN_REQUIRE(l->kv_heads > 0 && l->kv_heads <= 1024, "bad kv_heads in %s", what);
    RBN_REQUIRE(l->head_dim == 64 || l->head_dim == 128, "%s takes head_dim 64 or 128 (got %u)", what, l->head_dim);
    RBN_REQUIRE(aligned16(l->d_k) && aligned16(l->d_v) && aligned16(l->d_k_open) && aligned16(l->d_v_open),
                "the layer's code and open buffers of %s must be 16-byte aligned", what);
    *out = KvLayerArgs{(int)l->kv_heads, (uint8_t *)l->d_k, (uint8_t *)l->d_v, l->d_k_scale, l->d_v_scale,
                       (KvHalf *)l->d_k_open, (KvHalf *)l->d_v_open};
    return RBN_OK;
}

// The value a code stands for, before its scale.
template <int FMT>
__device__ __forceinline__ float kv_decode(uint8_t c) {
    if (FMT == RBN_KV_I8) return (float)(int8_t)c;
    return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
}
