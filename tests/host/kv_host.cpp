// kv_index.h compiled for the host: what the K/V kernels index with, for tests without a GPU.
#include "../../ronn_amd/csrc/kv_index.h"

extern "C" {

int kv_byte(int which, int head_dim, int t, int d) {
    if (head_dim == 128) return which ? kv_v_byte<128>(t, d) : kv_k_byte<128>(t, d);
    return which ? kv_v_byte<64>(t, d) : kv_k_byte<64>(t, d);
}

// out: row, first, n, pos, row_first, row_pos, row_n; returns whether the batch was found bad
int kv_unit_of(int rows, int max_blocks, int max_tokens, int32_t *start, int32_t *row, int32_t *pos, int32_t *unit,
               int32_t *count, int u, int *out) {
    KvTableArgs t{rows, max_blocks, 1, nullptr, nullptr, nullptr, nullptr};
    KvBatchArgs b{max_tokens, start, row, pos, nullptr, unit, count};
    bool bad = false;
    const KvUnit r = kv_resolve_unit(t, b, u, &bad, [](int) {});
    out[2] = r.n;
    if (r.n) {
        const int v[7] = {r.row, r.first, r.n, r.pos, r.row_first, r.row_pos, r.row_n};
        for (int i = 0; i < 7; ++i) out[i] = v[i];
    }
    return bad;
}

int kv_page_of(int rows, int max_blocks, int pages, int32_t *table, int row, int block) {
    KvTableArgs t{rows, max_blocks, pages, table, nullptr, nullptr, nullptr};
    return kv_page(t, row, block);
}

int kv_slot_page_of(int pages, int slot) {
    KvTableArgs t{1, 1, pages, nullptr, nullptr, nullptr, nullptr};
    return kv_slot_page(t, slot);
}

}  // extern "C"
