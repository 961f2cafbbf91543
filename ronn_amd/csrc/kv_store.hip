// Rotary embedding and the store into the paged 8-bit K/V cache, and reading it back.
#include "kv_common.hpp"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// f16 of a cache value: saturated, NaN to 0 (the cache holds finite values only, so that no masked
// position can turn 0 * value into NaN); *odd collects whether that changed a value.
__device__ __forceinline__ __half to_f16(float x, bool *odd) {
    if (!(fabsf(x) <= 65504.0f)) {
        // up to 65520 a value still rounds to the largest f16
        *odd |= !(fabsf(x) < 65520.0f);
        x = x != x ? 0.0f : copysignf(65504.0f, x);
    }
    return __float2half_rn(x);
}

template <int FMT>
__device__ __forceinline__ uint8_t encode(float x, float scale) {
    const float y = scale > 0.0f ? x / scale : 0.0f;
    if (FMT == RBN_KV_I8) return (uint8_t)(int8_t)(int)fminf(fmaxf(rintf(y), -127.0f), 127.0f);
    return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(fminf(fmaxf(y, -448.0f), 448.0f), 0.0f, 0, false) & 0xff);
}

__device__ __forceinline__ float group_max(float v, float *s_red) {
    for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off));
    if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s_red[0];
    for (int w = 1; w < kWaves; ++w) v = fmaxf(v, s_red[w]);
    __syncthreads();
    return v;
}

// One workgroup per (unit, K/V head): rotates the unit's q heads of the group and its k, completes
// the block from the row's open buffer if it starts inside it, and writes the page (full block) or
// the open buffer (unfinished).  The open buffer of a row is read by its first unit and written by
// its last: where the first has something to read, it also does the last one's K and V, after a
// barrier, so that nothing is overwritten before it was read.
template <int FMT, int HD>
__global__ __launch_bounds__(kThreads) void kv_store_kernel(const float *__restrict__ qkv, KvTableArgs t, KvBatchArgs b,
                                                            KvLayerArgs l, int heads, double log2_theta,
                                                            float *__restrict__ q_out, unsigned *flags) {
    constexpr int half = HD / 2;
    __shared__ float s_cs[kKvBlock][half], s_sn[kKvBlock][half];
    __shared__ __attribute__((aligned(16))) __half s_x[kKvBlock][HD + 8];
    __shared__ float s_red[kWaves];
    const int tid = threadIdx.x, kvh = blockIdx.y;
    const int group = heads / l.kv_heads;
    const size_t width = (size_t)(heads + 2 * l.kv_heads) * HD;
    KvUnit u = kv_unit(t, b, blockIdx.x, flags);
    if (u.n == 0) return;
    const int row_held = u.row_pos & (kKvBlock - 1);  // tokens of the row's first block that came earlier
    const int row_end = u.row_pos + u.row_n;
    const bool first = u.first == u.row_first;
    bool odd = false;

    for (int pass = 0; pass < 2; ++pass) {
        const int base = u.pos & (kKvBlock - 1);       // offset of the unit's first token in the block
        const bool full = (u.pos / kKvBlock + 1) * kKvBlock <= row_end;
        for (int i = tid; i < u.n * half; i += kThreads) {
            const int j = i / half, d = i - j * half;
            // turns = pos * theta^(-2d/hd) / 2 pi, reduced to [-1/2, 1/2] in 64 bits
            const double turns = (double)(u.pos + j) * exp2(log2_theta * (-2.0 * d / HD)) * 0.15915494309189533577;
            const float r = (float)(turns - rint(turns));
            s_cs[j][d] = cospif(2.0f * r);
            s_sn[j][d] = sinpif(2.0f * r);
        }
        __syncthreads();
        if (pass == 0)
            for (int i = tid; i < u.n * group * half; i += kThreads) {
                const int d = i % half, h = kvh * group + i / half % group, j = i / (half * group);
                const float *q = qkv + (size_t)(u.first + j) * width + (size_t)h * HD;
                float *o = q_out + ((size_t)(u.first + j) * heads + h) * HD;
                const float x = q[d], y = q[d + half], cs = s_cs[j][d], sn = s_sn[j][d];
                o[d] = x * cs - y * sn;
                o[d + half] = y * cs + x * sn;
            }
        // an unfinished block behind a first block that reads the open buffer belongs to the latter
        if (pass == 0 && !first && !full && row_held > 0) break;
        const int page = kv_slot_page(t, b.slot[u.first]);
        const bool page_ok = page >= 0;
        if (!page_ok && tid == 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
        for (int which = 0; which < 2; ++which) {
            const float *src = qkv + (size_t)u.first * width + (size_t)(heads + which * l.kv_heads + kvh) * HD;
            __half *open = (which ? l.v_open : l.k_open) + ((size_t)u.row * l.kv_heads + kvh) * kKvBlock * HD;
            for (int i = tid; i < u.n * half; i += kThreads) {
                const int j = i / half, d = i - j * half;
                float x = src[(size_t)j * width + d], y = src[(size_t)j * width + d + half];
                if (which == 0) {
                    const float cs = s_cs[j][d], sn = s_sn[j][d], z = x * cs - y * sn;
                    y = y * cs + x * sn;
                    x = z;
                }
                s_x[base + j][d] = to_f16(x, &odd);
                s_x[base + j][d + half] = to_f16(y, &odd);
            }
            if (full)
                for (int i = tid; i < base * HD; i += kThreads) s_x[i / HD][i % HD] = open[i];
            __syncthreads();
            if (full) {
                float m = 0.0f;
                for (int i = tid; i < kKvBlock * HD; i += kThreads) m = fmaxf(m, fabsf(__half2float(s_x[i / HD][i % HD])));
                m = group_max(m, s_red);
                const float scale = m / (FMT == RBN_KV_I8 ? 127.0f : 448.0f);
                if (page_ok) {
                    uint8_t *dst = (which ? l.v : l.k) + ((size_t)page * l.kv_heads + kvh) * kKvBlock * HD;
                    for (int i = tid; i < kKvBlock * HD; i += kThreads) {
                        const int tt = i / HD, d = i % HD;
                        dst[which ? kv_v_byte<HD>(tt, d) : kv_k_byte<HD>(tt, d)] =
                            encode<FMT>(__half2float(s_x[tt][d]), scale);
                    }
                    if (tid == 0) (which ? l.v_scale : l.k_scale)[(size_t)page * l.kv_heads + kvh] = scale;
                }
            } else {
                for (int i = tid; i < u.n * HD; i += kThreads) open[base * HD + i] = s_x[base + i / HD][i % HD];
            }
            __syncthreads();
        }
        // the first unit goes on to the row's last one if that is unfinished and was left to it
        const int last_pos = row_end - 1, last_block = last_pos / kKvBlock;
        if (pass == 1 || !first || row_held == 0 || last_block == u.pos / kKvBlock || row_end % kKvBlock == 0) break;
        u.first = u.row_first + (last_block * kKvBlock - u.row_pos);
        u.pos = last_block * kKvBlock;
        u.n = row_end - u.pos;
    }
    if (odd) atomicOr(flags, (unsigned)RBN_FLAG_KV_NONFINITE);
}

// One thread per value of a place.
template <int FMT, int HD>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(KvTableArgs t, KvLayerArgs l, const int32_t *__restrict__ row,
                                                           const int32_t *__restrict__ pos, int count,
                                                           __half *__restrict__ k, __half *__restrict__ v,
                                                           unsigned *flags) {
    const int i = blockIdx.x;
    const int r = row[i], p = pos[i];
    const int len = r >= 0 && r < t.rows ? min(t.len[r], t.max_blocks * kKvBlock) : 0;
    bool ok = p >= 0 && p < len;
    const int block = p / kKvBlock, tt = p % kKvBlock;
    const bool full = ok && (block + 1) * kKvBlock <= len;
    int page = 0;
    if (full) {
        page = kv_page(t, r, block);
        ok = page >= 0;
    }
    if (!ok && threadIdx.x == 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
    for (int j = threadIdx.x; j < l.kv_heads * HD; j += kThreads) {
        const int h = j / HD, d = j % HD;
        __half kx = __float2half_rn(0.0f), vx = kx;
        if (ok && full) {
            const size_t ph = (size_t)page * l.kv_heads + h;
            kx = __float2half_rn(kv_decode<FMT>(l.k[ph * kKvBlock * HD + kv_k_byte<HD>(tt, d)]) * l.k_scale[ph]);
            vx = __float2half_rn(kv_decode<FMT>(l.v[ph * kKvBlock * HD + kv_v_byte<HD>(tt, d)]) * l.v_scale[ph]);
        } else if (ok) {
            const size_t at = (((size_t)r * l.kv_heads + h) * kKvBlock + tt) * HD + d;
            kx = l.k_open[at];
            vx = l.v_open[at];
        }
        k[(size_t)i * l.kv_heads * HD + j] = kx;
        v[(size_t)i * l.kv_heads * HD + j] = vx;
    }
}

}  // namespace

extern "C" {

int rbn_rope_kv_store_q8(rbn_ctx *ctx, const float *d_qkv, const rbn_kv_table *table, const rbn_kv_batch *batch,
                         const rbn_kv_layer *layer, uint64_t heads, float theta, float *d_q) {
    rbn_clear_error();
    KvTableArgs t;
    KvBatchArgs b;
    KvLayerArgs l;
    RBN_CHECK(kv_check_table(table, &t, "rbn_rope_kv_store_q8"));
    RBN_CHECK(kv_check_batch(batch, &b, "rbn_rope_kv_store_q8"));
    RBN_CHECK(kv_check_layer(layer, &l, "rbn_rope_kv_store_q8"));
    RBN_REQUIRE(d_qkv && d_q, "null pointer in rbn_rope_kv_store_q8");
    RBN_REQUIRE(aligned16(d_qkv) && aligned16(d_q), "d_qkv and d_q of rbn_rope_kv_store_q8 must be 16-byte aligned");
    RBN_REQUIRE(heads > 0 && heads <= 1024 && heads % layer->kv_heads == 0,
                "heads (%llu) must be a multiple of kv_heads (%u), at most 1024", (unsigned long long)heads,
                layer->kv_heads);
    RBN_REQUIRE(theta > 0.0f && theta <= 3.4e38f, "theta must be positive and finite");
    RBN_ENTER(ctx);
    const dim3 grid(kv_max_units(batch->max_tokens, table->rows), layer->kv_heads);
    const double log2_theta = log2((double)theta);
    auto kernel = layer->format == RBN_KV_I8
                      ? (layer->head_dim == 128 ? kv_store_kernel<RBN_KV_I8, 128> : kv_store_kernel<RBN_KV_I8, 64>)
                      : (layer->head_dim == 128 ? kv_store_kernel<RBN_KV_E4M3, 128> : kv_store_kernel<RBN_KV_E4M3, 64>);
    kernel<<<grid, dim3(kThreads), 0, ctx->stream>>>(d_qkv, t, b, l, (int)heads, log2_theta, d_q, ctx->dev_flags);
    RBN_HIP(hipGetLastError());
    return RBN_OK;
}

int rbn_kv_read_f16(rbn_ctx *ctx, const rbn_kv_table *table, const rbn_kv_layer *layer, const int32_t *d_row,
                    const int32_t *d_pos, uint64_t count, void *d_k, void *d_v) {
    rbn_clear_error();
    KvTableArgs t;
    KvLayerArgs l;
    RBN_CHECK(kv_check_table(table, &t, "rbn_kv_read_f16"));
    RBN_CHECK(kv_check_layer(layer, &l, "rbn_kv_read_f16"));
    RBN_REQUIRE(d_row && d_pos && d_k && d_v, "null pointer in rbn_kv_read_f16");
    RBN_REQUIRE(count > 0 && count < (1ull << 31), "bad count in rbn_kv_read_f16");
    RBN_ENTER(ctx);
    auto kernel = layer->format == RBN_KV_I8
                      ? (layer->head_dim == 128 ? kv_read_kernel<RBN_KV_I8, 128> : kv_read_kernel<RBN_KV_I8, 64>)
                      : (layer->head_dim == 128 ? kv_read_kernel<RBN_KV_E4M3, 128> : kv_read_kernel<RBN_KV_E4M3, 64>);
    kernel<<<dim3((unsigned)count), dim3(kThreads), 0, ctx->stream>>>(t, l, d_row, d_pos, (int)count, (__half *)d_k,
                                                                     (__half *)d_v, ctx->dev_flags);
    RBN_HIP(hipGetLastError());
    return RBN_OK;
}

}  // extern "C"
