// Attention over the paged 8-bit K/V cache.
#include "kv_common.hpp"

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// One workgroup per (token, query head).  Each wave takes every fourth block with a running maximum
// and sum: scores with two lanes per key, then P.V with every lane on its own dimensions; the waves
// meet through LDS.
template <int FMT, int HD>
__global__ __launch_bounds__(kThreads) void attention_token_kernel(const float *__restrict__ q, KvTableArgs t,
                                                                   KvBatchArgs b, KvLayerArgs l, int heads,
                                                                   float *__restrict__ out, unsigned *flags) {
    constexpr int PER = HD / 64;  // dimensions a lane owns in P.V
    __shared__ float s_q[HD];
    __shared__ float s_p[kWaves][kKvBlock];
    __shared__ float s_m[kWaves], s_l[kWaves], s_o[kWaves][HD];
    const int i = blockIdx.x, h = blockIdx.y, kvh = h / (heads / l.kv_heads);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (i >= min(b.count[0], b.max_tokens)) return;
    const int row = b.row[i], pos = b.pos[i];
    const bool ok = row >= 0 && row < t.rows && pos >= 0 && pos < t.max_blocks * kKvBlock;
    int len = 0;
    if (ok) {
        const int end = b.start[row + 1];
        len = end > i && end <= b.max_tokens ? min(pos + (end - i), t.max_blocks * kKvBlock) : 0;
    }
    if (len == 0) {
        if (tid == 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
        return;
    }
    if (tid < HD) s_q[tid] = q[((size_t)i * heads + h) * HD + tid] * (HD == 128 ? 0.08838834764831845f : 0.125f);
    __syncthreads();
    float run_max = -INFINITY, run_sum = 0.0f, o[PER];
    for (int e = 0; e < PER; ++e) o[e] = 0.0f;
    for (int blk = wave; blk <= pos / kKvBlock; blk += kWaves) {
        const bool full = (blk + 1) * kKvBlock <= len;
        size_t ph = 0;
        if (full) {
            const int page = kv_page(t, row, blk);
            if (page < 0) {
                if (lane == 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
                continue;
            }
            ph = (size_t)page * l.kv_heads + kvh;
        }
        const size_t open = ((size_t)row * l.kv_heads + kvh) * kKvBlock * HD;
        const int key = lane & 31, part = lane >> 5;
        float s = 0.0f;
        for (int d = part * (HD / 2); d < (part + 1) * (HD / 2); ++d)
            s += s_q[d] * (full ? kv_decode<FMT>(l.k[ph * kKvBlock * HD + kv_k_byte<HD>(key, d)])
                                : __half2float(l.k_open[open + key * HD + d]));
        s += __shfl_xor(s, 32);
        if (full) s *= l.k_scale[ph];
        const bool seen = blk * kKvBlock + key <= pos;
        s = seen ? s : -INFINITY;
        float m = s;
        for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
        const float new_max = fmaxf(run_max, m);
        const float p = seen ? __expf(s - new_max) : 0.0f;
        float sum = p;
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
        const float corr = __expf(run_max - new_max);
        run_sum = run_sum * corr + sum;
        run_max = new_max;
        if (part == 0) s_p[wave][key] = p;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        for (int e = 0; e < PER; ++e) {
            const int d = lane * PER + e;
            float acc = 0.0f;
            for (int j = 0; j < kKvBlock; ++j) {
                if (blk * kKvBlock + j > pos) break;  // what lies behind may be anything
                acc += s_p[wave][j] * (full ? kv_decode<FMT>(l.v[ph * kKvBlock * HD + kv_v_byte<HD>(j, d)])
                                            : __half2float(l.v_open[open + j * HD + d]));
            }
            if (full) acc *= l.v_scale[ph];
            o[e] = o[e] * corr + acc;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    if (lane == 0) {
        s_m[wave] = run_max;
        s_l[wave] = run_sum;
    }
    for (int e = 0; e < PER; ++e) s_o[wave][lane * PER + e] = o[e];
    __syncthreads();
    if (tid < HD) {
        float m = -INFINITY, num = 0.0f, den = 0.0f;
        for (int w = 0; w < kWaves; ++w) m = fmaxf(m, s_m[w]);
        for (int w = 0; w < kWaves; ++w) {
            const float c = s_m[w] == -INFINITY ? 0.0f : __expf(s_m[w] - m);
            num += c * s_o[w][tid];
            den += c * s_l[w];
        }
        out[((size_t)i * heads + h) * HD + tid] = den > 0.0f || den != den ? num / den : 0.0f;
    }
}

}  // namespace

extern "C" {

int rbn_attention_q8kv(rbn_ctx *ctx, const float *d_q, const rbn_kv_table *table, const rbn_kv_batch *batch,
                       const rbn_kv_layer *layer, uint64_t heads, uint64_t max_new, float *d_out) {
    rbn_clear_error();
    KvTableArgs t;
    KvBatchArgs b;
    KvLayerArgs l;
    RBN_CHECK(kv_check_table(table, &t, "rbn_attention_q8kv"));
    RBN_CHECK(kv_check_batch(batch, &b, "rbn_attention_q8kv"));
    RBN_CHECK(kv_check_layer(layer, &l, "rbn_attention_q8kv"));
    RBN_REQUIRE(d_q && d_out, "null pointer in rbn_attention_q8kv");
    RBN_REQUIRE(aligned16(d_q) && aligned16(d_out), "d_q and d_out of rbn_attention_q8kv must be 16-byte aligned");
    RBN_REQUIRE(heads > 0 && heads <= 1024 && heads % layer->kv_heads == 0,
                "heads (%llu) must be a multiple of kv_heads (%u), at most 1024", (unsigned long long)heads,
                layer->kv_heads);
    RBN_REQUIRE(max_new > 0, "max_new of rbn_attention_q8kv is 0");
    RBN_ENTER(ctx);
    auto kernel =
        layer->format == RBN_KV_I8
            ? (layer->head_dim == 128 ? attention_token_kernel<RBN_KV_I8, 128> : attention_token_kernel<RBN_KV_I8, 64>)
            : (layer->head_dim == 128 ? attention_token_kernel<RBN_KV_E4M3, 128> : attention_token_kernel<RBN_KV_E4M3, 64>);
    kernel<<<dim3((unsigned)batch->max_tokens, (unsigned)heads), dim3(kThreads), 0, ctx->stream>>>(
        d_q, t, b, l, (int)heads, d_out, ctx->dev_flags);
    RBN_HIP(hipGetLastError());
    return RBN_OK;
}

}  // extern "C"
