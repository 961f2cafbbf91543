// Log probabilities of given tokens, entropy and the top alternatives of rows of logits.
#include "common.hpp"

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;

// Orders logits by value, then by the lower index, in one 64-bit number: the value's bits made
// monotonic (NaN below everything, -0 equal to +0) above the complement of the index.
__device__ __forceinline__ uint64_t order_key(float x, unsigned index) {
    unsigned u = __float_as_uint(x == 0.0f ? 0.0f : x);
    u = u & 0x80000000u ? ~u : u | 0x80000000u;
    if (x != x) u = 0;
    return ((uint64_t)u << 32) | (uint32_t)~index;
}

__device__ __forceinline__ uint64_t wave_max_u64(uint64_t v) {
    for (int off = 32; off > 0; off >>= 1) {
        const uint64_t o = __shfl_xor((unsigned long long)v, off);
        v = o > v ? o : v;
    }
    return v;
}

// (max, sum of exp(x - max), sum of (x - max) exp(x - max)) of two disjoint sets of logits.
struct Stat {
    float m, s, w;
};
__device__ __forceinline__ Stat join(Stat a, Stat b) {
    const float m = a.m > b.m || a.m != a.m ? a.m : b.m;
    if (m == -INFINITY) return Stat{m, 0.0f, 0.0f};
    // a part that vanishes against the other (one of nothing but -inf among them) adds nothing, not 0 * -inf
    const float da = a.m - m, db = b.m - m, ca = expf(da), cb = expf(db);
    return Stat{m, a.s * ca + b.s * cb,
                (ca == 0.0f ? 0.0f : ca * (a.w + da * a.s)) + (cb == 0.0f ? 0.0f : cb * (b.w + db * b.s))};
}

// One workgroup per row.
__global__ __launch_bounds__(kThreads) void logprobs_kernel(const float *__restrict__ logits, int vocab, size_t pitch,
                                                            const int32_t *__restrict__ target, int top,
                                                            float *__restrict__ logprob, float *__restrict__ entropy,
                                                            int32_t *__restrict__ top_token,
                                                            float *__restrict__ top_logprob) {
    __shared__ Stat s_stat[kWaves];
    __shared__ uint64_t s_key[kWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t r = blockIdx.x;
    const float *x = logits + r * pitch;
    float m = -INFINITY;
    bool nan = false;
    for (int i = tid; i < vocab; i += kThreads) {
        m = fmaxf(m, x[i]);
        nan |= x[i] != x[i];
    }
    Stat st{nan ? NAN : m, 0.0f, 0.0f};
    if (m != -INFINITY)
        for (int i = tid; i < vocab; i += kThreads) {
            const float d = x[i] - m, e = expf(d);
            st.s += e;
            st.w += e > 0.0f || e != e ? e * d : 0.0f;
        }
    for (int off = 32; off > 0; off >>= 1)
        st = join(st, Stat{__shfl_xor(st.m, off), __shfl_xor(st.s, off), __shfl_xor(st.w, off)});
    if (lane == 0) s_stat[wave] = st;
    __syncthreads();
    st = s_stat[0];
    for (int w = 1; w < kWaves; ++w) st = join(st, s_stat[w]);
    const float log_s = logf(st.s);
    const bool none = st.m == -INFINITY;  // nothing but -inf
    auto lp = [&](float v) { return none ? -INFINITY : (v - st.m) - log_s; };
    if (tid == 0) {
        if (logprob) {
            const int y = target[r];
            logprob[r] = y >= 0 && y < vocab ? lp(x[y]) : 0.0f;
        }
        if (entropy) entropy[r] = none ? 0.0f : log_s - st.w / st.s;
    }
    uint64_t below = ~0ull;
    for (int j = 0; j < top; ++j) {
        uint64_t best = 0;
        for (int i = tid; i < vocab; i += kThreads) {
            const uint64_t k = order_key(x[i], (unsigned)i);
            if (k < below && k > best) best = k;
        }
        best = wave_max_u64(best);
        if (lane == 0) s_key[wave] = best;
        __syncthreads();
        best = s_key[0];
        for (int w = 1; w < kWaves; ++w) best = s_key[w] > best ? s_key[w] : best;
        __syncthreads();
        if (tid == 0) {
            const int i = j < vocab ? (int)~(uint32_t)best : -1;
            top_token[r * top + j] = i;
            top_logprob[r * top + j] = i >= 0 ? lp(x[i]) : -INFINITY;
        }
        below = best;
    }
}

}  // namespace

extern "C" {

int rbn_token_logprobs_f32(rbn_ctx *ctx, const float *d_logits, uint64_t rows, uint64_t vocab, uint64_t pitch,
                           const int32_t *d_target, uint64_t top, float *d_logprob, float *d_entropy,
                           int32_t *d_top_token, float *d_top_logprob) {
    rbn_clear_error();
    RBN_REQUIRE(d_logits != nullptr, "null pointer in rbn_token_logprobs_f32");
    RBN_REQUIRE(rows > 0 && rows < (1u << 20) && vocab > 0 && vocab < (1u << 30) && pitch >= vocab &&
                    pitch < (1ull << 40),
                "bad sizes in rbn_token_logprobs_f32 (rows %llu, vocab %llu, pitch %llu)", (unsigned long long)rows,
                (unsigned long long)vocab, (unsigned long long)pitch);
    RBN_REQUIRE(top <= RBN_TOP_MAX, "top is at most %d", RBN_TOP_MAX);
    RBN_REQUIRE((d_logprob == nullptr) == (d_target == nullptr), "d_logprob and d_target go together");
    RBN_REQUIRE(top == 0 || (d_top_token && d_top_logprob), "top needs d_top_token and d_top_logprob");
    RBN_ENTER(ctx);
    logprobs_kernel<<<dim3((unsigned)rows), dim3(kThreads), 0, ctx->stream>>>(
        d_logits, (int)vocab, (size_t)pitch, d_target, (int)top, d_logprob, d_entropy, d_top_token, d_top_logprob);
    RBN_HIP(hipGetLastError());
    return RBN_OK;
}

}  // extern "C"
