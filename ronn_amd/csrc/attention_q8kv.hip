// Attention over the paged 8-bit K/V cache.
#include "kv_common.hpp"

namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

// Eight codes as f16, exactly: int8 c is the f16 with bits 0x6400 | (c + 128) (that is 1024 + c +
// 128) minus 1152; e4m3 has a conversion.
template <int FMT>
__device__ __forceinline__ v8h codes_to_f16(unsigned a, unsigned b) {
    v2h p[4];
    if (FMT == RBN_KV_I8) {
        const v2h bias = {(_Float16)1152.0f, (_Float16)1152.0f};
        a ^= 0x80808080u;
        b ^= 0x80808080u;
        p[0] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, a, 0x04010400u)) - bias;
        p[1] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, a, 0x04030402u)) - bias;
        p[2] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u)) - bias;
        p[3] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u)) - bias;
    } else {
        p[0] = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false));
        p[1] = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true));
        p[2] = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false));
        p[3] = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true));
    }
    return __builtin_shufflevector(__builtin_shufflevector(p[0], p[1], 0, 1, 2, 3),
                                   __builtin_shufflevector(p[2], p[3], 0, 1, 2, 3), 0, 1, 2, 3, 4, 5, 6, 7);
}

// The value of the lane eight away in the same row of sixteen.
__device__ __forceinline__ float other_half(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, false));  // row_ror:8
}

__device__ __forceinline__ float load_agent(const float *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_agent(float *p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Power of two at or below |v| (exponent clamped to the normal range), as an exponent.
__device__ __forceinline__ int exponent_of(float v) {
    const int e = (int)((__float_as_uint(v) >> 23) & 0xff) - 127;
    return e < -126 ? -126 : e;
}

// ---- few query columns: decode steps ------------------------------------------------------------
// S^T = K . Q^T and O^T = V^T . P^T on v_mfma_f32_16x16x32_f16, a wave on one block of 32 keys at a time.
//  * The codes are exact in f16.  q (scaled to |q| < 2 by a power of two for each column) and the
//    probabilities go in as hi + lo f16 pairs, 22 bits: of the 16 columns of a tile, 0-7 carry the hi
//    parts of eight (token, head) columns and 8-15 their lo parts, so one instruction does both.
//  * A page is laid out as the instructions read it: a lane's operand bytes are consecutive, a wave's
//    loads are whole cache lines, and P^T comes out of the score tiles already in operand order
//    (slot e of lane group g is key 16 (e/4) + 4 g + e%4; V's layout follows).
//  * The running maximum is shared by the four lanes of a column and moves only when a score exceeds it
//    by 8 (powers of two): the usual block costs no cross-lane step.  Sums are per lane until the end.
//  * The blocks of an item (token or unit, K/V head, up to 8 NT columns) go round the 4 * splits
//    waves of its workgroups; the last workgroup of an item to finish joins the partial results in
//    a fixed order.  Bound by the reading of the codes.
constexpr int kTokenWaves = 4;
constexpr int kTokenThreads = kTokenWaves * 64;
constexpr int kMinBlocksPerWave = 2;  // before another workgroup shares an item
constexpr int kTargetGroups = 4096;

// floats of one split's partial result: columns x (out, max, sum)
template <int HD, int NT>
constexpr int partial_floats() {
    return 8 * NT * (HD + 2);
}

template <int FMT, int HD, int NT, bool PER_TOKEN>
__global__ __launch_bounds__(kTokenThreads, NT == 1 ? 3 : 2) void attention_token_kernel(
    const float *__restrict__ q, KvTableArgs t, KvBatchArgs b, KvLayerArgs l, int heads, int splits,
    float *__restrict__ partials, unsigned *__restrict__ tickets, float *__restrict__ out, unsigned *flags) {
    constexpr int KK = HD / 32;   // k steps of the scores
    constexpr int DT = HD / 16;   // tiles of dimensions of the output
    constexpr int LD = HD / 32;   // 16-byte loads per lane of 32 keys, K and V each
    constexpr int kPitch = HD + 8;
    __shared__ __attribute__((aligned(16))) float s_o[kTokenWaves][8 * NT][HD];
    __shared__ __attribute__((aligned(16))) _Float16 s_open[kKvBlock * kPitch];
    __shared__ float s_m[kTokenWaves][8 * NT], s_l[kTokenWaves][8 * NT];
    __shared__ int s_last;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int c16 = lane & 15, c8 = lane & 7, g = lane >> 4;
    const int group = heads / l.kv_heads;
    const int split = blockIdx.x % splits, item = blockIdx.x / splits, kvh = item % l.kv_heads, u = item / l.kv_heads;

    // the item's tokens: `first` .. `first + n`, at positions pos .. of `row`
    int row, first, n, pos, len;
    if (PER_TOKEN) {
        first = u;
        if (u >= min(b.count[0], b.max_tokens)) return;
        n = 1;
        row = b.row[u];
        pos = b.pos[u];
        if (row < 0 || row >= t.rows) pos = -1;
    } else {
        const KvUnit unit = kv_unit(t, b, u, flags);
        if (unit.n == 0) return;
        first = unit.first;
        n = unit.n;
        row = unit.row;
        pos = unit.pos;
    }
    len = pos >= 0 ? min(t.len[row], t.max_blocks * kKvBlock) : 0;
    if (pos < 0 || pos + n > len) {
        if (tid == 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
        return;
    }
    const int cols = n * group;
    const int nblocks = (pos + n - 1) / kKvBlock + 1, full_blocks = min(len / kKvBlock, nblocks);

    // More columns than the grid's z covers (only if the host's bound was too low): the item's first
    // workgroup does the rest alone.
    for (int cg = blockIdx.y; cg * 8 * NT < cols; cg += gridDim.y) {
        int shares = min(splits, (nblocks + kTokenWaves * kMinBlocksPerWave - 1) / (kTokenWaves * kMinBlocksPerWave));
        if (cg != (int)blockIdx.y) shares = 1;
        if (split >= shares) continue;
        const int stride = shares * kTokenWaves, w0 = split * kTokenWaves + wave;

        // Q^T operand and what belongs to a column
        v8h qf[NT][KK];
        float col_scale[NT];   // 2^e log2(e) / sqrt(hd): raw score x K scale x this is an exponent of two
        int col_pos[NT];
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) {
            const int c = min((cg * NT + ct) * 8 + c8, cols - 1);
            const int token = c / group;
            const float *src = q + ((size_t)(first + token) * heads + kvh * group + (c - token * group)) * HD + 8 * g;
            col_pos[ct] = pos + token;
            float x[KK][8], m = 0.0f;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                const float4 lo4 = *reinterpret_cast<const float4 *>(src + 32 * kk);
                const float4 hi4 = *reinterpret_cast<const float4 *>(src + 32 * kk + 4);
                x[kk][0] = lo4.x, x[kk][1] = lo4.y, x[kk][2] = lo4.z, x[kk][3] = lo4.w;
                x[kk][4] = hi4.x, x[kk][5] = hi4.y, x[kk][6] = hi4.z, x[kk][7] = hi4.w;
#pragma unroll
                for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[kk][e]));
            }
            m = fmaxf(m, __shfl_xor(m, 16));
            m = fmaxf(m, __shfl_xor(m, 32));
            const int ex = exponent_of(m);
            col_scale[ct] = ldexpf(HD == 128 ? 0.12751743082459868f : 0.18033688011112042f, ex);  // log2(e) / sqrt(hd)
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float v = ldexpf(x[kk][e], -ex);
                    const _Float16 hi = (_Float16)v, lo = (_Float16)(v - (float)hi);
                    qf[ct][kk][e] = c16 < 8 ? hi : lo;
                }
        }

        float run_max[NT], run_sum[NT];
        v4f o[NT][DT];
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) {
            run_max[ct] = -INFINITY;
            run_sum[ct] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[ct][d] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        }
        // Scores of 32 keys from t0 on (tile a, register r: key 16 a + 4 g + r), their softmax and P.V.
        auto attend = [&](const v4f (&s)[NT][2], auto value, float kscale, float vscale, int t0) {
            const bool masked = t0 + kKvBlock - 1 > pos;
            v8h pf[NT];
#pragma unroll
            for (int ct = 0; ct < NT; ++ct) {
                const float f = kscale * col_scale[ct];
                float x[8], m = -INFINITY;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = s[ct][e >> 2][e & 3];
                    x[e] = (x[e] + other_half(x[e])) * f;
                    if (masked) x[e] = t0 + 16 * (e >> 2) + 4 * g + (e & 3) <= col_pos[ct] ? x[e] : -INFINITY;
                    m = fmaxf(m, x[e]);
                }
                if (__any(m > run_max[ct] + 8.0f)) {
                    m = fmaxf(m, __shfl_xor(m, 16));
                    m = fmaxf(m, __shfl_xor(m, 32));
                    const float top = fmaxf(run_max[ct], m);
                    const float corr = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(run_max[ct] - top);
                    run_max[ct] = top;
                    run_sum[ct] *= corr;
#pragma unroll
                    for (int d = 0; d < DT; ++d) o[ct][d] *= corr;
                }
                const float ref = run_max[ct] == -INFINITY ? 0.0f : run_max[ct];  // nothing seen yet: p = 0
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float p = __builtin_amdgcn_exp2f(x[e] - ref);
                    run_sum[ct] += p;
                    const _Float16 hi = (_Float16)p, lo = (_Float16)(p - (float)hi);
                    pf[ct][e] = c16 < 8 ? hi : lo;
                }
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                const v8h vf = value(d);
#pragma unroll
                for (int ct = 0; ct < NT; ++ct) {
                    const v4f z = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[ct], v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[ct][d][r] = fmaf(z[r], vscale, o[ct][d][r]);
                }
            }
        };

        // full blocks: this wave's w0, w0 + stride, ...
        const int mine = full_blocks > w0 ? (full_blocks - w0 + stride - 1) / stride : 0;
        v4u kc[LD], vc[LD];
        // (an invalid page loads page 0 and is skipped)
        auto load = [&](v4u (&to)[LD], const uint8_t *codes, int page) {
            const v4u *src =
                reinterpret_cast<const v4u *>(codes + ((size_t)max(page, 0) * l.kv_heads + kvh) * (kKvBlock * HD)) + lane;
#pragma unroll
            for (int j = 0; j < LD; ++j) to[j] = src[64 * j];
        };
        for (int base = 0; base < mine; base += 64) {
            // pages and scales of the next 64 blocks, one per lane
            const int steps = min(64, mine - base);
            int page = -1;
            float ks = 0.0f, vs = 0.0f;
            if (lane < steps) {
                page = kv_page(t, row, w0 + (base + lane) * stride);
                const size_t ph = (size_t)max(page, 0) * l.kv_heads + kvh;
                ks = l.k_scale[ph];
                vs = l.v_scale[ph];
                if (page < 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
            }
            load(kc, l.k, __builtin_amdgcn_readlane(page, 0));
            load(vc, l.v, __builtin_amdgcn_readlane(page, 0));
            for (int i = 0; i < steps; ++i) {
                const int here = __builtin_amdgcn_readlane(page, i), next = __builtin_amdgcn_readlane(page, min(i + 1, steps - 1));
                v4f s[NT][2];
#pragma unroll
                for (int a = 0; a < 2; ++a) {
#pragma unroll
                    for (int ct = 0; ct < NT; ++ct) s[ct][a] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int kk = 0; kk < KK; ++kk) {
                        const v4u w = kc[a * (KK / 2) + kk / 2];
                        const v8h kf = kk & 1 ? codes_to_f16<FMT>(w.z, w.w) : codes_to_f16<FMT>(w.x, w.y);
#pragma unroll
                        for (int ct = 0; ct < NT; ++ct)
                            s[ct][a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[ct][kk], s[ct][a], 0, 0, 0);
                    }
                }
                load(kc, l.k, next);  // the next block's keys travel during the softmax, its values during its scores
                if (here >= 0)
                    attend(s,
                           [&](int d) {
                               const v4u w = vc[d / 2];
                               return d & 1 ? codes_to_f16<FMT>(w.z, w.w) : codes_to_f16<FMT>(w.x, w.y);
                           },
                           __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ks), i)),
                           __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vs), i)),
                           (w0 + (base + i) * stride) * kKvBlock);
                load(vc, l.v, next);
            }
        }
        // the unfinished block, f16: K straight from the buffer, V transposed through LDS; rows behind
        // the end may hold anything, so V's are zeroed (K's scores are masked)
        if (nblocks > full_blocks && full_blocks % stride == w0) {
            const size_t at = ((size_t)row * l.kv_heads + kvh) * kKvBlock * HD;
            const _Float16 *ko = reinterpret_cast<const _Float16 *>(l.k_open) + at;
            const _Float16 *vo = reinterpret_cast<const _Float16 *>(l.v_open) + at;
            const int valid = len - full_blocks * kKvBlock;
            v8h kf[2][KK];
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int kk = 0; kk < KK; ++kk)
                    kf[a][kk] = *reinterpret_cast<const v8h *>(ko + (size_t)(16 * a + c16) * HD + 32 * kk + 8 * g);
#pragma unroll
            for (int j = 0; j < kKvBlock * HD / 512; ++j) {
                const int e = j * 512 + lane * 8, key = e / HD, d = e % HD;
                v8h x = *reinterpret_cast<const v8h *>(vo + e);
                if (key >= valid) x = v8h{0, 0, 0, 0, 0, 0, 0, 0};
                *reinterpret_cast<v8h *>(s_open + key * kPitch + d) = x;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            v4f s[NT][2];
#pragma unroll
            for (int ct = 0; ct < NT; ++ct)
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    s[ct][a] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int kk = 0; kk < KK; ++kk)
                        s[ct][a] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[a][kk], qf[ct][kk], s[ct][a], 0, 0, 0);
                }
            attend(s,
                   [&](int d) {
                       v8h vf;
#pragma unroll
                       for (int e = 0; e < 8; ++e) vf[e] = s_open[(16 * (e >> 2) + 4 * g + (e & 3)) * kPitch + 16 * d + c16];
                       return vf;
                   },
                   1.0f, 1.0f, full_blocks * kKvBlock);
        }

        // the waves meet
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) {
            run_sum[ct] += __shfl_xor(run_sum[ct], 16);
            run_sum[ct] += __shfl_xor(run_sum[ct], 32);
            if (lane < 8) {
                s_m[wave][ct * 8 + lane] = run_max[ct];
                s_l[wave][ct * 8 + lane] = run_sum[ct];
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                v4f z = o[ct][d];
#pragma unroll
                for (int r = 0; r < 4; ++r) z[r] += other_half(z[r]);
                if (c16 < 8) *reinterpret_cast<v4f *>(&s_o[wave][ct * 8 + c8][16 * d + 4 * g]) = z;
            }
        }
        __syncthreads();
        const int ncols = min(8 * NT, cols - cg * 8 * NT);
        const int slot = item * gridDim.y + cg;  // used by shared items only
        float *part = partials + (size_t)slot * splits * partial_floats<HD, NT>();
        auto write_out = [&](int c, int d, float num, float den) {
            const int col = cg * 8 * NT + c, token = col / group;
            out[((size_t)(first + token) * heads + kvh * group + (col - token * group)) * HD + d] =
                den > 0.0f || den != den ? num / den : 0.0f;
        };
        for (int i = tid; i < ncols * HD; i += kTokenThreads) {
            const int c = i / HD, d = i % HD;
            float m = -INFINITY, num = 0.0f, den = 0.0f;
#pragma unroll
            for (int w = 0; w < kTokenWaves; ++w) m = fmaxf(m, s_m[w][c]);
#pragma unroll
            for (int w = 0; w < kTokenWaves; ++w) {
                // a wave that saw no key has sum 0; one that saw a NaN only has maximum -inf and a NaN sum
                const float k = s_m[w][c] == -INFINITY ? (s_l[w][c] != 0.0f ? 1.0f : 0.0f)
                                                       : __builtin_amdgcn_exp2f(s_m[w][c] - m);
                num += k * s_o[w][c][d];
                den += k * s_l[w][c];
            }
            if (shares == 1) {
                write_out(c, d, num, den);
            } else {
                float *p = part + (size_t)split * partial_floats<HD, NT>() + c * (HD + 2);
                store_agent(p + d, num);
                if (d == 0) {
                    store_agent(p + HD, m);
                    store_agent(p + HD + 1, den);
                }
            }
        }
        if (shares > 1) {
            // published once the stores have completed (vmcnt(0): this wave's, the barrier: everybody's)
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            if (tid == 0) {
                const int is_last = atomicAdd(&tickets[slot], 1u) == (unsigned)shares - 1;
                if (is_last) atomicExch(&tickets[slot], 0u);  // ready for the next launch
                s_last = is_last;
            }
            __syncthreads();
            if (s_last)
                for (int i = tid; i < ncols * HD; i += kTokenThreads) {
                    const int c = i / HD, d = i % HD;
                    const float *p = part + c * (HD + 2);
                    float m = -INFINITY, num = 0.0f, den = 0.0f;
                    for (int sp = 0; sp < shares; ++sp) m = fmaxf(m, load_agent(p + (size_t)sp * partial_floats<HD, NT>() + HD));
                    for (int sp = 0; sp < shares; ++sp) {
                        const float *ps = p + (size_t)sp * partial_floats<HD, NT>();
                        const float pm = load_agent(ps + HD), pl = load_agent(ps + HD + 1);
                        const float k = pm == -INFINITY ? (pl != 0.0f ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(pm - m);
                        num += k * load_agent(ps + d);
                        den += k * pl;
                    }
                    write_out(c, d, num, den);
                }
        }
        __syncthreads();
    }
}

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;

// One workgroup per (token, query head).  Each wave takes every fourth block with a running maximum
// and sum: scores with two lanes per key, then P.V with every lane on its own dimensions; the waves
// meet through LDS.
template <int FMT, int HD>
__global__ __launch_bounds__(kThreads) void attention_simple_kernel(const float *__restrict__ q, KvTableArgs t,
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


template <int FMT, int HD, int NT, bool PER_TOKEN>
int launch_token_as(rbn_ctx *ctx, const float *d_q, const KvTableArgs &t, const KvBatchArgs &b, const KvLayerArgs &l,
                    int heads, uint64_t max_new, float *d_out) {
    const uint64_t group = heads / l.kv_heads;
    const uint64_t items = (uint64_t)(PER_TOKEN ? (unsigned)b.max_tokens : kv_max_units(b.max_tokens, t.rows)) * l.kv_heads;
    const uint64_t columns = group * (PER_TOKEN ? 1 : max_new < kKvBlock ? max_new : kKvBlock);
    const uint64_t tiles = (columns + 8 * NT - 1) / (8 * NT);
    // Workgroups that share an item: enough to fill the chip several times over (rows differ in length, and
    // short ones leave their share early), as far as tickets and partial results have room.
    uint64_t splits = kTargetGroups / (items * tiles);
    const uint64_t most = ((uint64_t)t.max_blocks + kTokenWaves * kMinBlocksPerWave - 1) / (kTokenWaves * kMinBlocksPerWave);
    const uint64_t room = (uint64_t)RBN_SPLITK_TILES * 1024 / (items * tiles * partial_floats<HD, NT>());
    splits = splits < most ? splits : most;
    splits = splits < room ? splits : room;
    if (splits < 1 || items * tiles > RBN_ATTENTION_ITEMS) splits = 1;
    RBN_REQUIRE(items * splits < (1ull << 31), "too many tokens in rbn_attention_q8kv");
    attention_token_kernel<FMT, HD, NT, PER_TOKEN>
        <<<dim3((unsigned)(items * splits), (unsigned)tiles), dim3(kTokenThreads), 0, ctx->stream>>>(
            d_q, t, b, l, heads, (int)splits, (float *)ctx->splitk_partials, ctx->attention_tickets, d_out, ctx->dev_flags);
    RBN_HIP(hipGetLastError());
    return RBN_OK;
}

template <int FMT, int HD>
int launch_token_of(rbn_ctx *ctx, const float *d_q, const KvTableArgs &t, const KvBatchArgs &b, const KvLayerArgs &l,
                    int heads, uint64_t max_new, float *d_out) {
    const uint64_t group = heads / l.kv_heads;
    if (max_new == 1)
        return group <= 8 ? launch_token_as<FMT, HD, 1, true>(ctx, d_q, t, b, l, heads, max_new, d_out)
                          : launch_token_as<FMT, HD, 2, true>(ctx, d_q, t, b, l, heads, max_new, d_out);
    return group * max_new <= 8 ? launch_token_as<FMT, HD, 1, false>(ctx, d_q, t, b, l, heads, max_new, d_out)
                                : launch_token_as<FMT, HD, 2, false>(ctx, d_q, t, b, l, heads, max_new, d_out);
}

int launch_token(rbn_ctx *ctx, const float *d_q, const KvTableArgs &t, const KvBatchArgs &b, const KvLayerArgs &l,
                 const rbn_kv_layer &layer, int heads, uint64_t max_new, float *d_out) {
    auto f = layer.format == RBN_KV_I8
                 ? (layer.head_dim == 128 ? launch_token_of<RBN_KV_I8, 128> : launch_token_of<RBN_KV_I8, 64>)
                 : (layer.head_dim == 128 ? launch_token_of<RBN_KV_E4M3, 128> : launch_token_of<RBN_KV_E4M3, 64>);
    return f(ctx, d_q, t, b, l, heads, max_new, d_out);
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
    const uint64_t group = heads / layer->kv_heads;
    if (max_new * group <= 16) {
        return launch_token(ctx, d_q, t, b, l, *layer, (int)heads, max_new, d_out);
    }
    auto kernel =
        layer->format == RBN_KV_I8
            ? (layer->head_dim == 128 ? attention_simple_kernel<RBN_KV_I8, 128> : attention_simple_kernel<RBN_KV_I8, 64>)
            : (layer->head_dim == 128 ? attention_simple_kernel<RBN_KV_E4M3, 128> : attention_simple_kernel<RBN_KV_E4M3, 64>);
    kernel<<<dim3((unsigned)batch->max_tokens, (unsigned)heads), dim3(kThreads), 0, ctx->stream>>>(
        d_q, t, b, l, (int)heads, d_out, ctx->dev_flags);
    RBN_HIP(hipGetLastError());
    return RBN_OK;
}

}  // extern "C"
