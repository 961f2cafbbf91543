// Log probabilities of given tokens, entropy and the top alternatives of rows of logits.
#include "common.hpp"
#include "wave_ops.hpp"

namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kVecs = 4;                             // 16-byte loads of a thread in one sweep of 8192 logits
constexpr int kGroups = kThreads / 8;                // groups of eight lanes, for the first threshold
constexpr int kCandidates = 2048;
constexpr int kMaxSegments = 16;
constexpr int kMinSegment = 8192;                    // logits of one sweep
constexpr int kTargetGroups = 512;
static_assert(kGroups == 64, "a lane per group maximum");
static_assert(kGroups >= RBN_TOP_MAX, "the top-th largest group maximum bounds the top-th largest logit");

// Orders logits by value, then by the lower index, in one 64-bit number: the value's bits made
// monotonic (NaN below everything, -0 equal to +0) above the complement of the index.
__device__ __forceinline__ uint64_t order_key(float x, unsigned index) {
    unsigned u = __float_as_uint(x == 0.0f ? 0.0f : x);
    u = u & 0x80000000u ? ~u : u | 0x80000000u;
    if (x != x) u = 0;
    return ((uint64_t)u << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(uint64_t key) {
    const unsigned u = (unsigned)(key >> 32);
    return u == 0 ? NAN : __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int key_index(uint64_t key) { return (int)~(uint32_t)key; }

template <int CTRL>
__device__ __forceinline__ float lane_max(float v) {
    const int i = __float_as_int(v);
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, false)));
}

// (max, sum of exp(x - max), sum of (x - max) exp(x - max)) of a set of logits.
struct Stat {
    float m, s, w;
};
// The sets of all lanes as one: each is moved to the common maximum, then the sums are added.
__device__ __forceinline__ Stat join(Stat a) {
    const float m = wave_max(a.m);
    if (m == -INFINITY) return Stat{m, wave_sum(a.s), 0.0f};  // nothing but -inf (s = 0) or NaN (s = NaN)
    // a set that vanishes against the others (one of nothing but -inf among them) adds nothing, not 0 * -inf;
    // a NaN in its sum stays
    const float d = a.m - m, c = expf(d);
    return Stat{m, wave_sum(a.s * c), wave_sum(c == 0.0f ? 0.0f : c * (a.w + d * a.s))};
}

// The largest `top` of the n keys in cand, sorted, to out: each key's place is the number of larger ones
// (keys differ, their indices do).
__device__ __forceinline__ void rank_keys(const uint64_t *cand, int n, int top, uint64_t *out) {
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const uint64_t key = cand[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += cand[j] > key;
        if (rank < top) out[rank] = key;
    }
}

typedef float v4f __attribute__((ext_vector_type(4)));
__device__ __forceinline__ float4 load_once(const float *p) {
    const v4f x = __builtin_nontemporal_load(reinterpret_cast<const v4f *>(p));
    return {x[0], x[1], x[2], x[3]};
}

// A row is one segment, or a few that workgroups share if there are few rows; the last workgroup of a row
// to finish joins them (in the order of the segments).  One pass over the logits:
//  * 16-byte loads, four in flight per thread; the exponentials' running maximum per thread.
//  * The top alternatives: the first sweep is held in registers; the top-th largest of the maxima of 64 groups of eight
//    lanes bounds the top-th largest logit from below, and only logits at or above it (typically no more
//    than twice `top`) go to a list in LDS, which is ranked by counting.  Later sweeps add what exceeds the
//    list's last entry (their indices are higher, so equals lose).  A sweep with too many of them is looked at once
//    more, with a bound of its own and no more equals than can count (1000 rows of 100003 with all but 20 logits at one
//    value: 85 us, before that 2.4 ms by the way below; in ascending order 0.76 ms).
//  * Where the list overflows even so, or comes out short (NaN), the segment's alternatives are found one by one
//    instead, each a pass over the segment.
// Bound by the reading of the logits; with few rows by latency.  1000 rows of 100003: 73 us, 5.5 TB/s with four workgroups on a
// CU (8 waves per SIMD; 93 with the 66 registers of twice the loads in flight, 81 with those loads in 64; 100 with the next
// sweep's loads ahead of the ranking: its registers spill).  16 rows of 32000: 8.4 us in four segments of 8000, a sweep
// each (8.9 in six, 9.2 in eight, 11.3 in three of two sweeps).
__global__ __launch_bounds__(kThreads, 8) void logprobs_kernel(const float *__restrict__ logits, int vocab, size_t pitch,
                                                               int segments, int seg_len,
                                                               const int32_t *__restrict__ target, int top,
                                                               float *__restrict__ logprob, float *__restrict__ entropy,
                                                               int32_t *__restrict__ top_token,
                                                               float *__restrict__ top_logprob, char *parts,
                                                               unsigned *__restrict__ tickets) {
    __shared__ uint64_t s_cand[kCandidates];
    __shared__ uint64_t s_top[RBN_TOP_MAX];
    __shared__ Stat s_stat[kWaves];
    __shared__ uint64_t s_best[kWaves];
    __shared__ float s_group[kGroups];
    __shared__ int s_rank[kGroups];
    __shared__ int s_equals[kWaves];
    __shared__ int s_count, s_last;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // the same in every lane
    const size_t r = blockIdx.x / segments;
    const int seg = blockIdx.x % segments;
    const float *x = logits + r * pitch;
    const int lo = seg * seg_len, hi = min(lo + seg_len, vocab), n = hi - lo;

    // up to three logits before the first 16-byte boundary and behind the last: a thread each
    const int head = min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(x + lo) & 15)) & 15) / 4));
    const int vecs = (n - head) / 4, tail = n - head - 4 * vecs;
    const int vec_lo = lo + head, tail_lo = vec_lo + 4 * vecs;
    const int sweeps = max(1, (vecs + kThreads * kVecs - 1) / (kThreads * kVecs));

    const int y = logprob && tid == 64 ? target[r] : -1;  // (of use to the row's last workgroup)
    const float xy = y >= 0 && y < vocab ? x[y] : 0.0f;

    Stat st{-INFINITY, 0.0f, 0.0f};
    const int want = min(top, n);
    bool slow = false;
    int held = 0;             // entries of s_top
    float bound = -INFINITY;  // value of the last of `want` entries
    for (int sweep = 0; sweep < sweeps; ++sweep) {
        float4 v[kVecs];
        const int v0 = sweep * kThreads * kVecs + tid;
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
            const int k = v0 + j * kThreads;
            v[j] = k < vecs ? load_once(x + vec_lo + 4 * (size_t)k)
                            : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        }
        int extra = -1;  // this thread's logit outside the 16-byte part
        if (sweep == 0 && tid < head) extra = lo + tid;
        if (sweep == sweeps - 1 && tid >= 4 && tid < 4 + tail) extra = tail_lo + tid - 4;
        const float xe = extra >= 0 ? x[extra] : -INFINITY;

        float m = xe;
#pragma unroll
        for (int j = 0; j < kVecs; ++j) m = fmaxf(fmaxf(fmaxf(m, v[j].x), fmaxf(v[j].y, v[j].z)), v[j].w);
        const float here = fmaxf(m, -INFINITY);  // (not NaN)
        if (here > st.m) {
            // the old sums at the new maximum; w counts from the maximum too
            const float d = st.m - here, c = expf(d);
            st.w = c == 0.0f ? 0.0f : c * (st.w + d * st.s);
            st.s *= c;
            st.m = here;
        }
        const float ref = st.m == -INFINITY ? 0.0f : st.m;
        auto add = [&](float a) {
            const float d = a - ref, e = __builtin_amdgcn_exp2f(d * 1.44269504088896341f);
            st.s += e;
            st.w += e * fmaxf(d, -1e4f);  // e = 0 there; keeps 0 * -inf out
        };
#pragma unroll
        for (int j = 0; j < kVecs; ++j) add(v[j].x), add(v[j].y), add(v[j].z), add(v[j].w);
        add(xe);
        if (top == 0 || slow) continue;

        const bool first = sweep == 0;
        // The want-th largest of the maxima of 64 groups of eight lanes in this sweep; sets the count to `entries`.
        auto threshold = [&](int entries) {
            float gm = lane_max<0xB1>(here);  // quad_perm [1,0,3,2]
            gm = lane_max<0x4E>(gm);          // quad_perm [2,3,0,1]
            gm = lane_max<0x141>(gm);         // row_half_mirror: the other four of the eight
            if ((lane & 7) == 0) s_group[tid >> 3] = gm;
            if (tid < kGroups) s_rank[tid] = 0;
            if (tid == 0) s_count = entries;
            __syncthreads();
            // the maxima as unsigned numbers in the same order, the last six bits for their places: all differ.  Each
            // wave compares them with eight of them.
            const unsigned u = __float_as_uint(s_group[lane]);
            const unsigned key = ((u & 0x80000000u ? ~u : u | 0x80000000u) & ~63u) | (unsigned)(63 - lane);
            int above = 0;
#pragma unroll
            for (int j = 0; j < kGroups / kWaves; ++j)
                above += (unsigned)__builtin_amdgcn_readlane((int)key, wave * (kGroups / kWaves) + j) > key;
            atomicAdd(&s_rank[lane], above);
            __syncthreads();
            // (equal but for those bits may stand in any order: the least of the first `want` it is)
            return wave_min(s_rank[lane] < want ? s_group[lane] : INFINITY);
        };
        if (tid < held) s_cand[tid] = s_top[tid];
        if (first) {
            bound = threshold(0);
        } else {
            if (tid == 0) s_count = held;
            __syncthreads();
        }
        auto put = [&](float a, int i) {
            const int at = atomicAdd(&s_count, 1);
            if (at < kCandidates) s_cand[at] = order_key(a, (unsigned)i);
        };
        if (first ? here >= bound : here > bound) {
            auto take = [&](float a, int i) {
                if (first ? a >= bound : a > bound) put(a, i);
            };
#pragma unroll
            for (int j = 0; j < kVecs; ++j) {
                const int k = v0 + j * kThreads, i = vec_lo + 4 * k;
                if (k < vecs) take(v[j].x, i), take(v[j].y, i + 1), take(v[j].z, i + 2), take(v[j].w, i + 3);
            }
            if (extra >= 0) take(xe, extra);
        }
        __syncthreads();
        int found = s_count;
        const int so_far = min(n, (sweep == sweeps - 1 ? n : head + 4 * kThreads * kVecs * (sweep + 1)));
        if (found > kCandidates) {
            // too many at the bound (masked logits, say) or above it (a row in ascending order): the sweep once more, with
            // the bound that it gives itself: what is above it, and the first `want` equals in the order of their indices
            // (a wave takes an eighth of the sweep; what the waves before it have gives its equals their ranks).  `want`
            // logits of the sweep are at that bound or above, so the list is short of nothing that counts.
            __syncthreads();
            bound = fmaxf(bound, threshold(held));
            const int from = first ? lo : vec_lo + 4 * kThreads * kVecs * sweep, to = lo + so_far;
            const int each = (to - from + kWaves - 1) / kWaves;
            const int mine = min(from + wave * each, to), behind = min(mine + each, to);
            if (tid < held) s_cand[tid] = s_top[tid];
            float a[4];
            auto load = [&](int i) {
#pragma unroll
                for (int j = 0; j < 4; ++j) a[j] = i + 64 * j + lane < behind ? x[i + 64 * j + lane] : NAN;
            };
            int rank = 0;
            for (int i = mine; i < behind && rank < want; i += 256) {  // (more than `want` need not be told apart)
                load(i);
#pragma unroll
                for (int j = 0; j < 4; ++j) rank += __popcll(__ballot(a[j] == bound));
            }
            if (lane == 0) s_equals[wave] = rank;
            __syncthreads();
            rank = 0;
            for (int w = 0; w < wave; ++w) rank += s_equals[w];
            for (int i = mine; i < behind; i += 256) {
                load(i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned long long equals = __ballot(a[j] == bound);
                    const int before =
                        __builtin_amdgcn_mbcnt_hi((unsigned)(equals >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)equals, 0));
                    if (a[j] > bound || (a[j] == bound && rank + before < want)) put(a[j], i + 64 * j + lane);
                    rank += __popcll(equals);
                }
            }
            __syncthreads();
            found = s_count;
        }
        if (found > kCandidates || found < min(want, so_far)) {
            slow = true;
        } else if (first || found > held) {
            rank_keys(s_cand, found, want, s_top);
            held = min(found, want);
            __syncthreads();
            bound = held == want ? key_value(s_top[want - 1]) : -INFINITY;
        }
        __syncthreads();
    }
    if (slow) {
        uint64_t below = ~0ull;
        for (int j = 0; j < want; ++j) {
            uint64_t best = 0;
            for (int i = lo + tid; i < hi; i += kThreads) {
                const uint64_t k = order_key(x[i], (unsigned)i);
                if (k < below && k > best) best = k;
            }
            for (int off = 32; off > 0; off >>= 1) {
                const uint64_t o = __shfl_xor((unsigned long long)best, off);
                best = o > best ? o : best;
            }
            if (lane == 0) s_best[wave] = best;
            __syncthreads();
            best = s_best[0];
            for (int w = 1; w < kWaves; ++w) best = s_best[w] > best ? s_best[w] : best;
            if (tid == 0) s_top[j] = best;
            below = best;
            __syncthreads();
        }
    }

    const Stat none{-INFINITY, 0.0f, 0.0f};
    st = join(st);
    if (lane == 0) s_stat[wave] = st;
    __syncthreads();
    st = join(lane < kWaves ? s_stat[lane] : none);
    int entries = want;

    if (segments > 1) {
        // partial result of a segment: keys (padded with 0, which is below every key), then the sums
        constexpr size_t kPart = RBN_TOP_MAX * 8 + 16;
        char *mine = parts + (size_t)blockIdx.x * kPart;
        if (tid < top)
            __hip_atomic_store(reinterpret_cast<uint64_t *>(mine) + tid, tid < want ? s_top[tid] : 0ull, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_AGENT);
        float *ms = reinterpret_cast<float *>(mine + RBN_TOP_MAX * 8);
        if (tid < 3)
            __hip_atomic_store(ms + tid, tid == 0 ? st.m : tid == 1 ? st.s : st.w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        // published once the stores have completed (vmcnt(0): this wave's, the barrier: everybody's)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) {
            const int is_last = atomicAdd(&tickets[r], 1u) == (unsigned)segments - 1;
            if (is_last) atomicExch(&tickets[r], 0u);  // ready for the next launch
            s_last = is_last;
        }
        __syncthreads();
        if (!s_last) return;
        const char *all = parts + r * segments * kPart;
        static_assert(kMaxSegments * RBN_TOP_MAX <= kThreads, "one thread per key of a partial result");
        const int keys = segments * top;
        if (tid < keys) {
            const int p = tid / top, j = tid % top;
            s_cand[tid] = __hip_atomic_load(reinterpret_cast<const uint64_t *>(all + p * kPart) + j, __ATOMIC_RELAXED,
                                            __HIP_MEMORY_SCOPE_AGENT);
        }
        static_assert(kMaxSegments <= 64, "a lane per partial result");
        Stat part = none;
        if (lane < segments) {
            const float *f = reinterpret_cast<const float *>(all + lane * kPart + RBN_TOP_MAX * 8);
            part.m = __hip_atomic_load(f, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            part.s = __hip_atomic_load(f + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            part.w = __hip_atomic_load(f + 2, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        st = join(part);
        __syncthreads();
        entries = min(top, vocab);
        if (tid < keys && s_cand[tid] != 0) {
            const uint64_t key = s_cand[tid];
            int rank = 0;
            // (padding is below every key)
#pragma unroll 8
            for (int j = 0; j < keys; ++j) rank += s_cand[j] > key;
            if (rank < entries) s_top[rank] = key;
        }
        __syncthreads();
    }

    const float log_s = logf(st.s);
    const bool empty = st.m == -INFINITY && st.s == 0.0f;  // nothing but -inf
    auto lp = [&](float v) { return empty ? -INFINITY : (v - st.m) - log_s; };
    if (tid < top) {
        const bool there = tid < entries;
        const uint64_t key = there ? s_top[tid] : 0;
        top_token[r * top + tid] = there ? key_index(key) : -1;
        top_logprob[r * top + tid] = there ? lp(key_value(key)) : -INFINITY;
    }
    if (tid == 64 && logprob) logprob[r] = y >= 0 && y < vocab ? lp(xy) : 0.0f;
    if (tid == 128 && entropy) entropy[r] = empty ? 0.0f : log_s - st.w / st.s;
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
    // few rows: workgroups share a row, as long as each has enough to read
    uint64_t segments = kTargetGroups / rows;
    const uint64_t most = (vocab + kMinSegment - 1) / kMinSegment;
    segments = segments < most ? segments : most;
    segments = segments < kMaxSegments ? segments : kMaxSegments;
    segments = segments > 1 ? segments : 1;
    static_assert(kTargetGroups / 2 <= RBN_SPLITK_GROUPS, "a ticket for every row that is shared");
    const uint64_t seg_len = (vocab + segments - 1) / segments;
    segments = (vocab + seg_len - 1) / seg_len;
    logprobs_kernel<<<dim3((unsigned)(rows * segments)), dim3(kThreads), 0, ctx->stream>>>(
        d_logits, (int)vocab, (size_t)pitch, (int)segments, (int)seg_len, d_target, (int)top, d_logprob, d_entropy,
        d_top_token, d_top_logprob, (char *)ctx->splitk_partials, ctx->splitk_tickets);
    RBN_HIP(hipGetLastError());
    return RBN_OK;
}

}  // extern "C"
