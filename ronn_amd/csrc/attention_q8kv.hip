// Attention over the paged 8-bit K/V cache.
#include <type_traits>

#include "kv_common.hpp"

namespace {

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef unsigned v2u __attribute__((ext_vector_type(2)));
template <int BYTES>
struct CodeVec {
    typedef v4u type;
};
template <>
struct CodeVec<8> {
    typedef v2u type;
};

constexpr float kLog2eBySqrt128 = 0.12751743082459868f, kLog2eBySqrt64 = 0.18033688011112042f;

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

// The maximum of the four lanes of a column, sixteen apart.
__device__ __forceinline__ float column_max(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

__device__ __forceinline__ float load_agent(const float *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_agent(float *p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_agent(float *p, v4f v) {  // 8-byte aligned
    unsigned long long *to = reinterpret_cast<unsigned long long *>(p);
    typedef unsigned long long v2q __attribute__((ext_vector_type(2)));
    const v2q w = __builtin_bit_cast(v2q, v);
    __hip_atomic_store(to, w.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(to + 1, w.y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Power of two at or below |v| (exponent clamped to the normal range), as an exponent.
__device__ __forceinline__ int exponent_of(float v) {
    const int e = (int)((__float_as_uint(v) >> 23) & 0xff) - 127;
    return e < -126 ? -126 : e;
}

// ---- who does what ------------------------------------------------------------------------------
// A workgroup's task: an entry of the batch (a token, or a unit), and a share of its blocks.
struct Task {
    int entry;         // -1: none
    int split, shares; // this workgroup is number `split` of `shares`
    int place;         // shares of the entries before this one that are shared: where the partial results go
    KvUnit unit;       // of a token: n = 1, no row_*
};

// Deals the batch out in shares of equal size, so that rows of any mix of lengths fill the chip evenly.  Every
// wave does it for itself: the blocks of all entries give the size of a share, and a running sum of the shares
// tells whose turn workgroup `block` is: one trip through the batch's arrays for up to 256 entries, no barrier, no idle
// workgroups between the busy ones.  Rows with fewer columns than min_columns or more than max_columns get no
// turn.  `each`: workgroups with the same share of an entry; `target`: shares times `each` wanted in all (one more
// for each entry can come out, and no more than 2 target belong to entries that are shared); least, most: blocks of
// a share at least, while that gives no more than a workgroup per CU and beyond; weigh: a unit's blocks (0: no turn).
constexpr int kComputeUnits = 256;
constexpr int kLook = 4;  // rounds of 64 entries looked at together

// Where nothing is shared, an entry for each workgroup, found without looking at the others: a token, a unit, or, for
// rows with few columns, the first or second of a row's at most two blocks.
template <bool PER_TOKEN, typename Weigh>
__device__ __forceinline__ Task deal_one(const KvTableArgs &t, const KvBatchArgs &b, int turn, int tokens, int count, int group,
                                         int min_columns, int max_columns, unsigned *flags, Weigh weigh) {
    Task r;
    r.entry = -1;
    r.split = r.place = 0;
    r.shares = 1;
    if (PER_TOKEN) {
        if (turn >= count) return r;
        r.entry = r.unit.first = turn;
        r.unit.n = 1;
        r.unit.row = b.row[turn];
        r.unit.pos = b.pos[turn];
        return r;
    }
    int i, row;
    if (max_columns == INT32_MAX) {
        if (turn >= count) return r;
        i = b.unit[turn];
        row = i >= 0 && i < b.max_tokens ? b.row[i] : -1;
    } else {
        row = turn >> 1;
        if (row >= t.rows) return r;
        i = b.start[row];
    }
    const bool known = row >= 0 && row < t.rows && i >= 0 && i < b.max_tokens;
    const int first = known ? b.start[row] : -1, end = known ? b.start[row + 1] : -1;
    int pos = known ? b.pos[i] : -1;
    if (max_columns < INT32_MAX) {
        if (end <= first) return r;  // no tokens
        if (turn & 1) {
            i += kKvBlock - (pos & (kKvBlock - 1));
            pos += kKvBlock - (pos & (kKvBlock - 1));
            if (i >= end) return r;
        }
    }
    r.unit = kv_make_unit(t, tokens, i, row, pos, first, end);
    if (r.unit.n == 0) {
        if (threadIdx.x == 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
        return r;
    }
    const int64_t columns = (int64_t)r.unit.row_n * group;
    if (columns >= min_columns && columns <= max_columns && weigh(r.unit) > 0) r.entry = turn;
    return r;
}

template <bool PER_TOKEN, typename Weigh>
__device__ __forceinline__ Task deal(const KvTableArgs &t, const KvBatchArgs &b, int block, int group, int min_columns,
                                     int max_columns, int each, int max_shares, int target, int least, int most,
                                     unsigned *flags, Weigh weigh) {
    const int lane = threadIdx.x & 63;
    const int tokens = min(b.count[0], b.max_tokens), count = PER_TOKEN ? tokens : min(b.count[1], b.max_tokens);
    // (read up to what there can be: no wait for the count)
    const int limit = PER_TOKEN ? b.max_tokens : kv_max_units(b.max_tokens, t.rows);
    Task r;
    r.entry = -1;
    KvUnit mine[kLook];
    int blocks[kLook];
    // round k of the entries from `base` on has any (the same in all lanes: small batches skip the others' work)
    auto any_in = [&](int base, int k) { return base + 64 * k < limit; };
    auto look = [&](int base) __attribute__((always_inline)) {
        int at[kLook], row[kLook], pos[kLook], s0[kLook], s1[kLook];
#pragma unroll
        for (int k = 0; k < kLook; ++k) {
            const int i = base + 64 * k + lane;
            at[k] = i >= limit ? -1 : PER_TOKEN ? i : b.unit[i];
        }
#pragma unroll
        for (int k = 0; k < kLook; ++k) {
            const bool in = at[k] >= 0 && at[k] < b.max_tokens;  // (behind the count anything may stand there)
            row[k] = in ? b.row[at[k]] : -1;
            pos[k] = in ? b.pos[at[k]] : -1;
        }
        if (!PER_TOKEN) {
#pragma unroll
            for (int k = 0; k < kLook; ++k) {
                const bool known = row[k] >= 0 && row[k] < t.rows;
                s0[k] = known ? b.start[row[k]] : -1;
                s1[k] = known ? b.start[row[k] + 1] : -1;
            }
        }
#pragma unroll
        for (int k = 0; k < kLook; ++k) {
            blocks[k] = 0;
            if (!any_in(base, k)) continue;
            const int i = base + 64 * k + lane;
            if (PER_TOKEN) {
                mine[k].row = row[k];
                mine[k].pos = pos[k];
                blocks[k] = pos[k] >= 0 && pos[k] < t.max_blocks * kKvBlock ? pos[k] / kKvBlock + 1 : 1;
            } else {
                mine[k] = kv_make_unit(t, tokens, at[k], row[k], pos[k], s0[k], s1[k]);
                if (i < count && mine[k].n == 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
                const int64_t columns = mine[k].n > 0 ? (int64_t)mine[k].row_n * group : -1;
                blocks[k] = columns >= min_columns && columns <= max_columns ? weigh(mine[k]) : 0;
            }
            if (i >= count) blocks[k] = 0;
        }
    };
    if (max_shares == 1) return deal_one<PER_TOKEN>(t, b, block / each, tokens, count, group, min_columns, max_columns, flags, weigh);
    if (!PER_TOKEN && (max_columns < INT32_MAX || limit > 64 * kLook)) {
        // often no row is for this kind of workgroup: one look at the rows alone tells
        bool any = false;
        for (int i = lane; i < t.rows; i += 64) {
            const int64_t columns = ((int64_t)b.start[i + 1] - b.start[i]) * group;
            any |= columns > 0 && columns >= min_columns && columns <= max_columns;
        }
        if (!__any(any)) return r;
    }
    int64_t all = 0;
    int longest = 0;  // of the entries of this lane
    for (int base = 0; base < limit; base += 64 * kLook) {
        look(base);
        int sum = 0;
#pragma unroll
        for (int k = 0; k < kLook; ++k) sum += blocks[k], longest = max(longest, blocks[k]);
        all += wave_sum_i(sum);
    }
    if (all == 0) return r;
    all *= each;
    const int share = (int)max(min((int64_t)most, max((int64_t)least, all / kComputeUnits)), (all + target - 1) / target);
    int turn = block / each;  // counts down to the entry
    r.place = 0;
    auto pick = [&](int base, int k, int owner) {
        auto of = [&](int v) { return __builtin_amdgcn_readlane(v, owner); };
        r.entry = base + 64 * k + owner;
        r.unit.row = of(mine[k].row);
        r.unit.pos = of(mine[k].pos);
        if (PER_TOKEN) {
            r.unit.first = r.entry;
            r.unit.n = 1;
        } else {
            r.unit.first = of(mine[k].first);
            r.unit.n = of(mine[k].n);
            r.unit.row_first = of(mine[k].row_first);
            r.unit.row_pos = of(mine[k].row_pos);
            r.unit.row_n = of(mine[k].row_n);
        }
    };
    // Shared entries first, then the others, the large before the small if they are in registers: what is
    // dispatched last should be small.
    const bool sorted = limit <= 64 * kLook;
    for (int kind = __any(longest > share) ? 0 : 1; kind < (sorted ? 1 : 2); ++kind)
        for (int base = 0; base < limit; base += 64 * kLook) {
            if (limit > 64 * kLook) look(base);
#pragma unroll
            for (int k = 0; k < kLook; ++k) {
                if (!any_in(base, k)) continue;
                int parts = min(max_shares, (int)((unsigned)(blocks[k] + share - 1) / (unsigned)share));
                if ((parts > 1) != (kind == 0)) parts = 0;
                const int upto = wave_scan_i(parts);
                const unsigned long long behind = __ballot(turn < upto);
                if (r.entry < 0 && behind) {
                    const int owner = (int)__builtin_ctzll(behind);
                    r.shares = __builtin_amdgcn_readlane(parts, owner);
                    r.split = turn - (__builtin_amdgcn_readlane(upto, owner) - r.shares);
                    r.place += __builtin_amdgcn_readlane(upto, owner) - r.shares;  // (counts for shared ones only)
                    pick(base, k, owner);
                }
                if (r.entry < 0) {
                    turn -= __builtin_amdgcn_readlane(upto, 63);
                    r.place += __builtin_amdgcn_readlane(upto, 63);
                }
            }
            if (r.entry >= 0) return r;
        }
    if (!sorted) return r;
    // the entry of one share each that has `turn` such entries before it in the order of their blocks: its number of
    // blocks by bisection, then its place among equals
    auto at_least = [&](int n) {
        int c = 0;
#pragma unroll
        for (int k = 0; k < kLook; ++k)
            if (any_in(0, k)) c += __popcll(__ballot(blocks[k] >= n && blocks[k] <= share));
        return c;
    };
    if (turn >= at_least(1)) return r;
    int lo = 1, hi = share + 1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (at_least(mid) > turn) lo = mid; else hi = mid;
    }
    turn -= at_least(lo + 1);
    r.split = 0;
    r.shares = 1;
#pragma unroll
    for (int k = 0; k < kLook; ++k) {
        if (!any_in(0, k)) continue;
        const unsigned long long equal = __ballot(blocks[k] == lo);
        if (r.entry < 0 && turn < __popcll(equal)) {
            const int before = __builtin_amdgcn_mbcnt_hi((unsigned)(equal >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)equal, 0));
            pick(0, k, (int)__builtin_ctzll(__ballot(blocks[k] == lo && before == turn)));
        }
        turn -= __popcll(equal);
    }
    return r;
}

// ---- few query columns: decode steps ------------------------------------------------------------
// S^T = K . Q^T and O^T = V^T . P^T on v_mfma_f32_16x16x32_f16, a wave on one block of 32 keys at a time.
//  * The codes are exact in f16.  q (scaled to |q| < 2 by a power of two for each column) and the
//    probabilities go in as hi + lo f16 pairs, 22 bits: of the 16 columns of a tile, 0-7 carry the hi
//    parts of eight (token, head) columns and 8-15 their lo parts, so one instruction does both.
//  * A column's probabilities of a block are scaled by a power of two that puts the largest of them into [2^14, 2^15): f16's
//    smallest step is 2^-38 of that, so a block far below the maximum keeps its 22 bits and many of them add up to what they
//    should.  The scale comes out with V's, when the block's output is added.
//  * A page is laid out as the instructions read it: a lane's operand bytes are consecutive, a wave's
//    loads are whole cache lines, and P^T comes out of the score tiles already in operand order
//    (slot e of lane group g is key 16 (e/4) + 4 g + e%4; V's layout follows).
//  * The running maximum, in whole powers of two, moves only when a score exceeds it by 8 of them: the usual block does not
//    touch the output but to add to it.  Sums are per lane until the end.
//  * The blocks of an item (token or unit, K/V head, up to 8 NT columns) go round the waves of the
//    workgroups that share it.  How many share is decided on the device, where the lengths are: a share is
//    what gives kTargetGroups shares in all, so that rows of any mix of lengths fill the chip evenly.
//    The last workgroup of an item to finish joins the partial results in a fixed order.
// Bound by the reading of the codes where there are many: 64 ragged rows up to 30000, 8 K/V heads, 377 MB: 71.5 us, 5.3 TB/s, 6.6
// between start and join (non-temporal loads; 82 with ordinary ones); one row of 131000: 50.5 us.  With few by round trips: 1 row of
// 1000, 20 heads: 10.3 us (task 2, q and pages 2.7, two blocks 2.7, publishing 1.8, joining 2.5).  A second block on its way per
// wave changed nothing (71.6, 51.6, 10.6 us): a wave has some 1800 cycles of vector work per block.
constexpr int kTokenWaves = 4;
constexpr int kTokenThreads = kTokenWaves * 64;
// Blocks a workgroup takes at least before another shares the item: 8 while that gives no more than a
// workgroup per CU, up to twice as many beyond (1 x 1000 tokens, 20 heads: 10.9 us with 8, 12.4 with 16; 16 rows of 500 to
// 4000, 5 heads: 21.0 us with 8, 17.0 with 16).  Half or twice both numbers: 1 x 4000, 8 heads, 12.8 and 12.1 us (11.4 as they
// are), 16 x 2500, 5 heads, 25.2 and 20.2 (20.8), 8 x 8000, 8 heads, 35.3 and 28.1 (33.3), 1 x 300, 20 heads, 9.6 and 7.3 (9.9).
constexpr int kMinShare = 8;
constexpr int kTargetGroups = 1536;   // workgroups that share the batch's blocks evenly
constexpr int kMaxShares = 64;        // one lane for each when they are joined; more cost more there than they gain
constexpr int kMostItems = 2048;      // more items fill the chip without sharing
constexpr int kFewColumns = 16;        // rows with no more are taken here even if others have more

// floats of one split's partial result: columns x (out, max, sum)
template <int HD, int NT>
constexpr int partial_floats() {
    return 8 * NT * (HD + 2);  // outputs by column, then maxima, then sums
}
static_assert(kMostItems <= RBN_ATTENTION_ITEMS, "a ticket for every item that is shared");

template <int HD, int NT>
struct TokenShared {
    float o[kTokenWaves][8 * NT][HD];
    _Float16 open[kKvBlock * (HD + 8)];
    v8h q[NT][HD / 32][64];
    float m[kTokenWaves][8 * NT], l[kTokenWaves][8 * NT];
    float weight[8 * NT][kMaxShares], den[8 * NT];
    int last;
};

// A share of an item, the one that deal_it() says.  Of the partial results' place every share takes room for PART_NT tiles
// of columns.
template <int FMT, int HD, int NT, int PART_NT, typename Deal>
__device__ __forceinline__ void attend_task(TokenShared<HD, NT> &shared, Deal deal_it, const float *__restrict__ q,
                                            const KvTableArgs &t, const KvLayerArgs &l, int heads, int group, int each, int rest,
                                            int kvh, int cg, float *__restrict__ partials, unsigned *__restrict__ tickets,
                                            float *__restrict__ out, unsigned *flags) {
    constexpr int KK = HD / 32;   // k steps of the scores
    constexpr int DT = HD / 16;   // tiles of dimensions of the output
    constexpr int LD = HD / 32;   // 16-byte loads per lane of 32 keys, K and V each
    constexpr int kPitch = HD + 8;
    constexpr int kTile = kKvBlock * HD;
    auto &s_o = shared.o;
    auto &s_open = shared.open;
    auto &s_q = shared.q;
    auto &s_m = shared.m, &s_l = shared.l;
    auto &s_weight = shared.weight;
    auto &s_den = shared.den;
    int &s_last = shared.last;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // the same in every lane: branches on it are scalar
    const int c16 = lane & 15, c8 = lane & 7, g = lane >> 4;
    const Task task = deal_it();
    if (task.entry < 0) return;
    const int row = task.unit.row, pos = task.unit.pos, first = task.unit.first, n = task.unit.n;
    const int split = task.split, shares = task.shares;
    const int cols = n * group;
    if (cg * 8 * NT >= cols) return;
    if (row < 0 || row >= t.rows || pos < 0 || pos + n > t.max_blocks * kKvBlock) {
        if (tid == 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
        return;
    }
    const int nblocks = (pos + n - 1) / kKvBlock + 1;
    const int stride = shares * kTokenWaves, w0 = split * kTokenWaves + wave;

    float x[NT][KK][8];  // this lane's part of its columns of q
    auto load_q = [&]() {
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) {
            const int c = min((cg * NT + ct) * 8 + c8, n * group - 1);
            const int token = c / group;
            const float *src = q + ((size_t)(first + token) * heads + kvh * group + (c - token * group)) * HD + 8 * g;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                const float4 a = *reinterpret_cast<const float4 *>(src + 32 * kk);
                const float4 z = *reinterpret_cast<const float4 *>(src + 32 * kk + 4);
                x[ct][kk][0] = a.x, x[ct][kk][1] = a.y, x[ct][kk][2] = a.z, x[ct][kk][3] = a.w;
                x[ct][kk][4] = z.x, x[ct][kk][5] = z.y, x[ct][kk][6] = z.z, x[ct][kk][7] = z.w;
            }
        }
    };
    // pages of the wave's first 64 blocks and the row's length; the unfinished block has no page
    int page = -1;
    if (w0 + lane * stride < nblocks) page = kv_page(t, row, w0 + lane * stride);
    const int len = __builtin_amdgcn_readfirstlane(min(t.len[row], t.max_blocks * kKvBlock));
    load_q();
    if (pos + n > len) {
        if (tid == 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
        return;
    }
    const int full_blocks = min(len / kKvBlock, nblocks);
    const int mine = full_blocks > w0 ? (full_blocks - w0 + stride - 1) / stride : 0;

    // Codes of a block: LD 16-byte loads each for K and V (an invalid page loads page 0 and is skipped).
    v4u kc[LD], vc[LD];
    auto load = [&](v4u (&to)[LD], const uint8_t *codes, int pg) {
        const v4u *src =
            reinterpret_cast<const v4u *>(codes + ((size_t)max(pg, 0) * l.kv_heads + kvh) * (kKvBlock * HD)) + lane;
#pragma unroll
        for (int j = 0; j < LD; ++j) to[j] = __builtin_nontemporal_load(src + 64 * j);
    };
    float ks = 0.0f, vs = 0.0f;
    auto load_scales = [&](int steps) {
        if (lane < steps) {
            const size_t ph = (size_t)max(page, 0) * l.kv_heads + kvh;
            ks = l.k_scale[ph];
            vs = l.v_scale[ph];
            if (page < 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
        }
    };
    if (mine > 0) {
        load(kc, l.k, __builtin_amdgcn_readlane(page, 0));
        load(vc, l.v, __builtin_amdgcn_readlane(page, 0));
        load_scales(min(64, mine));
    }
    __builtin_amdgcn_sched_barrier(0);

    // Q^T operand and what belongs to a column.  A wave prepares every kTokenWaves-th k step for all.
    v8h qf[NT][KK];
    float col_scale[NT];   // 2^e log2(e) / sqrt(hd): raw score x K scale x this is an exponent of two
    int col_pos[NT];
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
        col_pos[ct] = pos + min((cg * NT + ct) * 8 + c8, cols - 1) / group;
        float m = 0.0f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[ct][kk][e]));
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        const int ex = exponent_of(m);
        col_scale[ct] = ldexpf(HD == 128 ? kLog2eBySqrt128 : kLog2eBySqrt64, ex);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
            if (wave == kk % kTokenWaves) {
                v8h z;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float v = ldexpf(x[ct][kk][e], -ex);
                    const float hi = (float)(_Float16)v;
                    z[e] = (_Float16)(c16 < 8 ? hi : v - hi);
                }
                s_q[ct][kk][lane] = z;
            }
    }
    __syncthreads();
#pragma unroll
    for (int ct = 0; ct < NT; ++ct)
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) qf[ct][kk] = s_q[ct][kk][lane];

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
        float vs_up[NT];
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
            m = floorf(column_max(m));
            if (__any(m > run_max[ct] + 8.0f)) {
                const float top = fmaxf(run_max[ct], m);
                const float corr = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(run_max[ct] - top);
                run_max[ct] = top;
                run_sum[ct] *= corr;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[ct][d] *= corr;
            }
            // the block's weights on a scale of their own, the largest in [2^14, 2^15), and that scale in units of the output
            // (scores beyond 2^24 have no bits left to take 14 off)
            const bool none = m == -INFINITY;
            const float unit = none ? 0.0f : m - (fabsf(m) < 16777216.0f ? 14.0f : 0.0f);
            const float up = none ? 0.0f : __builtin_amdgcn_exp2f(unit - run_max[ct]);
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float p = __builtin_amdgcn_exp2f(x[e] - unit);
                sum += p;
                const _Float16 hi = (_Float16)p, lo = (_Float16)(p - (float)hi);
                pf[ct][e] = c16 < 8 ? hi : lo;
            }
            run_sum[ct] = fmaf(sum, up, run_sum[ct]);
            vs_up[ct] = vscale * up;
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const v8h vf = value(d);
#pragma unroll
            for (int ct = 0; ct < NT; ++ct) {
                const v4f z = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[ct], v4f{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
                for (int r = 0; r < 4; ++r) o[ct][d][r] = fmaf(z[r], vs_up[ct], o[ct][d][r]);
            }
        }
    };

    // full blocks: this wave's w0, w0 + stride, ...
    for (int base = 0; base < mine; base += 64) {
        const int steps = min(64, mine - base);
        if (base > 0) {
            page = -1;
            if (lane < steps) page = kv_page(t, row, w0 + (base + lane) * stride);
            load(kc, l.k, __builtin_amdgcn_readlane(page, 0));
            load(vc, l.v, __builtin_amdgcn_readlane(page, 0));
            load_scales(steps);
        }
        auto step = [&](int i, auto more) {
            const int here = __builtin_amdgcn_readlane(page, i);
            const int next = more.value ? __builtin_amdgcn_readlane(page, i + 1) : 0;
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
            if (more.value) load(kc, l.k, next);
            if (here >= 0)
                attend(s,
                       [&](int d) {
                           const v4u w = vc[d / 2];
                           return d & 1 ? codes_to_f16<FMT>(w.z, w.w) : codes_to_f16<FMT>(w.x, w.y);
                       },
                       __int_as_float(__builtin_amdgcn_readlane(__float_as_int(ks), i)),
                       __int_as_float(__builtin_amdgcn_readlane(__float_as_int(vs), i)),
                       (w0 + (base + i) * stride) * kKvBlock);
            if (more.value) load(vc, l.v, next);
        };
        // the next block's keys travel during the softmax, its values during its scores
        for (int i = 0; i < steps - 1; ++i) step(i, std::true_type());
        step(steps - 1, std::false_type());
    }
    // the unfinished block, f16: K straight from the buffer, V transposed through LDS; rows behind
    // the end may hold anything, so V's are zeroed (K's scores are masked)
    if (nblocks > full_blocks && full_blocks % stride == w0) {
        const size_t at = ((size_t)row * l.kv_heads + kvh) * kKvBlock * HD;
        const _Float16 *ko = reinterpret_cast<const _Float16 *>(l.k_open) + at;
        const _Float16 *vo = reinterpret_cast<const _Float16 *>(l.v_open) + at;
        const int valid = len - full_blocks * kKvBlock;
        v8h kf[2][KK], vx[kTile / 512];
        const unsigned k0 = c16 * HD + 8 * g, v0 = lane * 8;
#pragma unroll
        for (int j = 0; j < kTile / 512; ++j) vx[j] = *reinterpret_cast<const v8h *>(vo + (v0 + j * 512));
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) kf[a][kk] = *reinterpret_cast<const v8h *>(ko + (k0 + 16 * a * HD + 32 * kk));
        __builtin_amdgcn_sched_barrier(0);  // all on their way before the first is waited for
#pragma unroll
        for (int j = 0; j < kTile / 512; ++j) {
            const int key = (v0 + j * 512) / HD, d = (v0 + j * 512) % HD;
            if (key >= valid) vx[j] = v8h{0, 0, 0, 0, 0, 0, 0, 0};
            *reinterpret_cast<v8h *>(s_open + key * kPitch + d) = vx[j];
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
    const int slot = task.entry * each + rest;  // used by shared items only
    float *part = partials + ((size_t)task.place * each + (size_t)rest * shares) * partial_floats<HD, PART_NT>();
    auto write_out = [&](int c, int d, v4f num, float den) {
        const int col = cg * 8 * NT + c, token = col / group;
        const float inv = den > 0.0f || den != den ? 1.0f / den : 0.0f;
        *reinterpret_cast<v4f *>(out + ((size_t)(first + token) * heads + kvh * group + (col - token * group)) * HD + d) =
            num * inv;
    };
    for (int i = tid; i < ncols * (HD / 4); i += kTokenThreads) {
        const int c = i / (HD / 4), d = i % (HD / 4) * 4;
        float wm[kTokenWaves], wl[kTokenWaves], m = -INFINITY, den = 0.0f;
        v4f num = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kTokenWaves; ++w) {
            wm[w] = s_m[w][c];
            wl[w] = s_l[w][c];
            m = fmaxf(m, wm[w]);
        }
#pragma unroll
        for (int w = 0; w < kTokenWaves; ++w) {
            // a wave that saw no key has sum 0; one that saw a NaN only has maximum -inf and a NaN sum
            const float k = wm[w] == -INFINITY ? (wl[w] != 0.0f ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(wm[w] - m);
            num += k * *reinterpret_cast<const v4f *>(&s_o[w][c][d]);
            den += k * wl[w];
        }
        if (shares == 1) {
            write_out(c, d, num, den);
        } else {
            float *p = part + (size_t)split * partial_floats<HD, NT>();
            store_agent(p + c * HD + d, num);
            if (d == 0) {
                store_agent(p + 8 * NT * HD + c, m);
                store_agent(p + 8 * NT * (HD + 1) + c, den);
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
        if (s_last) {
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
            // outputs in quads; `lots` threads share one and meet in LDS.  The first loads go out before
            // the weights are known.
            const int quads = ncols * (HD / 4), lots = max(1, kTokenThreads / quads);
            const int my_quad = tid % quads, my_lot = tid / quads;
            const v4f *p0 = reinterpret_cast<const v4f *>(part) + my_quad;
            constexpr int kAhead = 8;
            v4f ahead[kAhead];
            if (my_lot < lots)
#pragma unroll
                for (int j = 0; j < kAhead; ++j)
                    ahead[j] = p0[(size_t)min(my_lot + j * lots, shares - 1) * (partial_floats<HD, NT>() / 4)];
            // weights: a wave per column, a lane per share
            for (int c = wave; c < ncols; c += kTokenWaves) {
                float pm = -INFINITY, pl = 0.0f;
                if (lane < shares) {
                    const float *p = part + (size_t)lane * partial_floats<HD, NT>() + 8 * NT * HD + c;
                    pm = load_agent(p);
                    pl = load_agent(p + 8 * NT);
                }
                const float m = wave_max(pm);
                const float k = pm == -INFINITY ? (pl != 0.0f ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(pm - m);
                const float den = wave_sum(k * pl);
                s_weight[c][lane] = k;
                if (lane == 0) s_den[c] = den;
            }
            __syncthreads();
            v4f *s_acc = reinterpret_cast<v4f *>(&s_o[0][0][0]);
            for (int i = tid; i < quads * lots; i += kTokenThreads) {
                const int quad = i % quads, lot = i / quads, c = quad / (HD / 4);
                const v4f *p = reinterpret_cast<const v4f *>(part) + quad;
                v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
                auto add = [&](v4f z, int sp) {
                    const float k = s_weight[c][sp];
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[r] = fmaf(k, z[r], acc[r]);
                };
                int sp = lot;
                if (i == tid) {
#pragma unroll
                    for (int j = 0; j < kAhead; ++j)
                        if (lot + j * lots < shares) add(ahead[j], lot + j * lots);
                    sp += kAhead * lots;
                }
#pragma unroll 8
                for (; sp < shares; sp += lots) add(p[(size_t)sp * (partial_floats<HD, NT>() / 4)], sp);
                s_acc[i] = acc;
            }
            __syncthreads();
            for (int i = tid; i < quads; i += kTokenThreads) {
                const int c = i / (HD / 4), d = i % (HD / 4) * 4;
                v4f num = s_acc[i];
                for (int lot = 1; lot < lots; ++lot) num += s_acc[lot * quads + i];
                write_out(c, d, num, s_den[c]);
            }
        }
    }
}

// ---- many query columns: prompts -------------------------------------------------------------------
// The same products on v_mfma_f32_32x32x16_f16, a wave with 32 queries (one block of positions of one head)
// against blocks of 32 keys.
//  * The (block, head) pairs of a row and a K/V head are numbered block by block; the four waves of a
//    workgroup take four in a row and share the keys and values, which the workgroup converts
//    once to f16 in LDS, in operand order: every operand read is one conflict-free 16-byte read per lane.
//  * q and P in f16 as hi + lo, two instructions each (a tile has 32 columns of its own here).  V's scale goes
//    into P, as its logarithm in the exponent (off by 2^-20 of it at most, at 2^-32); the output is kept in units of a
//    power of two near the scales so far.  Scales within [2^-4, 4) of the unit use it as it is, others move it (the
//    store's scales span 2^-32 .. 2^9), the running maximum lags behind by up to 2^4, and P is shifted up by 2^9: its
//    parts reach at most 2^15.  Where V's scale is the unit, a weight is off by up to 2^-34 of the largest (half of f16's
//    smallest step), so L keys far below it by up to L 2^-34 of V's largest together: 128 u with 131072 keys, u = 2^-24, a
//    third of what sums of as many terms round by.  (The output is summed up inside the matrix instructions, so a block's
//    weights cannot have a scale of their own as they have above.)
//  * Every block before a wave's own is full and unmasked, its own is masked, later ones are skipped.
// Bound by the matrix instructions where there is much to do: five prompts of 268 to 1248 behind up to 1631 positions, 20 / 5 heads:
// 59 us, 345 TFLOP/s (690 with the lo parts); 2750 cycles for a block of a workgroup in the loop, 2110 of them matrix instructions
// of the SIMD's two waves.  One prompt of 512, 20 heads: 24.7 us, latency (task 4, q, pages and first codes 5, blocks 10, join 5).
constexpr int kPromptThreads = 256;
// Powers of two that the running maximum may lag behind, and log2 of what P is scaled up by.  A lag moves the output less often (five
// ragged prompts: 59.6 us with 8, 60.4 with 4, 60.9 with 3) and leaves P as many bits less.
constexpr int kLag = 4, kShift = 13 - kLag;
// Shares in all (five ragged prompts: 61.4 us with 256, 59.7 with 288; the same with either: 5 x 700 behind 900 positions, 20 / 5
// heads, 116 us, 8 x 300 behind 500, 20 heads, 57, 2 x 1500 behind 1000, 32 / 8 heads, 184).
constexpr int kPromptTargetGroups = 288;
// blocks a workgroup takes at least before another shares the tile: partial results cost some 10 us to write, wait for
// and join, a block 0.75 (one prompt of 512, 20 heads: 27.2 us with 4, 25.5 with 8, 24.7 with 12, 27.9 with 16 or none shared;
// 512, 20 / 5 heads: 24.1 with 8 and 12, 27.1 with 16; 1000, 20 heads: 42.5 with 8 and 12, 36.2 with 16)
constexpr int kPromptMinShare = 12;
constexpr int kPromptMaxShares = 16;

// floats of one workgroup's partial result: four waves' registers, maxima and sums, lane by lane
template <int HD>
constexpr int prompt_partial_floats() {
    return 4 * 64 * (HD / 2 + 2);
}

template <int HD>
struct PromptShared {
    _Float16 k[3][kKvBlock * HD], v[3][kKvBlock * HD];
    v4f scale[4][64];
    int page[4][64], ve[4][64], last;
};

template <int FMT, int HD>
__device__ __forceinline__ void attend_prompts(PromptShared<HD> &shared, int block, const float *__restrict__ q,
                                               const KvTableArgs &t, const KvBatchArgs &b, const KvLayerArgs &l, int heads,
                                               int max_shares, int min_columns, float *__restrict__ partials,
                                               unsigned *__restrict__ tickets, float *__restrict__ out, unsigned *flags) {
    constexpr int KK = HD / 16;   // k steps of the scores
    constexpr int NT = HD / 32;   // tiles of dimensions of the output
    constexpr int kTile = kKvBlock * HD;
    constexpr int PER = kTile / kPromptThreads;  // codes of K (and of V) a thread converts: 16 or 8
    auto &s_k = shared.k, &s_v = shared.v;
    auto &s_scale = shared.scale;
    auto &s_page = shared.page, &s_ve = shared.ve;
    int &s_last = shared.last;
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, g = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);  // the same in every lane: branches on it are scalar
    const int group = heads / l.kv_heads;
    const int per_unit = (group + 3) / 4;
    const int each = l.kv_heads * per_unit, rest = block % each, kvh = rest % l.kv_heads, z = rest / l.kv_heads;
    // a unit counts for the workgroups whose first pair is in it, with the blocks of the first of them
    auto weigh = [group](const KvUnit &u) {
        const int first_block = u.row_pos / kKvBlock, last_block = (u.row_pos + u.row_n - 1) / kKvBlock;
        const int nth = u.pos / kKvBlock - first_block, pair0 = ((nth * group + 3) >> 2) * 4;
        if (pair0 >= (nth + 1) * group) return 0;
        return first_block + min(pair0 + 3, (last_block - first_block + 1) * group - 1) / group + 1;
    };
    const Task task = deal<false>(t, b, block, group, min_columns, INT32_MAX, each, max_shares, kPromptTargetGroups,
                                  kPromptMinShare, kPromptMinShare, flags, weigh);
    if (task.entry < 0) return;
    const KvUnit unit = task.unit;
    const int item = task.entry * each + rest;  // used by shared tiles only
    // the workgroups whose first pair is in this unit
    const int first_block = unit.row_pos / kKvBlock, last_block = (unit.row_pos + unit.row_n - 1) / kKvBlock;
    const int nth = unit.pos / kKvBlock - first_block;
    const int pair0 = (((nth * group + 3) >> 2) + z) * 4;
    if (pair0 >= (nth + 1) * group) return;
    const int pairs = (last_block - first_block + 1) * group;
    const int pair = pair0 + wave;
    const bool idle = pair >= pairs;
    const int own = idle ? -1 : first_block + pair / group;               // this wave's block of positions
    const int top = first_block + min(pair0 + 3, pairs - 1) / group;      // the workgroup's last
    const int head = kvh * group + (idle ? 0 : pair % group);
    const int query = own * kKvBlock + col;                               // this lane's position
    const bool real = !idle && query >= unit.row_pos && query < unit.row_pos + unit.row_n;
    const int token = unit.row_first + min(max(query - unit.row_pos, 0), unit.row_n - 1);

    // this workgroup's share of blocks 0 .. top: `from` .. `to`; the last share also takes the unfinished block
    const int split = task.split, shares = task.shares;
    const int part_blocks = (top + shares) / shares;
    const int from = split * part_blocks;

    // q, the pages of the share's first blocks and the row's length together; then the first codes, and q is
    // made ready while those travel
    int first_pages = -1;
    if (lane < part_blocks && from + lane <= top) first_pages = kv_page(t, unit.row, from + lane);
    float x[KK][8];
    {
        const float *src = q + ((size_t)token * heads + head) * HD + 8 * g;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const float4 a = *reinterpret_cast<const float4 *>(src + 16 * kk);
            const float4 c = *reinterpret_cast<const float4 *>(src + 16 * kk + 4);
            x[kk][0] = a.x, x[kk][1] = a.y, x[kk][2] = a.z, x[kk][3] = a.w;
            x[kk][4] = c.x, x[kk][5] = c.y, x[kk][6] = c.z, x[kk][7] = c.w;
        }
    }
    const int len = __builtin_amdgcn_readfirstlane(min(t.len[unit.row], t.max_blocks * kKvBlock));
    if (unit.row_pos + unit.row_n > len) {
        if (tid == 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
        return;
    }
    const int full = min(len / kKvBlock, top + 1);                        // full blocks among 0 .. top
    const int to = min(from + part_blocks, full), last = to - 1;

    typedef typename CodeVec<PER>::type vcode;  // a thread's codes of one page head
    struct Codes {
        vcode k, v;
    };
    auto load = [&](Codes &c, int page) __attribute__((always_inline)) {  // (an invalid page loads page 0 and is skipped)
        const size_t at = ((size_t)max(page, 0) * l.kv_heads + kvh) * kTile;
        c.k = *reinterpret_cast<const vcode *>(l.k + at + tid * PER);
        c.v = *reinterpret_cast<const vcode *>(l.v + at + tid * PER);
    };
    // What is known of a block: page (-1: skipped), K's scale, and of V's the exponent (kNone: it is 0), logarithm
    // and reciprocal.  A wave keeps this of 64 blocks in LDS: in registers, their loads would be waited for
    // together with the codes that are on their way.
    struct Block {
        int page, ve;
        float ks, vlog, vinv;
    };
    constexpr int kNone = 1000;
    auto fetch = [&](int kb, Codes &c) __attribute__((always_inline)) {  // puts block kb's codes on their way
        const int at = (kb - from) & 63;
        float ks = 0.0f, vs = 0.0f;
        if (at == 0) {
            int page = kb == from ? first_pages : -1;
            if (kb != from && kb + lane < to) page = kv_page(t, unit.row, kb + lane);
            if (kb + lane < to) {
                const size_t ph = (size_t)max(page, 0) * l.kv_heads + kvh;
                ks = l.k_scale[ph];
                vs = l.v_scale[ph];
                if (page < 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
            }
            s_page[wave][lane] = page;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        Block x;
        x.page = __builtin_amdgcn_readfirstlane(s_page[wave][at]);
        load(c, x.page);
        if (at == 0) {
            const bool some = vs > 0.0f;
            s_ve[wave][lane] = some ? exponent_of(vs) : kNone;
            s_scale[wave][lane] = (v4f){ks, some ? __builtin_amdgcn_logf(vs) : 0.0f, some ? 1.0f / vs : 1.0f, 0.0f};
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
        x.ve = __builtin_amdgcn_readfirstlane(s_ve[wave][at]);
        const v4f z = s_scale[wave][at];
        x.ks = z[0];
        x.vlog = z[1];
        x.vinv = z[2];
        return x;
    };
    Codes even, odd;
    Block x0{-1, kNone, 0.0f, 0.0f, 1.0f}, x1 = x0;
    if (from < to) {
        x0 = fetch(from, even);
        x1 = fetch(min(from + 1, last), odd);
    }
    __builtin_amdgcn_sched_barrier(0);

    v8h qhi[KK], qlo[KK];
    float col_scale;
    {
        float m = 0.0f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(x[kk][e]));
        m = fmaxf(m, __shfl_xor(m, 32));
        const int ex = exponent_of(m);
        const float down = ldexpf(1.0f, -ex);
        col_scale = ldexpf(HD == 128 ? kLog2eBySqrt128 : kLog2eBySqrt64, ex);
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float v0 = x[kk][e] * down, v1 = x[kk][e + 1] * down;
                const v2h hi = __builtin_convertvector((v2f){v0, v1}, v2h);
                const v2h lo = __builtin_convertvector(((v2f){v0 - (float)hi[0], v1 - (float)hi[1]}), v2h);
                qhi[kk][e] = hi[0], qhi[kk][e + 1] = hi[1];
                qlo[kk][e] = lo[0], qlo[kk][e + 1] = lo[1];
            }
    }

    float run_max = -INFINITY, run_sum = 0.0f;
    float limit = -INFINITY;  // the running maximum follows scores above this
    int vexp = -200;  // exponent of the output's unit; none yet
    v16f o[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[nt][r] = 0.0f;

    // scores of the 32 keys in buffer `buf`: register r is key 8 (r/4) + 4 g + r%4
    auto scores = [&](int buf) __attribute__((always_inline)) {
        v16f s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.0f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const v8h ka = *reinterpret_cast<const v8h *>(&s_k[buf][(kk * 64 + lane) * 8]);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, qhi[kk], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x16_f16(ka, qlo[kk], s, 0, 0, 0);
        }
        return s;
    };
    auto max_of = [&](const v16f &s) __attribute__((always_inline)) {
        float m = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) m = fmaxf(m, s[r]);
        return m;
    };
    // What the softmax of a block needs besides its raw scores s and their maximum m (before the masks of a
    // diagonal block): masks, a running maximum that is near enough, the output's unit.
    // f: raw score times this is an exponent of two (at least the smallest normal, so that a masked -inf stays
    // one where the scale is 0); bias: minus the maximum plus log2 of P's shift; inverse: of that shift.
    float f, bias, inverse;
    auto settle = [&](v16f &s, float m, const Block &x, bool diagonal) __attribute__((always_inline)) {
        if (x.ve != kNone && (x.ve < vexp - 4 || x.ve > vexp + 1)) {  // the unit of the output follows V's scale
            if (vexp > -200) {
                const float by = ldexpf(1.0f, vexp - x.ve);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[nt][r] *= by;
            }
            vexp = x.ve;
        }
        f = fmaxf(x.ks * col_scale, 1.17549435e-38f);
        if (diagonal) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 8 * (r >> 2) + 4 * g + (r & 3) <= col ? s[r] : -INFINITY;
            m = max_of(s);
        }
        m *= f;
        bool apart = false;  // the maximum is off the scores already
        if (__any(m > limit)) {
            m = fmaxf(m, __shfl_xor(m, 32));
            const float mx = fmaxf(run_max, m);
            const float corr = mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(run_max - mx);
            run_max = mx;
            run_sum *= corr;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[nt][r] *= corr;
            const float ref = run_max == -INFINITY ? 0.0f : run_max;
            apart = __any(fabsf(ref) > 1048576.0f);
            limit = apart ? -INFINITY : run_max + (float)kLag;
            if (apart) {
                // with so large a maximum the bias would have too few bits left: it comes off the scores first, in every block
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = s[r] * f - ref;
                f = 1.0f;
            }
        }
        // (a block of V's that is all zero: any shift will do)
        const int shift = x.ve != kNone ? kShift - vexp : 0;
        bias = x.vlog + (float)shift - (run_max == -INFINITY || apart ? 0.0f : run_max);
        inverse = ldexpf(x.vinv, -shift);
    };
    // P of the raw scores r and r + 1 as f16 hi + lo; returns their sum.
    v8h phi[2], plo[2];
    auto soften = [&](const v16f &s, int r) __attribute__((always_inline)) {
        const float w0 = __builtin_amdgcn_exp2f(fmaf(s[r], f, bias)), w1 = __builtin_amdgcn_exp2f(fmaf(s[r + 1], f, bias));
        const v2h hi = __builtin_convertvector((v2f){w0, w1}, v2h);
        const v2h lo = __builtin_convertvector(((v2f){w0 - (float)hi[0], w1 - (float)hi[1]}), v2h);
        phi[r >> 3][r & 7] = hi[0];
        phi[r >> 3][(r & 7) + 1] = hi[1];
        plo[r >> 3][r & 7] = lo[0];
        plo[r >> 3][(r & 7) + 1] = lo[1];
        return w0 + w1;
    };
    auto key_operand = [&](int buf, int kk) __attribute__((always_inline)) {
        return *reinterpret_cast<const v8h *>(&s_k[buf][(kk * 64 + lane) * 8]);
    };
    auto value_operand = [&](int buf, int i) __attribute__((always_inline)) {  // dimensions 32 (i/2) .., key slots of step i%2
        return *reinterpret_cast<const v8h *>(&s_v[buf][(i * 64 + lane) * 8]);
    };
    // Softmax and P.V of the block in buffer b0 whose raw scores are s; leaves the raw scores of the block in b1 in s
    // and their maximum in m;
    // `piece(i)`, i < 2 PER / 8, is other work for the vector units.  Written in the order it is to run in
    // (the barriers keep the compiler from gathering the operand reads right before their uses and the vector work
    // in one place): operands two reads ahead, the softmax between the matrix instructions of the scores,
    // the pieces between those of P.V.
    auto attend = [&](v16f &s, float &m, int b0, int b1, auto piece) __attribute__((always_inline)) {
        v16f z;
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] = 0.0f;
        v8h a[3];
        a[0] = key_operand(b1, 0);
        a[1] = key_operand(b1, 1);
        float sum = 0.0f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            a[(kk + 2) % 3] = kk + 2 < KK ? key_operand(b1, kk + 2) : value_operand(b0, kk + 2 - KK);
            z = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[kk % 3], qhi[kk], z, 0, 0, 0);
            z = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[kk % 3], qlo[kk], z, 0, 0, 0);
#pragma unroll
            for (int r = kk * 16 / KK; r < (kk + 1) * 16 / KK; r += 2) sum += soften(s, r);
            __builtin_amdgcn_sched_barrier(0);
        }
        run_sum = fmaf(sum, inverse, run_sum);  // the shift comes out of the sum as it went into P
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) {
            if (i + 2 < 2 * NT) a[(KK + i + 2) % 3] = value_operand(b0, i + 2);
            o[i / 2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[(KK + i) % 3], phi[i % 2], o[i / 2], 0, 0, 0);
            o[i / 2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[(KK + i) % 3], plo[i % 2], o[i / 2], 0, 0, 0);
            if (i % 2 == 0) piece(i / 2);
            // their maximum, with a delay that spares the wait for the last of the scores
            if (i >= 2 * NT - 2) {
                const int from = i == 2 * NT - 2 ? 0 : 8;
                if (from == 0) m = z[0];
#pragma unroll
                for (int r = from; r < from + 8; ++r) m = fmaxf(m, z[r]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        s = z;
    };

    // ---- the unfinished block first, if it is this share's: f16, rows behind the end zeroed
    if (top >= full && split == shares - 1) {
        const size_t at = ((size_t)unit.row * l.kv_heads + kvh) * kTile;
        const _Float16 *ko = reinterpret_cast<const _Float16 *>(l.k_open) + at;
        const _Float16 *vo = reinterpret_cast<const _Float16 *>(l.v_open) + at;
        const int valid = len - full * kKvBlock;
        for (int i = tid; i < kTile / 8; i += kPromptThreads) {
            const int key = i / (HD / 8), d = i % (HD / 8) * 8;
            v8h kx = *reinterpret_cast<const v8h *>(ko + key * HD + d), vx = *reinterpret_cast<const v8h *>(vo + key * HD + d);
            if (key >= valid) kx = vx = v8h{0, 0, 0, 0, 0, 0, 0, 0};
            *reinterpret_cast<v8h *>(&s_k[0][((d >> 4) * 64 + 32 * ((d >> 3) & 1) + key) * 8]) = kx;
            const int quad = (key & 15) >> 2, e = 4 * (quad >> 1) + (key & 3);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                s_v[0][(((d >> 5) * 2 + (key >> 4)) * 64 + 32 * (quad & 1) + ((d + j) & 31)) * 8 + e] = vx[j];
        }
        __syncthreads();
        if (own == top) {
            v16f s = scores(0);
            float m;
            settle(s, 0.0f, Block{0, 0, 1.0f, 0.0f, 1.0f}, true);
            attend(s, m, 0, 0, [](int) {});
        }
        __syncthreads();
    }

    // ---- the share's full blocks
    // Piece i of the conversion of a thread's codes: keys or values of its i/2-th eight (kv_k_byte, kv_v_byte).
    constexpr int kPieces = 2 * PER / 8;
    auto convert_piece = [&](const Codes &c, int buf, int piece) __attribute__((always_inline)) {
        const int h = piece >> 1, byte = tid * PER + 8 * h, chunk = byte >> 4, hh = (byte >> 3) & 1, i = chunk & 15;
        if (piece & 1) {
            const int quad = (chunk >> 4) & 3, p = chunk >> 6;
            const v8h x = codes_to_f16<FMT>(c.v[2 * h], c.v[2 * h + 1]);  // keys 4 quad .. +3, then 16 + 4 quad ..
#pragma unroll
            for (int a = 0; a < 2; ++a)
                *reinterpret_cast<v4h *>(&s_v[buf][((p * 2 + a) * 64 + 32 * (quad & 1) + 16 * hh + i) * 8 + 4 * (quad >> 1)]) =
                    a ? __builtin_shufflevector(x, x, 4, 5, 6, 7) : __builtin_shufflevector(x, x, 0, 1, 2, 3);
        } else {
            const int gg = (chunk >> 4) & 3, aj = chunk >> 6, a = aj / (HD / 64), j = aj % (HD / 64);
            const int kk = (2 * j + hh) * 2 + (gg >> 1);
            *reinterpret_cast<v8h *>(&s_k[buf][(kk * 64 + 32 * (gg & 1) + 16 * a + i) * 8]) =
                codes_to_f16<FMT>(c.k[2 * h], c.k[2 * h + 1]);
        }
    };
    auto convert = [&](const Codes &c, int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) convert_piece(c, buf, i);
    };
    static_assert(kPieces <= NT, "a piece for every second operand of P.V at most");
    // Pipeline, one barrier per block: while block i's softmax runs on the vector units the matrix units do the
    // scores of block i + 1, block i + 2 is converted into the third buffer, and blocks i + 3 and i + 4 are
    // on their way.
    if (from < to) {
        convert(even, 0);
        Block x2 = fetch(min(from + 2, last), even);
        convert(odd, 1);
        Block x3 = fetch(min(from + 3, last), odd);
        __syncthreads();
        v16f s = scores(0);
        float m = max_of(s);
        int b0 = 0, b1 = 1, b2 = 2;  // buffers of blocks i, i + 1, i + 2
        auto step = [&](int kb, Codes &c) __attribute__((always_inline)) {
            if (kb <= own && x0.page >= 0) {
                settle(s, m, x0, kb == own);
                // (behind the last block the codes are old ones, and never read)
                attend(s, m, b0, b1, [&](int i) __attribute__((always_inline)) {
                    if (i < kPieces) convert_piece(c, b2, i);
                });
            } else {
                if (kb < own) s = scores(b1), m = max_of(s);
                convert(c, b2);
            }
            x0 = x1, x1 = x2, x2 = x3;
            // (behind the last block its codes once more: without a branch the wait for a block's codes leaves
            // the next one's on their way)
            x3 = fetch(min(kb + 4, last), c);
            const int b = b0;
            b0 = b1, b1 = b2, b2 = b;
            __syncthreads();
        };
        int kb = from;
        for (; kb < last; kb += 2) {
            step(kb, even);
            step(kb + 1, odd);
        }
        if (kb == last) step(kb, even);
    }

    run_sum += __shfl_xor(run_sum, 32);
    const float unit_out = vexp > -200 ? ldexpf(1.0f, vexp - kShift) : 0.0f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[nt][r] *= unit_out;
    if (shares > 1) {
        float *part = partials + ((size_t)task.place * each + (size_t)rest * shares) * prompt_partial_floats<HD>();
        float *mine = part + (size_t)split * prompt_partial_floats<HD>() + wave * 64 * (HD / 2 + 2);
#pragma unroll
        for (int i = 0; i < 4 * NT; ++i)
            store_agent(mine + (i * 64 + lane) * 4,
                        (v4f){o[i / 4][i % 4 * 4], o[i / 4][i % 4 * 4 + 1], o[i / 4][i % 4 * 4 + 2], o[i / 4][i % 4 * 4 + 3]});
        store_agent(mine + 64 * (HD / 2) + lane, run_max);
        store_agent(mine + 64 * (HD / 2 + 1) + lane, run_sum);
        // published once the stores have completed (vmcnt(0): this wave's, the barrier: everybody's)
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (tid == 0) {
            const int is_last = atomicAdd(&tickets[item], 1u) == (unsigned)shares - 1;
            if (is_last) atomicExch(&tickets[item], 0u);  // ready for the next launch
            s_last = is_last;
        }
        __syncthreads();
        if (!s_last) return;
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
        const float *other = part + wave * 64 * (HD / 2 + 2);
        float m = -INFINITY, pm[kPromptMaxShares];
#pragma unroll
        for (int sp = 0; sp < kPromptMaxShares; ++sp)
            pm[sp] = sp < shares ? load_agent(other + (size_t)sp * prompt_partial_floats<HD>() + 64 * (HD / 2) + lane) : -INFINITY;
#pragma unroll
        for (int sp = 0; sp < kPromptMaxShares; ++sp) m = fmaxf(m, pm[sp]);
        run_sum = 0.0f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[nt][r] = 0.0f;
#pragma unroll 1
        for (int sp = 0; sp < shares; ++sp) {
            const float *p = other + (size_t)sp * prompt_partial_floats<HD>();
            v4f z[4 * NT];
#pragma unroll
            for (int i = 0; i < 4 * NT; ++i) z[i] = *reinterpret_cast<const v4f *>(p + (i * 64 + lane) * 4);
            const float pmax = p[64 * (HD / 2) + lane], pl = p[64 * (HD / 2 + 1) + lane];
            // a share without keys for this query has sum 0; one with nothing but NaN maximum -inf and a NaN sum
            const float k = pmax == -INFINITY ? (pl != 0.0f ? 1.0f : 0.0f) : __builtin_amdgcn_exp2f(pmax - m);
            run_sum = fmaf(k, pl, run_sum);
#pragma unroll
            for (int i = 0; i < 4 * NT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[i / 4][i % 4 * 4 + r] = fmaf(k, z[i][r], o[i / 4][i % 4 * 4 + r]);
        }
    }
    if (!real) return;
    const float inv = run_sum > 0.0f || run_sum != run_sum ? 1.0f / run_sum : 0.0f;
    float *dst = out + ((size_t)token * heads + head) * HD + 4 * g;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4)
            *reinterpret_cast<float4 *>(dst + 32 * nt + 8 * r4) =
                make_float4(o[nt][4 * r4] * inv, o[nt][4 * r4 + 1] * inv, o[nt][4 * r4 + 2] * inv, o[nt][4 * r4 + 3] * inv);
}

// The task of workgroup `block` of those for few columns: an item (token or unit, K/V head, tile of columns) and a share
// of its blocks.
template <bool PER_TOKEN>
__device__ __forceinline__ Task deal_tokens(const KvTableArgs &t, const KvBatchArgs &b, int block, int group, int max_columns,
                                            int each, int max_shares, unsigned *flags) {
    return deal<PER_TOKEN>(t, b, block, group, 0, max_columns, each, max_shares, kTargetGroups, kMinShare, 2 * kMinShare, flags,
                           [](const KvUnit &u) { return u.pos / kKvBlock + 1; });
}

// One token per row.
template <int FMT, int HD, int NT>
__global__ __launch_bounds__(kTokenThreads, NT == 1 ? 3 : 2) void attention_token_kernel(
    const float *__restrict__ q, KvTableArgs t, KvBatchArgs b, KvLayerArgs l, int heads, int tiles, int max_shares,
    float *__restrict__ partials, unsigned *__restrict__ tickets, float *__restrict__ out, unsigned *flags) {
    __shared__ __attribute__((aligned(16))) TokenShared<HD, NT> shared;
    const int group = heads / l.kv_heads, each = l.kv_heads * tiles, rest = blockIdx.x % each;
    const int kvh = rest % l.kv_heads, cg = rest / l.kv_heads;
    auto deal_it = [&]() { return deal_tokens<true>(t, b, blockIdx.x, group, INT32_MAX, each, max_shares, flags); };
    attend_task<FMT, HD, NT, NT>(shared, deal_it, q, t, l, heads, group, each, rest, kvh, cg, partials, tickets, out, flags);
}

// Any number of tokens per row: the first `prompts` workgroups are for rows with more than kFewColumns columns, the
// others for the rest (a single tile where eight columns do: 64 rows of 4000, 4 heads per K/V head, called as if they had more
// than a token each: 136 us with two, 113 with one, 97 as what they are); one launch, so that a batch of both kinds runs at the same time and one of a
// single kind does not wait for a launch that finds nothing to do (4.5 us).
template <int FMT, int HD>
__global__ __launch_bounds__(kPromptThreads, 2) void attention_batch_kernel(
    const float *__restrict__ q, KvTableArgs t, KvBatchArgs b, KvLayerArgs l, int heads, int prompts, int prompt_shares,
    int token_shares, float *__restrict__ partials, unsigned *__restrict__ tickets, float *__restrict__ out,
    unsigned *flags) {
    constexpr int NT = kFewColumns / 8;
    constexpr size_t kPromptPartials = 2ull * kPromptTargetGroups * prompt_partial_floats<HD>();
    static_assert(kPromptPartials + 2ull * kTargetGroups * partial_floats<HD, NT>() <= RBN_SPLITK_TILES * 1024ull,
                  "the partial results of all shares must fit the workspace");
    static_assert(kTokenThreads == kPromptThreads, "both kinds of workgroup are of one launch");
    __shared__ union {
        TokenShared<HD, NT> tokens;
        TokenShared<HD, 1> few;
        PromptShared<HD> prompts;
    } shared;
    if ((int)blockIdx.x < prompts) {
        attend_prompts<FMT, HD>(shared.prompts, blockIdx.x, q, t, b, l, heads, prompt_shares, kFewColumns + 1, partials,
                                tickets, out, flags);
        return;
    }
    const int block = blockIdx.x - prompts, group = heads / l.kv_heads, each = l.kv_heads, rest = block % each;
    const Task task = deal_tokens<false>(t, b, block, group, kFewColumns, each, token_shares, flags);
    if (task.entry < 0) return;
    float *token_partials = partials + kPromptPartials;
    unsigned *token_tickets = tickets + RBN_ATTENTION_ITEMS;
    auto dealt = [&]() { return task; };
    if (task.unit.n * group <= 8)
        attend_task<FMT, HD, 1, NT>(shared.few, dealt, q, t, l, heads, group, each, rest, rest, 0, token_partials, token_tickets,
                                    out, flags);
    else
        attend_task<FMT, HD, NT, NT>(shared.tokens, dealt, q, t, l, heads, group, each, rest, rest, 0, token_partials,
                                     token_tickets, out, flags);
}

// The most workgroups that may share an item, as far as there are tickets; how many do is decided on the device,
// where `target` shares and one more for each of `busy` items come out at most.
struct Grid {
    uint64_t shares, groups;
};
Grid grid_for(uint64_t items, uint64_t busy, uint64_t most_items, uint64_t most_shares, uint64_t target) {
    Grid g;
    g.shares = items > most_items || most_shares < 1 ? 1 : most_shares;
    g.groups = busy * g.shares;
    if (g.groups > busy + target) g.groups = busy + target;
    if (g.shares == 1) g.groups = busy;
    return g;
}

uint64_t token_shares(const KvTableArgs &t) {
    const uint64_t most = ((uint64_t)t.max_blocks + kMinShare - 1) / kMinShare;
    return most < kMaxShares ? most : kMaxShares;
}

template <int FMT, int HD, int NT>
int launch_tokens(rbn_ctx *ctx, const float *d_q, const KvTableArgs &t, const KvBatchArgs &b, const KvLayerArgs &l, int heads,
                  float *d_out) {
    const uint64_t tiles = (heads / l.kv_heads + 8 * NT - 1) / (8 * NT), items = (uint64_t)b.max_tokens * l.kv_heads * tiles;
    const Grid g = grid_for(items, items, kMostItems, token_shares(t), kTargetGroups);
    attention_token_kernel<FMT, HD, NT><<<dim3((unsigned)g.groups), dim3(kTokenThreads), 0, ctx->stream>>>(
        d_q, t, b, l, heads, (int)tiles, (int)g.shares, (float *)ctx->splitk_partials, ctx->attention_tickets, d_out,
        ctx->dev_flags);
    RBN_HIP(hipGetLastError());
    return RBN_OK;
}

template <int FMT, int HD>
int launch_batch(rbn_ctx *ctx, const float *d_q, const KvTableArgs &t, const KvBatchArgs &b, const KvLayerArgs &l, int heads,
                 float *d_out) {
    const uint64_t units = kv_max_units(b.max_tokens, t.rows), per_unit = (heads / l.kv_heads + 3) / 4;
    const uint64_t items = units * l.kv_heads * per_unit;
    const Grid p = grid_for(items, items, RBN_ATTENTION_ITEMS, kPromptMaxShares, kPromptTargetGroups);
    // (a row with few columns has two units at most)
    const uint64_t few = units < 2ull * t.rows ? units : 2ull * t.rows;
    Grid k = grid_for(units * l.kv_heads, few * l.kv_heads, kMostItems, token_shares(t), kTargetGroups);
    if (k.shares == 1) k.groups = 2ull * t.rows * l.kv_heads;
    attention_batch_kernel<FMT, HD><<<dim3((unsigned)(p.groups + k.groups)), dim3(kPromptThreads), 0, ctx->stream>>>(
        d_q, t, b, l, heads, (int)p.groups, (int)p.shares, (int)k.shares, (float *)ctx->splitk_partials,
        ctx->attention_tickets, d_out, ctx->dev_flags);
    RBN_HIP(hipGetLastError());
    return RBN_OK;
}

template <int FMT, int HD>
int launch_as(rbn_ctx *ctx, const float *d_q, const KvTableArgs &t, const KvBatchArgs &b, const KvLayerArgs &l, int heads,
              uint64_t max_new, float *d_out) {
    // One token per row: token by token (if a row has more after all, so are they).  Otherwise by the rows' columns.
    if (max_new > 1) return launch_batch<FMT, HD>(ctx, d_q, t, b, l, heads, d_out);
    return heads / l.kv_heads <= 8 ? launch_tokens<FMT, HD, 1>(ctx, d_q, t, b, l, heads, d_out)
                                   : launch_tokens<FMT, HD, 2>(ctx, d_q, t, b, l, heads, d_out);
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
    // a launch holds fewer than 2^32 threads
    const uint64_t group = heads / layer->kv_heads, tile = group <= 8 ? 8 : 16;
    const uint64_t groups =
        max_new > 1 ? ((uint64_t)kv_max_units(b.max_tokens, t.rows) * ((group + 3) / 4) + 2ull * t.rows) * layer->kv_heads
                    : (uint64_t)b.max_tokens * ((group + tile - 1) / tile) * layer->kv_heads;
    RBN_REQUIRE(groups + kTargetGroups + kPromptTargetGroups < (1ull << 24),
                "too much for one call of rbn_attention_q8kv (max_tokens %llu, kv_heads %u, heads %llu)",
                (unsigned long long)batch->max_tokens, layer->kv_heads, (unsigned long long)heads);
    RBN_ENTER(ctx);
    auto launch = layer->format == RBN_KV_I8 ? (layer->head_dim == 128 ? launch_as<RBN_KV_I8, 128> : launch_as<RBN_KV_I8, 64>)
                                             : (layer->head_dim == 128 ? launch_as<RBN_KV_E4M3, 128> : launch_as<RBN_KV_E4M3, 64>);
    return launch(ctx, d_q, t, b, l, (int)heads, max_new, d_out);
}

}  // extern "C"
