// Page tables and slot maps of a batch, built on the device from the lengths of its rows.
#include "kv_common.hpp"

namespace {

constexpr int kThreads = 1024;
constexpr int kPerThread = RBN_KV_MAX_ROWS / kThreads;  // rows a thread owns, consecutive
constexpr int kWaves = kThreads / 64;
// Enough workgroups for a token per thread and a wave for every four rows, whose pages it may have to return.
constexpr int kTokensPerGroup = kThreads, kRowsPerGroup = 64;

__device__ __forceinline__ int blocks_of(int n) { return (n + kKvBlock - 1) / kKvBlock; }

// Exclusive prefix sums over the workgroup of N values per thread, totals in total[]; s_wave is used once.
template <int N>
__device__ __forceinline__ void group_scan(int (&v)[N], int (&total)[N], int (*s_wave)[kWaves]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int upto = wave_scan_i(v[j]);
        if (lane == 63) s_wave[j][wave] = upto;
        v[j] = upto - v[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int waves = wave_scan_i(lane < kWaves ? s_wave[j][lane] : 0);
        total[j] = __builtin_amdgcn_readlane(waves, kWaves - 1);
        v[j] += wave > 0 ? __builtin_amdgcn_readlane(waves, wave - 1) : 0;
    }
}

// Admission (prefix sums over the rows) is a few microseconds of latency and no work, so every
// workgroup does it for itself and then writes its own share of the tokens: one launch, no
// second pass over the rows.  If the pool and the batch hold all that is asked for, one scan gives every place
// (tokens, pages, units, returned pages together); only otherwise do refusals need the two before it.
// Nothing a workgroup reads before the ticket is written before the last workgroup has drawn its ticket, so
// lengths and ring state may be updated in place.
// Bound by the chain of dependent steps (lengths, scan, page, entries): a tick of 64 rows is 5.0 us,
// 1000 rows of which 100 return up to 250 pages each 6.1 us (10.3 and 24.4 us before the one scan, a
// token per thread and a wave per returned row; 15 workgroups each had seven rows' pages to return one after the other).
__global__ __launch_bounds__(kThreads) void kv_plan_kernel(KvTableArgs t, KvBatchArgs b,
                                                           const int32_t *__restrict__ fresh, int32_t *len_out,
                                                           int32_t *ring_state_out, unsigned *ticket,
                                                           unsigned *flags) {
    __shared__ int s_start[RBN_KV_MAX_ROWS + 1];  // first token of the row
    __shared__ int s_len[RBN_KV_MAX_ROWS];        // positions held before
    __shared__ int s_page[RBN_KV_MAX_ROWS];       // first free page of the row minus its first new block
    __shared__ int s_unit[RBN_KV_MAX_ROWS];       // first unit of the row minus its first block
    __shared__ int s_back[RBN_KV_MAX_ROWS];       // place of the row's returned pages behind the tail
    __shared__ int s_wave[9][kWaves];
    __shared__ int s_last;
    const int tid = threadIdx.x;
    const int cap = t.max_blocks * kKvBlock;
    int head = t.ring_state[0], count = t.ring_state[1];
    unsigned raise = 0;
    if (count < 0 || count > t.pages || head < 0 || head >= t.pages) {  // no pages to give or take
        raise |= RBN_FLAG_KV_BAD_INDEX;
        count = count < 0 || count > t.pages ? 0 : count;
        head = head < 0 || head >= t.pages ? 0 : head;
    }

    int len[kPerThread], n[kPerThread], need[kPerThread], back[kPerThread];
    bool bad[kPerThread];
    int fin[4], total[4];  // tokens, pages, units, returned pages
    auto add_up = [&]() {
        fin[0] = fin[1] = fin[2] = fin[3] = 0;
#pragma unroll
        for (int j = 0; j < kPerThread; ++j) {
            fin[0] += max(n[j], 0);
            fin[1] += need[j];
            fin[2] += n[j] > 0 ? blocks_of(len[j] + n[j]) - len[j] / kKvBlock : 0;
            fin[3] += back[j];
        }
    };
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int r = tid * kPerThread + j;
        len[j] = r < t.rows ? t.len[r] : 0;
        int want = r < t.rows ? fresh[r] : 0;
        bad[j] = len[j] < 0 || len[j] > cap;
        if (bad[j]) raise |= RBN_FLAG_KV_BAD_INDEX;
        back[j] = want < 0 && !bad[j] ? blocks_of(len[j]) : 0;
        n[j] = want > 0 && !bad[j] && want <= b.max_tokens && want <= cap - len[j] ? want : 0;
        if (want > 0 && n[j] == 0 && !bad[j]) raise |= RBN_FLAG_KV_REFUSED;
        if (want < 0 && !bad[j]) n[j] = -1;
        need[j] = n[j] > 0 ? blocks_of(len[j] + n[j]) - blocks_of(len[j]) : 0;
    }
    add_up();
    group_scan(fin, total, s_wave);
    if (total[0] > b.max_tokens || total[1] > count) {  // not all fit: pages first ...
        int upto = fin[1], tokens[1] = {0}, total1[1];
#pragma unroll
        for (int j = 0; j < kPerThread; ++j) {
            upto += need[j];
            if (n[j] > 0 && need[j] > 0 && upto > count) {
                n[j] = 0;
                raise |= RBN_FLAG_KV_REFUSED;
            }
            tokens[0] += max(n[j], 0);
        }
        // ... then the batch's capacity ...
        group_scan(tokens, total1, s_wave + 4);
        upto = tokens[0];
#pragma unroll
        for (int j = 0; j < kPerThread; ++j) {
            upto += max(n[j], 0);
            if (n[j] > 0 && upto > b.max_tokens) {
                n[j] = 0;
                raise |= RBN_FLAG_KV_REFUSED;
            }
            need[j] = n[j] > 0 ? need[j] : 0;
        }
        // ... then the places of what was admitted
        add_up();
        group_scan(fin, total, s_wave + 5);
    }
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int r = tid * kPerThread + j;
        s_start[r] = fin[0];
        s_len[r] = len[j];
        s_page[r] = fin[1] - blocks_of(len[j]);
        s_unit[r] = fin[2] - len[j] / kKvBlock;
        s_back[r] = back[j] > 0 ? fin[3] : -1;
        fin[0] += max(n[j], 0);
        fin[1] += need[j];
        fin[2] += n[j] > 0 ? blocks_of(len[j] + n[j]) - len[j] / kKvBlock : 0;
        fin[3] += back[j];
    }
    if (tid == 0) s_start[RBN_KV_MAX_ROWS] = total[0];
    __syncthreads();

    // the tokens of this workgroup: row by binary search, position, page
    const int first = blockIdx.x * kTokensPerGroup;
    const int last = min(first + kTokensPerGroup, total[0]);
    for (int i = first + tid; i < last; i += kThreads) {
        int lo = 0, hi = t.rows;  // s_start[lo] <= i < s_start[hi] (a row without tokens is skipped over)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_start[mid] <= i) lo = mid; else hi = mid;
        }
        const int off = i - s_start[lo], pos = s_len[lo] + off, block = pos / kKvBlock;
        int32_t *entry = t.table + (size_t)lo * t.max_blocks + block;
        int page;
        const int take = s_page[lo] + block;  // which of the call's pages, for a new block
        const bool is_new = block >= blocks_of(s_len[lo]);
        if (is_new) {
            const unsigned at = (unsigned)head + (unsigned)take;
            page = t.ring[at >= (unsigned)t.pages ? at - t.pages : at];
        } else {
            page = *entry;
        }
        if (page < 0 || page >= t.pages) {
            raise |= RBN_FLAG_KV_BAD_INDEX;
            page = -1;
        }
        const bool opens = pos % kKvBlock == 0;
        if (is_new && opens) *entry = page;
        b.row[i] = lo;
        b.pos[i] = pos;
        b.slot[i] = page < 0 ? -1 : page * kKvBlock + pos % kKvBlock;
        if (opens || off == 0) b.unit[s_unit[lo] + block] = i;
    }
    // returned pages, behind the tail: a wave for each row
    for (int r = blockIdx.x * kWaves + (tid >> 6); r < t.rows; r += gridDim.x * kWaves) {
        const int place = s_back[r];
        if (place < 0) continue;
        const int blocks = blocks_of(s_len[r]);
        for (int j = tid & 63; j < blocks; j += 64) {
            const unsigned behind = (unsigned)count + (unsigned)place + (unsigned)j;
            if (behind >= (unsigned)t.pages) {  // more pages than the pool has: some are in it already
                raise |= RBN_FLAG_KV_BAD_INDEX;
                continue;
            }
            const unsigned at = (unsigned)head + behind;
            t.ring[at >= (unsigned)t.pages ? at - t.pages : at] = t.table[(size_t)r * t.max_blocks + j];
        }
    }
    if (raise) atomicOr(flags, raise);

    if (gridDim.x > 1) {
        __syncthreads();  // every read of this workgroup is done
        if (tid == 0) {
            const int is_last = atomicAdd(ticket, 1u) == gridDim.x - 1;
            if (is_last) atomicExch(ticket, 0u);  // ready for the next launch
            s_last = is_last;
        }
        __syncthreads();
        if (!s_last) return;
    }
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int r = tid * kPerThread + j;
        if (r >= t.rows) break;
        b.start[r] = s_start[r];
        len_out[r] = n[j] < 0 ? 0 : len[j] + n[j];
    }
    if (tid == 0) {
        b.start[t.rows] = total[0];
        b.count[0] = total[0];
        b.count[1] = total[2];
        const unsigned at = (unsigned)head + (unsigned)total[1];
        ring_state_out[0] = (int)(at >= (unsigned)t.pages ? at - t.pages : at);
        // (unsigned: rows that claim more pages than there are may add up to 2^31)
        ring_state_out[1] = (int)min((unsigned)(count - total[1]) + (unsigned)total[3], (unsigned)t.pages);
    }
}

}  // namespace

extern "C" {

size_t rbn_kv_code_bytes(uint64_t pages, uint64_t kv_heads, uint64_t head_dim) {
    if (pages >= (1ull << 31) / RBN_KV_BLOCK || kv_heads > 1024 || (head_dim != 64 && head_dim != 128)) return 0;
    return (size_t)(pages * kv_heads * RBN_KV_BLOCK * head_dim);
}

size_t rbn_kv_scale_bytes(uint64_t pages, uint64_t kv_heads) {
    if (pages >= (1ull << 31) / RBN_KV_BLOCK || kv_heads > 1024) return 0;
    return (size_t)(pages * kv_heads * sizeof(float));
}

size_t rbn_kv_open_bytes(uint64_t rows, uint64_t kv_heads, uint64_t head_dim) {
    if (rows > RBN_KV_MAX_ROWS || kv_heads > 1024 || (head_dim != 64 && head_dim != 128)) return 0;
    return (size_t)(rows * kv_heads * RBN_KV_BLOCK * head_dim * 2);
}

int rbn_kv_plan(rbn_ctx *ctx, const rbn_kv_table *table, const int32_t *d_new, const rbn_kv_batch *batch,
                int32_t *d_len_out, int32_t *d_ring_state_out) {
    rbn_clear_error();
    KvTableArgs t;
    KvBatchArgs b;
    RBN_CHECK(kv_check_table(table, &t, "rbn_kv_plan"));
    RBN_CHECK(kv_check_batch(batch, &b, "rbn_kv_plan"));
    RBN_REQUIRE(d_new && d_len_out && d_ring_state_out && t.ring && t.ring_state, "null pointer in rbn_kv_plan");
    RBN_ENTER(ctx);
    const uint64_t by_tokens = (batch->max_tokens + kTokensPerGroup - 1) / kTokensPerGroup;
    const uint64_t by_rows = (table->rows + kRowsPerGroup - 1) / kRowsPerGroup;
    const unsigned groups = (unsigned)(by_tokens > by_rows ? by_tokens : by_rows);
    kv_plan_kernel<<<dim3(groups), dim3(kThreads), 0, ctx->stream>>>(t, b, d_new, d_len_out, d_ring_state_out,
                                                                     ctx->splitk_tickets, ctx->dev_flags);
    RBN_HIP(hipGetLastError());
    return RBN_OK;
}

}  // extern "C"
