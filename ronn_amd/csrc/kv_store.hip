// Rotary embedding and the store into the paged 8-bit K/V cache, and reading it back.
#include "kv_common.hpp"

namespace {

// f16 of a cache value: saturated, NaN to 0 (the cache holds finite values only, so that no masked
// position can turn 0 * value into NaN); *odd collects whether that changed a value.
__device__ __forceinline__ float saturated(float x, bool *odd) {
    if (!(fabsf(x) <= 65504.0f)) {
        // up to 65520 a value still rounds to the largest f16
        *odd |= !(fabsf(x) < 65520.0f);
        x = x != x ? 0.0f : copysignf(65504.0f, x);
    }
    return x;
}

__device__ __forceinline__ void to_f16_values(float4 &x, bool *odd) {
    const bool fits = fabsf(x.x) <= 65504.0f & fabsf(x.y) <= 65504.0f & fabsf(x.z) <= 65504.0f & fabsf(x.w) <= 65504.0f;
    if (!fits) x = {saturated(x.x, odd), saturated(x.y, odd), saturated(x.z, odd), saturated(x.w, odd)};
    x.x = __half2float(__float2half_rn(x.x));
    x.y = __half2float(__float2half_rn(x.y));
    x.z = __half2float(__float2half_rn(x.z));
    x.w = __half2float(__float2half_rn(x.w));
}

typedef _Float16 v4h __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float4 load_open(const __half *p) {
    const v4h h = *reinterpret_cast<const v4h *>(p);
    return {(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
}
__device__ __forceinline__ void store_open(__half *p, float4 x) {  // f16 values already
    const v4h h = {(_Float16)x.x, (_Float16)x.y, (_Float16)x.z, (_Float16)x.w};
    *reinterpret_cast<v4h *>(p) = h;
}

__device__ __forceinline__ float max_of(float m, float4 x) {
    return fmaxf(fmaxf(m, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
}

// x / scale, correctly rounded, from 1 / scale correctly rounded: the quotient's remainder is exact in one fma
// and corrects it (Markstein 1990); f16 values and their scales are far from the ends of the f32 range.
__device__ __forceinline__ float quotient(float x, float scale, float inverse) {
    const float y = x * inverse;
    return fmaf(fmaf(-y, scale, x), inverse, y);
}

// Four codes.  No clamp is needed: |x| <= max and scale is max / 127 (448) but for two roundings, so that a
// quotient passes 127 (448) by a few units in the last place at most, and both conversions round that down.
template <int FMT>
__device__ __forceinline__ unsigned encode(float4 x, float scale, float inverse) {
    const float a = quotient(x.x, scale, inverse), b = quotient(x.y, scale, inverse);
    const float c = quotient(x.z, scale, inverse), d = quotient(x.w, scale, inverse);
    if (FMT == RBN_KV_I8) {
        // adding 1.5 * 2^23 rounds to the nearest even integer and leaves it in the low byte
        constexpr float kInt = 12582912.0f;
        const unsigned ab = __builtin_amdgcn_perm(__float_as_uint(b + kInt), __float_as_uint(a + kInt), 0x0c0c0400u);
        const unsigned cd = __builtin_amdgcn_perm(__float_as_uint(d + kInt), __float_as_uint(c + kInt), 0x04000c0cu);
        return ab | cd;
    }
    return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}

// 2/pi theta^(-2 d / head_dim), the quarter turns per position, as a product: one factor per bit of d and 2/pi.
struct RopeFactors {
    double bit[6], turn;
};

// cos and sin of pos * per_position quarter turns: what is left of the nearest whole one, in 64 bits, and minimax
// polynomials on [-pi/4, pi/4] (relative error 4e-9 and less; with the roundings, 0.7 units in the last place).
__device__ __forceinline__ void rotation(int pos, double per_position, float &c, float &s) {
    constexpr double kInt = 6755399441055744.0;  // 1.5 * 2^52: the integer stands in the low bits of the sum
    const double quarters = (double)pos * per_position, near = quarters + kInt;
    const int whole = (int)__double_as_longlong(near);
    const float a = (float)((quarters - (near - kInt)) * 1.5707963267948966);
    const float z = a * a;
    const float sn = fmaf(a * z, fmaf(z, fmaf(z, -1.9515215535648167e-4f, 8.33216030150652e-3f), -0.16666655242443085f), a);
    const float cs = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 2.443307857902255e-5f, -1.3887315290048718e-3f), 4.166664555668831e-2f), -0.5f), 1.0f);
    c = whole & 1 ? sn : cs;
    s = whole & 1 ? cs : sn;
    c = __uint_as_float(__float_as_uint(c) ^ (unsigned)(whole + 1 & 2) << 30);
    s = __uint_as_float(__float_as_uint(s) ^ (unsigned)(whole & 2) << 30);
}

__device__ __forceinline__ void rotate(float4 &x, float4 &y, const float (&c)[4], const float (&s)[4]) {
    const float4 a = x, b = y;
    x = {fmaf(-b.x, s[0], a.x * c[0]), fmaf(-b.y, s[1], a.y * c[1]), fmaf(-b.z, s[2], a.z * c[2]), fmaf(-b.w, s[3], a.w * c[3])};
    y = {fmaf(a.x, s[0], b.x * c[0]), fmaf(a.y, s[1], b.y * c[1]), fmaf(a.z, s[2], b.z * c[2]), fmaf(a.w, s[3], b.w * c[3])};
}

// qkv is read once: 54.7 us for four prompts of 3300 tokens in all, 20 heads, with ordinary loads, 47.6 with these.
typedef float v4f __attribute__((ext_vector_type(4)));
__device__ __forceinline__ float4 load_once(const float *p) {
    const v4f x = __builtin_nontemporal_load(reinterpret_cast<const v4f *>(p));
    return {x[0], x[1], x[2], x[3]};
}

// One workgroup per (unit, K/V head): rotates the unit's q heads of the group and its k, completes
// the block from the row's open buffer if it starts inside it, and writes the page (full block) or
// the open buffer (unfinished).  The open buffer of a row is read by its first unit and written by
// its last: where the first has something to read, it also does the last one's K and V, after a
// barrier, so that nothing is overwritten before it was read.
//  * For q and k a thread has four dimensions and their four partners, of two positions sixteen apart, so the
//    rotation stays in registers; for v it has four dimensions of four consecutive positions, whose codes stand
//    next to each other in a page.  Codes meet in LDS and leave as whole pages, 16 bytes per thread.
//  * A unit of a single token has the threads of the other positions take the other q heads.
//  * In a decode step the token's q, k and v are requested before its row is known: one round trip less (16 rows, 20 / 5 heads: 3.8 us,
//    5.2 without).
//  * The angle is reduced to an eighth of a turn in 64 bits, all loads are under way before the sines are computed.
// Bound by memory: 3300 tokens, 20 heads and as many K/V heads, 153 MB: 33 us with the loads above, 4.6 TB/s.
template <int FMT, int HD>
__global__ __launch_bounds__(2 * HD) void kv_store_kernel(const float *__restrict__ qkv, KvTableArgs t, KvBatchArgs b,
                                                          KvLayerArgs l, int heads, RopeFactors factors,
                                                          float *__restrict__ q_out, unsigned *flags) {
    constexpr int kThreads = 2 * HD, kWaves = kThreads / 64, kTile = kKvBlock * HD, half = HD / 2;
    constexpr int kSteps = 16;  // positions between a thread's two
    __shared__ __attribute__((aligned(16))) uint8_t s_code[2][kTile];
    __shared__ float s_max[2][kWaves];
    const int tid = threadIdx.x, kvh = blockIdx.x % l.kv_heads;
    const int d = tid % (half / 4) * 4, slot = tid / (half / 4);   // q and k: dimensions d .. d+3 (+ half), slots slot (+ 16)
    const int vd = tid % (HD / 4) * 4, vslot = tid / (HD / 4) * 4;  // v: dimensions vd .. vd+3, slots vslot .. vslot+3
    const int group = heads / l.kv_heads;
    const size_t width = (size_t)(heads + 2 * l.kv_heads) * HD;
    const float4 none = {0.0f, 0.0f, 0.0f, 0.0f};
    // A call with no more tokens than rows is a decode step: its units are single tokens (nearly all), whose q, k and v
    // can be on their way before it is known where they go.
    float4 step_q[2] = {none, none}, step_k[2] = {none, none}, step_v = none;
    int step_slot = -1;
    const bool step = b.max_tokens <= t.rows;
    bool bad = false;
    KvUnit u = kv_resolve_unit(t, b, blockIdx.x / l.kv_heads, &bad, [&](int i) __attribute__((always_inline)) {
        if (!step || i < 0) return;
        __builtin_amdgcn_sched_barrier(0);  // behind the loads that the unit's row is waited for with
        const float *from = qkv + (size_t)i * width;
        step_slot = b.slot[i];
        if (slot < group) {
            step_q[0] = load_once(from + (size_t)(kvh * group + slot) * HD + d);
            step_q[1] = load_once(from + (size_t)(kvh * group + slot) * HD + d + half);
        }
        if (slot == 0) {
            step_k[0] = load_once(from + (size_t)(heads + kvh) * HD + d);
            step_k[1] = load_once(from + (size_t)(heads + kvh) * HD + d + half);
        }
        if (vslot == 0) step_v = load_once(from + (size_t)(heads + l.kv_heads + kvh) * HD + vd);
        __builtin_amdgcn_sched_barrier(0);
    });
    if (bad && tid == 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
    if (u.n == 0) return;
    const int row_held = u.row_pos & (kKvBlock - 1);  // tokens of the row's first block that came earlier
    const int row_end = u.row_pos + u.row_n;
    const bool first = u.first == u.row_first;
    bool odd = false;
    double per_position[4];  // quarter turns
    per_position[0] = factors.turn;
#pragma unroll
    for (int i = 2; (1 << i) < half; ++i) per_position[0] *= (d >> i) & 1 ? factors.bit[i] : 1.0;
    per_position[1] = per_position[0] * factors.bit[0];
    per_position[2] = per_position[0] * factors.bit[1];
    per_position[3] = per_position[1] * factors.bit[1];
    __half *const open_k = l.k_open + ((size_t)u.row * l.kv_heads + kvh) * kTile;
    __half *const open_v = l.v_open + ((size_t)u.row * l.kv_heads + kvh) * kTile;

    if (step && u.n == 1 && (u.pos & (kKvBlock - 1)) != kKvBlock - 1) {
        // a single token that does not complete its block: k and v go to the open buffer (by the row's first unit, if
        // that reads the buffer: below)
        const int at = (u.pos & (kKvBlock - 1)) * HD;
        float c[4], s[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) rotation(u.pos, per_position[k], c[k], s[k]);
        for (int h = slot; h < group; h += kSteps) {
            if (h != slot) {
                const float *from = qkv + (size_t)u.first * width + (size_t)(kvh * group + h) * HD + d;
                step_q[0] = load_once(from);
                step_q[1] = load_once(from + half);
            }
            rotate(step_q[0], step_q[1], c, s);
            float *to = q_out + ((size_t)u.first * heads + kvh * group + h) * HD + d;
            *reinterpret_cast<float4 *>(to) = step_q[0];
            *reinterpret_cast<float4 *>(to + half) = step_q[1];
        }
        if (!first && row_held > 0) return;
        if (kv_slot_page(t, step_slot) < 0 && tid == 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
        if (slot == 0) {
            rotate(step_k[0], step_k[1], c, s);
            to_f16_values(step_k[0], &odd);
            to_f16_values(step_k[1], &odd);
            store_open(open_k + at + d, step_k[0]);
            store_open(open_k + at + d + half, step_k[1]);
        }
        if (vslot == 0) {
            to_f16_values(step_v, &odd);
            store_open(open_v + at + vd, step_v);
        }
        if (odd) atomicOr(flags, (unsigned)RBN_FLAG_KV_NONFINITE);
        return;
    }

    for (int pass = 0; pass < 2; ++pass) {
        const int base = u.pos & (kKvBlock - 1);       // slot of the unit's first token in the block
        const bool full = (u.pos / kKvBlock + 1) * kKvBlock <= row_end;
        const bool single = u.n == 1;
        // an unfinished block behind a first block that reads the open buffer belongs to the latter
        const bool keep = pass == 1 || first || full || row_held == 0;
        const float *const src = qkv + (size_t)u.first * width;
        int page = 0;
        float4 kx[2][2], vx[4], qx[2][2] = {{none, none}, {none, none}};
        if (keep) {
            page = kv_slot_page(t, b.slot[u.first]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int j = slot + kSteps * i - base;
                const float *from = src + (size_t)j * width + (size_t)(heads + kvh) * HD + d;
                kx[i][0] = kx[i][1] = none;
                if (j >= 0 && j < u.n) {
                    kx[i][0] = load_once(from);
                    kx[i][1] = load_once(from + half);
                } else if (j < 0 && full) {
                    kx[i][0] = load_open(open_k + (j + base) * HD + d);
                    kx[i][1] = load_open(open_k + (j + base) * HD + d + half);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = vslot + r - base;
                vx[r] = none;
                if (j >= 0 && j < u.n)
                    vx[r] = load_once(src + (size_t)j * width + (size_t)(heads + l.kv_heads + kvh) * HD + vd);
                else if (j < 0 && full)
                    vx[r] = load_open(open_v + (j + base) * HD + vd);
            }
        }
        // q: all heads of the positions slot and slot + 16, or every sixteenth head of a single token
        int h = single ? slot : 0;
        const int h_step = single ? kSteps : 1;
        auto token = [&](int i) { return single ? i : slot + kSteps * i - base; };
        auto load_q = [&]() {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int j = token(i);
                const float *from = src + (size_t)j * width + (size_t)(kvh * group + h) * HD + d;
                if (h < group && j >= 0 && j < u.n) {
                    qx[i][0] = load_once(from);
                    qx[i][1] = load_once(from + half);
                }
            }
        };
        if (pass == 0) load_q();

        float c[2][4], s[2][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) rotation(single ? u.pos : u.pos + token(0), per_position[k], c[0][k], s[0][k]);
        if (single) {
#pragma unroll
            for (int k = 0; k < 4; ++k) c[1][k] = c[0][k], s[1][k] = s[0][k];
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) rotation(u.pos + token(1), per_position[k], c[1][k], s[1][k]);
        }

        if (pass == 0)
            for (; h < group;) {
                float4 now[2][2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    now[i][0] = qx[i][0], now[i][1] = qx[i][1];
                    rotate(now[i][0], now[i][1], c[i], s[i]);
                }
                const int head = kvh * group + h;
                h += h_step;
                load_q();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int j = token(i);
                    if (j < 0 || j >= u.n) continue;
                    float *to = q_out + ((size_t)(u.first + j) * heads + head) * HD + d;
                    *reinterpret_cast<float4 *>(to) = now[i][0];
                    *reinterpret_cast<float4 *>(to + half) = now[i][1];
                }
            }
        if (!keep) break;

        const bool page_ok = page >= 0;
        if (!page_ok && tid == 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int j = slot + kSteps * i - base;
            if (j < 0 || j >= u.n) continue;
            rotate(kx[i][0], kx[i][1], c[i], s[i]);
            to_f16_values(kx[i][0], &odd);
            to_f16_values(kx[i][1], &odd);
            if (!full) {
                store_open(open_k + (j + base) * HD + d, kx[i][0]);
                store_open(open_k + (j + base) * HD + d + half, kx[i][1]);
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int j = vslot + r - base;
            if (j < 0 || j >= u.n) continue;
            to_f16_values(vx[r], &odd);
            if (!full) store_open(open_v + (j + base) * HD + vd, vx[r]);
        }
        if (full) {
            float km = max_of(max_of(max_of(max_of(0.0f, kx[0][0]), kx[0][1]), kx[1][0]), kx[1][1]);
            float vm = max_of(max_of(max_of(max_of(0.0f, vx[0]), vx[1]), vx[2]), vx[3]);
            km = wave_max(km);
            vm = wave_max(vm);
            if ((tid & 63) == 0) s_max[0][tid >> 6] = km, s_max[1][tid >> 6] = vm;
            __syncthreads();  // also: the open buffer has been read
#pragma unroll
            for (int w = 0; w < kWaves; ++w) km = fmaxf(km, s_max[0][w]), vm = fmaxf(vm, s_max[1][w]);
            constexpr float kPart = FMT == RBN_KV_I8 ? 1.0f / 127.0f : 1.0f / 448.0f;
            const float k_scale = km * kPart, v_scale = vm * kPart;
            const float k_inverse = k_scale > 0.0f ? 1.0f / k_scale : 0.0f;
            const float v_inverse = v_scale > 0.0f ? 1.0f / v_scale : 0.0f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int z = 0; z < 2; ++z)
                    *reinterpret_cast<unsigned *>(&s_code[0][kv_k_byte<HD>(slot + kSteps * i, d + half * z)]) =
                        encode<FMT>(kx[i][z], k_scale, k_inverse);
            // a dimension's codes of the four positions, next to each other
            *reinterpret_cast<unsigned *>(&s_code[1][kv_v_byte<HD>(vslot, vd)]) =
                encode<FMT>({vx[0].x, vx[1].x, vx[2].x, vx[3].x}, v_scale, v_inverse);
            *reinterpret_cast<unsigned *>(&s_code[1][kv_v_byte<HD>(vslot, vd + 1)]) =
                encode<FMT>({vx[0].y, vx[1].y, vx[2].y, vx[3].y}, v_scale, v_inverse);
            *reinterpret_cast<unsigned *>(&s_code[1][kv_v_byte<HD>(vslot, vd + 2)]) =
                encode<FMT>({vx[0].z, vx[1].z, vx[2].z, vx[3].z}, v_scale, v_inverse);
            *reinterpret_cast<unsigned *>(&s_code[1][kv_v_byte<HD>(vslot, vd + 3)]) =
                encode<FMT>({vx[0].w, vx[1].w, vx[2].w, vx[3].w}, v_scale, v_inverse);
            __syncthreads();
            if (page_ok) {
                const size_t at = (size_t)page * l.kv_heads + kvh;
                static_assert(kThreads * 16 == kTile, "a thread writes 16 bytes of each page");
                reinterpret_cast<uint4 *>(l.k + at * kTile)[tid] = reinterpret_cast<const uint4 *>(s_code[0])[tid];
                reinterpret_cast<uint4 *>(l.v + at * kTile)[tid] = reinterpret_cast<const uint4 *>(s_code[1])[tid];
                if (tid == 0) l.k_scale[at] = k_scale, l.v_scale[at] = v_scale;
            }
        }
        // the first unit goes on to the row's last one if that is unfinished and was left to it (its own block is full then)
        const int last_pos = row_end - 1, last_block = last_pos / kKvBlock;
        if (pass == 1 || !first || row_held == 0 || last_block == u.pos / kKvBlock || row_end % kKvBlock == 0) break;
        u.first = u.row_first + (last_block * kKvBlock - u.row_pos);
        u.pos = last_block * kKvBlock;
        u.n = row_end - u.pos;
    }
    if (odd) atomicOr(flags, (unsigned)RBN_FLAG_KV_NONFINITE);
}

// A workgroup has 64 places and a head, a lane a place: places are usually positions in a row, whose codes share the
// cache lines of a page.  The values turn round in LDS and leave 16 bytes per thread, a place's head at a time
// (3300 places, 20 heads: 14.3 us, 3.6 TB/s; 26 with a thread for eight dimensions of a place).
constexpr int kReadThreads = 256, kReadPlaces = 64;

template <int FMT, int HD>
__global__ __launch_bounds__(kReadThreads) void kv_read_kernel(KvTableArgs t, KvLayerArgs l, const int32_t *__restrict__ row,
                                                               const int32_t *__restrict__ pos, int count,
                                                               __half *__restrict__ k, __half *__restrict__ v,
                                                               unsigned *flags) {
    typedef _Float16 v8h __attribute__((ext_vector_type(8)));
    constexpr int kTile = kKvBlock * HD, kPitch = HD + 8, kWaves = kReadThreads / 64;
    __shared__ __attribute__((aligned(16))) _Float16 s_x[2][kReadPlaces * kPitch];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = blockIdx.x % l.kv_heads;
    const int64_t first = (int64_t)(blockIdx.x / l.kv_heads) * kReadPlaces;
    const int places = (int)min((int64_t)kReadPlaces, count - first);
    const bool place = lane < places;
    const int r = place ? row[first + lane] : 0, p = place ? pos[first + lane] : 0;
    const int len = place && r >= 0 && r < t.rows ? min(t.len[r], t.max_blocks * kKvBlock) : 0;
    bool ok = p >= 0 && p < len;
    const int block = p / kKvBlock, tt = p % kKvBlock;
    const bool full = ok && (block + 1) * kKvBlock <= len;
    int page = 0;
    if (full) {
        page = kv_page(t, r, block);
        ok = page >= 0;
    }
    if (place && !ok && wave == 0 && h == 0) atomicOr(flags, (unsigned)RBN_FLAG_KV_BAD_INDEX);
    const size_t ph = (size_t)page * l.kv_heads + h;
    const size_t open = ((size_t)r * l.kv_heads + h) * kTile + tt * HD;
    const bool coded = ok && full;
    const float ks = coded ? l.k_scale[ph] : 0.0f, vs = coded ? l.v_scale[ph] : 0.0f;
    constexpr int kEach = HD / 8 / kWaves;
    v8h kx[kEach], vx[kEach];
    if (coded) {
        uint2 kc[kEach];
        uint8_t vc[kEach][8];
#pragma unroll
        for (int z = 0; z < kEach; ++z) {
            const int d = 8 * (wave + kWaves * z);
            kc[z] = *reinterpret_cast<const uint2 *>(l.k + ph * kTile + kv_k_byte<HD>(tt, d));
#pragma unroll
            for (int j = 0; j < 8; ++j) vc[z][j] = l.v[ph * kTile + kv_v_byte<HD>(tt, d + j)];
        }
#pragma unroll
        for (int z = 0; z < kEach; ++z)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint8_t kb = (uint8_t)((j < 4 ? kc[z].x : kc[z].y) >> (8 * (j & 3)));
                kx[z][j] = (_Float16)(kv_decode<FMT>(kb) * ks);
                vx[z][j] = (_Float16)(kv_decode<FMT>(vc[z][j]) * vs);
            }
    } else {
#pragma unroll
        for (int z = 0; z < kEach; ++z) {
            const int d = 8 * (wave + kWaves * z);
            kx[z] = vx[z] = v8h{0, 0, 0, 0, 0, 0, 0, 0};
            if (ok) {
                kx[z] = *reinterpret_cast<const v8h *>(l.k_open + open + d);
                vx[z] = *reinterpret_cast<const v8h *>(l.v_open + open + d);
            }
        }
    }
#pragma unroll
    for (int z = 0; z < kEach; ++z) {
        const int d = 8 * (wave + kWaves * z);
        *reinterpret_cast<v8h *>(&s_x[0][lane * kPitch + d]) = kx[z];
        *reinterpret_cast<v8h *>(&s_x[1][lane * kPitch + d]) = vx[z];
    }
    __syncthreads();
    for (int i = tid; i < places * (HD / 8); i += kReadThreads) {
        const int at = i / (HD / 8), d = i % (HD / 8) * 8;
        const size_t to = ((size_t)(first + at) * l.kv_heads + h) * HD + d;
        *reinterpret_cast<v8h *>(k + to) = *reinterpret_cast<const v8h *>(&s_x[0][at * kPitch + d]);
        *reinterpret_cast<v8h *>(v + to) = *reinterpret_cast<const v8h *>(&s_x[1][at * kPitch + d]);
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
    // rotation() holds the whole quarter turns in 51 bits (theta < 1 has pairs that turn more than a radian per position)
    RBN_REQUIRE((double)table->max_blocks * RBN_KV_BLOCK * exp2(-(1.0 - 2.0 / layer->head_dim) * log2((double)theta)) < 0x1p50,
                "theta %g is too small for rows of %llu blocks", (double)theta, (unsigned long long)table->max_blocks);
    RBN_ENTER(ctx);
    const unsigned groups = (unsigned)kv_max_units(batch->max_tokens, table->rows) * layer->kv_heads;
    static_assert((RBN_KV_MAX_TOKENS / RBN_KV_BLOCK + 2ull * RBN_KV_MAX_ROWS) * 1024 * 256 < 1ull << 32, "threads of a launch");
    RopeFactors factors;
    factors.turn = 0.63661977236758134308;
    for (int i = 0; i < 6; ++i) factors.bit[i] = exp2(-2.0 * (1 << i) / layer->head_dim * log2((double)theta));
    auto kernel = layer->format == RBN_KV_I8
                      ? (layer->head_dim == 128 ? kv_store_kernel<RBN_KV_I8, 128> : kv_store_kernel<RBN_KV_I8, 64>)
                      : (layer->head_dim == 128 ? kv_store_kernel<RBN_KV_E4M3, 128> : kv_store_kernel<RBN_KV_E4M3, 64>);
    kernel<<<dim3(groups), dim3(2 * layer->head_dim), 0, ctx->stream>>>(d_qkv, t, b, l, (int)heads, factors, d_q,
                                                                       ctx->dev_flags);
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
    RBN_REQUIRE(aligned16(d_k) && aligned16(d_v), "d_k and d_v of rbn_kv_read_f16 must be 16-byte aligned");
    const uint64_t groups = (count + kReadPlaces - 1) / kReadPlaces * layer->kv_heads;
    RBN_REQUIRE(groups < (1ull << 24), "too many places in rbn_kv_read_f16");  // a launch holds fewer than 2^32 threads
    RBN_ENTER(ctx);
    auto kernel = layer->format == RBN_KV_I8
                      ? (layer->head_dim == 128 ? kv_read_kernel<RBN_KV_I8, 128> : kv_read_kernel<RBN_KV_I8, 64>)
                      : (layer->head_dim == 128 ? kv_read_kernel<RBN_KV_E4M3, 128> : kv_read_kernel<RBN_KV_E4M3, 64>);
    kernel<<<dim3((unsigned)groups), dim3(kReadThreads), 0, ctx->stream>>>(t, l, d_row, d_pos, (int)count,
                                                                          (__half *)d_k, (__half *)d_v, ctx->dev_flags);
    RBN_HIP(hipGetLastError());
    return RBN_OK;
}

}  // extern "C"
