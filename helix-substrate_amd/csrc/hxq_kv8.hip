// The KV cache in 8 bits: rows in, one token's attention over it, eviction.
//
// Format: blocks of 64 tokens per sequence and kv head, e4m3 with one power-of-two scale for the
// block's keys and one for its values; the unfinished block in 16 bits.
//  - e4m3 rather than 8-bit integers: keys have channels tens of times larger than the rest (the
//    key bias of Qwen2 models); a shared integer step would leave the others a few levels, e4m3
//    keeps 2^-4 relative down to 2^-15 of the largest.
//  - power-of-two scales: x / scale is exact, so a stored value is x rounded once, and
//    e4m3 * scale is exact in bf16, so MFMA operands carry no second rounding.
#include <algorithm>

#include "hxq_attn.h"

namespace hxq {

constexpr int kBlk = HXQ_KV8_BLOCK;
constexpr int kThr = 256;

// exponent e of the smallest 2^e >= 2^-110 with amax <= 448 * 2^e (448 = 1.75 * 2^8)
__device__ __forceinline__ int scale_exp(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return max(e, -110);
}

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

__device__ __forceinline__ float finite_abs(float v) {
    const float a = fabsf(v);
    return a < INFINITY ? a : 0.f;  // NaN and infinities count as 0
}

// four values times 2^-e, rounded to e4m3 (|v| 2^-e <= 448, or not finite: NaN)
__device__ __forceinline__ uint32_t pack_e4m3(float a, float b, float c, float d, float inv) {
    const auto fix = [inv](float v) { return fabsf(v) < INFINITY ? v * inv : __uint_as_float(0x7fc00000u); };
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(fix(a), fix(b), 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(fix(c), fix(d), w, true));
}

template <bool BF16>
__device__ __forceinline__ float up16(uint16_t v) { return BF16 ? bf16_to_f32(v) : f16_to_f32(v); }

// maximum over the block; every thread gets it
template <int THR>
__device__ __forceinline__ float block_amax(float v, float *red) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, kWave));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < THR / kWave; ++i) v = fmaxf(v, red[i]);
    return v;
}

// One block's 64 * D values, in the order of the cache (rows of COLS values, PITCH apart in src), to
// e4m3 and its scale.
template <bool BF16, int D, int COLS, int PITCH, int THR>
__device__ __forceinline__ void store_block(const uint16_t *src, uint8_t *dst, float *scale, float *red) {
    constexpr int CH = kBlk * D / 16, NC = (CH + THR - 1) / THR;   // 16-value chunks, in all and a thread
    u32x4 x[NC][2];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = min(static_cast<int>(threadIdx.x) + i * THR, CH - 1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            x[i][h] = *reinterpret_cast<const u32x4 *>(src + 16 * c / COLS * PITCH + 16 * c % COLS + 8 * h);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                top = fmaxf(top, finite_abs(up16<BF16>(static_cast<uint16_t>(x[i][h][j] & 0xffffu))));
                top = fmaxf(top, finite_abs(up16<BF16>(static_cast<uint16_t>(x[i][h][j] >> 16))));
            }
        }
    }
    top = block_amax<THR>(top, red);
    const int e = scale_exp(top);
    const float inv = pow2f(-e);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int c = threadIdx.x + i * THR;
        if (CH % THR && c >= CH) break;
        u32x4 w;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t lo = x[i][q >> 1][2 * (q & 1)], hi = x[i][q >> 1][2 * (q & 1) + 1];
            w[q] = pack_e4m3(up16<BF16>(static_cast<uint16_t>(lo & 0xffffu)),
                             up16<BF16>(static_cast<uint16_t>(lo >> 16)),
                             up16<BF16>(static_cast<uint16_t>(hi & 0xffffu)),
                             up16<BF16>(static_cast<uint16_t>(hi >> 16)), inv);
        }
        *reinterpret_cast<u32x4 *>(dst + 16 * c) = w;
    }
    if (threadIdx.x == 0) *scale = pow2f(e);
}

template <int DT>
__device__ __forceinline__ void load8(const void *p, int64_t at, float (&v)[8]) {
    if constexpr (DT == HXQ_F32) {
        const float4 a = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at);
        const float4 b = *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(static_cast<const uint16_t *>(p) + at);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[2 * j] = up16<DT == HXQ_BF16>(static_cast<uint16_t>(w[j] & 0xffffu));
            v[2 * j + 1] = up16<DT == HXQ_BF16>(static_cast<uint16_t>(w[j] >> 16));
        }
    }
}

template <bool BF16>
__device__ __forceinline__ u32x4 pack8(const float (&v)[8]) {
    return u32x4{pack16<BF16>(v[0], v[1]), pack16<BF16>(v[2], v[3]), pack16<BF16>(v[4], v[5]),
                 pack16<BF16>(v[6], v[7])};
}

// ---------------------------------------------------------------------------------------------
// Rows into the cache
// ---------------------------------------------------------------------------------------------
struct AppendArgs {
    HeadRows q, k, v;
    const int32_t *cu, *cached, *pos;
    RopeTable rope;
    int32_t rows, n_heads;
    hxq_kv8 c;
    void *q_out, *k_out, *v_out;
};

constexpr int kQHeads = 4;   // query heads a block of rows is rotated for at once

// HBM bound in large calls: 28 + 8 heads, 48 ragged pieces in fp32 (581 MB) 123 us, 4.7 TB/s; a prompt of 1000
// rows (11 MB) 9.8 us, a chain of offsets, rows, rotation, maximum, store.
// One block per (64 cache slots of a sequence, kv head or kQHeads query heads).  A thread owns 8
// neighbouring pairs (i, i + D/2) of a row, so that every access is 16 bytes.
// The block that completes the unfinished one reads the tail; the sequence's last, again unfinished
// block writes it: where there are both, the first block of the sequence does both, in that order.
template <int DT, bool BF16, int D>
__global__ __launch_bounds__(kThr) void kv8_append_kernel(const AppendArgs a) {
    constexpr int HALF = D / 2, TPR = HALF / 8, RPP = kThr / TPR;   // threads a row, rows a pass
    constexpr int VP = kBlk + 8;   // pitch of the transposed values: 16-byte rows, 4 banks apart
    __shared__ double turns[HALF];
    __shared__ float red[kThr / kWave];
    __shared__ __attribute__((aligned(16))) uint16_t sk[kBlk * D];
    __shared__ __attribute__((aligned(16))) uint16_t sv[D * VP];
    const int n_kv = a.c.n_kv_heads;
    int seq, tile;
    const auto n_rows = [&](int s) {
        return max(seq_off(a.cu, s + 1, a.rows) - seq_off(a.cu, s, a.rows), 0);
    };
    const auto tiles = [&](int s) {
        const int n = n_rows(s), held = a.cached[s];
        return n == 0 || held < 0 ? 0 : (held % kBlk + n + kBlk - 1) / kBlk;
    };
    if (!seq_tile(a.c.batch, blockIdx.x, tiles, seq, tile)) return;
    const int row0 = seq_off(a.cu, seq, a.rows), n = n_rows(seq);
    const int cached = a.cached[seq], held = cached % kBlk, full0 = cached / kBlk;
    const int total = held + n, last = (total - 1) / kBlk;
    const int pos0 = a.pos ? a.pos[seq] : cached;
    const bool rope = a.rope.on;
    if (rope && threadIdx.x < HALF) turns[threadIdx.x] = rope_turns(a.rope, threadIdx.x);
    __syncthreads();
    const int i0 = (threadIdx.x % TPR) * 8, r0 = threadIdx.x / TPR;
    const auto cos_sin = [&](int r, float (&c)[8], float (&s)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (rope) rope_cs(pos0 + r, turns[i0 + j], c[j], s[j]);
        }
    };
    const auto turn = [&](const void *p, int64_t at, const float (&c)[8], const float (&s)[8],
                          u32x4 &lo, u32x4 &hi) {
        float x1[8], x2[8], y1[8], y2[8];
        load8<DT>(p, at + i0, x1);
        load8<DT>(p, at + i0 + HALF, x2);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            y1[j] = x1[j];
            y2[j] = x2[j];
            if (rope) rope_turn(x1[j], x2[j], c[j], s[j], y1[j], y2[j]);
        }
        lo = pack8<BF16>(y1);
        hi = pack8<BF16>(y2);
    };
    if (static_cast<int>(blockIdx.y) >= n_kv) {
        if (!a.q_out) return;
        const int h0 = (blockIdx.y - n_kv) * kQHeads, h1 = min(h0 + kQHeads, a.n_heads);
        for (int t = r0; t < kBlk; t += RPP) {
            const int r = tile * kBlk + t - held;
            if (r < 0 || r >= n) continue;
            float c[8], s[8];
            cos_sin(r, c, s);
            for (int h = h0; h < h1; ++h) {
                u32x4 lo, hi;
                turn(a.q.p, (row0 + r) * a.q.row + h * a.q.head, c, s, lo, hi);
                uint16_t *o = static_cast<uint16_t *>(a.q_out) + ((int64_t)(row0 + r) * a.n_heads + h) * D;
                *reinterpret_cast<u32x4 *>(o + i0) = lo;
                *reinterpret_cast<u32x4 *>(o + i0 + HALF) = hi;
            }
        }
        return;
    }
    const int h = blockIdx.y;
    const bool has_tail = total % kBlk != 0;
    const bool both = last > 0 && has_tail && held > 0;   // tail read by the first, written by the last
    const bool store = a.c.k != nullptr;
    if (store && both && tile == last) return;            // the first block does it
    const int64_t bh = (int64_t)seq * n_kv + h;
    uint16_t *k_tail = static_cast<uint16_t *>(a.c.k_tail) + bh * kBlk * D;
    uint16_t *v_tail = static_cast<uint16_t *>(a.c.v_tail) + bh * kBlk * D;
    for (int pass = 0; pass < 2; ++pass) {
        const int tl = pass ? last : tile;
        const bool done = (tl + 1) * kBlk <= total;
        for (int t = r0; t < kBlk; t += RPP) {
            const int r = tl * kBlk + t - held;
            if (r >= n) continue;
            u32x4 lo, hi, vlo, vhi;
            if (r >= 0) {
                float c[8], s[8];
                cos_sin(r, c, s);
                turn(a.k.p, (row0 + r) * a.k.row + h * a.k.head, c, s, lo, hi);
                float x[8];
                load8<DT>(a.v.p, (row0 + r) * a.v.row + h * a.v.head + i0, x);
                vlo = pack8<BF16>(x);
                load8<DT>(a.v.p, (row0 + r) * a.v.row + h * a.v.head + i0 + HALF, x);
                vhi = pack8<BF16>(x);
                const int64_t at = ((int64_t)(row0 + r) * n_kv + h) * D + i0;
                if (a.k_out) {
                    *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.k_out) + at) = lo;
                    *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.k_out) + at + HALF) = hi;
                }
                if (a.v_out) {
                    *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.v_out) + at) = vlo;
                    *reinterpret_cast<u32x4 *>(static_cast<uint16_t *>(a.v_out) + at + HALF) = vhi;
                }
            } else if (store && done) {
                lo = *reinterpret_cast<const u32x4 *>(k_tail + t * D + i0);
                hi = *reinterpret_cast<const u32x4 *>(k_tail + t * D + i0 + HALF);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint16_t *p = v_tail + (i0 + 2 * j) * kBlk + t;
                    vlo[j] = p[0] | static_cast<uint32_t>(p[kBlk]) << 16;
                    vhi[j] = p[HALF * kBlk] | static_cast<uint32_t>(p[(HALF + 1) * kBlk]) << 16;
                }
            } else continue;
            if (!store) continue;
            *reinterpret_cast<u32x4 *>(sk + t * D + i0) = lo;
            *reinterpret_cast<u32x4 *>(sk + t * D + i0 + HALF) = hi;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                sv[(i0 + 2 * j) * VP + t] = static_cast<uint16_t>(vlo[j]);
                sv[(i0 + 2 * j + 1) * VP + t] = static_cast<uint16_t>(vlo[j] >> 16);
                sv[(i0 + HALF + 2 * j) * VP + t] = static_cast<uint16_t>(vhi[j]);
                sv[(i0 + HALF + 2 * j + 1) * VP + t] = static_cast<uint16_t>(vhi[j] >> 16);
            }
        }
        if (!store) return;
        __syncthreads();
        const int j = full0 + tl;
        if (j < a.c.n_blocks) {
            if (done) {
                const int at = a.c.blocks ? a.c.blocks[bh * a.c.n_blocks + j] : j;
                if (at >= 0 && at < a.c.n_blocks) {
                    const int64_t b = bh * a.c.n_blocks + at;
                    store_block<BF16, D, D, D, kThr>(sk, a.c.k + b * kBlk * D, a.c.k_scale + b, red);
                    store_block<BF16, D, kBlk, VP, kThr>(sv, a.c.v + b * kBlk * D, a.c.v_scale + b, red);
                }
            } else {
                // only the new tokens' slots: the others keep what they hold
                const int t0 = tl ? 0 : held, t1 = total - tl * kBlk;
                for (int e = threadIdx.x; e < (t1 - t0) * D; e += kThr)
                    k_tail[t0 * D + e] = sk[t0 * D + e];
                for (int e = threadIdx.x; e < kBlk * D; e += kThr) {
                    const int t = e % kBlk;
                    if (t >= t0 && t < t1) v_tail[e] = sv[e / kBlk * VP + t];
                }
            }
        }
        if (!(both && tile == 0) || pass) return;
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------
// One token of each sequence over its cache
// ---------------------------------------------------------------------------------------------
struct DecodeArgs {
    HeadRows q, k, v;
    const int32_t *cached, *pos;
    RopeTable rope;
    float scale2;                    // scale * log2(e): the softmax is in powers of two
    int32_t out_dtype, n_heads, splits, group, htiles;
    hxq_kv8 c;
    const float *w_in;
    float *w_out;
    void *out;
    float *part;                     // [batch * n_heads][splits][D]: sums of p v
    float2 *ml;                      // [batch * n_heads][splits]: maximum of the scores, sum of p
    float2 *share;                   // [batch * n_heads][n_blocks]: a block's sum of p and the maximum in it
};

constexpr int kHT = 8;               // query heads of a tile
constexpr int kDThr = 512;           // 8 waves

__device__ __forceinline__ void store_any(void *p, int64_t i, float v, int dt) {
    if (dt == HXQ_F32) store_act<HXQ_F32>(p, i, v);
    else if (dt == HXQ_BF16) store_act<HXQ_BF16>(p, i, v);
    else store_act<HXQ_F16>(p, i, v);
}

// A sequence's units: its full blocks and the unfinished one (with the new token), dealt to the
// splits in runs of `per`.  At least 8 units a split, one for each wave.
__device__ __forceinline__ int units_per_split(int units, int splits) {
    return max((units + splits - 1) / splits, kDThr / kWave);
}

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// 8 e4m3 values times a power of two, as bf16 (exact)
__device__ __forceinline__ u32x4 e4m3_bf16(uint32_t lo, uint32_t hi, float scale) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true))};
}

// value of lane ^ 8 in its row of 16
__device__ __forceinline__ float ror8(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, false));
}

__device__ __forceinline__ float rows_max(float v) {   // over lanes l, l ^ 16, l ^ 32, l ^ 48
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float rows_sum(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// One block: 8 waves over the units of a split of one (sequence, kv head, tile of 8 query heads).
// HBM bound: 64 sequences of 800 to 16000 tokens, 28 heads over 4 (564 MB) 124 us, 4.55 TB/s; one of 131000,
// 16 over 2 (67 MB) 15.8 us, of which 3 to 5 are the start (arguments, counts, token, rotation); one of 500
// 9.7 us.
//
// A wave takes a unit of 64 tokens by itself, in registers, with v_mfma_f32_16x16x32_bf16:
//   S^T = K q^T: rows are tokens, columns are heads.  Row 4 k + r of tile j is given the token
//     16 k + 4 j + r (k = lane / 16), so that a lane ends with the 16 consecutive tokens 16 k ..
//     16 k + 15 of one head;
//   O^T = V^T P^T: the lane's 16 tokens are the k slots of two steps of the product as they are,
//     and the 16 bytes that V^T wants of a lane are neighbours in the cache (values are stored
//     transposed): no shuffle, no shared memory between the two products.
// 16 columns hold 8 heads twice: q = hi + mid + lo in bf16 (24 bits; hi and mid in the two halves of
// one operand, lo in a second), p = hi + lo (16 bits), their products added across the halves.  So q
// keeps its fp32 bits and p 2^-17, at no cost where the cache's bytes bound the time.
template <int DT, bool BF16, int D, bool W>
__global__ __launch_bounds__(kDThr, 1) void kv8_decode_kernel(const DecodeArgs a) {
    constexpr int HALF = D / 2, NC = D / 64, NT = D / 16, NW = kDThr / kWave;
    constexpr int QP = D + 8, NP = ((kHT + 1) * HALF + kDThr - 1) / kDThr;   // pitch of q's rows; pairs a thread
    __shared__ __attribute__((aligned(16))) uint16_t q_hm[2 * kHT][QP], q_lo[kHT][QP];   // hi | mid, lo
    __shared__ __attribute__((aligned(16))) uint16_t kn[D], vn[D];   // the new token
    __shared__ float cs[HALF], sn[HALF];
    __shared__ __attribute__((aligned(16))) float so[NW][kHT][D];
    __shared__ float sm[NW][kHT], sl[NW][kHT], red[NW];
    // Everything that the first loads need in one round of scalar loads: left to itself each value is
    // fetched where it is used, and eight round trips come before the first byte of the cache.
    asm volatile("" ::"s"(a.cached), "s"(a.pos), "s"(a.q.p), "s"(a.q.row), "s"(a.q.head), "s"(a.k.p), "s"(a.k.row), "s"(a.k.head),
                 "s"(a.v.p), "s"(a.v.row), "s"(a.v.head), "s"(a.c.k), "s"(a.c.v), "s"(a.c.k_scale), "s"(a.c.v_scale),
                 "s"(a.c.blocks), "s"(a.c.n_blocks), "s"(a.c.n_kv_heads), "s"(a.n_heads), "s"(a.group), "s"(a.htiles), "s"(a.splits));
    const int n_kv = a.c.n_kv_heads, group = a.group, htiles = a.htiles;
    const int ht = blockIdx.y % htiles, kvh = blockIdx.y / htiles, b = blockIdx.z;
    const int h0 = kvh * group + ht * kHT, nh = min(kHT, group - ht * kHT);
    // the new token's values are asked for first: they are needed first, and loads return in order
    float x1[NP], x2[NP], xv = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int e = threadIdx.x + i * kDThr, h = min(e / HALF, kHT), hq = min(h, nh - 1);
        const void *p = h == kHT ? a.k.p : a.q.p;
        const int64_t at = (h == kHT ? b * a.k.row + kvh * a.k.head : b * a.q.row + (h0 + hq) * a.q.head) + e % HALF;
        x1[i] = load_act<DT>(p, at);
        x2[i] = load_act<DT>(p, at + HALF);
    }
    xv = load_act<DT>(a.v.p, b * a.v.row + kvh * a.v.head + threadIdx.x % D);
    const int cached = a.cached[b];
    if (cached < 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lh = lane & 15, kq = lane >> 4;
    const int full = cached / kBlk, held = cached % kBlk, units = full + 1;
    if (full >= a.c.n_blocks) {      // no room
        if (blockIdx.x == 0)
            for (int e = threadIdx.x; e < nh * D; e += kDThr)
                store_any(a.out, ((int64_t)b * a.n_heads + h0) * D + e, __uint_as_float(0x7fc00000u), a.out_dtype);
        return;
    }
    const int per = units_per_split(units, a.splits), u0 = blockIdx.x * per, u1 = min(u0 + per, units);
    if (u0 >= units) return;
    const int64_t bh = (int64_t)b * n_kv + kvh;
    const int32_t *table = a.c.blocks ? a.c.blocks + bh * a.c.n_blocks : nullptr;

    // A unit's bytes: K of step (j, c) and V of 16 dimensions, 16 bytes a lane.  They are asked for
    // one unit ahead, K when the scores no longer need its registers, V after the second product.
    const int uf = min(u1, full);
    u32x4 kr[4][NC], vr[NT];
    float ks = 1.f, vs = 1.f, bad = 0.f;
    int64_t blk = 0;
    const auto find = [&](int u) {
        int at = table ? table[u] : u;
        bad = at < 0 || at >= a.c.n_blocks ? __uint_as_float(0x7fc00000u) : 0.f;
        blk = bh * a.c.n_blocks + min(max(at, 0), a.c.n_blocks - 1);
    };
    const auto load_k = [&] {
        const u32x4 *kp = reinterpret_cast<const u32x4 *>(a.c.k + blk * kBlk * D);
        ks = a.c.k_scale[blk];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int c = 0; c < NC; ++c) kr[j][c] = kp[((lh >> 2) * 16 + 4 * j + (lh & 3)) * (D / 16) + 4 * c + kq];
    };
    const auto load_v = [&] {
        const u32x4 *vp = reinterpret_cast<const u32x4 *>(a.c.v + blk * kBlk * D);
        vs = a.c.v_scale[blk];
#pragma unroll
        for (int i = 0; i < NT; ++i) vr[i] = vp[(16 * i + lh) * 4 + kq];
    };
    // Every wave asks, also one that has no unit (for a block that another reads): with loads behind a
    // branch the wait for the token's values, asked for before, would be for all of them.
    find(max(min(u0 + wave, uf - 1), 0));
    load_k();
    load_v();

    // the new token: rotation in fp32, q in three bf16 (24 bits)
    const bool rope = a.rope.on;
    if (rope && threadIdx.x < HALF)
        rope_cs(a.pos ? a.pos[b] : cached, rope_turns(a.rope, threadIdx.x), cs[threadIdx.x], sn[threadIdx.x]);
    lds_barrier();
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const int e = threadIdx.x + i * kDThr, h = e / HALF, d = e % HALF;
        if (h > kHT) break;
        float y1 = x1[i], y2 = x2[i];
        if (rope) rope_turn(x1[i], x2[i], cs[d], sn[d], y1, y2);
        if (h == kHT) {
            const uint32_t w = pack16<BF16>(y1, y2);
            kn[d] = static_cast<uint16_t>(w);
            kn[d + HALF] = static_cast<uint16_t>(w >> 16);
            continue;
        }
        if (h >= nh) y1 = y2 = 0.f;
        const uint32_t hi = pack16<true>(y1, y2);
        y1 -= __uint_as_float(hi << 16);
        y2 -= __uint_as_float(hi & 0xffff0000u);
        const uint32_t mid = pack16<true>(y1, y2);
        const uint32_t lo = pack16<true>(y1 - __uint_as_float(mid << 16), y2 - __uint_as_float(mid & 0xffff0000u));
        q_hm[h][d] = static_cast<uint16_t>(hi);
        q_hm[h][d + HALF] = static_cast<uint16_t>(hi >> 16);
        q_hm[h + kHT][d] = static_cast<uint16_t>(mid);
        q_hm[h + kHT][d + HALF] = static_cast<uint16_t>(mid >> 16);
        q_lo[h][d] = static_cast<uint16_t>(lo);
        q_lo[h][d + HALF] = static_cast<uint16_t>(lo >> 16);
    }
    if (threadIdx.x < D) vn[threadIdx.x] = static_cast<uint16_t>(pack16<BF16>(xv, 0.f));
    lds_barrier();

    // q as B operands: d = 64 c + 16 kq + 8 e + 0..7 of step (c, e), as the 16-byte loads of K give it
    u32x4 q1[NC][2], q2[NC][2];
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int d = 64 * c + 16 * kq + 8 * e;
            q1[c][e] = *reinterpret_cast<const u32x4 *>(&q_hm[lh][d]);
            q2[c][e] = *reinterpret_cast<const u32x4 *>(&q_lo[lh & 7][d]);
            if (lh >= kHT) q2[c][e] = u32x4{0u, 0u, 0u, 0u};
        }

    f32x4 o[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;

    // scores of the lane's 16 tokens -> p in B-operand form
    const auto soften = [&](f32x4 (&s)[4], int unit, float bad, int n, u32x4 (&p)[2]) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float x = fmaf(s[j][r] + ror8(s[j][r]), a.scale2, bad);
                if (16 * kq + 4 * j + r >= n) x = -INFINITY;
                s[j][r] = x;
                mx = fmaxf(mx, x);
            }
        const float mn = fmaxf(m, rows_max(mx));
        if (__any(mn > m)) {
            const float al = __builtin_amdgcn_exp2f(m - mn);
            l *= al;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) o[i][r] *= al;
        }
        m = mn;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[j][r] = __builtin_amdgcn_exp2f(s[j][r] - m);
                sum += s[j][r];
            }
#pragma unroll
            for (int r = 0; r < 4; r += 2) {
                const uint32_t hi = pack16<true>(s[j][r], s[j][r + 1]);
                const uint32_t lo = pack16<true>(s[j][r] - __uint_as_float(hi << 16),
                                                 s[j][r + 1] - __uint_as_float(hi & 0xffff0000u));
                p[j >> 1][2 * (j & 1) + (r >> 1)] = lh < 8 ? hi : lo;
            }
        }
        l += sum;
        if constexpr (W) {
            sum = rows_sum(sum);
            if (lane < nh) a.share[((int64_t)b * a.n_heads + h0 + lane) * a.c.n_blocks + unit] = float2{sum, m};
        }
    };

    for (int u = u0 + wave; u < uf; u += NW) {
        const bool more = u + NW < uf;
        const float bad_now = bad;
        f32x4 s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const u32x4 k8 = e4m3_bf16(kr[j][c][2 * e], kr[j][c][2 * e + 1], ks);
                    s[j] = mfma16(k8, q1[c][e], s[j]);
                    s[j] = mfma16(k8, q2[c][e], s[j]);
                }
        }
        if (more) {
            find(u + NW);
            load_k();
        }
        u32x4 p[2];
        soften(s, u, bad_now, kBlk, p);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) o[i] = mfma16(e4m3_bf16(vr[i][2 * e], vr[i][2 * e + 1], vs), p[e], o[i]);
        if (more) load_v();
    }

    // the unfinished block in 16 bits, its last token from shared memory; fp16 as the sum of two bf16
    const bool tail = u1 == units;
    uint16_t *k_tail = static_cast<uint16_t *>(a.c.k_tail) + bh * kBlk * D;
    uint16_t *v_tail = static_cast<uint16_t *>(a.c.v_tail) + bh * kBlk * D;
    const auto split16 = [](const u32x4 &w, u32x4 &hi, u32x4 &lo) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = f16_to_f32(static_cast<uint16_t>(w[i])), y = f16_to_f32(static_cast<uint16_t>(w[i] >> 16));
            hi[i] = pack16<true>(x, y);
            lo[i] = pack16<true>(x - __uint_as_float(hi[i] << 16), y - __uint_as_float(hi[i] & 0xffff0000u));
        }
    };
    if (tail && wave == (full - u0) % NW) {
        // every slot is asked for at once; what is behind the last token is dropped afterwards
        u32x4 kt[4][NC][2], vt[NT][2];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    kt[j][c][e] = *reinterpret_cast<const u32x4 *>(k_tail + ((lh >> 2) * 16 + 4 * j + (lh & 3)) * D + 64 * c + 16 * kq + 8 * e);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) vt[i][e] = *reinterpret_cast<const u32x4 *>(v_tail + (16 * i + lh) * kBlk + 16 * kq + 8 * e);
        f32x4 s[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j] = f32x4{0.f, 0.f, 0.f, 0.f};
            const int t = (lh >> 2) * 16 + 4 * j + (lh & 3);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    u32x4 w = kt[j][c][e];
                    if (t == held) w = *reinterpret_cast<const u32x4 *>(kn + 64 * c + 16 * kq + 8 * e);
                    if constexpr (BF16) {
                        s[j] = mfma16(w, q1[c][e], s[j]);
                        s[j] = mfma16(w, q2[c][e], s[j]);
                    } else {
                        u32x4 hi, lo;
                        split16(w, hi, lo);
                        s[j] = mfma16(hi, q1[c][e], s[j]);
                        s[j] = mfma16(hi, q2[c][e], s[j]);
                        s[j] = mfma16(lo, q1[c][e], s[j]);
                    }
                }
        }
        u32x4 p[2];
        soften(s, full, 0.f, held + 1, p);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = 16 * i + lh, t0 = 16 * kq + 8 * e;
                const uint32_t nv = vn[d];
                u32x4 w = vt[i][e];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int t = t0 + 2 * j;
                    const uint32_t x = t < held ? w[j] & 0xffffu : t == held ? nv : 0u;
                    const uint32_t y = t + 1 < held ? w[j] >> 16 : t + 1 == held ? nv : 0u;
                    w[j] = x | y << 16;
                }
                if constexpr (BF16) {
                    o[i] = mfma16(w, p[e], o[i]);
                } else {
                    u32x4 hi, lo;
                    split16(w, hi, lo);
                    o[i] = mfma16(hi, p[e], o[i]);
                    o[i] = mfma16(lo, p[e], o[i]);
                }
            }
    }

    // the waves' results
    l = rows_sum(l);
    if (kq == 0 && lh < kHT) {
        sm[wave][lh] = m;
        sl[wave][lh] = l;
    }
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        f32x4 x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = o[i][r] + ror8(o[i][r]);
        if (lh < kHT) *reinterpret_cast<f32x4 *>(&so[wave][lh][16 * i + 4 * kq]) = x;
    }
    __syncthreads();
    const bool alone = per >= units;
    for (int e = threadIdx.x; e < nh * D; e += kDThr) {
        const int h = e / D, d = e % D;
        float mm = sm[0][h];
#pragma unroll
        for (int w = 1; w < NW; ++w) mm = fmaxf(mm, sm[w][h]);
        float x = 0.f, ll = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(sm[w][h] - mm);
            x = fmaf(f, so[w][h][d], x);
            ll = fmaf(f, sl[w][h], ll);
        }
        const int64_t row = (int64_t)b * a.n_heads + h0 + h;
        if (alone) store_any(a.out, row * D + d, x / ll, a.out_dtype);
        else a.part[(row * a.splits + blockIdx.x) * D + d] = x;
        if ((!alone || W) && d == 0) a.ml[row * a.splits + blockIdx.x] = float2{mm, ll};
    }

    // the token into the cache (no other block of the launch reads its place)
    if (!tail || ht != 0) return;
    for (int e = threadIdx.x; e < D; e += kDThr) {
        k_tail[held * D + e] = kn[e];
        v_tail[e * kBlk + held] = vn[e];
    }
    if (held != kBlk - 1) return;
    const int at = table ? table[full] : full;
    if (at < 0 || at >= a.c.n_blocks) return;
    __syncthreads();
    blk = bh * a.c.n_blocks + at;
    store_block<BF16, D, D, D, kDThr>(k_tail, a.c.k + blk * kBlk * D, a.c.k_scale + blk, red);
    store_block<BF16, D, kBlk, kBlk, kDThr>(v_tail, a.c.v + blk * kBlk * D, a.c.v_scale + blk, red);
}

// The maximum and the sum over all splits of one query head's scores, by a wave.
__device__ __forceinline__ float2 join_ml(const float2 *ml, int n) {
    const int lane = threadIdx.x & 63;
    float mm = -INFINITY, ll = 0.f;
    for (int i = lane; i < n; i += kWave) mm = fmaxf(mm, ml[i].x);
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) mm = fmaxf(mm, __shfl_xor(mm, s, kWave));
    for (int i = lane; i < n; i += kWave) ll = fmaf(__builtin_amdgcn_exp2f(ml[i].x - mm), ml[i].y, ll);
    return float2{mm, wave_sum(ll)};
}

constexpr int kFewSplits = 16;   // up to here a wave joins a query head by itself, above it a block

// What is left when the splits are done.  The first `row_blocks` blocks join the splits of query heads:
// a wave each, with no exchange (64 sequences, 28 heads, 4 splits: 5.4 us against 8.7 with a block
// each), or a block each where there are many splits.  The others: weight_out = weight_in + every
// cache block's share of the softmax, kThr cache blocks of one (sequence, kv head) each.
template <int D>
__global__ __launch_bounds__(kThr) void kv8_join_kernel(const DecodeArgs a, const int row_blocks) {
    constexpr int Q = D / 4, NG = kThr / Q, NW = kThr / kWave;
    __shared__ __attribute__((aligned(16))) float sx[NG][D];
    __shared__ float2 tot[kHT];
    const int n_kv = a.c.n_kv_heads, group = a.n_heads / n_kv, n_rows = a.c.batch * a.n_heads;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const auto splits_of = [&](int units) {
        const int per = units_per_split(units, a.splits);
        return (units + per - 1) / per;
    };
    if (static_cast<int>(blockIdx.x) < row_blocks && a.splits <= kFewSplits) {
        constexpr int R = D / kWave;
        const int64_t row = (int64_t)blockIdx.x * NW + wave;
        if (row >= n_rows) return;
        const int cached = a.cached[row / a.n_heads];
        if (cached < 0 || cached / kBlk >= a.c.n_blocks) return;
        const int n = splits_of(cached / kBlk + 1);
        if (n == 1) return;    // written already
        const float2 e = lane < n ? a.ml[row * a.splits + lane] : float2{-INFINITY, 0.f};
        const float *pt = a.part + row * a.splits * D + lane * R;
        float p[kFewSplits][R];
#pragma unroll
        for (int i = 0; i < kFewSplits; ++i)
            if (i < n)
#pragma unroll
                for (int r = 0; r < R; ++r) p[i][r] = pt[i * D + r];
        float mm = e.x;
#pragma unroll
        for (int s = kFewSplits / 2; s >= 1; s >>= 1) mm = fmaxf(mm, __shfl_xor(mm, s, kWave));
        mm = __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(mm)));
        const float f = lane < n ? __builtin_amdgcn_exp2f(e.x - mm) : 0.f;
        const float ll = wave_sum(f * e.y);
        float x[R] = {};
#pragma unroll
        for (int i = 0; i < kFewSplits; ++i)
            if (i < n)
#pragma unroll
                for (int r = 0; r < R; ++r) x[r] = fmaf(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), i)), p[i][r], x[r]);
#pragma unroll
        for (int r = 0; r < R; ++r) store_any(a.out, row * D + lane * R + r, x[r] / ll, a.out_dtype);
        return;
    }
    if (static_cast<int>(blockIdx.x) < row_blocks) {
        const int64_t row = blockIdx.x;
        const int cached = a.cached[row / a.n_heads];
        if (cached < 0 || cached / kBlk >= a.c.n_blocks) return;
        const int n = splits_of(cached / kBlk + 1);
        if (n == 1) return;    // written already
        const float2 *ml = a.ml + row * a.splits;
        const float2 t = join_ml(ml, n);
        const float *pt = a.part + row * a.splits * D;
        const int d = threadIdx.x % Q * 4, g = threadIdx.x / Q;
        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int i = g; i < n; i += NG) {
            const float f = __builtin_amdgcn_exp2f(ml[i].x - t.x);
            const f32x4 p = *reinterpret_cast<const f32x4 *>(pt + (int64_t)i * D + d);
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = fmaf(f, p[r], x[r]);
        }
        *reinterpret_cast<f32x4 *>(&sx[g][d]) = x;
        __syncthreads();
        if (threadIdx.x >= D) return;
        float y = 0.f;
#pragma unroll
        for (int i = 0; i < NG; ++i) y += sx[i][threadIdx.x];
        store_any(a.out, row * D + threadIdx.x, y / t.y, a.out_dtype);
        return;
    }
    const int chunks = (a.c.n_blocks + kThr - 1) / kThr, id = blockIdx.x - row_blocks;
    const int64_t bh = id / chunks;
    const int b = static_cast<int>(bh / n_kv), kvh = static_cast<int>(bh % n_kv);
    const int cached = a.cached[b];
    if (cached < 0) return;
    const int units = cached / kBlk < a.c.n_blocks ? cached / kBlk + 1 : 0;   // no room: the weights stay
    const int n = splits_of(units), j = id % chunks * kThr + threadIdx.x;
    const int64_t row0 = (int64_t)b * a.n_heads + kvh * group, at = bh * a.c.n_blocks + min(j, a.c.n_blocks - 1);
    float w = a.w_in ? a.w_in[at] : 0.f;
    for (int g0 = 0; g0 < (units ? group : 0); g0 += kHT) {
        const int ng = min(group - g0, kHT);
        // asked for before the totals that they wait for (entries behind the units hold nothing)
        float2 s[kHT];
#pragma unroll
        for (int g = 0; g < kHT; ++g) s[g] = a.share[(row0 + g0 + min(g, ng - 1)) * a.c.n_blocks + min(j, units - 1)];
        __syncthreads();
        for (int g = wave; g < ng; g += NW) {
            const float2 t = join_ml(a.ml + (row0 + g0 + g) * a.splits, n);
            if (lane == 0) tot[g] = float2{t.x, 1.f / t.y};
        }
        __syncthreads();
        if (j < units)
#pragma unroll
            for (int g = 0; g < kHT; ++g)
                if (g < ng) w = fmaf(s[g].x * __builtin_amdgcn_exp2f(s[g].y - tot[g].x), tot[g].y, w);
    }
    if (j < a.c.n_blocks) a.w_out[at] = w;
}

// ---------------------------------------------------------------------------------------------
// Eviction
// ---------------------------------------------------------------------------------------------
constexpr int kEvThr = 1024;

// Order-preserving bits of a weight; NaN is the greatest, -0 is 0.
__device__ __forceinline__ uint32_t weight_key(float v) {
    if (v != v) return 0xffffffffu;
    const uint32_t u = __float_as_uint(v + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One block per (sequence, kv head): the least weight that stays by four passes over its bits
// (histograms of 8 bits), then one pass in order that gives every block its new place.  Latency bound: 256
// rows of 2047 blocks 8.5 us, 2 of 157 4.4 us.
__global__ __launch_bounds__(kEvThr) void kv8_evict_kernel(const float *weight, const int32_t *blocks,
                                                           const int32_t *cached, int32_t n_kv, int32_t n_blocks,
                                                           int32_t keep, int32_t sink, int32_t recent, float *w_out,
                                                           int32_t *b_out, int32_t *c_out) {
    __shared__ int hist[256];
    __shared__ uint32_t s_key;
    __shared__ int s_left, wsum[2][kEvThr / kWave];
    const int64_t base = (int64_t)blockIdx.x * n_blocks;
    const int b = blockIdx.x / n_kv, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // tokens past the cache were never stored: they do not come back when there is room again
    const int n = min(cached[b], n_blocks * kBlk), full = n / kBlk;
    const float *w = weight + base;
    if (n < 0) {   // skipped: its blocks and weights as they are
        for (int j = tid; j < n_blocks; j += kEvThr) {
            b_out[base + j] = blocks ? blocks[base + j] : j;
            w_out[base + j] = w[j];
        }
        if (tid == 0 && blockIdx.x % n_kv == 0) c_out[b] = n;
        return;
    }
    const bool cut = full > keep;
    uint32_t key = 0;      // bits of the least key that stays, and how many of that key stay
    int left = keep - sink - recent;
    if (cut && left > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
            for (int j = sink + tid; j < full - recent; j += kEvThr) {
                const uint32_t k = weight_key(w[j]);
                if ((k & mask) == key) atomicAdd(&hist[k >> shift & 255u], 1);
            }
            __syncthreads();
            if (tid < 64) {   // from the greatest digit down: lane i holds digits 255 - 4 i ...
                int c[4], t = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) t += c[i] = hist[255 - 4 * lane - i];
                int above = wave_scan(t) - t;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (above < left && left <= above + c[i]) {
                        s_key = key | static_cast<uint32_t>(255 - 4 * lane - i) << shift;
                        s_left = left - above;
                    }
                    above += c[i];
                }
            }
            __syncthreads();
            key = s_key;
            left = s_left;
        }
    }
    const int stay = cut ? keep : full;
    int n_kept = 0, n_tie = 0;     // of the blocks before this pass's
    for (int j0 = 0; j0 < n_blocks; j0 += kEvThr) {
        const int j = j0 + tid;
        const bool in = j < full, fixed = in && (!cut || j < sink || j >= full - recent);
        const float x = j < n_blocks ? w[j] : 0.f;
        const uint32_t k = weight_key(x);
        const bool mid = in && !fixed && keep > sink + recent;
        const bool tie = mid && k == key;
        const uint64_t ties = __ballot(tie);
        __syncthreads();
        if (lane == 0) wsum[0][wave] = __builtin_popcountll(ties);
        __syncthreads();
        int before = n_tie, tot = 0;
        for (int i = 0; i < kEvThr / kWave; ++i) {
            if (i < wave) before += wsum[0][i];
            tot += wsum[0][i];
        }
        n_tie += tot;
        before += __builtin_popcountll(ties & ((1ull << lane) - 1));
        const bool kept = fixed || (mid && (k > key || (tie && before < left)));
        const uint64_t keeps = __ballot(kept);
        if (lane == 0) wsum[1][wave] = __builtin_popcountll(keeps);
        __syncthreads();
        int at = n_kept;
        tot = 0;
        for (int i = 0; i < kEvThr / kWave; ++i) {
            if (i < wave) at += wsum[1][i];
            tot += wsum[1][i];
        }
        n_kept += tot;
        at += __builtin_popcountll(keeps & ((1ull << lane) - 1));   // kept blocks before j
        if (j < n_blocks) {
            const int to = kept ? at : stay + j - at;
            b_out[base + to] = blocks ? blocks[base + j] : j;
            if (kept) w_out[base + to] = x;
            else if (to > stay || full == n_blocks) w_out[base + to] = 0.f;
        }
    }
    if (tid == 0) {
        if (full < n_blocks) w_out[base + stay] = w[full];   // the unfinished block's
        if (blockIdx.x % n_kv == 0) c_out[b] = n - (full - stay) * kBlk;
    }
}

}  // namespace hxq

using namespace hxq;

namespace {

bool kv8_ok(const hxq_kv8 *c, bool need) {
    if (!c || !attn_dtype(c->dtype, false) || c->batch <= 0 || c->n_kv_heads <= 0) return false;
    if (c->head_dim != 64 && c->head_dim != 128) return false;
    if (!c->k) return !need;
    const auto al = [](const void *p) { return p && reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    return al(c->k) && al(c->v) && al(c->k_tail) && al(c->v_tail) && c->k_scale && c->v_scale && c->n_blocks > 0 &&
           c->n_blocks <= (1 << 24);
}

// go(row dtype, cache in bf16, head_dim) as constants
template <typename F>
void kv8_dispatch(int32_t dtype, const hxq_kv8 &c, F go) {
    const auto by_d = [&](auto dt, auto bf) {
        if (c.head_dim == 128) go(dt, bf, std::integral_constant<int, 128>{});
        else go(dt, bf, std::integral_constant<int, 64>{});
    };
    const auto by_c = [&](auto dt) {
        if (c.dtype == HXQ_BF16) by_d(dt, std::true_type{});
        else by_d(dt, std::false_type{});
    };
    if (dtype == HXQ_F32) by_c(std::integral_constant<int, HXQ_F32>{});
    else if (dtype == HXQ_BF16) by_c(std::integral_constant<int, HXQ_BF16>{});
    else by_c(std::integral_constant<int, HXQ_F16>{});
}

// Splits of one sequence's cache: enough for 4 blocks a compute unit (sequences of different lengths
// even out), down to 16 units each, two for a wave; where that leaves compute units idle, down to 8.
int kv8_splits(int64_t tiles, int32_t n_blocks) {
    const int64_t cus = device_cu_count();
    const int64_t even = std::min<int64_t>((4 * cus + tiles - 1) / tiles, (n_blocks + 15) / 16);
    const int64_t idle = std::min<int64_t>((cus + tiles - 1) / tiles, (n_blocks + 7) / 8);
    return static_cast<int>(std::max<int64_t>(1, std::max(even, idle)));
}

int64_t kv8_tiles(int32_t batch, int32_t n_heads, int32_t n_kv) {
    return (int64_t)batch * n_kv * ((n_heads / n_kv + kHT - 1) / kHT);
}

// Workspace: part, then ml, then share.
struct Kv8Ws {
    int64_t ml, share, bytes;
};

Kv8Ws kv8_ws(int32_t batch, int32_t n_heads, int splits, int32_t D, int32_t n_blocks, bool weights) {
    const int64_t rows = (int64_t)batch * n_heads;
    Kv8Ws w;
    w.ml = splits > 1 ? rows * splits * D * 4 : 0;
    w.share = w.ml + (splits > 1 || weights ? (rows * splits * 8 + 15) / 16 * 16 : 0);
    w.bytes = w.share + (weights ? rows * n_blocks * 8 : 0);
    return w;
}

}  // namespace

extern "C" int hxq_kv8_append(const void *q, int64_t q_row_stride, int64_t q_head_stride, const void *k,
                              int64_t k_row_stride, int64_t k_head_stride, const void *v, int64_t v_row_stride,
                              int64_t v_head_stride, int32_t dtype, const int32_t *cu_rows, int64_t rows,
                              int32_t n_heads, const int32_t *cached, const int32_t *pos, float theta,
                              const hxq_kv8 *cache, void *q_out, void *k_out, void *v_out, hipStream_t stream) {
    clear_error();
    HXQ_REQUIRE(kv8_ok(cache, false), "bad cache (dtype bf16 or fp16, head_dim 64 or 128, 16-byte aligned pointers)");
    HXQ_REQUIRE(cu_rows && cached && (rows == 0 || (k && v && (q || !q_out))), "q, k, v, cu_rows and cached are required");
    HXQ_REQUIRE(attn_dtype(dtype, true), "bad dtype");
    HXQ_REQUIRE(rows >= 0 && rows < (int64_t{1} << 31) - 2 * kBlk && n_heads > 0 && n_heads % cache->n_kv_heads == 0,
                "bad sizes (n_heads must be a multiple of n_kv_heads)");
    HXQ_REQUIRE(theta >= 0.f && theta < INFINITY, "theta must be finite and not negative");
    const HeadRows qr{q, q_row_stride, q_head_stride}, kr{k, k_row_stride, k_head_stride}, vr{v, v_row_stride, v_head_stride};
    HXQ_REQUIRE((!q_out || rows_aligned(qr, dtype)) && rows_aligned(kr, dtype) && rows_aligned(vr, dtype),
                "q, k and v need pointers and strides that are multiples of 16 bytes");
    for (const void *p : {q_out, k_out, v_out})
        HXQ_REQUIRE(reinterpret_cast<uintptr_t>(p) % 16 == 0, "outputs must be 16-byte aligned");
    if (rows == 0) return HXQ_OK;
    const AppendArgs a{qr, kr, vr, cu_rows, cached, pos, rope_table(theta, cache->head_dim), static_cast<int32_t>(rows), n_heads, *cache, q_out, k_out, v_out};
    const int64_t tiles = rows / kBlk + 2 * (int64_t)cache->batch;
    const int64_t heads = cache->n_kv_heads + (q_out ? (n_heads + kQHeads - 1) / kQHeads : 0);
    HXQ_REQUIRE(tiles * kThr < kMaxThreads && heads <= 65535, "too many rows, sequences or heads");
    const dim3 grid(static_cast<uint32_t>(tiles), static_cast<uint32_t>(heads));
    kv8_dispatch(dtype, *cache, [&](auto dt, auto bf, auto d) {
        hipLaunchKernelGGL((kv8_append_kernel<decltype(dt)::value, decltype(bf)::value, decltype(d)::value>), grid,
                           dim3(kThr), 0, stream, a);
    });
    HXQ_LAUNCH_CHECK();
    return HXQ_OK;
}

extern "C" int64_t hxq_kv8_attn_decode_workspace_bytes(int32_t batch, int32_t n_heads, int32_t n_kv_heads,
                                                       int32_t head_dim, int32_t n_blocks, int32_t weights) {
    if (batch <= 0 || n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads || n_blocks <= 0 ||
        (head_dim != 64 && head_dim != 128)) return -1;
    const int s = kv8_splits(kv8_tiles(batch, n_heads, n_kv_heads), n_blocks);
    return kv8_ws(batch, n_heads, s, head_dim, n_blocks, weights != 0).bytes;
}

extern "C" int hxq_kv8_attn_decode(const void *q, int64_t q_row_stride, int64_t q_head_stride, const void *k,
                                   int64_t k_row_stride, int64_t k_head_stride, const void *v, int64_t v_row_stride,
                                   int64_t v_head_stride, int32_t dtype, int32_t n_heads, const int32_t *cached,
                                   const int32_t *pos, float theta, float scale, const hxq_kv8 *cache,
                                   const float *weight_in, float *weight_out, void *out, int32_t out_dtype,
                                   void *workspace, int64_t workspace_bytes, hipStream_t stream) {
    clear_error();
    HXQ_REQUIRE(kv8_ok(cache, true), "bad cache (dtype bf16 or fp16, head_dim 64 or 128, 16-byte aligned pointers)");
    HXQ_REQUIRE(q && k && v && cached && out, "q, k, v, cached and out are required");
    HXQ_REQUIRE(attn_dtype(dtype, true) && attn_dtype(out_dtype, true), "bad dtype");
    HXQ_REQUIRE(n_heads > 0 && n_heads % cache->n_kv_heads == 0, "n_heads must be a multiple of n_kv_heads");
    HXQ_REQUIRE(theta >= 0.f && theta < INFINITY && fabsf(scale) <= 0x1p100f,
                "theta must be finite and not negative, scale finite and at most 2^100");
    HXQ_REQUIRE(weight_out || !weight_in, "weight_in without weight_out");
    const int64_t tiles = kv8_tiles(cache->batch, n_heads, cache->n_kv_heads);
    HXQ_REQUIRE(cache->batch <= 65535 && tiles / cache->batch <= 65535 && (int64_t)cache->batch * n_heads < (int64_t{1} << 31), "batch or heads too large");
    const int splits = kv8_splits(tiles, cache->n_blocks);
    const Kv8Ws w = kv8_ws(cache->batch, n_heads, splits, cache->head_dim, cache->n_blocks, weight_out != nullptr);
    HXQ_REQUIRE(w.bytes == 0 || (workspace && workspace_bytes >= w.bytes && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                "workspace too small or not 16-byte aligned");
    char *ws = static_cast<char *>(workspace);
    const DecodeArgs a{{q, q_row_stride, q_head_stride}, {k, k_row_stride, k_head_stride}, {v, v_row_stride, v_head_stride},
                       cached, pos, rope_table(theta, cache->head_dim), scale * 1.44269504088896340736f, out_dtype, n_heads, splits,
                       n_heads / cache->n_kv_heads, (n_heads / cache->n_kv_heads + kHT - 1) / kHT, *cache,
                       weight_in, weight_out, out, reinterpret_cast<float *>(ws),
                       reinterpret_cast<float2 *>(ws + w.ml), reinterpret_cast<float2 *>(ws + w.share)};
    // what the second launch has to do: rows to join, chunks of weights
    const int64_t rows = (int64_t)cache->batch * n_heads;
    const int64_t chunks = weight_out ? (int64_t)cache->batch * cache->n_kv_heads * ((cache->n_blocks + kThr - 1) / kThr) : 0;
    HXQ_REQUIRE((rows + chunks) * kThr < kMaxThreads, "batch * heads or blocks too large");
    const int64_t row_blocks = splits == 1 ? 0 : splits <= kFewSplits ? (rows + kThr / kWave - 1) / (kThr / kWave) : rows;
    const dim3 join(static_cast<uint32_t>(row_blocks + chunks));
    const dim3 grid(splits, static_cast<uint32_t>(tiles / cache->batch), cache->batch);
    const auto go = [&](auto dt, auto bf, auto dd) {
        constexpr int T = decltype(dt)::value, D = decltype(dd)::value;
        constexpr bool B = decltype(bf)::value;
        if (weight_out) hipLaunchKernelGGL((kv8_decode_kernel<T, B, D, true>), grid, dim3(kDThr), 0, stream, a);
        else hipLaunchKernelGGL((kv8_decode_kernel<T, B, D, false>), grid, dim3(kDThr), 0, stream, a);
        if (splits > 1 || weight_out) hipLaunchKernelGGL((kv8_join_kernel<D>), join, dim3(kThr), 0, stream, a, static_cast<int>(row_blocks));
    };
    kv8_dispatch(dtype, *cache, go);
    HXQ_LAUNCH_CHECK();
    return HXQ_OK;
}

extern "C" int hxq_kv8_evict(const float *weight, const int32_t *blocks_in, const int32_t *cached, int32_t batch,
                             int32_t n_kv_heads, int32_t n_blocks, int32_t keep, int32_t sink, int32_t recent,
                             float *weight_out, int32_t *blocks_out, int32_t *cached_out, hipStream_t stream) {
    clear_error();
    HXQ_REQUIRE(weight && cached && weight_out && blocks_out && cached_out, "weight, cached and the outputs are required");
    HXQ_REQUIRE(weight != weight_out && blocks_in != blocks_out && cached != cached_out, "outputs must not be the inputs");
    HXQ_REQUIRE(batch > 0 && n_kv_heads > 0 && n_blocks > 0 && n_blocks <= (1 << 24) &&
                    (int64_t)batch * n_kv_heads * kEvThr < kMaxThreads, "bad sizes");
    HXQ_REQUIRE(keep > 0 && sink >= 0 && recent >= 0 && (int64_t)sink + recent <= keep,
                "keep must be positive and hold the first `sink` and the last `recent` blocks");
    hipLaunchKernelGGL(kv8_evict_kernel, dim3(batch * n_kv_heads), dim3(kEvThr), 0, stream, weight, blocks_in, cached,
                       n_kv_heads, n_blocks, keep, sink, recent, weight_out, blocks_out, cached_out);
    HXQ_LAUNCH_CHECK();
    return HXQ_OK;
}
