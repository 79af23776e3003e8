// What the prompt attention and the 8-bit cache share: argument checks, packed
// sequences, rotation.
#pragma once

#include <math.h>

#include "hxq_common.h"

namespace hxq {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int64_t kMaxThreads = int64_t{1} << 32;   // a launch has fewer in x

// [rows, heads, head_dim] with strides in elements
struct HeadRows {
    const void *p;
    int64_t row, head;
};

inline bool attn_dtype(int32_t d, bool f32) {
    return d == HXQ_BF16 || d == HXQ_F16 || (f32 && d == HXQ_F32);
}

// pointer and strides are multiples of 16 bytes (the kernels load 16 bytes a lane)
inline bool rows_aligned(const HeadRows &r, int32_t dtype) {
    const int64_t e = dtype == HXQ_F32 ? 4 : 8;
    return reinterpret_cast<uintptr_t>(r.p) % 16 == 0 && r.row % e == 0 && r.head % e == 0;
}

// Offset i of a packed batch, inside [0, rows] whatever the array holds.
__device__ __forceinline__ int seq_off(const int32_t *cu, int i, int rows) {
    return min(max(cu[i], 0), rows);
}

// Tile t (counted over all sequences, count(s) of them in sequence s): its
// sequence and its number in it; false past the last.  Every wave computes it
// alike (lanes cover sequences s, s + 64, ...).
template <typename F>
__device__ __forceinline__ bool seq_tile(int n_seqs, int t, F count, int &seq, int &tile) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    for (int s0 = 0; s0 < n_seqs; s0 += 64) {
        const int n = s0 + lane < n_seqs ? count(s0 + lane) : 0;
        const int inc = wave_scan(n);
        const int tot = __builtin_amdgcn_readlane(inc, 63);
        if (t < base + tot) {
            const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(__ballot(base + inc > t)));
            seq = s0 + l;
            tile = t - base - __builtin_amdgcn_readlane(inc - n, l);
            return true;
        }
        base += tot;
    }
    return false;
}

// Turns per position of pair i of D/2: theta^(-i / (D/2)) / 2 pi, in 64 bits (at position 10^5 an fp32
// frequency is off by 10^5 2^-24 / 2 pi = 10^-3 turns).  p[k] = theta^(-2^k / (D/2)) comes from the
// host: the power is six products, not a 64-bit exp and log in every launch.
struct RopeTable {
    double p[6];
    bool on;
};

inline RopeTable rope_table(float theta, int head_dim) {
    RopeTable t{};
    t.on = theta > 0.f;
    if (t.on)
        for (int k = 0; k < 6; ++k) t.p[k] = pow(static_cast<double>(theta), -(1 << k) / (head_dim / 2.0));
    return t;
}

__device__ __forceinline__ double rope_turns(const RopeTable &t, int i) {
    double f = 0.15915494309189533577;
#pragma unroll
    for (int k = 0; k < 6; ++k) f *= i >> k & 1 ? t.p[k] : 1.0;
    return f;
}

// A prompt's rows and single tokens are rotated in different kernels and have to give the same bits: the
// two functions below say where products and sums are rounded once, and contract nothing by themselves.

// cos and sin of pos * turns (in turns), reduced to half a turn in 64 bits.
__device__ __forceinline__ void rope_cs(int pos, double turns, float &c, float &s) {
#pragma clang fp contract(off)
    const double p = pos;
    sincospif(2.f * static_cast<float>(fma(p, turns, -rint(p * turns))), &s, &c);
}

// The pair (x1, x2) turned.
__device__ __forceinline__ void rope_turn(float x1, float x2, float c, float s, float &y1, float &y2) {
#pragma clang fp contract(off)
    y1 = fmaf(x1, c, -(x2 * s));
    y2 = fmaf(x1, s, x2 * c);
}

}  // namespace hxq
