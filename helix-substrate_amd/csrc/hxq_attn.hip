// Attention of packed prompts: causal, grouped heads, sequences of different lengths.
#include "hxq_attn.h"

namespace hxq {

struct PromptArgs {
    HeadRows q, k, v;
    void *out;
    int64_t out_row, out_head;
    const int32_t *cu_q, *cu_k;
    int32_t n_seqs, rows_q, rows_k, n_heads, group, tiles;
    float scale2;   // scale * log2(e): the softmax is in powers of two
};

constexpr int kBM = 128;    // query rows of a block
constexpr int kBN = 64;     // keys of a step
constexpr int kPThr = 256;

template <bool BF16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Transposing read: in each group of 16 lanes, result lane 4 q + c gets as element e the element c
// of the 8 bytes addressed by lane 4 e + q.
__device__ __forceinline__ u32x2 lds_tr(const uint16_t *p) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(p)));
}

// Element offset of 16-byte chunk c of row r of a staged tile.  The chunk is XORed with the row's
// low bits: rows 0..15 at one chunk (the reads of K) and rows r..r+3 at four neighbouring chunks
// (the transposing reads of V) both hit distinct banks.
template <int D>
__device__ __forceinline__ int swz(int r, int c) {
    if constexpr (D == 128) return r * D + ((c ^ ((r & 3) << 2 | (r >> 2 & 3))) << 3);
    else return r * D + ((c ^ ((r & 2) << 1 | (r >> 1 & 2) | (r >> 3 & 1))) << 3);   // two rows share the banks
}

__device__ __forceinline__ float half_max(float v) {   // over lanes l, l ^ 32
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

__device__ __forceinline__ float half_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Both values of a pair finite?  If not, those that are not become 0 in w.
template <bool BF16>
__device__ __forceinline__ bool drop_nonfinite(uint32_t &w) {
    constexpr uint32_t E = BF16 ? 0x7f80u : 0x7c00u;
    const bool lo = (w & E) == E, hi = (w >> 16 & E) == E;
    if (lo) w &= 0xffff0000u;
    if (hi) w &= 0xffffu;
    return lo || hi;
}

// One block: 128 query rows of one head, a wave 32 of them; steps of 64 keys with the running
// maximum and sum of the softmax.  Both products are transposed, S^T = K Q^T and O^T = V^T P^T, so
// that a lane holds scores of one query (its column): the softmax is in the lane but for one
// exchange of halves, and P^T is the second product's operand in the lane's own registers.  For
// that, row 8 a + 4 h + c of a K tile is given the key 16 (a / 2) + 8 h + 4 (a % 2) + c.
// A weight of 0 does not undo an infinity or NaN of v: in the steps where some query of the block
// does not see some key, such values are staged as 0, their rows marked, and added to the queries
// that see them.
template <bool BF16, int D, bool CAUSAL>
__global__ __launch_bounds__(kPThr, 2) void attn_prompt_kernel(const PromptArgs a) {
    constexpr int NK = D / 16, ND = D / 32, CPR = D / 8, NL = kBN * CPR / kPThr;
    __shared__ __attribute__((aligned(16))) uint16_t sk[kBN * D], sv[kBN * D];
    __shared__ uint32_t odd_rows[2][2];   // of this step and the next: a bit for each key
    const int head = blockIdx.x % a.n_heads, t_id = a.tiles - 1 - blockIdx.x / a.n_heads;
    int seq, tile;
    const auto count = [&](int s) {
        return (max(seq_off(a.cu_q, s + 1, a.rows_q) - seq_off(a.cu_q, s, a.rows_q), 0) + kBM - 1) / kBM;
    };
    if (!seq_tile(a.n_seqs, t_id, count, seq, tile)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ql = lane & 31, hh = lane >> 5;
    const int q_beg = seq_off(a.cu_q, seq, a.rows_q), lq = seq_off(a.cu_q, seq + 1, a.rows_q) - q_beg;
    const int k_beg = seq_off(a.cu_k, seq, a.rows_k), lk = max(seq_off(a.cu_k, seq + 1, a.rows_k) - k_beg, 0);
    const int i0 = tile * kBM, iw = i0 + wave * 32, iq = iw + ql;   // in the sequence
    const int past = lk - lq;
    const int64_t kvh = head / a.group;
    const uint16_t *kp = static_cast<const uint16_t *>(a.k.p) + kvh * a.k.head + (int64_t)k_beg * a.k.row;
    const uint16_t *vp = static_cast<const uint16_t *>(a.v.p) + kvh * a.v.head + (int64_t)k_beg * a.v.row;
    u32x4 q[NK];
    {
        const uint16_t *p = static_cast<const uint16_t *>(a.q.p) + head * a.q.head + (int64_t)(q_beg + min(iq, lq - 1)) * a.q.row + 8 * hh;
#pragma unroll
        for (int s = 0; s < NK; ++s) q[s] = *reinterpret_cast<const u32x4 *>(p + 16 * s);
    }
    f32x16 o[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
    float m = -INFINITY, keep = -INFINITY, l = 0.f;
    const int last = min(i0 + kBM, lq) - 1;                           // the block's last query
    const int n_keys = CAUSAL ? min(lk, max(last + past + 1, 0)) : lk;   // keys that it sees
    const int lim = CAUSAL ? min(iq + past, lk - 1) : lk - 1;         // the lane's last key
    const int lim_b = min(i0 + past, lk - 1);                         // the least of the block's
    const int row_k = (ql & 0x13) | (ql & 4) << 1 | (ql & 8) >> 1;    // key of the lane's row
    if (threadIdx.x < 4) odd_rows[threadIdx.x >> 1][threadIdx.x & 1] = 0u;

    // a step's keys and values go through registers, asked for one step ahead
    u32x4 kr[NL], vr[NL];
    const uint32_t off_k = static_cast<uint32_t>((threadIdx.x / CPR) * a.k.row + threadIdx.x % CPR * 8) * 2;
    const uint32_t off_v = static_cast<uint32_t>((threadIdx.x / CPR) * a.v.row + threadIdx.x % CPR * 8) * 2;
    constexpr int RPP = kPThr / CPR;   // rows a pass
    const auto fetch = [&](int j0) {
        const char *kb = reinterpret_cast<const char *>(kp + j0 * a.k.row);
        const char *vb = reinterpret_cast<const char *>(vp + j0 * a.v.row);
        if (j0 + kBN <= lk) {
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                kr[i] = *reinterpret_cast<const u32x4 *>(kb + i * RPP * a.k.row * 2 + off_k);
                vr[i] = *reinterpret_cast<const u32x4 *>(vb + i * RPP * a.v.row * 2 + off_v);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                kr[i] = vr[i] = u32x4{0u, 0u, 0u, 0u};
                if (j0 + static_cast<int>(threadIdx.x / CPR) + i * RPP < lk) {
                    kr[i] = *reinterpret_cast<const u32x4 *>(kb + i * RPP * a.k.row * 2 + off_k);
                    vr[i] = *reinterpret_cast<const u32x4 *>(vb + i * RPP * a.v.row * 2 + off_v);
                }
            }
        }
    };
    // EDGE: some query of the block does not see some key of the step
    const auto step = [&](int j0, auto edge_c) {
        constexpr bool EDGE = decltype(edge_c)::value;
        uint32_t *odd = odd_rows[j0 / kBN & 1];
        lds_barrier();
        if constexpr (EDGE) {
            if (threadIdx.x < 2) odd_rows[(j0 / kBN & 1) ^ 1][threadIdx.x] = 0u;
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int r = (threadIdx.x + i * kPThr) / CPR;
                bool found = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t w = vr[i][e];
                    found |= drop_nonfinite<BF16>(w);
                    vr[i][e] = w;
                }
                if (found) atomicOr(&odd[r >> 5], 1u << (r & 31));
            }
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int c = threadIdx.x + i * kPThr;
            *reinterpret_cast<u32x4 *>(sk + swz<D>(c / CPR, c % CPR)) = kr[i];
            *reinterpret_cast<u32x4 *>(sv + swz<D>(c / CPR, c % CPR)) = vr[i];
        }
        lds_barrier();
        if (j0 + kBN < n_keys) fetch(j0 + kBN);
        f32x16 s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
#pragma unroll
            for (int x = 0; x < NK; ++x)
                s[t] = mfma32<BF16>(*reinterpret_cast<const u32x4 *>(sk + swz<D>(32 * t + row_k, 2 * x + hh)), q[x], s[t]);
        }
        float mx = -INFINITY;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                if (EDGE && j0 + 32 * t + 16 * (r / 8) + 8 * hh + r % 8 > lim) s[t][r] = -INFINITY;
                mx = fmaxf(mx, s[t][r]);
            }
        // The running maximum is kept while no score passes it by more than 2^8 in weight: the sums
        // stay far from fp32's range, and the accumulators are rescaled a few times in a row only.
        mx = half_max(mx);
        if (__any(mx > keep)) {
            const float mn = fmaxf(m, mx);
            const float al = m == mn ? 1.f : __builtin_amdgcn_exp2f((m - mn) * a.scale2);   // both may be -inf
            m = mn;
            keep = m + 8.f / a.scale2;
            l *= al;
#pragma unroll
            for (int i = 0; i < ND; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[i][r] *= al;
        }
        const float base = m == -INFINITY ? 0.f : m * a.scale2;   // nothing seen yet: p = 0
        u32x4 p[4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[t][r], a.scale2, -base));
                const float y = __builtin_amdgcn_exp2f(fmaf(s[t][r + 1], a.scale2, -base));
                l += x + y;
                p[2 * t + r / 8][r % 8 / 2] = pack16<BF16>(x, y);
            }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int i = 0; i < ND; ++i) {
                // keys 16 x + 8 hh + 0..7 of column 32 i + ql
                const int r = 16 * x + 8 * hh + (lane >> 2 & 3), c = 4 * i + 2 * (lane >> 4 & 1) + (lane >> 1 & 1);
                const u32x2 lo = lds_tr(sv + swz<D>(r, c) + 4 * (lane & 1)), hi = lds_tr(sv + swz<D>(r + 4, c) + 4 * (lane & 1));
                o[i] = mfma32<BF16>(u32x4{lo[0], lo[1], hi[0], hi[1]}, p[x], o[i]);
            }
        if constexpr (EDGE) {
            for (int t = 0; t < kBN; ++t) {
                if (!(odd[t >> 5] >> (t & 31) & 1u) || j0 + t > lim) continue;
                const uint16_t *row = vp + (int64_t)(j0 + t) * a.v.row + 4 * hh;
#pragma unroll
                for (int i = 0; i < ND; ++i)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const float x = BF16 ? bf16_to_f32(row[32 * i + 2 * (r & 12) + (r & 3)])
                                             : f16_to_f32(row[32 * i + 2 * (r & 12) + (r & 3)]);
                        if (!(fabsf(x) < INFINITY)) o[i][r] += x;
                    }
            }
        }
    };
    if (n_keys > 0) fetch(0);
    int j0 = 0;
    for (; j0 + kBN <= min(n_keys, lim_b + 1); j0 += kBN) step(j0, std::false_type{});
    for (; j0 < n_keys; j0 += kBN) step(j0, std::true_type{});
    l = half_sum(l);
    if (iq >= lq) return;
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;   // no key seen: zeros
    uint16_t *op = static_cast<uint16_t *>(a.out) + head * a.out_head + (int64_t)(q_beg + iq) * a.out_row;
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<u32x2 *>(op + 32 * i + 2 * r + 4 * hh) =
                u32x2{pack16<BF16>(o[i][r] * inv, o[i][r + 1] * inv), pack16<BF16>(o[i][r + 2] * inv, o[i][r + 3] * inv)};
}

}  // namespace hxq

using namespace hxq;

extern "C" int hxq_attn_prompt(const void *q, int64_t q_row_stride, int64_t q_head_stride, const void *k,
                               int64_t k_row_stride, int64_t k_head_stride, const void *v, int64_t v_row_stride,
                               int64_t v_head_stride, int32_t dtype, const int32_t *cu_q, const int32_t *cu_k,
                               int32_t n_seqs, int64_t rows_q, int64_t rows_k, int32_t n_heads, int32_t n_kv_heads,
                               int32_t head_dim, float scale, int32_t causal, void *out, int64_t out_row_stride,
                               int64_t out_head_stride, hipStream_t stream) {
    clear_error();
    HXQ_REQUIRE(attn_dtype(dtype, false), "q, k and v must be bf16 or fp16");
    HXQ_REQUIRE(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128");
    HXQ_REQUIRE(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0, "n_heads must be a multiple of n_kv_heads");
    HXQ_REQUIRE(n_seqs >= 0 && rows_q >= 0 && rows_k >= 0 && rows_q < (int64_t{1} << 31) - 4 * kBM &&
                    rows_k < (int64_t{1} << 31) - 4 * kBM, "bad sizes");
    HXQ_REQUIRE(scale == scale && scale > 0.f && scale < INFINITY, "scale must be positive and finite");
    if (n_seqs == 0 || rows_q == 0) return HXQ_OK;
    HXQ_REQUIRE(q && out && cu_q && (rows_k == 0 || (k && v)), "q, k, v, cu_q and out are required");
    const HeadRows qr{q, q_row_stride, q_head_stride}, kr{k, k_row_stride, k_head_stride}, vr{v, v_row_stride, v_head_stride},
        orow{out, out_row_stride, out_head_stride};
    HXQ_REQUIRE(k_row_stride < (1 << 24) && v_row_stride < (1 << 24) && k_row_stride >= 0 && v_row_stride >= 0,
                "row strides of k and v must be at least 0 and less than 2^24 elements");
    HXQ_REQUIRE(rows_aligned(qr, dtype) && rows_aligned(kr, dtype) && rows_aligned(vr, dtype) && rows_aligned(orow, dtype),
                "q, k, v and out need pointers and strides that are multiples of 16 bytes");
    const int64_t tiles = rows_q / kBM + n_seqs;
    HXQ_REQUIRE(tiles * n_heads < (int64_t{1} << 31), "too many rows");
    const PromptArgs a{qr, kr, vr, out, out_row_stride, out_head_stride, cu_q, cu_k ? cu_k : cu_q, n_seqs,
                       static_cast<int32_t>(rows_q), static_cast<int32_t>(rows_k), n_heads, n_heads / n_kv_heads,
                       static_cast<int32_t>(tiles), scale * 1.44269504088896340736f};
    const dim3 grid(static_cast<uint32_t>(tiles * n_heads));
    const auto go = [&](auto bf, auto dd) {
        constexpr bool B = decltype(bf)::value;
        constexpr int D = decltype(dd)::value;
        if (causal) hipLaunchKernelGGL((attn_prompt_kernel<B, D, true>), grid, dim3(kPThr), 0, stream, a);
        else hipLaunchKernelGGL((attn_prompt_kernel<B, D, false>), grid, dim3(kPThr), 0, stream, a);
    };
    const auto by_d = [&](auto bf) {
        if (head_dim == 128) go(bf, std::integral_constant<int, 128>{});
        else go(bf, std::integral_constant<int, 64>{});
    };
    if (dtype == HXQ_BF16) by_d(std::true_type{});
    else by_d(std::false_type{});
    HXQ_LAUNCH_CHECK();
    return HXQ_OK;
}
