// Attention of packed prompts: causal, grouped heads, sequences of different lengths.
#include <algorithm>

#include "hxq_attn.h"

namespace hxq {

struct PromptArgs {
    HeadRows q, k, v;
    void *out;
    int64_t out_row, out_head;
    const int32_t *cu_q, *cu_k;
    int32_t n_seqs, rows_q, rows_k, n_heads, group;
    float scale2;   // scale * log2(e): the softmax is in powers of two
    int32_t splits, by_die;
    float *part;    // [rows_q * n_heads][splits][D]: sums of p v of a split's keys
    float2 *ml;     // [rows_q * n_heads][splits]: their maximum (in powers of two) and sum of p
};

constexpr int kMaxSplits = 16;

// Steps of 64 keys of one split; at least 4, and even (steps are taken in pairs).
__device__ __forceinline__ int steps_per_split(int steps, int splits) { return max((steps + splits - 1) / splits + 1 & ~1, 4); }

// Keys that the queries up to `last` of a sequence see.
template <bool CAUSAL>
__device__ __forceinline__ int keys_seen(int last, int lq, int lk) {
    return CAUSAL ? min(lk, max(last + lk - lq + 1, 0)) : lk;
}

constexpr int kBN = 64;     // keys of a step

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

// 16 bytes a lane from `from` to LDS: lane l's to 16 l bytes behind `to` (the same in all lanes).
__device__ __forceinline__ void load_lds16(const uint16_t *from, uint16_t *to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                     (__attribute__((address_space(3))) void *)to, 16, 0, 0);
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

// A block's part of a packed batch.
struct PromptTile {
    int tile, q_beg, lq, k_beg, lk;   // tile of its sequence; the sequence's rows
};

// Tile t_id of a launch: tiles are dealt by the keys they see, the most first (the long ones do not
// come last), over all sequences.  Tile `tile` of BM queries of a sequence with `base` tiles of earlier
// keys has level base + tile; the number of tiles of a level or above is searched by halving.  The
// first 64 sequences are held one in a lane: one round of loads, then registers only.
template <int BM>
__device__ __forceinline__ bool prompt_tile(const PromptArgs &a, int t_id, PromptTile &at) {
    const int lane = threadIdx.x & 63;
    struct Seq {
        int q_beg, lq, k_beg, lk, n, base;
    };
    const auto load = [&](int s) {
        Seq x{0, 0, 0, 0, 0, 0};
        if (s >= a.n_seqs) return x;
        x.q_beg = seq_off(a.cu_q, s, a.rows_q);
        x.lq = max(seq_off(a.cu_q, s + 1, a.rows_q) - x.q_beg, 0);
        x.k_beg = seq_off(a.cu_k, s, a.rows_k);
        x.lk = max(seq_off(a.cu_k, s + 1, a.rows_k) - x.k_beg, 0);
        x.n = (x.lq + BM - 1) / BM;
        x.base = max(x.lk - x.lq, 0) / BM;
        return x;
    };
    const auto of_level = [](const Seq &x, int L) { return min(max(x.n + x.base - L, 0), x.n); };   // L or above
    const Seq first = load(lane);
    const auto above = [&](int L) {
        int v = of_level(first, L);
        for (int s = lane + 64; s - lane < a.n_seqs; s += 64) v += of_level(load(s), L);
        return __builtin_amdgcn_readlane(wave_scan(v), 63);
    };
    if (t_id >= above(0)) return false;
    int lo = 0, hi = first.n + first.base;   // above(lo) > t_id >= above(hi)
    if (a.n_seqs > 64) hi = a.rows_q / BM + a.rows_k / BM + 2;
    else {
#pragma unroll
        for (int m = 32; m >= 1; m >>= 1) hi = max(hi, __shfl_xor(hi, m, kWave));
    }
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (above(mid) > t_id) lo = mid;
        else hi = mid;
    }
    // among the sequences that have a tile of level lo, in order
    int left = t_id - above(lo + 1);
    for (int s0 = 0; s0 < a.n_seqs; s0 += 64) {
        const Seq x = s0 ? load(s0 + lane) : first;
        const uint64_t has = __ballot(lo >= x.base && lo < x.base + x.n);
        const int c = __builtin_popcountll(has);
        if (left < c) {
            // the lane with `left` others before it
            const int mine = __builtin_popcountll(has & ((1ull << lane) - 1));
            const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(__ballot((has >> lane & 1) && mine == left)));
            at = PromptTile{lo - __builtin_amdgcn_readlane(x.base, l), __builtin_amdgcn_readlane(x.q_beg, l),
                            __builtin_amdgcn_readlane(x.lq, l), __builtin_amdgcn_readlane(x.k_beg, l),
                            __builtin_amdgcn_readlane(x.lk, l)};
            return true;
        }
        left -= c;
    }
    return false;
}

// V^T as an operand: keys 16 x + 8 hh + 0..7 of column 32 i + lane % 32.
template <int D>
__device__ __forceinline__ u32x4 v_operand(const uint16_t *v, int x, int i, int lane) {
    const int r = 16 * x + 8 * (lane >> 5) + (lane >> 2 & 3), c = 4 * i + 2 * (lane >> 4 & 1) + (lane >> 1 & 1);
    const u32x2 lo = lds_tr(v + swz<D>(r, c) + 4 * (lane & 1)), hi = lds_tr(v + swz<D>(r + 4, c) + 4 * (lane & 1));
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

// Adds what is not finite in a row of v (which was staged as 0).
template <bool BF16, int ND>
__device__ __forceinline__ void add_odd(const uint16_t *row, bool seen, f32x16 (&o)[ND]) {
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const uint16_t w = row[32 * i + 2 * (r & 12) + (r & 3)];
            const float x = BF16 ? bf16_to_f32(w) : f16_to_f32(w);
            o[i][r] += seen && !(fabsf(x) < INFINITY) ? x : 0.f;
        }
}

// What the weights are divided by: no key seen gives zeros; keys seen but every score -inf, NaN as 0 / 0.
__device__ __forceinline__ float inv_sum(float sum, bool sees) {
    return sum > 0.f || sum != sum ? 1.f / sum : sees ? __uint_as_float(0x7fc00000u) : 0.f;
}

template <bool BF16, int ND>
__device__ __forceinline__ void store_rows(const f32x16 (&o)[ND], float inv, uint16_t *to) {
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<u32x2 *>(to + 32 * i + 2 * r) =
                u32x2{pack16<BF16>(o[i][r] * inv, o[i][r + 1] * inv), pack16<BF16>(o[i][r + 2] * inv, o[i][r + 3] * inv)};
}

// One block: 32 NW query rows of one head, a wave 32 of them; steps of 64 keys with the running
// maximum and sum of the softmax.  Both products are transposed, S^T = K Q^T and O^T = V^T P^T, so
// that a lane holds scores of one query (its column): the softmax is in the lane but for one
// exchange of halves, and P^T is the second product's operand in the lane's own registers.  For
// that, row 8 a + 4 h + c of a K tile is given the key 16 (a / 2) + 8 h + 4 (a % 2) + c.
// A weight of 0 does not undo an infinity or NaN of v: in the steps where some query of the block
// does not see some key, such values are staged as 0, their rows marked, and added at the end to the
// queries that see them.
//
// NW = 4: 128 queries, two blocks on a compute unit, two buffers that the next step's loads fill directly
// (twelve sequences 226 us, one buffer filled through registers 240); at head_dim 64 three blocks, one
// buffer, through registers (101 us; as above 106).  NW = 8: 256 queries, two buffers, through registers
// (992 us; directly 1003); half the bytes a query are staged.
// KW: 32 queries a block, its four waves take steps of 64 keys in turn, each with a tile of its own in
// LDS (loaded straight into it, no barrier), and join their sums at the end: for calls too small to fill
// the chip, where the chain of a block's steps is the time.
// SPLIT: blockIdx.y takes a part of the keys and leaves its sums for attn_join_kernel.
//
// Bound by the issue of MFMA, softmax and LDS reads together: the matrix pipe is busy 54 % of the cycles,
// LDS 34 %, without bank conflicts.  P in the operands' 16 bits: half a step of each weight, of the size of
// the output's own rounding.  Measured: 16 heads over 2, 16384 tokens 1007 us (1.09 PFLOP/s); 28 over 4,
// twelve sequences of 371 to 2048 226; fp16 at head_dim 64, six pieces over 7000 keys 98 and 6 of the join;
// 211 tokens 8.9 (KW).  Pairs of times above and in the rules below were measured side by side; cards differ
// by 3 %.
template <int NW, bool BF16, int D, bool CAUSAL, bool SPLIT, bool KW = false>
__global__ __launch_bounds__(64 * NW, 2) void attn_prompt_kernel(const PromptArgs a) {
    constexpr int THR = KW ? 64 : 64 * NW, BM = KW ? 32 : 32 * NW, NB = KW || D == 64 ? 1 : 2;
    constexpr bool STAGED = NW == 8 || !KW && D == 64;     // through registers
    constexpr int NK = D / 16, ND = D / 32, CPR = D / 8, NL = kBN * CPR / THR, RPP = THR / CPR;
    constexpr int ODD = BM / kBN + 3;    // steps in which some query does not see some key, at most
    __shared__ __attribute__((aligned(16))) uint16_t sk[KW ? NW : NB][kBN * D], sv[KW ? NW : NB][kBN * D];
    __shared__ uint32_t odd[ODD][2];     // a bit for each of their keys
    // Blocks go round the 8 dies.  In large calls the heads of one kv head and tile stay on a die, and with
    // them the tiles of a kv head on as few as there are: their keys and values come from its L2 (28 heads
    // over 4, twelve sequences: 82 % of the requests instead of 49).  8 dies hold 8 / n_kv tiles a row, the
    // most work first: every other row goes the other way round.  In small calls the heads go round.
    const int n_kv = a.n_heads / a.group;
    int unit, head;
    if (a.by_die) {
        const int die = blockIdx.x % 8, turn = blockIdx.x / 8, row = turn / a.group;
        unit = row * 8 + die;
        if (row & 1 && 8 % n_kv == 0) unit += 8 - n_kv - 2 * (die / n_kv * n_kv);
        head = unit % n_kv * a.group + turn % a.group;
    } else {
        head = blockIdx.x % a.n_heads;
        unit = blockIdx.x / a.n_heads * n_kv;
    }
    const int kvh = head / a.group;
    PromptTile at;
    if (!prompt_tile<BM>(a, unit / n_kv, at)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ql = lane & 31, hh = lane >> 5;
    const int q_beg = at.q_beg, lq = at.lq, k_beg = at.k_beg, lk = at.lk;
    const int i0 = at.tile * BM, iq = i0 + (KW ? 0 : wave * 32) + ql;   // in the sequence
    const int past = lk - lq;
    const uint16_t *kp = static_cast<const uint16_t *>(a.k.p) + kvh * a.k.head + (int64_t)k_beg * a.k.row;
    const uint16_t *vp = static_cast<const uint16_t *>(a.v.p) + kvh * a.v.head + (int64_t)k_beg * a.v.row;
    u32x4 q[NK];
    {
        const uint16_t *p = static_cast<const uint16_t *>(a.q.p) + head * a.q.head + (int64_t)(q_beg + min(iq, lq - 1)) * a.q.row + 8 * hh;
#pragma unroll
        for (int s = 0; s < NK; ++s) q[s] = *reinterpret_cast<const u32x4 *>(p + 16 * s);
    }
    const int last = min(i0 + BM, lq) - 1;                              // the block's last query
    const int n_keys = keys_seen<CAUSAL>(last, lq, lk);
    const int lim = CAUSAL ? min(iq + past, lk - 1) : lk - 1;            // the lane's last key
    const int lim_w = CAUSAL ? min(i0 + (KW ? 0 : wave * 32) + 31 + past, lk - 1) : lk - 1;   // the most of the wave's
    const int lim_b = CAUSAL ? min(i0 + past, lk - 1) : lk - 1;          // the least of the block's
    const int steps = (n_keys + kBN - 1) / kBN, clean = max(min(n_keys, lim_b + 1), 0) / kBN & -NB;
    const int row_k = (ql & 0x13) | (ql & 4) << 1 | (ql & 8) >> 1;       // key of the lane's row
    int t0 = 0, t1 = steps;
    if constexpr (SPLIT) {
        const int per = steps_per_split(steps, a.splits);
        t0 = min(static_cast<int>(blockIdx.y) * per, steps);
        t1 = min(t0 + per, steps);
        if (t0 == t1 && t0 > 0) {   // nothing to do; the first split is written also where nothing is seen
            if (iq < lq && hh == 0) a.ml[((int64_t)(q_beg + iq) * a.n_heads + head) * a.splits + blockIdx.y] = float2{-INFINITY, 0.f};
            return;
        }
    }
    if (threadIdx.x < 2 * ODD) odd[threadIdx.x >> 1][threadIdx.x & 1] = 0u;

    // a step's keys and values, asked for one step ahead
    u32x4 kr[NL], vr[NL];
    const int tr = (KW ? lane : threadIdx.x) / CPR, tc = (KW ? lane : threadIdx.x) % CPR;
    const int first = !STAGED ? swz<D>(tr, tc) - tr * D : tc * 8;   // in its row
    const uint32_t off_k = static_cast<uint32_t>(tr * a.k.row + first) * 2;
    const uint32_t off_v = static_cast<uint32_t>(tr * a.v.row + first) * 2;
    const auto fetch = [&](int t) {
        const char *kb = reinterpret_cast<const char *>(kp + t * kBN * a.k.row);
        const char *vb = reinterpret_cast<const char *>(vp + t * kBN * a.v.row);
        if ((t + 1) * kBN <= lk) {
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                kr[i] = *reinterpret_cast<const u32x4 *>(kb + i * RPP * a.k.row * 2 + off_k);
                vr[i] = *reinterpret_cast<const u32x4 *>(vb + i * RPP * a.v.row * 2 + off_v);
            }
        } else {   // rows behind the last are the last again: no query sees them
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int64_t r = min(tr + i * RPP, lk - 1 - t * kBN);
                kr[i] = *reinterpret_cast<const u32x4 *>(kb + (r * a.k.row + tc * 8) * 2);
                vr[i] = *reinterpret_cast<const u32x4 *>(vb + (r * a.v.row + tc * 8) * 2);
            }
        }
    };

    f32x16 o[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
    float m = -INFINITY, keep = -INFINITY, l = 0.f;
    const auto put = [&](int t, int b) {
        if (t >= clean) {
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int r = tr + i * RPP;
                bool found = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t w = vr[i][e];
                    found |= drop_nonfinite<BF16>(w);
                    vr[i][e] = w;
                }
                if (found) atomicOr(&odd[t - clean][r >> 5], 1u << (r & 31));
            }
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            *reinterpret_cast<u32x4 *>(sk[b] + swz<D>(tr + i * RPP, tc)) = kr[i];
            *reinterpret_cast<u32x4 *>(sv[b] + swz<D>(tr + i * RPP, tc)) = vr[i];
        }
    };
    // A tile straight into LDS (a load's lanes write 1 KB in a row: a lane has chunk tc of its row, so it asks
    // for the chunk that belongs there).
    const int tile_at = KW ? 0 : wave * (64 / CPR) * D;
    const auto fetch_lds = [&](const uint16_t *base, int64_t stride, uint32_t off, int t, uint16_t *to) {
        if (!KW && (t + 1) * kBN <= lk) {   // (RPP is a multiple of 16: the same chunk in all rows of a thread)
            const char *b = reinterpret_cast<const char *>(base + t * kBN * stride);
#pragma unroll
            for (int i = 0; i < NL; ++i)
                load_lds16(reinterpret_cast<const uint16_t *>(b + i * RPP * stride * 2 + off), to + tile_at + i * RPP * D);
            return;
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) {   // rows behind the last are the last again: no query sees them
            const int r = tr + i * RPP, c = (swz<D>(r, tc) - r * D) >> 3;
            load_lds16(base + min(t * kBN + r, lk - 1) * stride + c * 8, to + tile_at + i * RPP * D);
        }
    };
    // Waits for the thread's own part of a tile and takes what is not finite out of its values.
    const auto take_lds = [&](int t, uint16_t *v) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if (t < clean) return;
        constexpr uint32_t ONE = BF16 ? 0x00800080u : 0x04000400u;   // carries into bit 15 of a half that is not finite
        uint32_t any = 0u;
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(v + swz<D>(tr + i * RPP, tc));
#pragma unroll
            for (int e = 0; e < 4; ++e) any |= (w[e] & 0x7fff7fffu) + ONE;
        }
        if (!__any(any & 0x80008000u)) return;
#pragma unroll 1
        for (int i = 0; i < NL; ++i) {
            const int r = tr + i * RPP;
            u32x4 w = *reinterpret_cast<const u32x4 *>(v + swz<D>(r, tc));
            bool found = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t x = w[e];
                found |= drop_nonfinite<BF16>(x);
                w[e] = x;
            }
            if (found) {
                atomicOr(&odd[t - clean][r >> 5], 1u << (r & 31));
                *reinterpret_cast<u32x4 *>(v + swz<D>(r, tc)) = w;
            }
        }
    };
    // EDGE: some query of the block does not see some key of the step
    const auto compute = [&](int t, auto b_c, auto edge_c) {
        constexpr bool EDGE = decltype(edge_c)::value;
        const uint16_t *k = sk[KW ? wave : decltype(b_c)::value], *v = sv[KW ? wave : decltype(b_c)::value];
        if (!KW && EDGE && t * kBN > lim_w) return;   // nothing that the wave's queries see
        f32x16 s[2];
        // the wave that multiplies goes before the one that is in its softmax
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[h][r] = 0.f;
#pragma unroll
        for (int x = 0; x < NK; ++x)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                s[h] = mfma32<BF16>(*reinterpret_cast<const u32x4 *>(k + swz<D>(32 * h + row_k, 2 * x + hh)), q[x], s[h]);
        // operands are read four products ahead
        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
        for (int x = 0; x < 2 * NK - 4; ++x) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
        __builtin_amdgcn_s_setprio(0);
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                if (EDGE && t * kBN + 32 * h + 16 * (r / 8) + 8 * hh + r % 8 > lim) s[h][r] = -INFINITY;
                mx = fmaxf(mx, s[h][r]);
            }
        // The running maximum is kept while no score passes it by more than 2^8 in weight: the sums
        // stay far from fp32's range, and the accumulators are rescaled a few times in a row only.
        mx = half_max(mx);
        if (__any(mx > keep)) {
            const float mn = fmaxf(m, mx);
            const float al = m == mn ? 1.f : __builtin_amdgcn_exp2f((m - mn) * a.scale2);   // both may be -inf
            m = mn;
            keep = BF16 || fabsf(m * a.scale2) < 0x1p20f ? m + 8.f / a.scale2 : m;
            l *= al;
#pragma unroll
            for (int i = 0; i < ND; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[i][r] *= al;
        }
        // fp16 ends at 2^-24: weights below it would count in their sum but not in the product (5000 keys of
        // 2^-26 beside one of 1: 7.5e-5 of the output).  They, and with them sums and products, are taken 2^7
        // times as large: with the 2^8 above at most 2^15, inside 65504.  (Past scores of 2^20, where fp32 no
        // longer holds the exponents to 2^-4, no maximum is kept.)
        const float base = m == -INFINITY ? 0.f : BF16 ? m * a.scale2 : fmaf(m, a.scale2, -7.f);   // nothing seen yet: p = 0
        u32x4 p[4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 16; r += 2) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[h][r], a.scale2, -base));
                const float y = __builtin_amdgcn_exp2f(fmaf(s[h][r + 1], a.scale2, -base));
                l += x + y;
                p[2 * h + r / 8][r % 8 / 2] = pack16<BF16>(x, y);
            }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int i = 0; i < ND; ++i) o[i] = mfma32<BF16>(v_operand<D>(v, x, i, lane), p[x], o[i]);
        __builtin_amdgcn_sched_group_barrier(0x100, 6, 1);
        __builtin_amdgcn_sched_group_barrier(0x002, 36, 1);
#pragma unroll
        for (int x = 0; x < 4 * ND; ++x) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
            __builtin_amdgcn_sched_group_barrier(0x002, 7, 1);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
        }
    };
    const auto step = [&](int t, auto b_c, auto edge_c) {
        constexpr int other = decltype(b_c)::value ^ 1;
        const bool more = t + 1 < t1;
        if constexpr (NB == 1) {
            lds_barrier();
            put(t, 0);
            lds_barrier();
        }
        if constexpr (STAGED) {
            if (more) fetch(t + 1);
        } else if (more) {
            fetch_lds(kp, a.k.row, off_k, t + 1, sk[other]);
            fetch_lds(vp, a.v.row, off_v, t + 1, sv[other]);
        }
        compute(t, b_c, edge_c);
        if constexpr (NB == 2) {
            if (more) {
                if constexpr (STAGED) put(t + 1, other);
                else take_lds(t + 1, sv[other]);
            }
            lds_barrier();
        }
    };
    if (t0 < t1 && !KW) {
        if constexpr (STAGED) {
            fetch(t0);
        } else {
            fetch_lds(kp, a.k.row, off_k, t0, sk[0]);
            fetch_lds(vp, a.v.row, off_v, t0, sv[0]);
        }
        if constexpr (NB == 2) {
            lds_barrier();   // odd[] is cleared
            if constexpr (STAGED) put(t0, 0);
            else take_lds(t0, sv[0]);
            lds_barrier();
        }
    }
    using B0 = std::integral_constant<int, 0>;
    using B1 = std::integral_constant<int, NB - 1>;
    if constexpr (KW) {
        lds_barrier();   // odd[] is cleared
        for (int t = t0 + wave; t < t1; t += NW) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the last step's reads are done
            fetch_lds(kp, a.k.row, off_k, t, sk[wave]);
            fetch_lds(vp, a.v.row, off_v, t, sv[wave]);
            take_lds(t, sv[wave]);
            compute(t, B0{}, std::true_type{});
        }
    } else {
        int t = t0;
        for (; t < (SPLIT ? min(clean, t1) : clean); t += NB) {   // (with the min 3 % slower where it is not needed)
            step(t, B0{}, std::false_type{});
            if constexpr (NB == 2) step(t + 1, B1{}, std::false_type{});
        }
        for (; t < t1; t += NB) {
            step(t, B0{}, std::true_type{});
            if (NB == 2 && t + 1 < t1) step(t + 1, B1{}, std::true_type{});
        }
    }

    __syncthreads();
    for (int t = max(clean, t0); t < t1; ++t) {
        if (KW && (t - t0) % NW != wave) continue;
        uint64_t bits = odd[t - clean][0] | static_cast<uint64_t>(odd[t - clean][1]) << 32;
        if (lk - t * kBN < kBN) bits &= (1ull << (lk - t * kBN)) - 1;   // rows behind the last were staged as the last
        for (; bits; bits &= bits - 1) {
            const int j = t * kBN + __builtin_ctzll(bits);
            add_odd<BF16, ND>(vp + (int64_t)j * a.v.row + 4 * hh, j <= lim, o);
        }
    }
    l = half_sum(l);
    if constexpr (KW) {   // the waves' sums joined: a wave's in the place of its keys, chunks turned by the row
        __shared__ float2 wml[NW][32];
        float *so = reinterpret_cast<float *>(sk[wave]) + ql * D;
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<f32x4 *>(so + 4 * ((8 * i + r / 2 + hh) ^ (ql & 15))) = f32x4{o[i][r], o[i][r + 1], o[i][r + 2], o[i][r + 3]};
        if (hh == 0) wml[wave][ql] = float2{m * a.scale2, l};
        __syncthreads();
        const int j = threadIdx.x / 8, row = i0 + j;
        if (row >= lq) return;
        const bool sees = (CAUSAL ? min(row + past, lk - 1) : lk - 1) >= 0;
        float mm = -INFINITY, ll = 0.f, f[NW], y[NW];
#pragma unroll
        for (int w = 0; w < NW; ++w) mm = fmaxf(mm, wml[w][j].x);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            y[w] = wml[w][j].y;
            f[w] = y[w] == 0.f ? 0.f : __builtin_amdgcn_exp2f(wml[w][j].x - mm);
            ll = fmaf(f[w], y[w], ll);
        }
        const float inv = inv_sum(ll, sees);
        const int64_t to = ((int64_t)(q_beg + row) * a.n_heads + head) * a.splits + blockIdx.y;
#pragma unroll
        for (int e = 0; e < D / 32; ++e) {
            const int c = threadIdx.x % 8 + 8 * e;
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const f32x4 p = *reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(sk[w]) + j * D + 4 * (c ^ (j & 15)));
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = fmaf(f[w], y[w] == 0.f ? 0.f : p[r], x[r]);
            }
            if constexpr (SPLIT)
                *reinterpret_cast<f32x4 *>(a.part + to * D + 4 * c) = x;
            else
                *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(a.out) + head * a.out_head + (int64_t)(q_beg + row) * a.out_row + 4 * c) =
                    u32x2{pack16<BF16>(x[0] * inv, x[1] * inv), pack16<BF16>(x[2] * inv, x[3] * inv)};
        }
        if (SPLIT && threadIdx.x % 8 == 0) a.ml[to] = float2{mm, ll == 0.f && sees ? -0.f : ll};
        return;
    }
    if (iq >= lq) return;
    if constexpr (SPLIT) {
        const int64_t at = ((int64_t)(q_beg + iq) * a.n_heads + head) * a.splits + blockIdx.y;
        float *to = a.part + at * D + 4 * hh;
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int r = 0; r < 16; r += 4)
                *reinterpret_cast<f32x4 *>(to + 32 * i + 2 * r) = f32x4{o[i][r], o[i][r + 1], o[i][r + 2], o[i][r + 3]};
        if (hh == 0) a.ml[at] = float2{m * a.scale2, l == 0.f && lim >= 0 ? -0.f : l};   // -0: every score -inf
    } else {
        store_rows<BF16, ND>(o, inv_sum(l, lim >= 0), static_cast<uint16_t *>(a.out) + head * a.out_head + (int64_t)(q_beg + iq) * a.out_row + 4 * hh);
    }
}

// The splits (at most NS) of every query of a head joined, D / 4 lanes each.  No search for its
// sequence: a split that has no keys is marked by its sum 0, and rows between the first offset and the
// last belong to some sequence.  All loads are asked for at once, for splits past the last those of the
// last again (behind branches each waits for the one before: 8 queries in 15 splits 12 us, 3.9 so).
template <bool BF16, int D, int NS>
__global__ __launch_bounds__(256) void attn_join_kernel(const PromptArgs a) {
    constexpr int G = D / 4;
    const int lane = threadIdx.x % G, n = a.splits;
    const int rows = a.rows_q * a.n_heads, row = min(static_cast<int>(blockIdx.x * (256 / G) + threadIdx.x / G), rows - 1);
    const int64_t at = (int64_t)row * n;
    float2 e = a.ml[at + min(lane, n - 1)];
    f32x4 p[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) p[s] = *reinterpret_cast<const f32x4 *>(a.part + (at + min(s, n - 1)) * D + 4 * lane);
    if (lane >= n) e = float2{-INFINITY, 0.f};
    float mm = e.x;
#pragma unroll
    for (int s = NS / 2; s >= 1; s >>= 1) mm = fmaxf(mm, __shfl_xor(mm, s, NS));
    mm = __shfl(mm, 0, G);
    // a split of which the query sees nothing has sum 0 (and NaN where all that it sees is NaN)
    const float f = e.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(e.x - mm);
    float ll = f * e.y;
    int sees = e.y != 0.f || __float_as_int(e.y) < 0;
#pragma unroll
    for (int s = NS / 2; s >= 1; s >>= 1) {
        ll += __shfl_xor(ll, s, NS);
        sees |= __shfl_xor(sees, s, NS);
    }
    const float inv = inv_sum(__shfl(ll, 0, G), __shfl(sees, 0, G));
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        const float fs = __shfl(f, s, G);
        const bool has = __shfl(e.y, s, G) != 0.f;   // what is not written is not used
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = fmaf(fs, has ? p[s][r] : 0.f, x[r]);
    }
    const int i = row / a.n_heads, head = row % a.n_heads;
    if (i < seq_off(a.cu_q, 0, a.rows_q) || i >= seq_off(a.cu_q, a.n_seqs, a.rows_q)) return;
    *reinterpret_cast<u32x2 *>(static_cast<uint16_t *>(a.out) + head * a.out_head + (int64_t)i * a.out_row + 4 * lane) =
        u32x2{pack16<BF16>(x[0] * inv, x[1] * inv), pack16<BF16>(x[2] * inv, x[3] * inv)};
}

}  // namespace hxq

using namespace hxq;

namespace {

struct PromptPlan {
    int nw, bm, splits;
    int64_t part_bytes, bytes;   // workspace: part, then ml
};

// What depends on sizes that the host knows; lengths of sequences are on the device.
PromptPlan prompt_plan(int64_t rows_q, int64_t rows_k, int64_t n_seqs, int64_t n_heads, int32_t D) {
    PromptPlan p{4, 128, 1, 0, 0};
    const int64_t cus = device_cu_count(), held = (D == 64 ? 3 : 2) * cus;
    const int64_t seqs = std::min(rows_q, n_seqs);
    const int64_t keys = rows_k / seqs - rows_q / seqs / 2;   // that a query sees
    // 8 waves where queries see many keys and there are two blocks a compute unit, 4 for the others (16 heads
    // over 2, us with 4 and 8 waves: one of 16384 tokens 1063 and 1023, of 8192 292 and 272, of 4096 106 and 120,
    // eight of 2048 164 and 174, four of 2048 behind 4000 336 and 329): two blocks of 4 a unit hide each other's
    // start, 8 waves stage half the bytes.
    if (D == 128 && keys >= 4096 && rows_q / 256 * n_heads >= 2 * cus) p.nw = 8;
    if (p.nw == 8) {
        p.bm = 256;
        return p;
    }
    // Small calls: a block takes 32 queries and its four waves different keys, so that its chain of steps is a
    // quarter as long, and the keys are split while compute units idle.  It stages four times the bytes a query,
    // so not past some keys a split; above one block a unit (head_dim 64: two and a half) it pays from some keys
    // on.  us with 128 and 32 queries a block: 16 heads, a prompt of 211 13.2 and 8.2, of 512 20.7 and 10.8, of
    // 1024 30.2 and 22.9, 8 queries over 2000 keys 14.8 and 10.7, 64 of a prompt 6.8 and 7.8; 28 heads, 600 24.0
    // and 26.5, four of 100 10.1 and 15.2; at head_dim 64 512 12.3 and 7.4, two of 200 over 1200 16.2 and 11.4.
    const int64_t small = std::max(seqs, (rows_q + 16 * seqs + 15) / 32) * n_heads;
    if (rows_k / seqs > 96 && (small <= cus || (D == 64 ? 2 * small <= 5 * cus : small <= 2 * cus && keys >= 300))) {
        const int64_t each = D == 64 ? 512 : 256;
        const int64_t splits = std::max<int64_t>(1, std::min({cus / small, (keys + each - 1) / each, int64_t{kMaxSplits}}));
        if (keys <= splits * (D == 64 ? 1600 : 1100)) {
            p.bm = 32;
            p.splits = static_cast<int>(splits);
        }
    }
    // Few blocks of the others: the keys of each are split, to as many blocks as run at once (two a compute unit, at
    // head_dim 64 three), while a split keeps 192 keys (at head_dim 64 256, and 640 past one block a unit:
    // its steps are half the work).  16 heads, us with one block and split: 8 queries over 8000 keys 216
    // and 24, 512 over 8500 230 and 60, 2048 over 2048 61 and 51, 1000 over 1000 34 and 30; at head_dim 64
    // 2048 over 10000 137 and 115, 200 over 1200 22 and 18.
    const int64_t blocks = std::max(seqs, (rows_q + 64 * seqs) / 128) * n_heads;
    int64_t splits = std::max(std::min(cus / blocks, keys / 256), std::min(held / blocks, keys / (D == 64 ? 640 : 192)));
    // (one sequence: its blocks are alike, three splits take two rounds for three: 2304 over 3304 98 and 83)
    if (D == 128 && n_seqs == 1 && blocks > cus && blocks <= 2 * held / 3 && keys >= 3 * 512) splits = 3;
    if (p.bm == 128) p.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(splits, kMaxSplits)));
    if (p.splits > 1) {
        p.part_bytes = rows_q * n_heads * p.splits * D * 4;
        p.bytes = p.part_bytes + rows_q * n_heads * p.splits * 8;
    }
    return p;
}

}  // namespace

extern "C" int64_t hxq_attn_prompt_workspace_bytes(int64_t rows_q, int64_t rows_k, int32_t n_seqs, int32_t n_heads,
                                                   int32_t head_dim) {
    if (rows_q < 0 || rows_k < 0 || n_seqs < 0 || n_heads <= 0 || (head_dim != 64 && head_dim != 128)) return -1;
    return rows_q && n_seqs ? prompt_plan(rows_q, rows_k, n_seqs, n_heads, head_dim).bytes : 0;
}

extern "C" int hxq_attn_prompt(const void *q, int64_t q_row_stride, int64_t q_head_stride, const void *k,
                               int64_t k_row_stride, int64_t k_head_stride, const void *v, int64_t v_row_stride,
                               int64_t v_head_stride, int32_t dtype, const int32_t *cu_q, const int32_t *cu_k,
                               int32_t n_seqs, int64_t rows_q, int64_t rows_k, int32_t n_heads, int32_t n_kv_heads,
                               int32_t head_dim, float scale, int32_t causal, void *out, int64_t out_row_stride,
                               int64_t out_head_stride, void *workspace, int64_t workspace_bytes, hipStream_t stream) {
    clear_error();
    HXQ_REQUIRE(attn_dtype(dtype, false), "q, k and v must be bf16 or fp16");
    HXQ_REQUIRE(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128");
    HXQ_REQUIRE(n_heads > 0 && n_kv_heads > 0 && n_heads % n_kv_heads == 0, "n_heads must be a multiple of n_kv_heads");
    HXQ_REQUIRE(n_seqs >= 0 && rows_q >= 0 && rows_k >= 0 && rows_q < (int64_t{1} << 31) - 1024 &&
                    rows_k < (int64_t{1} << 31) - 1024, "bad sizes");
    HXQ_REQUIRE(scale >= 0x1p-100f && scale <= 0x1p100f, "scale must lie in 2^-100 .. 2^100");
    if (n_seqs == 0 || rows_q == 0) return HXQ_OK;
    HXQ_REQUIRE(q && out && cu_q && (rows_k == 0 || (k && v)), "q, k, v, cu_q and out are required");
    const HeadRows qr{q, q_row_stride, q_head_stride}, kr{k, k_row_stride, k_head_stride}, vr{v, v_row_stride, v_head_stride},
        orow{out, out_row_stride, out_head_stride};
    HXQ_REQUIRE(k_row_stride < (1 << 24) && v_row_stride < (1 << 24) && k_row_stride >= 0 && v_row_stride >= 0,
                "row strides of k and v must be at least 0 and less than 2^24 elements");
    HXQ_REQUIRE(rows_aligned(qr, dtype) && rows_aligned(kr, dtype) && rows_aligned(vr, dtype) && rows_aligned(orow, dtype),
                "q, k, v and out need pointers and strides that are multiples of 16 bytes");
    const PromptPlan plan = prompt_plan(rows_q, rows_k, n_seqs, n_heads, head_dim);
    HXQ_REQUIRE(plan.bytes == 0 || (workspace && workspace_bytes >= plan.bytes && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                "workspace too small or not 16-byte aligned");
    const int64_t tiles = rows_q / plan.bm + n_seqs;
    // eight tiles of a kv head a die: below that some dies would go short (8 queries, 8192 keys, 16 heads: 50
    // us by die, 23 round)
    const bool by_die = tiles * n_kv_heads >= 64;
    const int64_t blocks = by_die ? (tiles * n_kv_heads + 7) / 8 * 8 * (n_heads / n_kv_heads) : tiles * n_heads;
    const int64_t joins = plan.splits > 1 ? (rows_q * n_heads * (head_dim / 4) + 255) / 256 : 0;
    HXQ_REQUIRE(blocks * 64 * plan.nw < kMaxThreads && joins * 256 < kMaxThreads, "too many rows, sequences or heads");
    const PromptArgs a{qr, kr, vr, out, out_row_stride, out_head_stride, cu_q, cu_k ? cu_k : cu_q, n_seqs,
                       static_cast<int32_t>(rows_q), static_cast<int32_t>(rows_k), n_heads, n_heads / n_kv_heads,
                       scale * 1.44269504088896340736f, plan.splits, by_die, static_cast<float *>(workspace),
                       reinterpret_cast<float2 *>(static_cast<char *>(workspace) + plan.part_bytes)};
    const dim3 grid(static_cast<uint32_t>(blocks), plan.splits), join(static_cast<uint32_t>(joins));
    const auto go = [&](auto bf, auto dd) {
        constexpr bool B = decltype(bf)::value;
        constexpr int D = decltype(dd)::value;
        const auto by_c = [&](auto cc) {
            constexpr bool C = decltype(cc)::value;
            if (plan.splits > 1) {
                if (plan.bm == 32) hipLaunchKernelGGL((attn_prompt_kernel<4, B, D, C, true, true>), grid, dim3(256), 0, stream, a);
                else hipLaunchKernelGGL((attn_prompt_kernel<4, B, D, C, true>), grid, dim3(256), 0, stream, a);
                const auto joined = [&](auto ns) {
                    hipLaunchKernelGGL((attn_join_kernel<B, D, decltype(ns)::value>), join, dim3(256), 0, stream, a);
                };
                if (plan.splits <= 2) joined(std::integral_constant<int, 2>{});
                else if (plan.splits <= 4) joined(std::integral_constant<int, 4>{});
                else if (plan.splits <= 8) joined(std::integral_constant<int, 8>{});
                else joined(std::integral_constant<int, kMaxSplits>{});
                return;
            }
            if (plan.bm == 32) {
                hipLaunchKernelGGL((attn_prompt_kernel<4, B, D, C, false, true>), grid, dim3(256), 0, stream, a);
                return;
            }
            if constexpr (D == 128)
                if (plan.nw == 8) {
                    hipLaunchKernelGGL((attn_prompt_kernel<8, B, D, C, false>), grid, dim3(512), 0, stream, a);
                    return;
                }
            hipLaunchKernelGGL((attn_prompt_kernel<4, B, D, C, false>), grid, dim3(256), 0, stream, a);
        };
        if (causal) by_c(std::true_type{});
        else by_c(std::false_type{});
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
