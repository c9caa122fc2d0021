// The router's kernels (gfx950): the choice of experts, its gradient, the
// balance loss and its gradient.  Logits are [tokens, experts], experts <= 1024.
//
// Every kernel reads a token's logits once, 16 lanes a token (four tokens a
// wavefront), and reduces over the 16 lanes by row rotations, which cost an
// instruction each; a lane holds VPT logits in registers, four consecutive ones at
// every 64th, so that 16 lanes read 64 in one piece.  All arithmetic is f32.

#include <type_traits>

#include "iqk_host.h"
#include "iqk_mx.h"

namespace iqk {

constexpr int64_t kRouterMaxExperts = 1024;
constexpr int64_t kRouterMaxK = 64;
constexpr int kRowLanes = 16;

// ------------------------------------------------------------ 16-lane rows ---

// x of the lane N places on in the same 16 lanes (a rotation).
template <int N>
__device__ __forceinline__ uint32_t rotate(uint32_t x) {
    return uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x120 + N, 0xf, 0xf, false));
}
template <int N>
__device__ __forceinline__ float rotate(float x) {
    return __builtin_bit_cast(float, rotate<N>(__builtin_bit_cast(uint32_t, x)));
}

template <typename T, typename F>
__device__ __forceinline__ T row_reduce(T v, F f) {
    v = f(v, rotate<8>(v));
    v = f(v, rotate<4>(v));
    v = f(v, rotate<2>(v));
    return f(v, rotate<1>(v));
}
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    return row_reduce(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}
__device__ __forceinline__ uint32_t row_min(uint32_t v) {
    return row_reduce(v, [](uint32_t a, uint32_t b) { return min(a, b); });
}
__device__ __forceinline__ float row_max(float v) {
    return row_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float row_sum(float v) {
    return row_reduce(v, [](float a, float b) { return a + b; });
}

// exp(x) for x <= 0 or NaN: 2^(x log2 e) with the product's rounding error put back.
__device__ __forceinline__ float exp_neg(float x) {
    x = x < -200.f ? -200.f : x;  // 0 in f32; keeps NaN
    constexpr float kHi = 0x1.715476p+0f, kLo = 0x1.4ae0c0p-26f;  // log2 e
    const float t = x * kHi;
    const float lo = fmaf(x, kLo, fmaf(x, kHi, -t));
    return __builtin_amdgcn_exp2f(t) * fmaf(lo, 0x1.62e430p-1f, 1.0f);
}

template <int DT>
__device__ __forceinline__ void put_at(void *p, size_t i, float v) {
    if constexpr (DT == MX_F32)
        static_cast<float *>(p)[i] = v;
    else
        static_cast<uint16_t *>(p)[i] = uint16_t(DT == MX_F16 ? float_to_half_bits(v) : bf16_bits(v));
}

// The expert at place i of lane j.  QUADS: experts are a multiple of four and
// rows aligned to four of them; else a lane holds every 16th.
template <bool QUADS>
__device__ __forceinline__ constexpr uint32_t expert_of(uint32_t i, uint32_t j) {
    return QUADS ? (i / 4 * kRowLanes + j) * 4 + i % 4 : i * kRowLanes + j;
}

// The lane's VPT logits of a row as they stand (16-bit ones two a word).
template <int DT, int VPT>
using RowWords = uint32_t[DT == MX_F32 ? VPT : VPT / 2];

template <int DT, int VPT, bool QUADS>
__device__ __forceinline__ void load_words(const void *x, size_t row, uint32_t E, uint32_t j,
                                           RowWords<DT, VPT> &v) {
    const size_t base = row * E;
    if constexpr (QUADS) {
#pragma unroll
        for (int q = 0; q < VPT / 4; ++q) {
            const uint32_t e = expert_of<true>(4 * q, j);
            const size_t at = base + (e < E ? e : 0u);  // past the end: any, masked at use
            if constexpr (DT == MX_F32) {
                const uint4_t w = load_u4(static_cast<const float *>(x) + at);
                v[4 * q] = w.x, v[4 * q + 1] = w.y, v[4 * q + 2] = w.z, v[4 * q + 3] = w.w;
            } else {
                const uint2_t w = *reinterpret_cast<const uint2_t *>(static_cast<const uint16_t *>(x) + at);
                v[2 * q] = w.x, v[2 * q + 1] = w.y;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const uint32_t e = expert_of<false>(i, j);
            const size_t at = base + (e < E ? e : 0u);
            if constexpr (DT == MX_F32) {
                v[i] = static_cast<const uint32_t *>(x)[at];
            } else {
                const uint32_t h = static_cast<const uint16_t *>(x)[at];
                v[i / 2] = i & 1 ? v[i / 2] | h << 16 : h;
            }
        }
    }
}

// A 16-bit logit's bits.
template <int VPT>
__device__ __forceinline__ uint32_t half_of(const uint32_t (&v)[VPT], int i) {
    return i & 1 ? v[i / 2] >> 16 : v[i / 2] & 0xffffu;
}

template <int DT>
__device__ __forceinline__ float float_of(uint32_t bits) {
    return DT == MX_F32 ? __builtin_bit_cast(float, bits)
           : DT == MX_F16 ? half_bits_to_float(bits) : __builtin_bit_cast(float, bits << 16);
}

// As floats, -inf past E.
template <int DT, int VPT, bool QUADS>
__device__ __forceinline__ void to_floats(const RowWords<DT, VPT> &w, uint32_t E, uint32_t j, float (&v)[VPT]) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        uint32_t bits;
        if constexpr (DT == MX_F32)
            bits = w[i];
        else
            bits = half_of(w, i);
        v[i] = expert_of<QUADS>(i, j) < E ? float_of<DT>(bits) : -__builtin_inff();
    }
}

template <int DT, int VPT, bool QUADS>
__device__ __forceinline__ void store_row(void *y, size_t row, uint32_t E, uint32_t j, const float (&v)[VPT]) {
    const size_t base = row * E;
    if constexpr (QUADS) {
#pragma unroll
        for (int q = 0; q < VPT; q += 4) {
            const uint32_t e = expert_of<true>(q, j);
            if (e >= E) continue;
            if constexpr (DT == MX_F32) {
                *reinterpret_cast<float4_t *>(static_cast<float *>(y) + base + e) =
                    float4_t{v[q], v[q + 1], v[q + 2], v[q + 3]};
            } else {
                uint32_t h[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = DT == MX_F16 ? float_to_half_bits(v[q + i]) : bf16_bits(v[q + i]);
                *reinterpret_cast<uint2_t *>(static_cast<uint16_t *>(y) + base + e) =
                    uint2_t{h[0] | h[1] << 16, h[2] | h[3] << 16};
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (expert_of<false>(i, j) < E) put_at<DT>(y, base + expert_of<false>(i, j), v[i]);
    }
}

// Order of floats as unsigned: NaN highest, then +inf .. -inf; 0 is below all.
__device__ __forceinline__ uint32_t order_key(float f) {
    if (f != f) return 0xffffffffu;
    const uint32_t u = __builtin_bit_cast(uint32_t, f + 0.0f);  // -0 counts as +0
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __builtin_bit_cast(float, k >> 31 ? k == 0xffffffffu ? 0x7fc00000u : k & 0x7fffffffu : ~k);
}

// The same of a 16-bit float's bits, in the high half; the low half orders
// experts, the lowest highest, so that no two keys are equal.
template <int DT>
__device__ __forceinline__ uint32_t order_key16(uint32_t h, uint32_t e) {
    constexpr uint32_t kInf = DT == MX_F16 ? 0x7c00u : 0x7f80u;
    const uint32_t m = h & 0x7fffu;
    const uint32_t k = m > kInf ? 0xffffu : (h >> 15) ? 0x8000u - m : 0x8000u + m;  // -0 is +0
    return k << 16 | (0xffffu - e);
}
template <int DT>
__device__ __forceinline__ float key16_value(uint32_t key) {
    const uint32_t k = key >> 16;
    return float_of<DT>(k == 0xffffu ? 0x7fffu : k >= 0x8000u ? k - 0x8000u : (0x8000u - k) | 0x8000u);
}

// v -> softmax over the row's 16 lanes, in place (none of it where every
// logit is -inf: zeros).  A NaN makes the sum, and so the row, NaN, also where all
// else is -inf (places past E are) and the maximum, which skips NaN, is too.
template <int VPT>
__device__ __forceinline__ void row_softmax(float (&v)[VPT]) {
    float top = v[0];
#pragma unroll
    for (int i = 1; i < VPT; ++i) top = fmaxf(top, v[i]);
    top = row_max(top);
    if (top == -__builtin_inff()) top = 0.f;  // no logit but -inf, whose exponentials are 0, and NaN
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        v[i] = exp_neg(v[i] - top);
        s += v[i];
    }
    s = row_sum(s);
    const float inv = s == 0.f ? 0.f : 1.0f / s;
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] *= inv;
}

// -------------------------------------------------------------------- top k ---

struct TopkArgs {
    const void *logits;
    float *weights;
    int32_t *ids;
    const float *dweights;
    void *dlogits;
    uint32_t rows, E, k;
};

// The k highest logits, ties to the lowest expert, and their softmax weights:
// over the chosen (NORM) or over all.  k rounds of a maximum over the row, bound
// by their instructions.  16-bit logits and their expert make one key, and of
// the keys below the last choice the highest has the highest unsigned key -
// choice (those at or above it wrap to less), so that a round needs a
// subtraction and half a maximum a logit.  f32 logits need five instructions: the
// lowest of the experts that hold the maximum is a second reduction.  65536 tokens,
// bf16 and f32: top 4 of 60 6.4 and 7.6 us, 6 of 256 15.4 and 21.3 (2.4 and 3.3 TB/s), 12 of
// 256 19.9 and 34.9, 8 of 512 26.2 and 44.0; over all experts 4 to 9 more, for their
// exponentials.  One token in f32: 3.8, a launch.
template <int DT, int VPT, bool NORM, bool QUADS>
__global__ __launch_bounds__(256) void topk_kernel(TopkArgs a) {
    constexpr bool WIDE = DT == MX_F32;
    const uint32_t lane = threadIdx.x & 63u, j = lane & 15u;
    const uint32_t row = blockIdx.x * 16 + threadIdx.x / kRowLanes;
    const bool live = row < a.rows;
    RowWords<DT, VPT> words;
    load_words<DT, VPT, QUADS>(a.logits, live ? row : 0u, a.E, j, words);
    uint32_t key[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const uint32_t e = expert_of<QUADS>(i, j);
        if constexpr (WIDE)
            key[i] = e < a.E ? order_key(float_of<DT>(words[i])) : 0u;
        else
            key[i] = e < a.E ? order_key16<DT>(half_of(words, i), e) : 0u;
    }
    // lane j: choices j, 16 + j, ..
    uint32_t chosen[4], id[4];
    uint32_t best = 0, first = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        chosen[q] = id[q] = 0;
        if (16u * q >= a.k) break;  // uniform
        const uint32_t n = min(a.k - 16u * q, 16u);
        for (uint32_t c = 0; c < n; ++c) {
            uint32_t e = 0;
            if constexpr (WIDE) {
                uint32_t m = key[0];
#pragma unroll
                for (int i = 1; i < VPT; ++i) m = max(m, key[i]);
                best = row_max(m);
                uint32_t at = 0xffffu;
#pragma unroll
                for (int i = VPT - 1; i >= 0; --i) at = key[i] == best ? uint32_t(expert_of<QUADS>(i, j)) : at;
                e = row_min(at);
#pragma unroll
                for (int i = 0; i < VPT; ++i) key[i] = expert_of<QUADS>(i, j) == e ? 0u : key[i];
            } else {
                uint32_t m = key[0] - best;
#pragma unroll
                for (int i = 1; i < VPT; ++i) m = max(m, key[i] - best);
                best += row_max(m);
            }
            if (q == 0 && c == 0) first = best;
            if (j == c) {
                chosen[q] = best;
                id[q] = WIDE ? e : 0xffffu - (best & 0xffffu);
            }
        }
    }
    const auto value = [](uint32_t k) { return WIDE ? key_value(k) : key16_value<DT>(k); };
    const float top = value(first);
    float ex[4], sum = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        ex[q] = 16u * q + j < a.k ? exp_neg(value(chosen[q]) - top) : 0.f;
        if constexpr (NORM) sum += ex[q];
    }
    if constexpr (!NORM) {
        float v[VPT];
        to_floats<DT, VPT, QUADS>(words, a.E, j, v);
#pragma unroll
        for (int i = 0; i < VPT; ++i) sum += exp_neg(v[i] - top);
    }
    sum = row_sum(sum);
    const bool empty = top == -__builtin_inff();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint32_t c = 16u * q + j;
        if (!live || c >= a.k) continue;
        const size_t at = size_t(row) * a.k + c;
        a.weights[at] = empty ? 0.f : ex[q] / sum;
        a.ids[at] = int32_t(id[q]);
    }
}

// d loss / d logits from d loss / d weights.  With D = sum_j w_j dw_j:
//   NORM      w_i (dw_i - D) at the chosen, 0 elsewhere
//   otherwise p_e (dw_e - D), dw_e = 0 where e was not chosen.
// The chosen's values meet their place in the row through LDS.  Bound by the store of
// the rows: 65536 tokens of 256, bf16, NORM, 8.5 us (4.3 TB/s); over all experts, which
// reads the logits too, 15.9 (4.5 TB/s).
template <int DT, int VPT, bool NORM, bool QUADS>
__global__ __launch_bounds__(256) void topk_grad_kernel(TopkArgs a) {
    constexpr int PLACES = kRowLanes * VPT;
    __shared__ __attribute__((aligned(16))) float place[16][PLACES];
    const uint32_t lane = threadIdx.x & 63u, j = lane & 15u, r = threadIdx.x / kRowLanes;
    const uint32_t row = blockIdx.x * 16 + r;
    const bool live = row < a.rows;
    float w[4], dw[4];
    int32_t id[4];
    float dot = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint32_t c = 16u * q + j;
        const bool in = live && c < a.k;
        const size_t at = in ? size_t(row) * a.k + c : 0;
        w[q] = in ? a.weights[at] : 0.f;
        dw[q] = in ? a.dweights[at] : 0.f;
        id[q] = in ? a.ids[at] : -1;
        if (in) dot += w[q] * dw[q];
    }
    dot = row_sum(dot);
    // a row's places are written and read by the 16 lanes of one wavefront
    // only, whose LDS operations stay in order
#pragma unroll
    for (int q = 0; q < VPT / 4; ++q)
        *reinterpret_cast<float4_t *>(&place[r][(q * kRowLanes + j) * 4]) = float4_t{0, 0, 0, 0};
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (uint32_t(id[q]) < a.E) place[r][id[q]] = NORM ? w[q] * (dw[q] - dot) : dw[q];
    __builtin_amdgcn_wave_barrier();
    float d[VPT];
    if constexpr (QUADS) {
#pragma unroll
        for (int q = 0; q < VPT / 4; ++q) {
            const float4_t v = *reinterpret_cast<const float4_t *>(&place[r][(q * kRowLanes + j) * 4]);
#pragma unroll
            for (int i = 0; i < 4; ++i) d[4 * q + i] = v[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i) d[i] = place[r][expert_of<false>(i, j)];
    }
    if constexpr (!NORM) {
        RowWords<DT, VPT> words;
        load_words<DT, VPT, QUADS>(a.logits, live ? row : 0u, a.E, j, words);
        float p[VPT];
        to_floats<DT, VPT, QUADS>(words, a.E, j, p);
        row_softmax<VPT>(p);
#pragma unroll
        for (int i = 0; i < VPT; ++i) d[i] = p[i] * (d[i] - dot);
    }
    if (live) store_row<DT, VPT, QUADS>(a.dlogits, row, a.E, j, d);
}

// ------------------------------------------------------------- balance loss ---
//
// Of a group's n kept tokens, with c_e the pairs that name expert e and S_e the
// sum of its probabilities: loss = E / (k n^2) sum_e c_e S_e, and
//   d loss / d l_te = E / (k n^2) p_te (c_e - sum_j c_j p_tj).
// The sums run in two launches whose order never changes: workgroups over
// shares of a group's tokens, then one workgroup a group over the shares.
// 16 groups of 4096 tokens, 256 experts in f32 (67 MB): sums 18.2 us (3.7 TB/s),
// join 3.9, gradient 28.6 (4.7 TB/s read and written); one group of 500 tokens, 60
// experts: 3.6, 3.0 and 3.7, a launch each.  What bounds the sums is not shown: a workgroup
// has four turns between clearing its LDS and adding up through it.  The join is one
// workgroup a group: 65536 tokens of 256 in one group take it 18.3, as long as their sums.
constexpr int kBalanceThreads = 512;
constexpr int kBalanceRows = kBalanceThreads / kRowLanes;

struct BalanceArgs {
    const void *logits;
    const int32_t *ids;
    const uint8_t *mask;
    float *psum;      // [groups][shares][E]
    int32_t *pcount;  // [groups][shares][E]
    int32_t *pkept;   // [groups][shares]
    float *loss;
    int32_t *counts;
    int32_t *kept;
    const float *dloss;
    void *dlogits;
    uint32_t T, E, k, shares, share;  // share: tokens of one
};

// A wavefront loads its next four tokens before it works on the ones it has.
template <int DT, int VPT, bool QUADS>
__global__ __launch_bounds__(kBalanceThreads) void balance_sums_kernel(BalanceArgs a) {
    constexpr int PLACES = kRowLanes * VPT;
    __shared__ float sums[kBalanceThreads / 64][PLACES];
    __shared__ int32_t count[PLACES];
    __shared__ int32_t kept;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, j = lane & 15u, wave = tid >> 6;
    const uint32_t group = blockIdx.y, share = blockIdx.x;
    const uint32_t lo = share * a.share, hi = min(a.T, lo + a.share);
    for (uint32_t e = tid; e < uint32_t(PLACES); e += kBalanceThreads) count[e] = 0;
    if (tid == 0) kept = 0;
    __syncthreads();
    float s[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) s[i] = 0.f;
    const auto row_of = [&](uint32_t t) { return size_t(group) * a.T + (t < hi ? t : lo); };
    RowWords<DT, VPT> words;
    uint32_t t = lo + tid / kRowLanes;
    if (lo < hi) load_words<DT, VPT, QUADS>(a.logits, row_of(t), a.E, j, words);
    uint32_t mine = 0;
    for (uint32_t t0 = lo; t0 < hi; t0 += kBalanceRows, t += kBalanceRows) {
        float p[VPT];
        to_floats<DT, VPT, QUADS>(words, a.E, j, p);
        load_words<DT, VPT, QUADS>(a.logits, row_of(t + kBalanceRows), a.E, j, words);
        const size_t row = row_of(t);
        const bool keep = t < hi && (!a.mask || a.mask[row]);
        if (keep) {
            for (uint32_t c = j; c < a.k; c += kRowLanes) {
                const uint32_t e = uint32_t(a.ids[row * a.k + c]);
                if (e < a.E) atomicAdd(&count[e], 1);
            }
            mine += j == 0;
        }
        row_softmax<VPT>(p);
#pragma unroll
        for (int i = 0; i < VPT; ++i) s[i] += keep ? p[i] : 0.f;
    }
    if (mine) atomicAdd(&kept, int32_t(mine));
    // the four rows of a wavefront, then the wavefronts
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        s[i] += __shfl_xor(s[i], 16, 64);
        s[i] += __shfl_xor(s[i], 32, 64);
        if (lane < 16) sums[wave][expert_of<QUADS>(i, j)] = s[i];
    }
    __syncthreads();
    const size_t at = size_t(group) * a.shares + share;
    for (uint32_t e = tid; e < a.E; e += kBalanceThreads) {
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < kBalanceThreads / 64; ++w) v += sums[w][e];
        a.psum[at * a.E + e] = v;
        a.pcount[at * a.E + e] = count[e];
    }
    if (tid == 0) a.pkept[at] = kept;
}

// One workgroup a group: `slices` threads an expert, each over every slices-th
// share, four loads of both sums in flight.
constexpr int kJoinThreads = 1024;

__global__ __launch_bounds__(kJoinThreads) void balance_join_kernel(BalanceArgs a) {
    __shared__ float vsum[kJoinThreads];
    __shared__ int32_t csum[kJoinThreads];
    __shared__ float part[kJoinThreads / 64];
    __shared__ int32_t npart[kJoinThreads / 64];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, group = blockIdx.x;
    const size_t base = size_t(group) * a.shares;
    int32_t n = 0;
    for (uint32_t s = tid; s < a.shares; s += kJoinThreads) n += a.pkept[base + s];
    const uint32_t wide = (a.E + 63u) & ~63u, slices = kJoinThreads / wide;
    const uint32_t slice = tid / wide, e = tid % wide;
    float v = 0.f;
    int32_t c = 0;
    if (slice < slices && e < a.E) {
        for (uint32_t s0 = slice; s0 < a.shares; s0 += 4 * slices) {
            float lv[4];
            int32_t lc[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t s = s0 + i * slices;
                const size_t at = (base + (s < a.shares ? s : slice)) * a.E + e;
                lv[i] = a.psum[at];
                lc[i] = a.pcount[at];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = s0 + i * slices < a.shares;
                v += in ? lv[i] : 0.f;
                c += in ? lc[i] : 0;
            }
        }
    }
    vsum[tid] = v;
    csum[tid] = c;
    __syncthreads();
    float dot = 0.f;
    if (tid < a.E) {
        for (uint32_t i = 1; i < slices; ++i) {
            v += vsum[i * wide + tid];
            c += csum[i * wide + tid];
        }
        a.counts[size_t(group) * a.E + tid] = c;
        dot = float(c) * v;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        dot += __shfl_xor(dot, off, 64);
        n += __shfl_xor(n, off, 64);
    }
    if (lane == 0) {
        part[tid >> 6] = dot;
        npart[tid >> 6] = n;
    }
    __syncthreads();
    if (tid == 0) {
        v = 0.f;
        n = 0;
        for (int w = 0; w < kJoinThreads / 64; ++w) {
            v += part[w];
            n += npart[w];
        }
        const float fn = float(n);
        a.loss[group] = n ? v / fn * (float(a.E) / (float(a.k) * fn)) : 0.f;
        a.kept[group] = n;
    }
}

// A workgroup walks over every gridDim.x-th 16 tokens of its group, the experts'
// counts in registers.
template <int DT, int VPT, bool QUADS>
__global__ __launch_bounds__(256) void balance_grad_kernel(BalanceArgs a) {
    const uint32_t j = threadIdx.x & 15u, group = blockIdx.y, step = gridDim.x * 16;
    const int32_t n = a.kept[group];
    const float fn = float(n), scale = n > 0 ? a.dloss[group] / fn * (float(a.E) / (float(a.k) * fn)) : 0.f;
    float c[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const uint32_t e = expert_of<QUADS>(i, j);
        c[i] = e < a.E ? float(a.counts[size_t(group) * a.E + (e < a.E ? e : 0u)]) : 0.f;
    }
    const auto row_of = [&](uint32_t t) { return size_t(group) * a.T + (t < a.T ? t : 0u); };
    uint32_t t = blockIdx.x * 16 + threadIdx.x / kRowLanes;
    RowWords<DT, VPT> words;
    load_words<DT, VPT, QUADS>(a.logits, row_of(t), a.E, j, words);
    for (uint32_t t0 = blockIdx.x * 16; t0 < a.T; t0 += step, t += step) {
        float p[VPT];
        to_floats<DT, VPT, QUADS>(words, a.E, j, p);
        load_words<DT, VPT, QUADS>(a.logits, row_of(t + step < t ? a.T : t + step), a.E, j, words);
        row_softmax<VPT>(p);
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i) dot += c[i] * p[i];
        dot = row_sum(dot);
        const bool live = t < a.T;
        const size_t row = row_of(t);
        const bool keep = live && n > 0 && (!a.mask || a.mask[row]);
#pragma unroll
        for (int i = 0; i < VPT; ++i) p[i] = keep ? scale * p[i] * (c[i] - dot) : 0.f;
        if (live) store_row<DT, VPT, QUADS>(a.dlogits, row, a.E, j, p);
    }
}

// launch(a, workgroups) for each part of the rows that one launch holds (2^32 threads are
// too many), a's pointers moved to it; 16 rows, a workgroup's, keep every alignment.
template <typename F>
void by_rows(const TopkArgs &all, int64_t rows, int dtype, F &&launch) {
    constexpr int64_t kPart = int64_t(1) << 27;
    const int64_t size = dtype == MX_F32 ? 4 : 2;
    for (int64_t first = 0; first < rows; first += kPart) {
        TopkArgs a = all;
        const int64_t n = rows - first < kPart ? rows - first : kPart;
        a.rows = uint32_t(n);
        if (a.logits) a.logits = static_cast<const char *>(a.logits) + first * all.E * size;
        if (a.dlogits) a.dlogits = static_cast<char *>(a.dlogits) + first * all.E * size;
        a.weights += first * all.k;
        a.ids += first * all.k;
        if (a.dweights) a.dweights += first * all.k;
        launch(a, uint32_t((n + 15) / 16));
    }
}

// f(dtype, places a lane, quads) as compile-time constants.
template <typename F>
void by_shape(int dtype, int64_t experts, bool quads, F &&f) {
    const auto with = [&](auto dt, auto vpt) {
        if (quads)
            f(dt, vpt, std::true_type{});
        else
            f(dt, vpt, std::false_type{});
    };
    const auto sized = [&](auto dt) {
        if (experts <= 64)
            with(dt, std::integral_constant<int, 4>{});
        else if (experts <= 128)
            with(dt, std::integral_constant<int, 8>{});
        else if (experts <= 256)
            with(dt, std::integral_constant<int, 16>{});
        else if (experts <= 512)
            with(dt, std::integral_constant<int, 32>{});
        else
            with(dt, std::integral_constant<int, 64>{});
    };
    if (dtype == MX_F32)
        sized(std::integral_constant<int, MX_F32>{});
    else if (dtype == MX_F16)
        sized(std::integral_constant<int, MX_F16>{});
    else
        sized(std::integral_constant<int, MX_BF16>{});
}

bool router_shape_ok(int64_t rows, int64_t experts, int64_t k) {
    return experts > 0 && experts <= kRouterMaxExperts && k > 0 && k <= kRouterMaxK && k <= experts && rows >= 0 &&
           rows < (int64_t(1) << 31);
}

bool quads_ok(int dtype, int64_t experts, const void *a, const void *b) {
    const uintptr_t mask = dtype == MX_F32 ? 15u : 7u;
    return experts % 4 == 0 && ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & mask) == 0;
}

int64_t balance_shares(int64_t groups, int64_t tokens) {
    // a share is whole turns of the workgroup's rows; about two workgroups a CU
    const int64_t most = (tokens + kBalanceRows - 1) / kBalanceRows;
    const int64_t want = (512 + groups - 1) / groups;
    return most < want ? (most > 0 ? most : 1) : want;
}

}  // namespace iqk

extern "C" {

int iqk_router_topk(int dtype, const void *logits, int64_t rows, int64_t experts, int64_t k, int normalize,
                    float *weights, int32_t *ids, void *stream) {
    using namespace iqk;
    if (dtype < MX_F32 || dtype > MX_BF16) return IQK_ERR_ARGUMENT;
    if (!router_shape_ok(rows, experts, k)) return IQK_ERR_GEOMETRY;
    if (rows == 0) return IQK_OK;
    if (!logits || !weights || !ids) return IQK_ERR_ARGUMENT;
    TopkArgs a{};
    a.logits = logits;
    a.weights = weights;
    a.ids = ids;
    a.E = uint32_t(experts);
    a.k = uint32_t(k);
    const bool quads = quads_ok(dtype, experts, logits, nullptr);
    by_shape(dtype, experts, quads, [&](auto dt, auto vpt, auto qd) {
        constexpr int DT = decltype(dt)::value, VPT = decltype(vpt)::value;
        constexpr bool Q = decltype(qd)::value;
        by_rows(a, rows, dtype, [&](const TopkArgs &part, uint32_t blocks) {
            if (normalize)
                hipLaunchKernelGGL((topk_kernel<DT, VPT, true, Q>), dim3{blocks}, dim3{256}, 0, as_stream(stream), part);
            else
                hipLaunchKernelGGL((topk_kernel<DT, VPT, false, Q>), dim3{blocks}, dim3{256}, 0, as_stream(stream), part);
        });
    });
    return record_launch(hipGetLastError());
}

int iqk_router_topk_grad(int dtype, const void *logits, const float *weights, const int32_t *ids,
                         const float *dweights, int64_t rows, int64_t experts, int64_t k, int normalize, void *dlogits,
                         void *stream) {
    using namespace iqk;
    if (dtype < MX_F32 || dtype > MX_BF16) return IQK_ERR_ARGUMENT;
    if (!router_shape_ok(rows, experts, k)) return IQK_ERR_GEOMETRY;
    if (rows == 0) return IQK_OK;
    if ((!logits && !normalize) || !weights || !ids || !dweights || !dlogits) return IQK_ERR_ARGUMENT;
    TopkArgs a{};
    a.logits = logits;
    a.weights = const_cast<float *>(weights);
    a.ids = const_cast<int32_t *>(ids);
    a.dweights = dweights;
    a.dlogits = dlogits;
    a.E = uint32_t(experts);
    a.k = uint32_t(k);
    const bool quads = quads_ok(dtype, experts, normalize ? nullptr : logits, dlogits);
    by_shape(dtype, experts, quads, [&](auto dt, auto vpt, auto qd) {
        constexpr int DT = decltype(dt)::value, VPT = decltype(vpt)::value;
        constexpr bool Q = decltype(qd)::value;
        by_rows(a, rows, dtype, [&](const TopkArgs &part, uint32_t blocks) {
            if (normalize)
                hipLaunchKernelGGL((topk_grad_kernel<DT, VPT, true, Q>), dim3{blocks}, dim3{256}, 0, as_stream(stream), part);
            else
                hipLaunchKernelGGL((topk_grad_kernel<DT, VPT, false, Q>), dim3{blocks}, dim3{256}, 0, as_stream(stream), part);
        });
    });
    return record_launch(hipGetLastError());
}

int64_t iqk_balance_work(int64_t groups, int64_t tokens, int64_t experts) {
    using namespace iqk;
    if (groups <= 0 || groups > 65535 || !router_shape_ok(tokens, experts, 1)) return -1;
    return groups * balance_shares(groups, tokens) * (2 * experts + 1);
}

int iqk_balance(int dtype, const void *logits, const int32_t *ids, const uint8_t *mask, int64_t groups,
                int64_t tokens, int64_t experts, int64_t k, uint32_t *work, float *loss, int32_t *counts,
                int32_t *kept, void *stream) {
    using namespace iqk;
    if (dtype < MX_F32 || dtype > MX_BF16) return IQK_ERR_ARGUMENT;
    if (!router_shape_ok(tokens, experts, k) || groups < 0 || groups > 65535) return IQK_ERR_GEOMETRY;
    if (groups == 0) return IQK_OK;
    if ((tokens && (!logits || !ids)) || !work || !loss || !counts || !kept) return IQK_ERR_ARGUMENT;
    BalanceArgs a{};
    const int64_t shares = balance_shares(groups, tokens);
    a.logits = logits;
    a.ids = ids;
    a.mask = mask;
    a.psum = reinterpret_cast<float *>(work);
    a.pcount = reinterpret_cast<int32_t *>(work + groups * shares * experts);
    a.pkept = reinterpret_cast<int32_t *>(work + 2 * groups * shares * experts);
    a.loss = loss;
    a.counts = counts;
    a.kept = kept;
    a.T = uint32_t(tokens);
    a.E = uint32_t(experts);
    a.k = uint32_t(k);
    a.shares = uint32_t(shares);
    const int64_t turns = (tokens + kBalanceRows - 1) / kBalanceRows;
    a.share = uint32_t((turns + shares - 1) / shares * kBalanceRows);
    const bool quads = quads_ok(dtype, experts, logits, nullptr);
    by_shape(dtype, experts, quads, [&](auto dt, auto vpt, auto qd) {
        hipLaunchKernelGGL((balance_sums_kernel<decltype(dt)::value, decltype(vpt)::value, decltype(qd)::value>),
                           dim3(uint32_t(shares), uint32_t(groups)), dim3{kBalanceThreads}, 0, as_stream(stream), a);
    });
    if (const hipError_t err = hipGetLastError(); err != hipSuccess) return record_launch(err);
    hipLaunchKernelGGL(balance_join_kernel, dim3{uint32_t(groups)}, dim3{kJoinThreads}, 0, as_stream(stream), a);
    return record_launch(hipGetLastError());
}

int iqk_balance_grad(int dtype, const void *logits, const uint8_t *mask, const int32_t *counts, const int32_t *kept,
                     const float *dloss, int64_t groups, int64_t tokens, int64_t experts, int64_t k, void *dlogits,
                     void *stream) {
    using namespace iqk;
    if (dtype < MX_F32 || dtype > MX_BF16) return IQK_ERR_ARGUMENT;
    if (!router_shape_ok(tokens, experts, k) || groups < 0 || groups > 65535) return IQK_ERR_GEOMETRY;
    if (groups == 0 || tokens == 0) return IQK_OK;
    if (!logits || !counts || !kept || !dloss || !dlogits) return IQK_ERR_ARGUMENT;
    BalanceArgs a{};
    a.logits = logits;
    a.mask = mask;
    a.counts = const_cast<int32_t *>(counts);
    a.kept = const_cast<int32_t *>(kept);
    a.dloss = dloss;
    a.dlogits = dlogits;
    a.T = uint32_t(tokens);
    a.E = uint32_t(experts);
    a.k = uint32_t(k);
    const bool quads = quads_ok(dtype, experts, logits, dlogits);
    // 16 tokens a turn, about eight workgroups a CU
    const int64_t turns = (tokens + 15) / 16, most = (256 * 8 + groups - 1) / groups;
    by_shape(dtype, experts, quads, [&](auto dt, auto vpt, auto qd) {
        hipLaunchKernelGGL((balance_grad_kernel<decltype(dt)::value, decltype(vpt)::value, decltype(qd)::value>),
                           dim3(uint32_t(turns < most ? turns : most), uint32_t(groups)), dim3{256}, 0,
                           as_stream(stream), a);
    });
    return record_launch(hipGetLastError());
}

}  // extern "C"
