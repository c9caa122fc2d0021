// The router's kernels (gfx950): the choice of experts, its gradient, the
// balance loss and its gradient.  Logits are [tokens, experts], experts <= 1024.
//
// Every kernel reads a token's logits once, 16 lanes a token (four tokens a
// wavefront), a lane VPT consecutive ones in registers, and reduces over the 16
// lanes by row rotations.  All arithmetic is f32.

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

__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    v = max(v, rotate<8>(v));
    v = max(v, rotate<4>(v));
    v = max(v, rotate<2>(v));
    return max(v, rotate<1>(v));
}

// The same value in all 16 lanes: each step adds the two halves of a ring.
__device__ __forceinline__ float row_sum(float v) {
    v += rotate<8>(v);
    v += rotate<4>(v);
    v += rotate<2>(v);
    return v + rotate<1>(v);
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
__device__ __forceinline__ float value_at(const void *p, size_t i) {
    if constexpr (DT == MX_F32) return static_cast<const float *>(p)[i];
    const uint32_t u = static_cast<const uint16_t *>(p)[i];
    return DT == MX_F16 ? half_bits_to_float(u) : __builtin_bit_cast(float, u << 16);
}

template <int DT>
__device__ __forceinline__ void put_at(void *p, size_t i, float v) {
    if constexpr (DT == MX_F32)
        static_cast<float *>(p)[i] = v;
    else
        static_cast<uint16_t *>(p)[i] = uint16_t(DT == MX_F16 ? float_to_half_bits(v) : bf16_bits(v));
}

// The lane's VPT logits of a row, `none` past E.  quads: E is a multiple of
// four and rows are aligned to four elements.
template <int DT, int VPT>
__device__ __forceinline__ void load_row(const void *x, size_t row, uint32_t E, uint32_t j, bool quads, float none,
                                         float (&v)[VPT]) {
    const size_t base = row * E;
    if (quads) {
#pragma unroll
        for (int q = 0; q < VPT; q += 4) {
            const uint32_t e = j * VPT + q;
            const bool in = e < E;
            const size_t at = base + (in ? e : 0u);
            if constexpr (DT == MX_F32) {
                const float4_t f = *reinterpret_cast<const float4_t *>(static_cast<const float *>(x) + at);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[q + i] = in ? f[i] : none;
            } else {
                const uint2_t u = *reinterpret_cast<const uint2_t *>(static_cast<const uint16_t *>(x) + at);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t w = i < 2 ? u.x : u.y, h = i & 1 ? w >> 16 : w & 0xffffu;
                    const float f = DT == MX_F16 ? half_bits_to_float(h) : __builtin_bit_cast(float, h << 16);
                    v[q + i] = in ? f : none;
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const uint32_t e = j * VPT + i;
            v[i] = e < E ? value_at<DT>(x, base + (e < E ? e : 0u)) : none;
        }
    }
}

template <int DT, int VPT>
__device__ __forceinline__ void store_row(void *y, size_t row, uint32_t E, uint32_t j, bool quads,
                                          const float (&v)[VPT]) {
    const size_t base = row * E;
    if (quads) {
#pragma unroll
        for (int q = 0; q < VPT; q += 4) {
            const uint32_t e = j * VPT + q;
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
            if (j * VPT + i < E) put_at<DT>(y, base + j * VPT + i, v[i]);
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

// v -> softmax over the row's 16 lanes, in place (none of it where every
// logit is -inf: zeros).  Lanes' places past E hold -inf.
template <int VPT>
__device__ __forceinline__ void row_softmax(float (&v)[VPT]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) m = max(m, order_key(v[i]));
    const float top = key_value(row_max(m));
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        v[i] = exp_neg(v[i] - top);
        s += v[i];
    }
    s = row_sum(s);
    const float inv = 1.0f / s;
    const bool empty = top == -__builtin_inff();
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] = empty ? 0.f : v[i] * inv;
}

// -------------------------------------------------------------------- top k ---

struct TopkArgs {
    const void *logits;
    float *weights;
    int32_t *ids;
    const float *dweights;
    void *dlogits;
    uint32_t rows, E, k;
    uint32_t quads;
};

// The k highest logits, ties to the lowest expert, and their softmax weights:
// over the chosen (NORM) or over all.  k rounds of a maximum over the row;
// lanes hold consecutive experts, so of the lanes that hold the maximum the
// lowest has the lowest expert.
template <int DT, int VPT, bool NORM>
__global__ __launch_bounds__(256) void topk_kernel(TopkArgs a) {
    const uint32_t lane = threadIdx.x & 63u, j = lane & 15u;
    const uint32_t row = (blockIdx.x * 256 + threadIdx.x) / kRowLanes;
    const bool live = row < a.rows;
    float v[VPT];
    load_row<DT, VPT>(a.logits, live ? row : 0u, a.E, j, a.quads, -__builtin_inff(), v);
    uint32_t key[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) key[i] = j * VPT + i < a.E ? order_key(v[i]) : 0u;
    float chosen[4];  // lane j: choices j, 16 + j, ..
    int32_t id[4];
    float top = 0.f, sum = 0.f;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        if (16u * q >= a.k) break;  // uniform
        const uint32_t n = min(a.k - 16u * q, 16u);
        for (uint32_t c = 0; c < n; ++c) {
            uint32_t m = key[0];
#pragma unroll
            for (int i = 1; i < VPT; ++i) m = max(m, key[i]);
            const uint32_t best = row_max(m);
            const uint32_t has = uint32_t(__ballot(m == best) >> (lane & 48u)) & 0xffffu;
            const uint32_t win = uint32_t(__ffs(int(has))) - 1u;
            int32_t at = 0;
#pragma unroll
            for (int i = VPT - 1; i >= 0; --i) at = key[i] == best ? i : at;
            const int32_t e = __shfl(int32_t(j) * VPT + at, int(win), kRowLanes);
#pragma unroll
            for (int i = 0; i < VPT; ++i) key[i] = j == win && i == at ? 0u : key[i];
            const float value = key_value(best);
            if (q == 0 && c == 0) top = value;
            if constexpr (NORM) sum += exp_neg(value - top);
            if (j == c) {
                chosen[q] = value;
                id[q] = e;
            }
        }
    }
    if constexpr (!NORM) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) sum += exp_neg(v[i] - top);
        sum = row_sum(sum);
    }
    const bool empty = top == -__builtin_inff();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const uint32_t c = 16u * q + j;
        if (!live || c >= a.k) continue;
        const size_t at = size_t(row) * a.k + c;
        a.weights[at] = empty ? 0.f : exp_neg(chosen[q] - top) / sum;
        a.ids[at] = id[q];
    }
}

// d loss / d logits from d loss / d weights.  With D = sum_j w_j dw_j:
//   NORM      w_i (dw_i - D) at the chosen, 0 elsewhere
//   otherwise p_e (dw_e - D), dw_e = 0 where e was not chosen.
// The chosen's values meet their place in the row through LDS.
template <int DT, int VPT, bool NORM>
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
#pragma unroll
    for (int i = 0; i < VPT; ++i) place[r][j * VPT + i] = 0.f;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (uint32_t(id[q]) < a.E) place[r][id[q]] = NORM ? w[q] * (dw[q] - dot) : dw[q];
    __syncthreads();
    float d[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) d[i] = place[r][j * VPT + i];
    if constexpr (!NORM) {
        float p[VPT];
        load_row<DT, VPT>(a.logits, live ? row : 0u, a.E, j, a.quads, -__builtin_inff(), p);
        row_softmax<VPT>(p);
#pragma unroll
        for (int i = 0; i < VPT; ++i) d[i] = p[i] * (d[i] - dot);
    }
    if (live) store_row<DT, VPT>(a.dlogits, row, a.E, j, a.quads, d);
}

// ------------------------------------------------------------- balance loss ---
//
// Of a group's n kept tokens, with c_e the pairs that name expert e and S_e the
// sum of its probabilities: loss = E / (k n^2) sum_e c_e S_e, and
//   d loss / d l_te = E / (k n^2) p_te (c_e - sum_j c_j p_tj).
// The sums run in two launches whose order never changes: workgroups over
// shares of a group's tokens, then one workgroup a group over the shares.
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
    uint32_t T, E, k, shares, share, quads;  // share: tokens of one
};

template <int DT, int VPT>
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
    uint32_t mine = 0;
    for (uint32_t t0 = lo; t0 < hi; t0 += kBalanceRows) {
        const uint32_t t = t0 + tid / kRowLanes;
        const bool in = t < hi;
        const size_t row = size_t(group) * a.T + (in ? t : lo);
        const bool keep = in && (!a.mask || a.mask[row]);
        float p[VPT];
        load_row<DT, VPT>(a.logits, row, a.E, j, a.quads, -__builtin_inff(), p);
        row_softmax<VPT>(p);
#pragma unroll
        for (int i = 0; i < VPT; ++i) s[i] += keep ? p[i] : 0.f;
        if (keep) {
            for (uint32_t c = j; c < a.k; c += kRowLanes) {
                const uint32_t e = uint32_t(a.ids[row * a.k + c]);
                if (e < a.E) atomicAdd(&count[e], 1);
            }
            mine += j == 0;
        }
    }
    if (mine) atomicAdd(&kept, int32_t(mine));
    // the four rows of a wavefront, then the wavefronts
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        s[i] += __shfl_xor(s[i], 16, 64);
        s[i] += __shfl_xor(s[i], 32, 64);
        if (lane < 16) sums[wave][j * VPT + i] = s[i];
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

__global__ __launch_bounds__(1024) void balance_join_kernel(BalanceArgs a) {
    __shared__ float part[16];
    const uint32_t tid = threadIdx.x, group = blockIdx.x;
    const size_t base = size_t(group) * a.shares;
    int32_t n = 0;
    for (uint32_t s = 0; s < a.shares; ++s) n += a.pkept[base + s];
    float dot = 0.f;
    for (uint32_t e = tid; e < a.E; e += 1024) {
        float v = 0.f;
        int32_t c = 0;
        for (uint32_t s = 0; s < a.shares; ++s) {
            v += a.psum[(base + s) * a.E + e];
            c += a.pcount[(base + s) * a.E + e];
        }
        a.counts[size_t(group) * a.E + e] = c;
        dot += float(c) * v;
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) dot += __shfl_xor(dot, off, 64);
    if ((tid & 63u) == 0) part[tid >> 6] = dot;
    __syncthreads();
    if (tid == 0) {
        float v = 0.f;
        for (int w = 0; w < 16; ++w) v += part[w];
        const float fn = float(n);
        a.loss[group] = n ? v / fn * (float(a.E) / (float(a.k) * fn)) : 0.f;
        a.kept[group] = n;
    }
}

template <int DT, int VPT>
__global__ __launch_bounds__(256) void balance_grad_kernel(BalanceArgs a) {
    const uint32_t lane = threadIdx.x & 63u, j = lane & 15u;
    const uint32_t group = blockIdx.y, t = (blockIdx.x * 256 + threadIdx.x) / kRowLanes;
    const bool live = t < a.T;
    const size_t row = size_t(group) * a.T + (live ? t : 0u);
    const int32_t n = a.kept[group];
    const bool keep = live && n > 0 && (!a.mask || a.mask[row]);
    float p[VPT];
    load_row<DT, VPT>(a.logits, row, a.E, j, a.quads, -__builtin_inff(), p);
    row_softmax<VPT>(p);
    float c[VPT], dot = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const uint32_t e = j * VPT + i;
        c[i] = e < a.E ? float(a.counts[size_t(group) * a.E + (e < a.E ? e : 0u)]) : 0.f;
        dot += c[i] * p[i];
    }
    dot = row_sum(dot);
    const float fn = float(n), scale = a.dloss[group] / fn * (float(a.E) / (float(a.k) * fn));
#pragma unroll
    for (int i = 0; i < VPT; ++i) p[i] = keep ? scale * p[i] * (c[i] - dot) : 0.f;
    if (live) store_row<DT, VPT>(a.dlogits, row, a.E, j, a.quads, p);
}

// f(dtype, places a lane) as compile-time constants.
template <typename F>
void by_shape(int dtype, int64_t experts, F &&f) {
    const auto with = [&](auto dt) {
        if (experts <= 64)
            f(dt, std::integral_constant<int, 4>{});
        else if (experts <= 128)
            f(dt, std::integral_constant<int, 8>{});
        else if (experts <= 256)
            f(dt, std::integral_constant<int, 16>{});
        else if (experts <= 512)
            f(dt, std::integral_constant<int, 32>{});
        else
            f(dt, std::integral_constant<int, 64>{});
    };
    if (dtype == MX_F32)
        with(std::integral_constant<int, MX_F32>{});
    else if (dtype == MX_F16)
        with(std::integral_constant<int, MX_F16>{});
    else
        with(std::integral_constant<int, MX_BF16>{});
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
    // a share is whole turns of the workgroup's rows; about one workgroup a CU
    const int64_t most = (tokens + kBalanceRows - 1) / kBalanceRows;
    const int64_t want = (256 + groups - 1) / groups;
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
    a.rows = uint32_t(rows);
    a.E = uint32_t(experts);
    a.k = uint32_t(k);
    a.quads = quads_ok(dtype, experts, logits, nullptr);
    const dim3 grid{uint32_t((rows + 15) / 16)};
    by_shape(dtype, experts, [&](auto dt, auto vpt) {
        constexpr int DT = decltype(dt)::value, VPT = decltype(vpt)::value;
        if (normalize)
            hipLaunchKernelGGL((topk_kernel<DT, VPT, true>), grid, dim3{256}, 0, as_stream(stream), a);
        else
            hipLaunchKernelGGL((topk_kernel<DT, VPT, false>), grid, dim3{256}, 0, as_stream(stream), a);
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
    a.rows = uint32_t(rows);
    a.E = uint32_t(experts);
    a.k = uint32_t(k);
    a.quads = quads_ok(dtype, experts, normalize ? nullptr : logits, dlogits);
    const dim3 grid{uint32_t((rows + 15) / 16)};
    by_shape(dtype, experts, [&](auto dt, auto vpt) {
        constexpr int DT = decltype(dt)::value, VPT = decltype(vpt)::value;
        if (normalize)
            hipLaunchKernelGGL((topk_grad_kernel<DT, VPT, true>), grid, dim3{256}, 0, as_stream(stream), a);
        else
            hipLaunchKernelGGL((topk_grad_kernel<DT, VPT, false>), grid, dim3{256}, 0, as_stream(stream), a);
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
    a.quads = quads_ok(dtype, experts, logits, nullptr);
    by_shape(dtype, experts, [&](auto dt, auto vpt) {
        hipLaunchKernelGGL((balance_sums_kernel<decltype(dt)::value, decltype(vpt)::value>),
                           dim3(uint32_t(shares), uint32_t(groups)), dim3{kBalanceThreads}, 0, as_stream(stream), a);
    });
    if (const hipError_t err = hipGetLastError(); err != hipSuccess) return record_launch(err);
    hipLaunchKernelGGL(balance_join_kernel, dim3{uint32_t(groups)}, dim3{1024}, 0, as_stream(stream), a);
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
    a.quads = quads_ok(dtype, experts, logits, dlogits);
    by_shape(dtype, experts, [&](auto dt, auto vpt) {
        hipLaunchKernelGGL((balance_grad_kernel<decltype(dt)::value, decltype(vpt)::value>),
                           dim3(uint32_t((tokens + 15) / 16), uint32_t(groups)), dim3{256}, 0, as_stream(stream), a);
    });
    return record_launch(hipGetLastError());
}

}  // extern "C"
