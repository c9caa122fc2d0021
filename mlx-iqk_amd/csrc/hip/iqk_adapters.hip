// Low-rank adapters of many requests beside a shared projection (gfx950):
//   out[t] = y[t] + s_a B_a (A_a x[t]),  a = ids[t],
// A_a [rank, in], B_a [out, rank], 16-bit like x and y; an id of -1 leaves y[t], another one
// outside the bank gives a row of NaN.  Products are exact and summed in f32, A_a x and its
// product with s_a stay in f32, and the sum with y is rounded once.

#include <type_traits>

#include "iqk_host.h"
#include "iqk_mx.h"

namespace iqk {

constexpr int64_t kAdaptersMax = 1024;
constexpr int64_t kRankMax = 256;

typedef uint32_t chunk_t __attribute__((ext_vector_type(4), aligned(2)));

struct AdapterArgs {
    const uint16_t *x;
    const uint32_t *ids;
    const uint16_t *down, *up;
    const float *scales;
    float *t;                 // [T][rank]
    const uint16_t *y;
    uint16_t *out;
    uint32_t T, in, N, rank, adapters, wide, per_id;
};

// The adapter of row t: the bank's size for none, more for one that does not exist.
__device__ __forceinline__ uint32_t adapter_of(const AdapterArgs &a, uint32_t t) {
    const uint32_t i = t / a.per_id;
    if (a.wide) {
        const uint2_t id = reinterpret_cast<const uint2_t *>(a.ids)[i];
        if (id.y == 0 && id.x < a.adapters) return id.x;
        return (id.x & id.y) == 0xffffffffu ? a.adapters : a.adapters + 1;
    }
    const uint32_t id = a.ids[i];
    return id < a.adapters ? id : id == 0xffffffffu ? a.adapters : a.adapters + 1;
}

template <bool BF>
__device__ __forceinline__ float2v_t floats(uint32_t w) {
    if constexpr (BF)
        return float2v_t{__builtin_bit_cast(float, w << 16), __builtin_bit_cast(float, w & 0xffff0000u)};
    else
        return float2v_t{half_bits_to_float(w & 0xffffu), half_bits_to_float(w >> 16)};
}

template <bool BF>
__device__ __forceinline__ float float_of16(uint16_t h) {
    return BF ? __builtin_bit_cast(float, uint32_t(h) << 16) : half_bits_to_float(h);
}

// t[row][j] = s A_a[j] . x[row]: a wavefront each.
template <bool BF>
__global__ __launch_bounds__(256) void adapter_down_kernel(AdapterArgs a) {
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t groups = (a.rank + 3) / 4, row = blockIdx.x / groups, j = blockIdx.x % groups * 4 + wave;
    if (j >= a.rank) return;
    const uint32_t id = adapter_of(a, row);
    if (id >= a.adapters) return;
    const uint16_t *const x = a.x + size_t(row) * a.in, *const w = a.down + (size_t(id) * a.rank + j) * a.in;
    float sum = 0.f;
    for (uint32_t c = 8 * lane; c < a.in; c += 512) {
        const uint4_t xv = *reinterpret_cast<const chunk_t *>(x + c), wv = load_u4(w + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2v_t p = floats<BF>(xv[i]), q = floats<BF>(wv[i]);
            sum = fmaf(p.y, q.y, fmaf(p.x, q.x, sum));
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if (lane == 0) a.t[size_t(row) * a.rank + j] = sum * a.scales[id];
}

// out[row][n] = y[row][n] + B_a[n] . t[row]: a thread each.
template <bool BF>
__global__ __launch_bounds__(256) void adapter_up_kernel(AdapterArgs a) {
    const uint32_t groups = (a.N + 255) / 256, row = blockIdx.x / groups, n = blockIdx.x % groups * 256 + threadIdx.x;
    if (n >= a.N) return;
    const uint32_t id = adapter_of(a, row);
    const size_t at = size_t(row) * a.N + n;
    if (id >= a.adapters) {
        a.out[at] = id == a.adapters ? a.y[at] : BF ? uint16_t(0x7fc0) : kHalfNaN;
        return;
    }
    const uint16_t *const w = a.up + (size_t(id) * a.N + n) * a.rank;
    const float *const t = a.t + size_t(row) * a.rank;
    float sum = 0.f;
    for (uint32_t c = 0; c < a.rank; c += 8) {
        const uint4_t wv = load_u4(w + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2v_t q = floats<BF>(wv[i]);
            sum = fmaf(t[c + 2 * i + 1], q.y, fmaf(t[c + 2 * i], q.x, sum));
        }
    }
    sum += float_of16<BF>(a.y[at]);
    a.out[at] = uint16_t(BF ? bf16_bits(sum) : float_to_half_bits(sum));
}

bool adapters_shape_ok(int64_t in, int64_t out, int64_t rank, int64_t adapters, int64_t rows) {
    constexpr int64_t kLim = int64_t(1) << 31;
    return in > 0 && in < kLim && in % 8 == 0 && out > 0 && out < kLim && rank > 0 && rank <= kRankMax && rank % 8 == 0 &&
           adapters > 0 && adapters <= kAdaptersMax && rows >= 0 && rows < kLim;
}

}  // namespace iqk

extern "C" {

int64_t iqk_adapters_work(int64_t in_features, int64_t out_features, int64_t rank, int64_t num_adapters, int64_t rows) {
    using namespace iqk;
    if (!adapters_shape_ok(in_features, out_features, rank, num_adapters, rows)) return -1;
    return rows * rank;
}

int iqk_adapters(int dtype, int64_t in_features, int64_t out_features, int64_t rank, int64_t num_adapters,
                 const void *x, int64_t rows, const void *ids, int wide_ids, int64_t rows_per_id, const void *down,
                 const void *up, const float *scales, uint32_t *work, const void *y, void *out, void *stream) {
    using namespace iqk;
    if (dtype != MX_F16 && dtype != MX_BF16) return IQK_ERR_ARGUMENT;
    if (!adapters_shape_ok(in_features, out_features, rank, num_adapters, rows)) return IQK_ERR_GEOMETRY;
    if (rows == 0) return IQK_OK;
    if (!x || !ids || rows_per_id <= 0 || rows_per_id >= (int64_t(1) << 31) || !down || !up || !scales || !work || !y ||
        !out)
        return IQK_ERR_ARGUMENT;
    if ((reinterpret_cast<uintptr_t>(down) | reinterpret_cast<uintptr_t>(up)) & 15u) return IQK_ERR_ARGUMENT;
    AdapterArgs a{};
    a.x = static_cast<const uint16_t *>(x);
    a.ids = static_cast<const uint32_t *>(ids);
    a.down = static_cast<const uint16_t *>(down);
    a.up = static_cast<const uint16_t *>(up);
    a.scales = scales;
    a.t = reinterpret_cast<float *>(work);
    a.y = static_cast<const uint16_t *>(y);
    a.out = static_cast<uint16_t *>(out);
    a.T = uint32_t(rows);
    a.in = uint32_t(in_features);
    a.N = uint32_t(out_features);
    a.rank = uint32_t(rank);
    a.adapters = uint32_t(num_adapters);
    a.wide = wide_ids != 0;
    a.per_id = uint32_t(rows_per_id);
    const int64_t downs = rows * ((rank + 3) / 4), ups = rows * ((out_features + 255) / 256);
    if (!grid_ok(downs, 256) || !grid_ok(ups, 256)) return IQK_ERR_GEOMETRY;
    const auto run = [&](auto kernel, int64_t blocks) {
        hipLaunchKernelGGL(kernel, dim3{uint32_t(blocks)}, dim3{256}, 0, as_stream(stream), a);
        return hipGetLastError();
    };
    const bool bf = dtype == MX_BF16;
    if (const hipError_t err = bf ? run(adapter_down_kernel<true>, downs) : run(adapter_down_kernel<false>, downs);
        err != hipSuccess)
        return record_launch(err);
    return record_launch(bf ? run(adapter_up_kernel<true>, ups) : run(adapter_up_kernel<false>, ups));
}

}  // extern "C"
