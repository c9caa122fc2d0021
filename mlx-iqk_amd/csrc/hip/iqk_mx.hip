// 4-bit microscaled quantisation, its inverse, and the weights' layout (gfx950).
//
// Quantisation of a block of 32: with 2^p the power of two at or below its
// largest magnitude, the scale is 2^(p - 2), at least 2^-127, so the largest
// value lands in [4, 8) on a grid whose top is 6; values round to nearest,
// ties to the even code, and those above 6 to 6.  A block that holds a NaN or
// an infinity gets the NaN scale.  p is the exponent field of the largest
// magnitude's bits, and v_cvt_scalef32_pk_fp4_f32 scales, rounds and saturates
// two values at once, so both directions are bound by memory: a lane moves
// eight values (16 or 32 bytes), four lanes a block.  [131072 x 4096] in bf16: 302
// us to codes (4.5 TB/s read and written), 250 back (5.4); [8 x 4096]: 2.5 us
// each, a launch.

#include "iqk_host.h"
#include "iqk_mx.h"

namespace iqk {

constexpr int kCastThreads = 256;

template <int DT>
struct Eight {
    float v[8];
    __device__ __forceinline__ void load(const void *x, size_t i) {
        if constexpr (DT == MX_F32) {
            const float *p = static_cast<const float *>(x) + i;
            const float4_t a = *reinterpret_cast<const float4_t *>(p), b = *reinterpret_cast<const float4_t *>(p + 4);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                v[k] = a[k];
                v[4 + k] = b[k];
            }
        } else {
            const uint4_t a = load_u4(static_cast<const uint16_t *>(x) + i);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if constexpr (DT == MX_F16) {
                    v[2 * k] = half_bits_to_float(a[k] & 0xffffu);
                    v[2 * k + 1] = half_bits_to_float(a[k] >> 16);
                } else {
                    v[2 * k] = __builtin_bit_cast(float, a[k] << 16);
                    v[2 * k + 1] = __builtin_bit_cast(float, a[k] & 0xffff0000u);
                }
            }
        }
    }
};

__device__ __forceinline__ uint32_t magnitude(float f) { return __builtin_bit_cast(uint32_t, f) & 0x7fffffffu; }

struct CastArgs {
    const void *x;
    uint8_t *codes;
    uint8_t *scales;
    int64_t stride, scale_stride;  // elements between rows of x, bytes between rows of scales
    uint32_t eights;               // cols / 8
    uint64_t total;                // rows * cols / 8
};

template <int DT>
__global__ __launch_bounds__(kCastThreads) void mx_quantize_kernel(CastArgs a) {
    const uint64_t step = uint64_t(gridDim.x) * kCastThreads;
    // total is a multiple of four (a row is whole blocks) and so is step, so a
    // block's four lanes run the same turns
    for (uint64_t i = uint64_t(blockIdx.x) * kCastThreads + threadIdx.x; i < a.total; i += step) {
        const uint64_t row = i / a.eights;
        const uint32_t at = uint32_t(i - row * a.eights);
        Eight<DT> e;
        e.load(a.x, size_t(row) * a.stride + 8u * size_t(at));
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) top = max(top, magnitude(e.v[k]));
        top = max(top, uint32_t(__shfl_xor(int(top), 1, 64)));
        top = max(top, uint32_t(__shfl_xor(int(top), 2, 64)));
        const uint32_t p = top >> 23;  // exponent field: 255 for infinities and NaN
        const bool bad = p == 255u;
        const uint32_t byte = bad ? 255u : p > 2u ? p - 2u : 0u;
        // a scale below 2^-126 is no normal float: block and scale are moved up
        // by 2^64, exactly
        const bool low = byte < 64u;
        const float s = scale_float(low ? byte + 64u : byte), up = low ? 0x1p64f : 1.0f;
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, e.v[0] * up, e.v[1] * up, s, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, e.v[2] * up, e.v[3] * up, s, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, e.v[4] * up, e.v[5] * up, s, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, e.v[6] * up, e.v[7] * up, s, 3);
        reinterpret_cast<uint32_t *>(a.codes)[i] = bad ? 0u : c;
        if ((at & 3u) == 0u) a.scales[size_t(row) * a.scale_stride + (at >> 2)] = uint8_t(byte);
    }
}

// Two of a word's codes times the scale as floats.
template <int BYTE>
__device__ __forceinline__ float2v_t pair32(uint32_t codes, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, BYTE);
}

template <int DT>
__device__ __forceinline__ void store_eight(void *y, size_t i, uint32_t c, float s) {
    if constexpr (DT == MX_F32) {
        float2v_t v[4] = {pair32<0>(c, s), pair32<1>(c, s), pair32<2>(c, s), pair32<3>(c, s)};
        float *p = static_cast<float *>(y) + i;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            *reinterpret_cast<float4_t *>(p + 4 * h) = float4_t{v[2 * h].x, v[2 * h].y, v[2 * h + 1].x, v[2 * h + 1].y};
    } else {
        *reinterpret_cast<uint4_t *>(static_cast<uint16_t *>(y) + i) = eight16<DT == MX_BF16>(c, s);
    }
}

template <int DT>
__global__ __launch_bounds__(kCastThreads) void mx_dequantize_kernel(CastArgs a) {
    const uint64_t step = uint64_t(gridDim.x) * kCastThreads;
    for (uint64_t i = uint64_t(blockIdx.x) * kCastThreads + threadIdx.x; i < a.total; i += step) {
        const uint64_t row = i / a.eights;
        const uint32_t at = uint32_t(i - row * a.eights);
        const uint32_t c = reinterpret_cast<const uint32_t *>(a.codes)[i];
        const float s = scale_float(a.scales[size_t(row) * a.scale_stride + (at >> 2)]);
        store_eight<DT>(const_cast<void *>(a.x), 8u * size_t(i), c, s);
    }
}

struct PackArgs {
    const uint8_t *codes;
    const uint8_t *scales;
    uint4_t *tiles;
    uint8_t *tscale;
    int32_t *rexp;
    uint32_t out, rows, blocks, steps, quads;  // rows: out up to 16; blocks: in / 32; steps: in / 128 up; quads: out / 64 up
    int64_t scale_stride;
};

constexpr int kPackThreads = 256;

// The power of two that is taken out of a row whose blocks with a value have scale
// bytes least .. most.
__device__ __forceinline__ int row_exponent(int least, int most) {
    return most - min(max(most, kMxLow + most - least), kMxTop);
}

// 64 experts [2048 x 4096]: 161 us, 5.2 TB/s of 838 MB moved, the codes read once for
// the rows' scales and once for the tiles (once a checkpoint, so not kept between the two).
// One block of 256 threads a tile row (16 rows of one expert), thread (r, j):
// first the row's smallest and largest scale among blocks with a value, then the tiles.
__global__ __launch_bounds__(kPackThreads) void mx_pack_kernel(PackArgs a) {
    __shared__ int least_of[kMxRows][16], most_of[kMxRows][16];
    __shared__ int taken[kMxRows];
    const uint32_t trows = a.rows / kMxRows, e = blockIdx.x / trows, t = blockIdx.x % trows;
    const uint32_t tid = threadIdx.x, r = tid >> 4, j = tid & 15u, row = kMxRows * t + r;
    const size_t src = size_t(e) * a.out + row;
    const uint4_t *const codes = reinterpret_cast<const uint4_t *>(a.codes) + src * a.blocks;
    const uint8_t *const scales = a.scales + src * a.scale_stride;
    int least = 255, most = -1;
    if (row < a.out)
        for (uint32_t b = j; b < a.blocks; b += 16) {
            const int s = scales[b];
            const uint4_t c = codes[b];
            if (s != 255 && ((c.x | c.y | c.z | c.w) & 0x77777777u)) {
                least = min(least, s);
                most = max(most, s);
            }
        }
    least_of[r][j] = least;
    most_of[r][j] = most;
    __syncthreads();
    if (tid < kMxRows) {
        least = 255, most = -1;
        for (int k = 0; k < 16; ++k) {
            least = min(least, least_of[tid][k]);
            most = max(most, most_of[tid][k]);
        }
        taken[tid] = most < 0 ? 0 : row_exponent(least, most);
        a.rexp[size_t(e) * a.rows + kMxRows * t + tid] = taken[tid];
    }
    __syncthreads();
    // thread -> lane 16 g + rr of step s
    const uint32_t lane = tid & 63u, g = lane >> 4, rr = lane & 15u;
    const uint32_t row2 = kMxRows * t + rr;
    const size_t src2 = size_t(e) * a.out + row2;
    for (uint32_t s = tid >> 6; s < a.steps; s += 4) {
        const uint32_t b = 4 * s + g;
        uint4_t c = {0, 0, 0, 0};
        uint32_t byte = 127u;
        if (row2 < a.out && b < a.blocks) {
            c = reinterpret_cast<const uint4_t *>(a.codes)[src2 * a.blocks + b];
            const int raw = a.scales[src2 * a.scale_stride + b], kept = raw - taken[rr];
            // a block of zeros may have any scale, also one above the largest
            if (raw == 255)
                byte = 255u;
            else if (kept < 0 || !((c.x | c.y | c.z | c.w) & 0x77777777u))
                c = uint4_t{0, 0, 0, 0};
            else
                byte = uint32_t(kept);
        }
        a.tiles[((size_t(e) * trows + t) * a.steps + s) * 64 + lane] = c;
        a.tscale[(((size_t(e) * a.steps + s) * a.quads + t / 4) * 64 + lane) * 4 + t % 4] = uint8_t(byte);
    }
}

struct UnpackArgs {
    const uint4_t *tiles;
    const uint8_t *tscale;
    const int32_t *rexp;
    void *y;
    uint32_t out, rows, blocks, steps, quads;
    uint64_t total;  // num_experts * out * blocks * 4
};

// The tiles' weights as a dense stack: a lane eight values.  For checks and exports:
// 64 experts [2048 x 4096] take 453 us in f16 (3.0 TB/s) and 790 in f32; the lanes of a row
// read 16 bytes in a piece, as the tiles have them.
template <int DT>
__global__ __launch_bounds__(kCastThreads) void mx_unpack_kernel(UnpackArgs a) {
    const uint64_t step = uint64_t(gridDim.x) * kCastThreads;
    for (uint64_t i = uint64_t(blockIdx.x) * kCastThreads + threadIdx.x; i < a.total; i += step) {
        const uint64_t block = i >> 2, orow = block / a.blocks;
        const uint32_t b = uint32_t(block - orow * a.blocks), q = uint32_t(i) & 3u;
        const uint32_t e = uint32_t(orow / a.out), row = uint32_t(orow - uint64_t(e) * a.out);
        const uint32_t s = b >> 2, g = b & 3u;
        const uint4_t *const tile =
            a.tiles + ((size_t(e) * (a.rows / kMxRows) + row / kMxRows) * a.steps + s) * 64 + 16 * g + row % kMxRows;
        const uint32_t c = reinterpret_cast<const uint32_t *>(tile)[q];
        const uint32_t rel =
            a.tscale[(((size_t(e) * a.steps + s) * a.quads + row / 64) * 64 + 16 * g + row % 16) * 4 + row / 16 % 4];
        // back to the format's byte
        const int byte = rel == 255u ? 255 : int(rel) + a.rexp[size_t(e) * a.rows + row];
        store_eight<DT>(a.y, 8u * size_t(i), c, scale_float(uint32_t(min(max(byte, 0), 255))));
    }
}

uint32_t cast_blocks(uint64_t total) {
    // eight blocks a CU, each striding over the rest: the launch ends without a
    // tail of short blocks
    const uint64_t blocks = (total + kCastThreads - 1) / kCastThreads;
    return uint32_t(blocks < 256 * 8 ? blocks : 256 * 8);
}

bool mx_shape_ok(int64_t in, int64_t out, int64_t experts) {
    return in > 0 && in % kMxBlock == 0 && in < (int64_t(1) << 24) && out > 0 && out < (int64_t(1) << 24) &&
           experts > 0 && experts < (int64_t(1) << 20) &&
           grid_ok((out + 15) / 16 * experts, kPackThreads);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace iqk

extern "C" {

int iqk_mx_quantize(int dtype, const void *x, int64_t rows, int64_t cols, int64_t row_stride, uint8_t *codes,
                    uint8_t *scales, int64_t scale_stride, void *stream) {
    using namespace iqk;
    if (dtype < MX_F32 || dtype > MX_BF16) return IQK_ERR_ARGUMENT;
    if (cols <= 0 || cols % kMxBlock || cols >= (int64_t(1) << 32)) return IQK_ERR_GEOMETRY;
    if (rows < 0 || rows >= (int64_t(1) << 43) / cols || row_stride < 0 || scale_stride < cols / kMxBlock)
        return IQK_ERR_ARGUMENT;
    if (rows == 0) return IQK_OK;
    const int64_t per16 = dtype == MX_F32 ? 4 : 8;  // elements of 16 bytes
    if (!x || !codes || !scales || !aligned16(x) || (reinterpret_cast<uintptr_t>(codes) & 3u) || row_stride % per16)
        return IQK_ERR_ARGUMENT;
    CastArgs a{x, codes, scales, row_stride, scale_stride, uint32_t(cols / 8), uint64_t(rows) * uint64_t(cols / 8)};
    const dim3 grid{cast_blocks(a.total)}, block{kCastThreads};
    if (dtype == MX_F32)
        hipLaunchKernelGGL((mx_quantize_kernel<MX_F32>), grid, block, 0, as_stream(stream), a);
    else if (dtype == MX_F16)
        hipLaunchKernelGGL((mx_quantize_kernel<MX_F16>), grid, block, 0, as_stream(stream), a);
    else
        hipLaunchKernelGGL((mx_quantize_kernel<MX_BF16>), grid, block, 0, as_stream(stream), a);
    return record_launch(hipGetLastError());
}

int iqk_mx_dequantize(int dtype, const uint8_t *codes, const uint8_t *scales, int64_t rows, int64_t cols,
                      int64_t scale_stride, void *y, void *stream) {
    using namespace iqk;
    if (dtype < MX_F32 || dtype > MX_BF16) return IQK_ERR_ARGUMENT;
    if (cols <= 0 || cols % kMxBlock || cols >= (int64_t(1) << 32)) return IQK_ERR_GEOMETRY;
    if (rows < 0 || rows >= (int64_t(1) << 43) / cols || scale_stride < cols / kMxBlock) return IQK_ERR_ARGUMENT;
    if (rows == 0) return IQK_OK;
    if (!y || !codes || !scales || !aligned16(y) || (reinterpret_cast<uintptr_t>(codes) & 3u)) return IQK_ERR_ARGUMENT;
    CastArgs a{y, const_cast<uint8_t *>(codes), const_cast<uint8_t *>(scales), cols, scale_stride, uint32_t(cols / 8),
               uint64_t(rows) * uint64_t(cols / 8)};
    const dim3 grid{cast_blocks(a.total)}, block{kCastThreads};
    if (dtype == MX_F32)
        hipLaunchKernelGGL((mx_dequantize_kernel<MX_F32>), grid, block, 0, as_stream(stream), a);
    else if (dtype == MX_F16)
        hipLaunchKernelGGL((mx_dequantize_kernel<MX_F16>), grid, block, 0, as_stream(stream), a);
    else
        hipLaunchKernelGGL((mx_dequantize_kernel<MX_BF16>), grid, block, 0, as_stream(stream), a);
    return record_launch(hipGetLastError());
}

int iqk_mx_pack(int64_t in_features, int64_t out_features, int64_t num_experts, const uint8_t *codes,
                const uint8_t *scales, int64_t scale_stride, void *tiles, uint8_t *tile_scales, int32_t *row_exps,
                void *stream) {
    using namespace iqk;
    if (!mx_shape_ok(in_features, out_features, num_experts)) return IQK_ERR_GEOMETRY;
    if (!codes || !scales || !tiles || !tile_scales || !row_exps || !aligned16(codes) || !aligned16(tiles) ||
        scale_stride < in_features / kMxBlock)
        return IQK_ERR_ARGUMENT;
    const uint32_t rows = uint32_t((out_features + 15) / 16 * 16);
    PackArgs a{codes, scales, static_cast<uint4_t *>(tiles), tile_scales, row_exps, uint32_t(out_features), rows,
               uint32_t(in_features / kMxBlock), uint32_t((in_features + kMxStep - 1) / kMxStep),
               uint32_t((out_features + 63) / 64), scale_stride};
    hipLaunchKernelGGL(mx_pack_kernel, dim3{uint32_t(num_experts * (rows / kMxRows))}, dim3{kPackThreads}, 0,
                       as_stream(stream), a);
    return record_launch(hipGetLastError());
}

int iqk_mx_unpack(int dtype, int64_t in_features, int64_t out_features, int64_t num_experts, const void *tiles,
                  const uint8_t *tile_scales, const int32_t *row_exps, void *y, void *stream) {
    using namespace iqk;
    if (dtype < MX_F32 || dtype > MX_BF16) return IQK_ERR_ARGUMENT;
    if (!mx_shape_ok(in_features, out_features, num_experts)) return IQK_ERR_GEOMETRY;
    if (!tiles || !tile_scales || !row_exps || !y || !aligned16(tiles) || !aligned16(y)) return IQK_ERR_ARGUMENT;
    const uint32_t rows = uint32_t((out_features + 15) / 16 * 16), blocks = uint32_t(in_features / kMxBlock);
    UnpackArgs a{static_cast<const uint4_t *>(tiles), tile_scales, row_exps, y, uint32_t(out_features), rows, blocks,
                 uint32_t((in_features + kMxStep - 1) / kMxStep), uint32_t((out_features + 63) / 64),
                 uint64_t(num_experts) * uint64_t(out_features) * blocks * 4};
    const dim3 grid{cast_blocks(a.total)}, block{kCastThreads};
    if (dtype == MX_F32)
        hipLaunchKernelGGL((mx_unpack_kernel<MX_F32>), grid, block, 0, as_stream(stream), a);
    else if (dtype == MX_F16)
        hipLaunchKernelGGL((mx_unpack_kernel<MX_F16>), grid, block, 0, as_stream(stream), a);
    else
        hipLaunchKernelGGL((mx_unpack_kernel<MX_BF16>), grid, block, 0, as_stream(stream), a);
    return record_launch(hipGetLastError());
}

}  // extern "C"
