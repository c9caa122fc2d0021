// What the 4-bit microscaled kernels share (gfx950).
//
// The format: 32 consecutive values along the reduction axis share a scale
// 2^(byte - 127) (byte 255: the block is NaN) and hold four bits each, sign
// and the magnitude's index in {0, 1/2, 1, 3/2, 2, 3, 4, 6}; two codes a byte,
// the even position's in the low half.
//
// The products read weights laid out in tiles of 16 rows by 128 columns, the
// operand of v_mfma_scale_f32_16x16x128_f8f6f4: lane 16 g + r of a wavefront
// holds the 16 code bytes of row r, block g, and a tile is those 64 x 16
// bytes in lane order, so that a wavefront's load is 1 KiB in one piece.
//   tiles  u8  [E][rows / 16][steps][64][16]   (steps = columns / 128)
//   tscale u8  [E][steps][rows / 64][64][4]    byte i of lane 16 g + r: row 16 i + r, block g
//   rexp   i32 [E][rows]
// so a lane's word of scales serves a wavefront's 64 rows, the MFMA selecting
// the byte.  rows and columns round up to 16 (of tscale to 64) and 128 (codes 0,
// scale 1).  A row's scales are kept as byte - rexp, and its products' f32 sums are
// multiplied by 2^rexp at the end.  rexp brings the row into fp16: it is 0 where every
// block with a value has a scale of 2^-13 .. 2^13, whose weights are normal numbers
// there, and otherwise the one nearest to 0 with which that holds.  So the sums are
// those of the values themselves, and reach as far as f32 does, in every row but
// those.  Where the row's scales are more than 2^26 apart its largest becomes 2^13:
// weights down to 2^-36 of the largest scale are exact (fp16's smallest value
// is 2^-24), and a block below that rounds to multiples of 2^-24, under 2^-38 of the
// row's largest weight; below 2^-27 of it they are subnormal, and the matrix cores
// add them as exactly as values of 2^-27.  bf16 and the scaled MFMA hold all of them; a
// block more than 2^140 below its row's largest counts as zero.
#ifndef IQK_MX_H
#define IQK_MX_H

#include "iqk_device.h"

namespace iqk {

constexpr int kMxBlock = 32;          // values of one scale
constexpr int kMxStep = 128;          // columns of a tile
constexpr int kMxRows = 16;           // rows of a tile
constexpr int kMxTileBytes = 1024;
constexpr int kMxTop = 140;           // the stored scale of a row's largest block, at most
constexpr int kMxLow = 114;           // of its smallest, at least, where kMxTop leaves room

enum MxDtype : int { MX_F32 = 0, MX_F16 = 1, MX_BF16 = 2 };

typedef __bf16 bf16_t;
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef int int8v_t __attribute__((ext_vector_type(8)));
typedef int int4v_t __attribute__((ext_vector_type(4)));
typedef float float2v_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float scale_float(uint32_t byte) { return __builtin_bit_cast(float, byte << 23); }

__device__ __forceinline__ uint32_t bf16_bits(float f) {
    return uint32_t(__builtin_bit_cast(uint16_t, bf16_t(f)));
}

// Two of a word's eight codes (byte BYTE) times the scale, rounded once to
// 16 bits: v_cvt_scalef32_pk_{f16,bf16}_fp4 takes the scale's exponent field,
// so 0 stands for 2^-127 and 255 for NaN, as in the format.
template <bool BF, int BYTE>
__device__ __forceinline__ uint32_t pair16(uint32_t codes, float scale) {
    if constexpr (BF)
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, BYTE));
    else
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, BYTE));
}

// A word's eight values in 16 bits.
template <bool BF>
__device__ __forceinline__ uint4_t eight16(uint32_t codes, float scale) {
    return uint4_t{pair16<BF, 0>(codes, scale), pair16<BF, 1>(codes, scale), pair16<BF, 2>(codes, scale),
                   pair16<BF, 3>(codes, scale)};
}

}  // namespace iqk

#endif  // IQK_MX_H
