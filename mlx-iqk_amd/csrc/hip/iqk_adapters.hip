// Low-rank adapters of many requests beside a shared projection (gfx950):
//   out[t] = y[t] + s_a B_a (A_a x[t]),  a = ids[t],
// A_a [rank, in], B_a [out, rank], 16-bit like x and y; an id of -1 leaves y[t], another one
// outside the bank gives a row of NaN.  Products are exact and summed in f32, A_a x and its
// product with s_a stay in f32, and the sum with y is rounded once.

#include <type_traits>
#include <utility>

#include "iqk_host.h"
#include "iqk_mx.h"
#include "iqk_sort.h"

namespace iqk {

constexpr int64_t kAdaptersMax = kSortMaxExperts;
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
    // grouped form
    const uint32_t *offs;     // first slots of each adapter, then of the rows without one
    const uint32_t *rows;     // [T] each slot's row
    uint4_t *tiles;           // adapter, first slot, slots
    uint4_t *pieces;          // A x of a tile's slots, split, as operand B of the second product
    float *powers;            // [tile][slots] what the pieces are multiplied with
    uint32_t chunks;          // operands B of a slot: of 32 ranks, a power of two of them
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

// ------------------------------------------------------------- many rows ---
//
// Rows sorted by adapter, in tiles of 64 slots of one adapter; both products on the
// 16x16x32 MFMAs, operand A the adapter's (16 ranks, 16 outputs), operand B 16 slots'.  The
// first kernel leaves A x split into 16-bit pieces that give f32 back: a bf16 product takes three
// pieces of eight bits (truncated, so that their sum is exact), an f16 product two of eleven
// bits over a power of two of the slot's largest, which is multiplied back in f32.

constexpr int kTileSlots = 64, kTileGroups = kTileSlots / 16;

template <bool BF>
constexpr int kPieces = BF ? 3 : 2;

template <bool BF>
__device__ __forceinline__ float4_t mfma(uint4_t a, uint4_t b, float4_t c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                       c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c,
                                                      0, 0, 0);
}

struct Tile {
    uint32_t adapter, first, slots;  // slots 0: none
};

// Tile t of the list in which each adapter's slots, and the rows without one (adapter: the
// bank's size), take whole tiles in order.  All threads of a workgroup of THREADS call it.
template <int THREADS>
__device__ __forceinline__ Tile find_tile(const AdapterArgs &a, uint32_t t, uint32_t (&sums)[THREADS / 64], uint32_t (&found)[3]) {
    constexpr int PER = (int(kAdaptersMax) + THREADS) / THREADS;  // consecutive groups of a thread
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, g0 = threadIdx.x * PER;
    uint32_t first[PER + 1], mine = 0;
#pragma unroll
    for (int i = 0; i <= PER; ++i) first[i] = g0 + i <= a.adapters ? a.offs[g0 + i] : a.T;
#pragma unroll
    for (int i = 0; i < PER; ++i) mine += (first[i + 1] - first[i] + kTileSlots - 1) / kTileSlots;
    uint32_t incl = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t up = __shfl_up(incl, off, 64);
        if (lane >= uint32_t(off)) incl += up;
    }
    if (lane == 63) sums[wave] = incl;
    if (threadIdx.x == 0) found[2] = 0;
    __syncthreads();
    uint32_t at = incl - mine;
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w)
        if (uint32_t(w) < wave) at += sums[w];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const uint32_t n = first[i + 1] - first[i], tiles = (n + kTileSlots - 1) / kTileSlots;
        if (t >= at && t < at + tiles) {
            const uint32_t begin = (t - at) * kTileSlots;
            found[0] = g0 + i;
            found[1] = first[i] + begin;
            found[2] = min(n - begin, uint32_t(kTileSlots));
        }
        at += tiles;
    }
    __syncthreads();
    return {found[0], found[1], found[2]};
}

// A x of 16 CT slots of a tile: WAVES wavefronts take 32 KH columns in turn, DEPTH such steps on
// their way at once, and their sums meet in LDS.
template <bool BF, int RT, int CT, int WAVES, int KH, int DEPTH>
__global__ __launch_bounds__(64 * WAVES) void adapter_down_tiles_kernel(AdapterArgs a) {
    constexpr int SLOTS = 16 * CT, RANKS = 16 * RT, THREADS = 64 * WAVES, KC = (RT + 1) / 2, PARTS = kTileGroups / CT;
    __shared__ float part[WAVES][SLOTS][RANKS + 4];
    __shared__ uint32_t sums[WAVES], found[3];
    const uint32_t t = blockIdx.x / PARTS, group = blockIdx.x % PARTS * CT;  // the first of its groups of 16
    Tile tile = find_tile<THREADS>(a, t, sums, found);
    if (threadIdx.x == 0 && group == 0) a.tiles[t] = uint4_t{tile.adapter, tile.first, tile.slots, 0};
    if (tile.slots <= 16 * group || tile.adapter >= a.adapters) return;  // uniform
    tile.first += 16 * group;
    tile.slots = min(tile.slots - 16 * group, uint32_t(SLOTS));
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, m = lane & 15u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint16_t *w[RT], *x[CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)  // ranks past the last: it again, its sums not used
        w[r] = a.down + (size_t(tile.adapter) * a.rank + min(16u * r + m, a.rank - 1u)) * a.in;
#pragma unroll
    for (int c = 0; c < CT; ++c) x[c] = a.x + size_t(a.rows[tile.first + min(16u * c + m, tile.slots - 1u)]) * a.in;
    float4_t acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[r][c] = float4_t{0, 0, 0, 0};
    uint4_t xv[DEPTH][KH][CT], wv[DEPTH][KH][RT];
    constexpr uint32_t STEP = 32 * KH * WAVES;
    const auto load = [&](int d, uint32_t k0) {
#pragma unroll
        for (int h = 0; h < KH; ++h) {
            const uint32_t k = k0 + 32 * h + 8 * g;
            const bool in = k < a.in;
            const uint32_t at = in ? k : 0u;
#pragma unroll
            for (int c = 0; c < CT; ++c) xv[d][h][c] = *reinterpret_cast<const chunk_t *>(x[c] + at);
#pragma unroll
            for (int r = 0; r < RT; ++r) wv[d][h][r] = load_u4(w[r] + at);
        }
    };
    const auto multiply = [&](int d, uint32_t k0) {
#pragma unroll
        for (int h = 0; h < KH; ++h) {
            if (k0 + 32 * h + 32 > a.in && k0 + 32 * h + 8 * g >= a.in) {  // past the row: zeros on both sides
#pragma unroll
                for (int c = 0; c < CT; ++c) xv[d][h][c] = uint4_t{0, 0, 0, 0};
#pragma unroll
                for (int r = 0; r < RT; ++r) wv[d][h][r] = uint4_t{0, 0, 0, 0};
            }
#pragma unroll
            for (int r = 0; r < RT; ++r)
#pragma unroll
                for (int c = 0; c < CT; ++c) acc[r][c] = mfma<BF>(wv[d][h][r], xv[d][h][c], acc[r][c]);
        }
    };
    uint32_t k0 = 32 * KH * wave;
#pragma unroll
    for (int d = 0; d < DEPTH - 1; ++d) load(d, k0 + d * STEP);
    for (; k0 < a.in; k0 += DEPTH * STEP) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
            load((d + DEPTH - 1) % DEPTH, k0 + (d + DEPTH - 1) * STEP);
            if (k0 + d * STEP < a.in) multiply(d, k0 + d * STEP);  // uniform
        }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < CT; ++c) *reinterpret_cast<float4_t *>(&part[wave][16 * c + m][16 * r + 4 * g]) = acc[r][c];
    __syncthreads();
    const float scale = a.scales[tile.adapter];
    constexpr int UNITS = 4 * KC;  // eights of a slot's ranks, rounded up to whole operands
    for (uint32_t u = threadIdx.x; u < SLOTS * UNITS; u += THREADS) {
        const uint32_t slot = u / UNITS, unit = u % UNITS, r0 = 8 * unit;
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
        if (r0 < a.rank) {  // whole eights
#pragma unroll
            for (int k = 0; k < WAVES; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += part[k][slot][r0 + i];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= scale;
        }
        // operand B of chunk kc: lane 16 g + n has slot n's ranks 32 kc + 8 g ..
        const size_t at = ((size_t(t) * kTileGroups + group + slot / 16) * KC + unit / 4) * kPieces<BF> * 64 +
                          16 * (unit & 3u) + (slot & 15u);
        if constexpr (BF) {
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                uint4_t out;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t bits = __builtin_bit_cast(uint32_t, v[i]);
                    const bool finite = (bits & 0x7f800000u) != 0x7f800000u;
                    uint32_t top = bits >> 16;
                    if (!finite && (bits & 0x7fffffu)) top |= 0x40u;  // a NaN stays one
                    v[i] = finite ? v[i] - __builtin_bit_cast(float, bits & 0xffff0000u) : 0.f;
                    out[i / 2] = i & 1 ? out[i / 2] | top << 16 : top;
                }
                a.pieces[at + 64 * p] = out;
            }
        } else {
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[i]));
#pragma unroll
            for (int off = 1; off < UNITS; off <<= 1) most = fmaxf(most, __shfl_xor(most, off, 64));
            // the largest to 2^14 .. 2^15; with an infinity (or nothing) as it is
            const int e = most > 0.f && most < __builtin_inff() ? 14 - ilogbf(most) : 0;
            uint4_t hi, lo;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float scaled = ldexpf(v[i], e);
                const uint32_t top = float_to_half_bits(scaled);
                const float rest = fabsf(scaled) < __builtin_inff() ? scaled - half_bits_to_float(top) : 0.f;
                const uint32_t low = float_to_half_bits(rest);
                hi[i / 2] = i & 1 ? hi[i / 2] | top << 16 : top;
                lo[i / 2] = i & 1 ? lo[i / 2] | low << 16 : low;
            }
            a.pieces[at] = hi;
            a.pieces[at + 64] = lo;
            if (unit == 0) a.powers[size_t(t) * kTileSlots + 16 * group + slot] = ldexpf(1.f, -e);
        }
    }
}

// Two outputs in 16 bits.
template <bool BF>
__device__ __forceinline__ uint32_t pair_bits(float lo, float hi) {
    return BF ? bf16_bits(lo) | bf16_bits(hi) << 16 : float_to_half_bits(lo) | float_to_half_bits(hi) << 16;
}

// 256 outputs of a tile: a wavefront takes 64 of them for all slots, lane 16 g + n sixteen
// consecutive ones (16 g ..) of slot n of each group, so that y is read and written 32 bytes a
// lane.  The slots' operands go through LDS, which all four wavefronts read.
template <bool BF>
__global__ __launch_bounds__(256) void adapter_up_tiles_kernel(AdapterArgs a) {
    constexpr int P = kPieces<BF>, CT = kTileGroups, STAGE = 2;  // chunks of 32 ranks in LDS at once
    __shared__ uint4_t operands[STAGE][CT][P][64];
    const uint32_t columns = (a.N + 255) / 256, t = blockIdx.x / columns;
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, m = lane & 15u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t n0 = blockIdx.x % columns * 256 + 64 * wave;
    const uint4_t tile = a.tiles[t];
    const uint32_t adapter = tile.x, first = tile.y, slots = tile.z;
    if (slots == 0) return;  // uniform
    const uint32_t mine = n0 + 16 * g;  // the lane's first output
    const uint32_t have = mine < a.N ? min(a.N - mine, 16u) : 0u;
    size_t at[CT];
    uint32_t row[CT];
    uint4_t y[CT][2];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        row[c] = a.rows[first + min(16u * c + m, slots - 1u)];
        at[c] = size_t(row[c]) * a.N + mine;
        y[c][0] = y[c][1] = uint4_t{0, 0, 0, 0};
        if (have == 16 && 16u * c < slots) {
            y[c][0] = *reinterpret_cast<const chunk_t *>(a.y + at[c]);
            y[c][1] = *reinterpret_cast<const chunk_t *>(a.y + at[c] + 8);
        }
    }
    if (adapter >= a.adapters) {  // rows without an adapter; uniform
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            if (16 * c + m >= slots) continue;
            const bool bare = adapter_of(a, row[c]) == a.adapters;
            const uint32_t nan = BF ? 0x7fc07fc0u : 0x7e007e00u;
            if (have == 16) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    *reinterpret_cast<chunk_t *>(a.out + at[c] + 8 * h) = bare ? y[c][h] : uint4_t{nan, nan, nan, nan};
            } else {
                for (uint32_t i = 0; i < have; ++i) a.out[at[c] + i] = bare ? a.y[at[c] + i] : uint16_t(nan);
            }
        }
        return;
    }
    // operand A's row m of tile j is output 16 (m / 4) + 4 j + m % 4
    const uint16_t *w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        w[j] = a.up + (size_t(adapter) * a.N + min(n0 + 16 * (m >> 2) + 4 * j + (m & 3u), a.N - 1u)) * a.rank;
    float4_t acc[4][CT];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[j][c] = float4_t{0, 0, 0, 0};
    for (uint32_t k0 = 0; k0 < a.rank; k0 += 32 * STAGE) {
        uint4_t wv[STAGE][4];
#pragma unroll
        for (int s = 0; s < STAGE; ++s) {
            const uint32_t k = k0 + 32 * s + 8 * g;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                wv[s][j] = uint4_t{0, 0, 0, 0};
                if (k < a.rank) wv[s][j] = load_u4(w[j] + k);
            }
        }
        if (k0) __syncthreads();  // the stage before has been read
#pragma unroll
        for (int s = 0; s < STAGE; ++s) {
            if (k0 + 32 * s >= a.rank) continue;  // uniform
#pragma unroll
            for (int i = 0; i < (CT * P * 64) / 256; ++i) {  // a group's pieces of a chunk lie together
                const uint32_t u = 256 * i + threadIdx.x, c = u / (P * 64), rest = u % (P * 64);
                const size_t from = ((size_t(t) * CT + c) * a.chunks + k0 / 32 + s) * P * 64 + rest;
                if (16 * c < slots) operands[s][c][rest / 64][rest % 64] = a.pieces[from];
            }
        }
        __syncthreads();
#pragma unroll
        for (int s = 0; s < STAGE; ++s) {
            if (k0 + 32 * s >= a.rank) continue;  // uniform
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                if (16u * c >= slots) continue;  // uniform
#pragma unroll
                for (int p = P - 1; p >= 0; --p) {  // the small pieces first
                    const uint4_t b = operands[s][c][p][lane];
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[j][c] = mfma<BF>(wv[s][j], b, acc[j][c]);
                }
            }
        }
    }
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        if (16 * c + m >= slots) continue;
        const float power = BF ? 1.f : a.powers[size_t(t) * kTileSlots + 16 * c + m];
        float v[16];
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * j + i] = BF ? acc[j][c][i] : acc[j][c][i] * power;
        if (have == 16) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint4_t out;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t word = y[c][h][i];
                    const float2v_t old = floats<BF>(word);
                    out[i] = pair_bits<BF>(old.x + v[8 * h + 2 * i], old.y + v[8 * h + 2 * i + 1]);
                }
                *reinterpret_cast<chunk_t *>(a.out + at[c] + 8 * h) = out;
            }
        } else {
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i) {
                if (i >= have) continue;
                const float sum = float_of16<BF>(a.y[at[c] + i]) + v[i];
                a.out[at[c] + i] = uint16_t(BF ? bf16_bits(sum) : float_to_half_bits(sum));
            }
        }
    }
}

namespace {

bool adapters_shape_ok(int64_t in, int64_t out, int64_t rank, int64_t adapters, int64_t rows) {
    constexpr int64_t kLim = int64_t(1) << 31;
    return in > 0 && in < kLim && in % 8 == 0 && out > 0 && out < kLim && rank > 0 && rank <= kRankMax && rank % 8 == 0 &&
           adapters > 0 && adapters <= kAdaptersMax && rows >= 0 && rows < kLim;
}

constexpr int64_t kRowsAlone = 64;  // rows up to which each is computed on its own

// The grouped form's workspace, in words: where each part begins.
struct GroupPlan {
    int64_t tiles, chunks, hist, offs, rows, desc, pieces, powers, words;
};

GroupPlan group_plan(int64_t rank, int64_t adapters, int64_t rows) {
    GroupPlan p{};
    // every adapter and the rows without one may end in a part of a tile
    const int64_t most = rows / kTileSlots + adapters + 1;
    p.tiles = most < rows ? most : rows;
    for (p.chunks = 1; 32 * p.chunks < rank;) p.chunks *= 2;
    const auto take = [&](int64_t words) {
        const int64_t at = p.words;
        p.words += (words + 3) / 4 * 4;  // 16-byte steps
        return at;
    };
    p.hist = take(sort_plan(rows, adapters).words);
    p.offs = take(adapters + 1);
    p.rows = take(rows);
    p.desc = take(4 * p.tiles);
    p.pieces = take(p.tiles * kTileGroups * p.chunks * 3 * 64 * 4);
    p.powers = take(p.tiles * kTileSlots);
    return p;
}

// f(16s of ranks, groups of slots, wavefronts, 32s of columns a step, steps on their way)
template <typename F>
void by_ranks(int64_t rank, F &&f) {
    using std::integer_sequence;
    if (rank <= 16)
        f(integer_sequence<int, 1, 2, 8, 2, 4>{});
    else if (rank <= 32)
        f(integer_sequence<int, 2, 2, 8, 2, 4>{});
    else if (rank <= 64)
        f(integer_sequence<int, 4, 2, 8, 2, 2>{});
    else if (rank <= 128)
        f(integer_sequence<int, 8, 2, 4, 1, 2>{});
    else
        f(integer_sequence<int, 16, 1, 4, 1, 2>{});
}

template <bool BF, int RT, int CT, int WAVES, int KH, int DEPTH>
void launch_down(const AdapterArgs &a, int64_t tiles, hipStream_t stream, std::integer_sequence<int, RT, CT, WAVES, KH, DEPTH>) {
    hipLaunchKernelGGL((adapter_down_tiles_kernel<BF, RT, CT, WAVES, KH, DEPTH>), dim3{uint32_t(tiles * (kTileGroups / CT))},
                       dim3{64 * WAVES}, 0, stream, a);
}

int rows_alone(const AdapterArgs &a, bool bf, hipStream_t stream) {
    const int64_t downs = int64_t(a.T) * ((a.rank + 3) / 4), ups = int64_t(a.T) * ((int64_t(a.N) + 255) / 256);
    if (!grid_ok(downs, 256) || !grid_ok(ups, 256)) return IQK_ERR_GEOMETRY;
    const auto run = [&](auto kernel, int64_t blocks) {
        hipLaunchKernelGGL(kernel, dim3{uint32_t(blocks)}, dim3{256}, 0, stream, a);
        return hipGetLastError();
    };
    if (const hipError_t err = bf ? run(adapter_down_kernel<true>, downs) : run(adapter_down_kernel<false>, downs);
        err != hipSuccess)
        return record_launch(err);
    return record_launch(bf ? run(adapter_up_kernel<true>, ups) : run(adapter_up_kernel<false>, ups));
}

int rows_grouped(AdapterArgs a, bool bf, uint32_t *work, hipStream_t stream) {
    const GroupPlan p = group_plan(a.rank, a.adapters, a.T);
    const int64_t ups = p.tiles * ((int64_t(a.N) + 255) / 256);
    if (!grid_ok(ups, 256) || !grid_ok(p.tiles * kTileGroups, 512)) return IQK_ERR_GEOMETRY;
    SortCall c{};
    c.ids = a.ids;
    c.wide = a.wide;
    c.pairs = a.T;
    c.experts = a.adapters;
    c.per_token = 1;
    c.per_id = a.per_id;
    c.work = work + p.hist;
    c.offsets = reinterpret_cast<int32_t *>(work + p.offs);
    c.tokens = reinterpret_cast<int32_t *>(work + p.rows);
    if (const int rc = sort_launch(c, stream); rc != IQK_OK) return rc;
    a.offs = work + p.offs;
    a.rows = work + p.rows;
    a.tiles = reinterpret_cast<uint4_t *>(work + p.desc);
    a.pieces = reinterpret_cast<uint4_t *>(work + p.pieces);
    a.powers = reinterpret_cast<float *>(work + p.powers);
    a.chunks = uint32_t(p.chunks);
    by_ranks(a.rank, [&](auto shape) {
        if (bf)
            launch_down<true>(a, p.tiles, stream, shape);
        else
            launch_down<false>(a, p.tiles, stream, shape);
    });
    if (const hipError_t err = hipGetLastError(); err != hipSuccess) return record_launch(err);
    if (bf)
        hipLaunchKernelGGL(adapter_up_tiles_kernel<true>, dim3{uint32_t(ups)}, dim3{256}, 0, stream, a);
    else
        hipLaunchKernelGGL(adapter_up_tiles_kernel<false>, dim3{uint32_t(ups)}, dim3{256}, 0, stream, a);
    return record_launch(hipGetLastError());
}

}  // namespace
}  // namespace iqk

extern "C" {

int64_t iqk_adapters_work(int64_t in_features, int64_t out_features, int64_t rank, int64_t num_adapters, int64_t rows) {
    using namespace iqk;
    if (!adapters_shape_ok(in_features, out_features, rank, num_adapters, rows)) return -1;
    return rows <= kRowsAlone ? rows * rank : group_plan(rank, num_adapters, rows).words;
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
    if ((reinterpret_cast<uintptr_t>(down) | reinterpret_cast<uintptr_t>(up) | reinterpret_cast<uintptr_t>(work)) & 15u)
        return IQK_ERR_ARGUMENT;
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
    const bool bf = dtype == MX_BF16;
    return rows <= kRowsAlone ? rows_alone(a, bf, as_stream(stream)) : rows_grouped(a, bf, work, as_stream(stream));
}

}  // extern "C"
