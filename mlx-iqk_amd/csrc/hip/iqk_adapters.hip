// Low-rank adapters of many requests beside a shared projection (gfx950):
//   out[t] = y[t] + s_a B_a (A_a x[t]),  a = ids[t],
// A_a [rank, in], B_a [out, rank], 16-bit like x and y.  Both are kept with eight consecutive
// values of their reduction axis together, so that lanes that take one rank or output each read
// consecutive 16 bytes: down [in / 8][rank][8], up [rank / 8][out][8].  An id of -1 leaves y[t], another one
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
    const uint16_t *y;
    uint16_t *out;
    uint32_t T, in, N, rank, adapters, wide, per_id;
    // grouped form
    const uint4_t *tiles;      // adapter (the bank's size: none), -, slots (0: no such tile), -
    const uint32_t *tile_rows; // [tile][slots] their rows
    float *sums;              // [splits][tile][slots][rank] A x, in parts
    uint32_t n_tiles, splits;
    uint32_t columns;         // 256s of outputs of a workgroup
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

// Two values in 16 bits.
template <bool BF>
__device__ __forceinline__ uint32_t pair_bits(float lo, float hi) {
    return BF ? bf16_bits(lo) | bf16_bits(hi) << 16 : float_to_half_bits(lo) | float_to_half_bits(hi) << 16;
}

template <bool BF>
constexpr uint16_t kNaN16 = BF ? 0x7fc0 : kHalfNaN;

// ------------------------------------------------------------- rows alone ---
//
// A workgroup computes A x of one row, then up to 1024 of its outputs, a thread each; that A x
// is computed again in every 1024 outputs' workgroup costs less than a second launch (the
// adapter comes from L2).  Of A's units of eight columns 16 lanes take 16 ranks each and a
// wavefront four units at a time; B's and y's loads, which wait for nothing, are on their way from the start.
// [8192 x 4096] of rank 16: one row 5.2 us, of which the launch takes 2.2 and three latencies (id, A,
// the sum over the wavefronts) the rest; 32 rows of 32 adapters 8.0 us, A from L2 eight times over (first
// in two launches: 6.6 and 9.4, and a gap).
constexpr int kAloneWaves = 16, kAloneThreads = 64 * kAloneWaves;

// GROUPS of 16 ranks and AHEAD units at once; UP: eights of ranks whose B is loaded ahead (0: none).
template <bool BF, int GROUPS, int AHEAD, int UP>
__global__ __launch_bounds__(kAloneThreads) void adapter_row_kernel(AdapterArgs a) {
    __shared__ float part[kAloneWaves][kRankMax];
    __shared__ __attribute__((aligned(16))) float t[kRankMax];
    const uint32_t columns = (a.N + kAloneThreads - 1) / kAloneThreads, row = blockIdx.x / columns;
    const uint32_t n = blockIdx.x % columns * kAloneThreads + threadIdx.x;
    const uint32_t id = __builtin_amdgcn_readfirstlane(adapter_of(a, row));
    const size_t at = size_t(row) * a.N + min(n, a.N - 1u);
    const uint16_t old = a.y[at];
    if (id >= a.adapters) {  // uniform
        if (n < a.N) a.out[at] = id == a.adapters ? old : kNaN16<BF>;
        return;
    }
    const uint32_t eights = a.rank / 8, units = a.in / 8;
    const uint16_t *const up = a.up + (size_t(id) * eights * a.N + min(n, a.N - 1u)) * 8;
    uint4_t ahead[UP ? UP : 1];
#pragma unroll
    for (int i = 0; i < UP; ++i) ahead[i] = load_u4(up + size_t(min(uint32_t(i), eights - 1u)) * a.N * 8);
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint16_t *const x = a.x + size_t(row) * a.in, *const down = a.down + size_t(id) * units * a.rank * 8;
    for (uint32_t r0 = 0; r0 < a.rank; r0 += 16 * GROUPS) {
        const uint32_t r = r0 + (lane & 15u);
        float sum[GROUPS] = {};
        for (uint32_t c0 = 4 * wave + (lane >> 4); c0 < units + (lane >> 4); c0 += 4 * kAloneWaves * AHEAD) {
            uint4_t xv[AHEAD], wv[AHEAD][GROUPS];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                if (c0 - (lane >> 4) + 4 * kAloneWaves * i >= units) continue;  // uniform
                const uint32_t c = min(c0 + 4 * kAloneWaves * i, units - 1u);
                xv[i] = *reinterpret_cast<const chunk_t *>(x + 8 * size_t(c));
#pragma unroll
                for (int q = 0; q < GROUPS; ++q)
                    if (r0 + 16 * q < a.rank)  // uniform
                        wv[i][q] = load_u4(down + (size_t(c) * a.rank + min(r + 16 * q, a.rank - 1u)) * 8);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                if (c0 + 4 * kAloneWaves * i >= units) continue;
#pragma unroll
                for (int q = 0; q < GROUPS; ++q) {
                    if (r0 + 16 * q >= a.rank) continue;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float2v_t p = floats<BF>(xv[i][k]), w = floats<BF>(wv[i][q][k]);
                        sum[q] = fmaf(p.y, w.y, fmaf(p.x, w.x, sum[q]));
                    }
                }
            }
        }
#pragma unroll
        for (int q = 0; q < GROUPS; ++q) {
            if (r0 + 16 * q >= a.rank) continue;
            sum[q] += __shfl_xor(sum[q], 16, 64);
            sum[q] += __shfl_xor(sum[q], 32, 64);
            if (lane < 16 && r + 16 * q < a.rank) part[wave][r + 16 * q] = sum[q];
        }
    }
    __syncthreads();
    if (threadIdx.x < a.rank) {
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kAloneWaves; ++w) sum += part[w][threadIdx.x];
        t[threadIdx.x] = sum * a.scales[id];
    }
    __syncthreads();
    if (n >= a.N) return;
    float sum = 0.f;
    const auto add = [&](uint4_t w, uint32_t i) {
        const float4_t lo = *reinterpret_cast<const float4_t *>(&t[8 * i]), hi = *reinterpret_cast<const float4_t *>(&t[8 * i + 4]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float2v_t b = floats<BF>(w[k]);
            const float t0 = k < 2 ? lo[2 * k] : hi[2 * k - 4], t1 = k < 2 ? lo[2 * k + 1] : hi[2 * k - 3];
            sum = fmaf(t1, b.y, fmaf(t0, b.x, sum));
        }
    };
    if constexpr (UP > 0) {
#pragma unroll
        for (int i = 0; i < UP; ++i)
            if (uint32_t(i) < eights) add(ahead[i], i);
    } else {
#pragma unroll 8
        for (uint32_t i = 0; i < eights; ++i) add(load_u4(up + size_t(i) * a.N * 8), i);
    }
    sum += float_of16<BF>(old);
    a.out[at] = uint16_t(BF ? bf16_bits(sum) : float_to_half_bits(sum));
}

// ------------------------------------------------------------- many rows ---
//
// Rows sorted by adapter, in tiles of 64 slots of one adapter; both products on the
// 16x16x32 MFMAs, operand A the adapter's (16 ranks, 16 outputs), operand B 16 slots'.  The
// first kernel leaves A x in f32, a sum for each part of the columns; the second adds these
// and splits each value into three 16-bit pieces.  bf16 has f32's exponents: pieces of eight bits,
// truncated, whose sum is the value.  f16 has fewer: a slot's values are multiplied with a power of
// two that brings the largest to 2^14 .. 2^15 (their sums are divided by it), and two pieces of
// eleven bits leave a rest of at most 2^-23 of the value or 2^-25, the third piece, times 2^24.  That
// is off by at most 2^-12 of the rest, so that the sum is off by 2^-24 of a value, an f32
// rounding, down to 2^-13, 2^27 below the slot's largest.  (Two pieces are off by 2^-23, and lose more from
// 2^17 below the largest on; rank 64 as below, 88.9 us with two, 90.1 with three.)  Where a rank of
// 16 slots is smaller still, or finite beside an infinity, their chunk of 32 ranks stays f32 and goes through
// the 16x16x4 f32 MFMAs (146 us with such a rank in every tile).

// Parts of the columns, at most.  us with 1, 2, 4 and (of 256 columns) 8, [8192 x 4096] of rank 16: 256 rows of 64
// adapters 34.5, 28.1, 24.6, 25.5, 2048 rows 51.2, 43.0, 39.4, 41.8; [256 x 8192], 4096 rows of 4 adapters
// 52.6, 36.7, 29.5, 26.7.
constexpr uint32_t kMaxSplits = 4;
constexpr int kTileSlots = int(kSortTile), kTileGroups = kTileSlots / 16;

constexpr int kPieces = 3;
constexpr float kThird = 0x1p24f;  // what f16's third piece is multiplied with
constexpr uint32_t kLeastBits = 0x39000000u;  // 2^-13, the smallest value that f16 pieces stand for

template <bool BF>
__device__ __forceinline__ float4_t mfma(uint4_t a, uint4_t b, float4_t c) {
    if constexpr (BF)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                       c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c,
                                                      0, 0, 0);
}

// Lanes of a wavefront read what others of it wrote to LDS.
__device__ __forceinline__ void wavefront_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A x of 16 CT slots of a tile over one of a.splits parts of the columns.  WAVES wavefronts take 64
// columns in turn and their sums meet in LDS.  A wavefront reads 128 bytes of a row together and
// turns them into operand B in its own part of LDS (rows read as the operand wants them, 16 of
// them 64 bytes each in an instruction, kept the loads waiting for the cache: 8192 rows of 4096,
// rank 16, 34 us; 17 now).  Nothing is loaded a step ahead: the registers that it takes keep other
// wavefronts off the CU, whose loads do as well (24 us with four steps on their way).
template <bool BF, int RT, int CT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void adapter_down_tiles_kernel(AdapterArgs a) {
    constexpr int SLOTS = 16 * CT, RANKS = 16 * RT, THREADS = 64 * WAVES, PARTS = kTileGroups / CT;
    constexpr int SUMS = SLOTS * (RANKS + 4), STAGE = SLOTS * 32;  // floats of a wavefront's sums, of its turned rows
    __shared__ __attribute__((aligned(16))) float shared[WAVES][SUMS > STAGE ? SUMS : STAGE];
    const uint32_t split = blockIdx.x % a.splits, block = blockIdx.x / a.splits;
    const uint32_t t = block / PARTS, group = block % PARTS * CT;  // the first of its groups of 16
    const uint4_t tile = a.tiles[t];
    const uint32_t adapter = tile.x;
    if (tile.z <= 16 * group || adapter >= a.adapters) return;  // uniform
    const uint32_t slots = min(tile.z - 16 * group, uint32_t(SLOTS));
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, m = lane & 15u, c8 = lane & 7u, r8 = lane >> 3;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint16_t *w[RT], *x[2 * CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)  // ranks past the last: it again, its sums not used
        w[r] = a.down + size_t(adapter) * a.rank * a.in + 8 * min(16u * r + m, a.rank - 1u);
#pragma unroll
    for (int c = 0; c < 2 * CT; ++c) {
        const uint32_t slot = 8 * c + r8, row = a.tile_rows[t * kTileSlots + 16 * group + slot];
        x[c] = a.x + size_t(slot < slots && row < a.T ? row : 0u) * a.in;  // past the tile's: row 0, its sums not used
    }
    float4_t acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[r][c] = float4_t{0, 0, 0, 0};
    constexpr uint32_t STEP = 64 * WAVES;
    uint4_t *const turned = reinterpret_cast<uint4_t *>(shared[wave]);  // [slot][8 chunks], chunk c at c ^ slot % 8
    // Each workgroup begins at another step: in step with each other they would all read the same
    // part of rows that lie a power of two apart, from few of the memory's channels.
    const uint32_t units = (a.in + 63) / 64, each = (units + a.splits - 1) / a.splits;
    const uint32_t first = min(units, split * each), last = min(units, first + each);
    const uint32_t steps = (last - first + WAVES - 1) / WAVES, turn = steps ? block % steps : 0u;
    const auto column = [&](uint32_t i) {
        return 64 * (first + wave) + STEP * (i + turn < steps ? i + turn : i + turn - steps);
    };
    const auto run = [&](auto live) {  // LIVE groups of 16 slots
        constexpr int LIVE = decltype(live)::value;
        for (uint32_t i = 0; i < steps; ++i) {
            const uint32_t k0 = column(i);
            if (k0 >= 64 * last) continue;  // uniform
            const bool rest = k0 + 64 > a.in;  // uniform: columns past the row, zeros on both sides
            uint4_t xv[2 * LIVE], wv[2][RT];
            const uint32_t kx = k0 + 8 * c8;
#pragma unroll
            for (int c = 0; c < 2 * LIVE; ++c)
                xv[c] = __builtin_nontemporal_load(reinterpret_cast<const chunk_t *>(x[c] + (kx < a.in ? kx : 0u)));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t kw = k0 + 32 * h + 8 * g;
#pragma unroll
                for (int r = 0; r < RT; ++r) wv[h][r] = load_u4(w[r] + size_t(kw < a.in ? kw : 0u) * a.rank);
            }
            wavefront_fence();
#pragma unroll
            for (int c = 0; c < 2 * LIVE; ++c) {
                if (rest && kx >= a.in) xv[c] = uint4_t{0, 0, 0, 0};
                turned[(8 * c + r8) * 8 + (c8 ^ r8)] = xv[c];
            }
            wavefront_fence();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint4_t b[LIVE];
#pragma unroll
                for (int c = 0; c < LIVE; ++c) b[c] = turned[(16 * c + m) * 8 + ((4 * h + g) ^ (m & 7u))];
                if (rest && k0 + 32 * h + 8 * g >= a.in) {
#pragma unroll
                    for (int r = 0; r < RT; ++r) wv[h][r] = uint4_t{0, 0, 0, 0};
                }
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int c = 0; c < LIVE; ++c) acc[r][c] = mfma<BF>(wv[h][r], b[c], acc[r][c]);
            }
        }
    };
    if (CT == 1 || slots <= 16)
        run(std::integral_constant<int, 1>{});
    else if (CT == 2 || slots <= 32)
        run(std::integral_constant<int, CT < 2 ? CT : 2>{});
    else
        run(std::integral_constant<int, CT>{});
    wavefront_fence();
    const auto part = [&](uint32_t w, uint32_t slot, uint32_t rank) -> float & { return shared[w][slot * (RANKS + 4) + rank]; };
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < CT; ++c) *reinterpret_cast<float4_t *>(&part(wave, 16 * c + m, 16 * r + 4 * g)) = acc[r][c];
    __syncthreads();
    for (uint32_t u = threadIdx.x; u < SLOTS * 2 * RT; u += THREADS) {
        const uint32_t slot = u / (2 * RT), r0 = 8 * (u % (2 * RT));
        if (r0 >= a.rank || slot >= slots) continue;
        float4_t lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < WAVES; ++k) {
            lo += *reinterpret_cast<const float4_t *>(&part(k, slot, r0));
            hi += *reinterpret_cast<const float4_t *>(&part(k, slot, r0 + 4));
        }
        float4_t *const out = reinterpret_cast<float4_t *>(
            a.sums + ((size_t(split) * a.n_tiles + t) * kTileSlots + 16 * group + slot) * a.rank + r0);
        out[0] = lo;
        out[1] = hi;
    }
}

// Outputs of a tile: 256 at a time, of which a wavefront takes 64 for all slots, the next 256's
// y and B on their way meanwhile.  The slots' operands are made once, in LDS (KC chunks of 32 ranks), and the sums go through it: the matrix cores leave four outputs of 16 slots to
// 64 lanes, memory wants 64 outputs of a slot together.  x, y and the outputs pass through once
// and do not stay in the caches in place of A, B and the sums (8192 rows of rank 64 [8192 x 4096]: 101 us, 96 so;
// 89 now, of which this kernel 62, 4.3 TB/s of y read and written).
template <bool BF, int KC>
__global__ __launch_bounds__(256, KC <= 4 ? 2 : 1) void adapter_up_tiles_kernel(AdapterArgs a) {
    constexpr int P = kPieces, CT = kTileGroups, STAGE = KC < 2 ? KC : 2;  // chunks of B in registers at once
    // B is loaded with the column before's, or (more registers than there are) with its own, once for
    // all slots, or (more than those) for each group of slots again; y always is ahead
    constexpr bool AHEAD = KC == 1, ONCE = KC <= 2;
    __shared__ uint4_t operands[CT][KC][P][64];
    __shared__ float powers[kTileSlots];  // what an f16 slot's sums are multiplied with
    __shared__ uint32_t chunks_in_f32[4];
    __shared__ __attribute__((aligned(16))) float turned[4][16][64 + 4];
    const uint32_t groups = (a.N + 256 * a.columns - 1) / (256 * a.columns), t = blockIdx.x / groups;
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, m = lane & 15u, s8 = lane >> 3;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t begin = blockIdx.x % groups * 256 * a.columns, end = min(a.N, begin + 256 * a.columns);
    const uint4_t tile = a.tiles[t];
    const uint32_t adapter = tile.x, slots = min(tile.z, uint32_t(kTileSlots));
    if (slots == 0) return;  // uniform
    uint32_t row[CT][2];  // a lane's outputs are of slots s8 and s8 + 8 of each group
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t slot = 16 * c + 8 * h + s8, of = a.tile_rows[t * kTileSlots + slot];
            row[c][h] = slot < slots && of < a.T ? of : 0u;  // past the tile's: read, not written
        }
    const uint32_t mine = 8 * (lane & 7u);
    if (adapter >= a.adapters) {  // rows without an adapter; uniform
        for (uint32_t n0 = begin + 64 * wave; n0 < end; n0 += 256) {
            const uint32_t n = n0 + mine, have = n < a.N ? min(a.N - n, 8u) : 0u;
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if (16u * c + 8 * h + s8 >= slots) continue;
                    const size_t at = size_t(row[c][h]) * a.N + n;
                    const bool bare = adapter_of(a, row[c][h]) == a.adapters;
                    const uint32_t nan = kNaN16<BF> * 0x10001u;
                    if (have == 8)
                        *reinterpret_cast<chunk_t *>(a.out + at) =
                            bare ? uint4_t(*reinterpret_cast<const chunk_t *>(a.y + at)) : uint4_t{nan, nan, nan, nan};
                    else
                        for (uint32_t i = 0; i < have; ++i) a.out[at + i] = bare ? a.y[at + i] : kNaN16<BF>;
                }
        }
        return;
    }
    const uint16_t *const up = a.up + size_t(adapter) * a.rank * a.N;
    uint4_t y[2][CT][2], w[AHEAD ? 2 : 1][STAGE][4];
    // Nothing is loaded under a condition, as in the first product.  Outputs past the last, and of rows of
    // fewer than eight, are not used: any others stand in for them.
    const auto load_y = [&](auto live, int d, uint32_t n0) __attribute__((always_inline)) {
        const uint32_t n = a.N < 8 ? 0u : min(n0 + mine, a.N - 8u);
#pragma unroll
        for (int c = 0; c < decltype(live)::value; ++c)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint16_t *const from = a.N < 8 ? up : a.y + size_t(row[c][h]) * a.N + n;
                y[d][c][h] = __builtin_nontemporal_load(reinterpret_cast<const chunk_t *>(from));
            }
    };
    const auto load_w = [&](int d, uint32_t n0, uint32_t k0) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < STAGE; ++s) {
            const uint32_t k = k0 + 32 * s + 8 * g, eight = min(k / 8, a.rank / 8 - 1u);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[d][s][j] = load_u4(up + (size_t(eight) * a.N + min(n0 + 16 * j + m, a.N - 1u)) * 8);
        }
    };
    // tiles begin at different columns, as their A x does
    const uint32_t turns = (end - begin + 255) / 256, turn = t % turns;
    const auto column = [&](uint32_t i) { return begin + 64 * wave + 256 * (i + turn < turns ? i + turn : i + turn - turns); };
    const auto by_live = [&](auto &&f) {
        if (slots <= 16)
            f(std::integral_constant<int, 1>{});
        else if (slots <= 32)
            f(std::integral_constant<int, 2>{});
        else
            f(std::integral_constant<int, 4>{});
    };
    by_live([&](auto live) { load_y(live, 0, column(0)); });
    if (ONCE) load_w(0, column(0), 0);
    __builtin_amdgcn_sched_barrier(0);
    // A x: the parts' sum, scaled, in pieces; a thread has eight ranks of a slot, 4 KC threads a slot
    constexpr int EIGHTS = 4 * KC;
    const float scale = a.scales[adapter];
    uint32_t in_f32 = 0;  // f16: the chunks of a group of slots (bit KC c + chunk) that stay f32
    const auto values = [&](uint32_t slot, uint32_t eight, float(&v)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 0.f;
        if (8 * eight >= a.rank || slot >= slots) return;
        const float *const from = a.sums + (size_t(t) * kTileSlots + slot) * a.rank + 8 * eight;
        float4_t parts[kMaxSplits][2];  // all on their way at once; past the last: it again
#pragma unroll
        for (uint32_t p = 0; p < kMaxSplits; ++p) {
            const float4_t *const part = reinterpret_cast<const float4_t *>(
                from + size_t(min(p, a.splits - 1u)) * a.n_tiles * kTileSlots * a.rank);
            parts[p][0] = part[0];
            parts[p][1] = part[1];
        }
#pragma unroll
        for (uint32_t p = 0; p < kMaxSplits; ++p) {
            if (p >= a.splits) continue;  // uniform
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] += parts[p][0][k], v[4 + k] += parts[p][1][k];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] *= scale;
    };
    // f16: the slot's power of two, and the values times it.  The largest comes to 2^14 .. 2^15; with an
    // infinity (or nothing) all stay as they are.
    const auto by_power = [&](float(&v)[8], float &most) __attribute__((always_inline)) {
        most = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) most = fmaxf(most, fabsf(v[k]));
#pragma unroll
        for (int off = 1; off < EIGHTS; off <<= 1) most = fmaxf(most, __shfl_xor(most, off, 64));
        const int e = most > 0.f && most < __builtin_inff() ? 14 - ilogbf(most) : 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = ldexpf(v[k], e);
        return e;
    };
    // operand B of a chunk of 32 ranks: lane 16 g + n has slot n's ranks 8 g ..
    const auto place = [&](uint32_t slot, uint32_t eight, int p) -> uint4_t & {
        return operands[slot / 16][eight / 4][p][16 * (eight & 3u) + (slot & 15u)];
    };
#pragma unroll
    for (int i = 0; i < kTileSlots * EIGHTS / 256; ++i) {
        const uint32_t u = 256 * i + threadIdx.x, slot = u / EIGHTS, eight = u % EIGHTS;
        float v[8];
        values(slot, eight, v);
        if constexpr (BF) {
#pragma unroll
            for (int p = 0; p < P; ++p) {
                uint4_t out;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint32_t bits = __builtin_bit_cast(uint32_t, v[k]);
                    const bool finite = (bits & 0x7f800000u) != 0x7f800000u;
                    uint32_t top = bits >> 16;
                    if (!finite && (bits & 0x7fffffu)) top |= 0x40u;  // a NaN stays one
                    v[k] = finite ? v[k] - __builtin_bit_cast(float, bits & 0xffff0000u) : 0.f;
                    out[k / 2] = k & 1 ? out[k / 2] | top << 16 : top;
                }
                place(slot, eight, p) = out;
            }
        } else {
            float most;
            const int e = by_power(v, most);
            uint32_t least = ~0u;  // bits of the smallest value but zeros, less 1
#pragma unroll
            for (int k = 0; k < 8; ++k) least = min(least, (__builtin_bit_cast(uint32_t, v[k]) & 0x7fffffffu) - 1u);
            // zeros are all ones here, NaN goes through the pieces
            if (least < kLeastBits - 1u || most == __builtin_inff()) in_f32 |= 1u << (slot / 16 * KC + eight / 4);
            if (eight == 0) powers[slot] = ldexpf(1.f, -e);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                uint4_t out;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const uint32_t top = float_to_half_bits(v[k]);
                    v[k] = (v[k] - half_bits_to_float(top)) * (p == 1 ? kThird : 1.f);
                    out[k / 2] = k & 1 ? out[k / 2] | top << 16 : top;
                }
                place(slot, eight, p) = out;
            }
        }
    }
    if constexpr (!BF) {
        if (__ballot(in_f32 != 0)) {
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) in_f32 |= uint32_t(__shfl_xor(int(in_f32), off, 64));
        }
        if (lane == 0) chunks_in_f32[wave] = in_f32;
    }
    __syncthreads();
    if constexpr (!BF) {
        in_f32 = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) in_f32 |= chunks_in_f32[i];
        in_f32 = __builtin_amdgcn_readfirstlane(in_f32);
        if (in_f32) {
            for (int i = 0; i < kTileSlots * EIGHTS / 256; ++i) {
                const uint32_t u = 256 * i + threadIdx.x, slot = u / EIGHTS, eight = u % EIGHTS;
                float v[8], most;
                values(slot, eight, v);
                by_power(v, most);
                if (in_f32 >> (slot / 16 * KC + eight / 4) & 1u) {
#pragma unroll
                    for (int p = 0; p < 2; ++p)
                        place(slot, eight, p) = __builtin_bit_cast(uint4_t, float4_t{v[4 * p], v[4 * p + 1], v[4 * p + 2], v[4 * p + 3]});
                }
            }
            __syncthreads();
        }
    }
    // WHOLE: every slot and output of the columns is there, and stored without a condition.  ANY_F32: a chunk
    // may be in f32 (a loop of its own with nothing ahead: the others have no registers left)
    const auto compute = [&](auto live, auto whole, auto any_f32, uint32_t n0) __attribute__((always_inline)) {
        constexpr int LIVE = decltype(live)::value;
        constexpr bool WHOLE = decltype(whole)::value, ANY_F32 = decltype(any_f32)::value;
        const uint32_t n = n0 + mine, have = n < a.N ? min(a.N - n, 8u) : 0u;
        if constexpr (ONCE) {  // past the ranks: zeros, as in the slots' operands
#pragma unroll
            for (int s = 0; s < STAGE; ++s)
                if (32 * s + 8 * g >= a.rank) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[0][s][j] = uint4_t{0, 0, 0, 0};
                }
        }
#pragma unroll
        for (int c = 0; c < LIVE; ++c) {
            float4_t acc[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = float4_t{0, 0, 0, 0};
#pragma unroll
            for (int k0 = 0; k0 < 32 * KC; k0 += 32 * STAGE) {
                if (k0 && uint32_t(k0) >= a.rank) continue;  // uniform
                if constexpr (!ONCE) {
                    load_w(0, n0, k0);
#pragma unroll
                    for (int s = 0; s < STAGE; ++s)
                        if (k0 + 32 * s + 8 * g >= a.rank) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) w[0][s][j] = uint4_t{0, 0, 0, 0};
                        }
                }
                // Sums as large as the third pieces, by a power of two: of slots without an infinity, whose chunks all
                // are f32, they are far from f32's end.
                constexpr uint32_t CHUNKS = (1u << STAGE) - 1u;
                const bool third = !BF && (!ANY_F32 || (in_f32 >> (KC * c + k0 / 32) & CHUNKS) != CHUNKS);
                if (third && k0) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[j] *= kThird;
                }
#pragma unroll
                for (int p = P - 1; p >= 0; --p) {  // the small pieces first
#pragma unroll
                    for (int s = 0; s < STAGE; ++s) {
                        if (ANY_F32 && (in_f32 >> (KC * c + k0 / 32 + s) & 1u)) continue;  // uniform
                        const uint4_t b = operands[c][k0 / 32 + s][p][lane];
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[j] = mfma<BF>(w[0][s][j], b, acc[j]);
                    }
                    if (third && p == 2) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[j] *= 1 / kThird;
                    }
                }
                if constexpr (ANY_F32) {
#pragma unroll
                    for (int s = 0; s < STAGE; ++s) {
                        if (!(in_f32 >> (KC * c + k0 / 32 + s) & 1u)) continue;  // uniform
                        const auto *const operand = operands[c][k0 / 32 + s];
                        const float4_t b[2] = {__builtin_bit_cast(float4_t, operand[0][lane]),
                                               __builtin_bit_cast(float4_t, operand[1][lane])};
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                uint32_t pair = w[0][s][j][k / 2];
                                asm volatile("" : "+v"(pair));  // made f32 here, not once for all groups and kept
                                acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                    float_of16<BF>(uint16_t(k & 1 ? pair >> 16 : pair)), b[k / 4][k % 4], acc[j], 0, 0, 0);
                            }
                        }
                    }
                }
            }
            wavefront_fence();
            const float power = BF ? 1.f : powers[16 * c + m];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float4_t v = acc[j];
                if constexpr (!BF) v *= power;
                *reinterpret_cast<float4_t *>(&turned[wave][m][16 * j + 4 * g]) = v;
            }
            wavefront_fence();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (!WHOLE && 16u * c + 8 * h + s8 >= slots) continue;
                const float *const v = &turned[wave][8 * h + s8][mine];
                const size_t at = size_t(row[c][h]) * a.N + n;
                if (WHOLE || have == 8) {
                    const float4_t lo = *reinterpret_cast<const float4_t *>(v), hi = *reinterpret_cast<const float4_t *>(v + 4);
                    uint4_t out;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2v_t old = floats<BF>(y[0][c][h][i]);
                        const float v0 = i < 2 ? lo[2 * i] : hi[2 * i - 4], v1 = i < 2 ? lo[2 * i + 1] : hi[2 * i - 3];
                        out[i] = pair_bits<BF>(old.x + v0, old.y + v1);
                    }
                    __builtin_nontemporal_store(chunk_t(out), reinterpret_cast<chunk_t *>(a.out + at));
                } else {
                    for (uint32_t i = 0; i < have; ++i) {
                        const float sum = float_of16<BF>(a.y[at + i]) + v[i];
                        a.out[at + i] = uint16_t(BF ? bf16_bits(sum) : float_to_half_bits(sum));
                    }
                }
            }
        }
    };
    const auto all = [&](auto live, auto whole) __attribute__((always_inline)) {
        for (uint32_t i = 0; i + 1 < turns; ++i) {
            if (ONCE && !AHEAD && i) load_w(0, column(i), 0);
            __builtin_amdgcn_sched_barrier(0);
            load_y(live, 1, column(i + 1));
            if (AHEAD) load_w(AHEAD ? 1 : 0, column(i + 1), 0);
            __builtin_amdgcn_sched_barrier(0);
            compute(live, whole, std::false_type{}, column(i));
#pragma unroll
            for (int c = 0; c < decltype(live)::value; ++c)
#pragma unroll
                for (int h = 0; h < 2; ++h) y[0][c][h] = y[1][c][h];
            if constexpr (AHEAD) {
#pragma unroll
                for (int s = 0; s < STAGE; ++s)
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[0][s][j] = w[1][s][j];
            }
        }
        if (ONCE && !AHEAD && turns > 1) load_w(0, column(turns - 1), 0);
        compute(live, whole, std::false_type{}, column(turns - 1));
    };
    if constexpr (!BF) {
        if (in_f32) {
            const std::integral_constant<int, CT> live{};
            for (uint32_t i = 0; i < turns; ++i) {
                load_y(live, 0, column(i));
                if (ONCE) load_w(0, column(i), 0);
                compute(live, std::false_type{}, std::true_type{}, column(i));
            }
            return;
        }
    }
    if (slots == kTileSlots && (end - begin) % 256 == 0)
        all(std::integral_constant<int, 4>{}, std::true_type{});
    else
        by_live([&](auto live) { all(live, std::false_type{}); });
}

namespace {

bool adapters_shape_ok(int64_t in, int64_t out, int64_t rank, int64_t adapters, int64_t rows) {
    constexpr int64_t kLim = int64_t(1) << 31;
    return in > 0 && in < kLim && in % 8 == 0 && out > 0 && out < kLim && rank > 0 && rank <= kRankMax && rank % 8 == 0 &&
           adapters > 0 && adapters <= kAdaptersMax && rows >= 0 && rows < kLim;
}

// Whether rows are computed each on its own, by what its workgroups read of the adapters, each and
// together.  us alone and grouped, bf16, 64 adapters, from a graph: [8192 x 4096] of rank 16, 64 rows (80 MiB) 13.0,
// 20.4, 128 rows (160 MiB) 21.6, 23.4; of rank 32, 32 rows (80 MiB) 13.1, 17.8, 64 rows (160 MiB) 23.1, 21.8; of
// rank 64, 16 rows (80 MiB) 15.2, 15.8, 32 rows (160 MiB) 21.6, 21.2; [4096 x 4096] of rank 128, one row
// (1.3 MiB a workgroup) 16.5, 15.3.  Adapters that are small beside the launches: [512 x 512] of rank 8, 1024 rows
// 6.5, 13.8, 1536 rows 8.7, 16.4, 4096 rows 20.5, 19.3; [1024 x 512] of rank 32, 1024 rows 14.0, 15.3, 1280 rows
// 17.0, 16.6: beyond 1024 workgroups it depends on their size, and is left to the tiles.
bool rows_stand_alone(int64_t in, int64_t out, int64_t rank, int64_t rows) {
    const int64_t groups = rows * ((out + kAloneThreads - 1) / kAloneThreads), each = rank * (in + kAloneThreads) * 2;
    return groups <= 1024 && each <= int64_t(1) << 20 && groups * each <= int64_t(128) << 20;
}

// The grouped form's workspace, in words: where each part begins.
struct GroupPlan {
    int64_t tiles, splits, hist, desc, tile_rows, sums, words;
};

GroupPlan group_plan(int64_t in, int64_t rank, int64_t adapters, int64_t rows) {  // of a row at least
    GroupPlan p{};
    p.tiles = sort_tiles(rows, adapters);
    // the columns in parts where the tiles leave CUs empty: two workgroups a CU, 512 columns each at least
    const int64_t want = 512 / p.tiles, most = in / 512;
    p.splits = want < 1 || most < 1 ? 1 : want < most ? want : most;
    if (p.splits > kMaxSplits) p.splits = kMaxSplits;
    const auto take = [&](int64_t words) {
        const int64_t at = p.words;
        p.words += (words + 3) / 4 * 4;  // 16-byte steps
        return at;
    };
    p.hist = take(sort_plan(rows, adapters).words);
    p.desc = take(4 * p.tiles);
    p.tile_rows = take(p.tiles * kTileSlots);
    p.sums = take(p.splits * p.tiles * kTileSlots * rank);
    return p;
}

// f(16s of ranks, groups of slots, wavefronts)
template <typename F>
void by_ranks(int64_t rank, F &&f) {
    using std::integer_sequence;
    if (rank <= 16)
        f(integer_sequence<int, 1, 4, 4>{});
    else if (rank <= 32)
        f(integer_sequence<int, 2, 4, 4>{});
    else if (rank <= 64)
        f(integer_sequence<int, 4, 4, 4>{});
    else if (rank <= 128)
        f(integer_sequence<int, 8, 2, 4>{});
    else
        f(integer_sequence<int, 16, 1, 4>{});
}

template <bool BF, int RT, int CT, int WAVES>
hipError_t launch_tiles(const AdapterArgs &a, int64_t tiles, hipStream_t stream,
                        std::integer_sequence<int, RT, CT, WAVES>) {
    const int64_t ups = tiles * ((int64_t(a.N) + 256 * a.columns - 1) / (256 * a.columns));
    hipLaunchKernelGGL((adapter_down_tiles_kernel<BF, RT, CT, WAVES>),
                       dim3{uint32_t(tiles * a.splits * (kTileGroups / CT))}, dim3{64 * WAVES}, 0, stream, a);
    if (const hipError_t err = hipGetLastError(); err != hipSuccess) return err;
    hipLaunchKernelGGL((adapter_up_tiles_kernel<BF, (RT + 1) / 2>), dim3{uint32_t(ups)}, dim3{256}, 0, stream, a);
    return hipGetLastError();
}

int rows_alone(const AdapterArgs &a, bool bf, hipStream_t stream) {
    const int64_t blocks = int64_t(a.T) * ((int64_t(a.N) + kAloneThreads - 1) / kAloneThreads);
    if (!grid_ok(blocks, kAloneThreads)) return IQK_ERR_GEOMETRY;
    const auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3{uint32_t(blocks)}, dim3{kAloneThreads}, 0, stream, a);
    };
    if (a.rank <= 16)
        bf ? run(adapter_row_kernel<true, 1, 2, 2>) : run(adapter_row_kernel<false, 1, 2, 2>);
    else if (a.rank <= 32)
        bf ? run(adapter_row_kernel<true, 2, 2, 4>) : run(adapter_row_kernel<false, 2, 2, 4>);
    else
        bf ? run(adapter_row_kernel<true, 4, 4, 0>) : run(adapter_row_kernel<false, 4, 4, 0>);
    return record_launch(hipGetLastError());
}

int rows_grouped(AdapterArgs a, bool bf, uint32_t *work, hipStream_t stream) {
    const GroupPlan p = group_plan(a.in, a.rank, a.adapters, a.T);
    // workgroups of up to 4 x 256 outputs, about eight a CU: with two that stay, a last one makes
    // a CU take half as long again (8192 rows [8192 x 512] of rank 16: 83 us, 75 so).  Beyond rank 64
    // the slots' operands, made anew by each, cost more than that.
    const int64_t wide = (int64_t(a.N) + 255) / 256, all = p.tiles * wide, each = a.rank > 64 ? all / 512 : all / 2048;
    const int64_t most = a.rank > 64 ? 8 : 4;
    a.columns = uint32_t(each < 1 ? 1 : each > most ? most : each);
    const int64_t ups = p.tiles * ((int64_t(a.N) + 256 * a.columns - 1) / (256 * a.columns));
    if (!grid_ok(ups, 256) || !grid_ok(p.tiles * p.splits * kTileGroups, 256)) return IQK_ERR_GEOMETRY;
    SortCall c{};
    c.ids = a.ids;
    c.wide = a.wide;
    c.pairs = a.T;
    c.experts = a.adapters;
    c.per_token = 1;
    c.per_id = a.per_id;
    c.work = work + p.hist;
    c.tiles = work + p.desc;
    c.tile_pairs = work + p.tile_rows;
    c.n_tiles = p.tiles;
    if (const int rc = sort_launch(c, stream); rc != IQK_OK) return rc;
    a.tiles = reinterpret_cast<const uint4_t *>(work + p.desc);
    a.tile_rows = work + p.tile_rows;
    a.sums = reinterpret_cast<float *>(work + p.sums);
    a.n_tiles = uint32_t(p.tiles);
    a.splits = uint32_t(p.splits);
    hipError_t err = hipSuccess;
    by_ranks(a.rank, [&](auto shape) {
        err = bf ? launch_tiles<true>(a, p.tiles, stream, shape) : launch_tiles<false>(a, p.tiles, stream, shape);
    });
    return record_launch(err);
}

}  // namespace
}  // namespace iqk

extern "C" {

int64_t iqk_adapters_work(int64_t in_features, int64_t out_features, int64_t rank, int64_t num_adapters, int64_t rows) {
    using namespace iqk;
    if (!adapters_shape_ok(in_features, out_features, rank, num_adapters, rows)) return -1;
    return rows == 0 || rows_stand_alone(in_features, out_features, rank, rows)
               ? 0 : group_plan(in_features, rank, num_adapters, rows).words;
}

int iqk_adapters(int dtype, int64_t in_features, int64_t out_features, int64_t rank, int64_t num_adapters,
                 const void *x, int64_t rows, const void *ids, int wide_ids, int64_t rows_per_id, const void *down,
                 const void *up, const float *scales, uint32_t *work, const void *y, void *out, void *stream) {
    using namespace iqk;
    if (dtype != MX_F16 && dtype != MX_BF16) return IQK_ERR_ARGUMENT;
    if (!adapters_shape_ok(in_features, out_features, rank, num_adapters, rows)) return IQK_ERR_GEOMETRY;
    if (rows == 0) return IQK_OK;
    const bool alone = rows_stand_alone(in_features, out_features, rank, rows);
    if (!x || !ids || rows_per_id <= 0 || rows_per_id >= (int64_t(1) << 31) || !down || !up || !scales || !y || !out ||
        (!alone && !work))
        return IQK_ERR_ARGUMENT;
    if ((reinterpret_cast<uintptr_t>(down) | reinterpret_cast<uintptr_t>(up) | reinterpret_cast<uintptr_t>(work)) & 15u)
        return IQK_ERR_ARGUMENT;
    AdapterArgs a{};
    a.x = static_cast<const uint16_t *>(x);
    a.ids = static_cast<const uint32_t *>(ids);
    a.down = static_cast<const uint16_t *>(down);
    a.up = static_cast<const uint16_t *>(up);
    a.scales = scales;
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
    return alone ? rows_alone(a, bf, as_stream(stream)) : rows_grouped(a, bf, work, as_stream(stream));
}

}  // extern "C"
