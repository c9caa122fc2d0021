// Products with 4-bit microscaled weights (gfx950): y[p] = x[row(p)] W[e(p)]^T.
//
// Activations come in 16 bits, which enter exactly: the weights' codes are
// scaled into the same type (v_cvt_scalef32_pk_{f16,bf16}_fp4, two values an
// instruction, exact but for the tiny blocks that iqk_mx.h names) and
// contracted on the 16x16x32 MFMAs; or as 4-bit microscaled rows, where both
// operands go to v_mfma_scale_f32_16x16x128_f8f6f4 as they are, at four times
// the rate.  Sums are f32; the row's scale and one rounding end them.
//
// In every MFMA the weights are operand A (16 rows), the activations operand B
// (16 slots): a lane's accumulators are four consecutive outputs of one slot.
// Lane 16 g + r holds block g (32 columns) of row r in both operands; the
// 16-bit form splits a tile's 128 columns into four MFMAs of 32, the j-th taking
// values 8 j .. 8 j + 7 of each block.

#include <type_traits>

#include "iqk_host.h"
#include "iqk_mx.h"

namespace iqk {

// How a call's activations come, and so its outputs' type.
enum MxAct : int { ACT_F16 = 0, ACT_BF16 = 1, ACT_MX_F16 = 2, ACT_MX_BF16 = 3 };

constexpr bool act_mx(int act) { return act >= ACT_MX_F16; }
constexpr bool act_bf16(int act) { return act & 1; }

struct MxArgs {
    const uint8_t *x;        // 16-bit rows, or 4-bit codes
    const uint8_t *xscale;   // 4-bit rows' scales
    int64_t xscale_stride;
    const uint4_t *tiles;
    const uint32_t *tscale;  // words of a lane
    const int32_t *rexp;
    const uint32_t *ids;     // pairs: expert ids, or null: all expert 0
    const uint32_t *offs;    // groups: first slots, or null: one group
    const uint32_t *xr;      // groups: activation rows, or null: the slots'
    const uint32_t *yr;      // groups: output rows, or null: the slots'
    uint16_t *y;
    uint32_t K, N, rows, steps, quads, E, n_slots, n_x_rows, per_row, wide, set, run;
};

template <int ACT>
__device__ __forceinline__ uint32_t out16(float v) {
    if constexpr (act_bf16(ACT))
        return bf16_bits(v);
    else
        return float_to_half_bits(v);
}

template <int ACT>
constexpr uint16_t kOutNaN = act_bf16(ACT) ? 0x7fc0 : kHalfNaN;

template <int ACT>
__device__ __forceinline__ float4_t mfma16(uint4_t a, uint4_t b, float4_t c) {
    if constexpr (act_bf16(ACT))
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                       c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c,
                                                      0, 0, 0);
}

// Both operands four bits (format code 4), each lane's scale its words' low byte.
__device__ __forceinline__ float4_t mfma4(uint4_t a, uint32_t sa, uint4_t b, uint32_t sb, float4_t c) {
    const int8v_t av = {int(a.x), int(a.y), int(a.z), int(a.w), 0, 0, 0, 0};
    const int8v_t bv = {int(b.x), int(b.y), int(b.z), int(b.w), 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, int(sa), 0, int(sb));
}

// One 16-byte (4-byte) load per lane from global memory into LDS at lds + 16
// (4) lane, M0 holding the wavefront's base.  Inline asm, so that the compiler
// sees no load to wait for: the waits are written out below.  An LDS DMA right
// after the write of M0 needs one wait state.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void to_lds16(uint32_t lds, const void *src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(src)
                 : "memory", "m0");
}
__device__ __forceinline__ void to_lds4(uint32_t lds, const void *src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(src)
                 : "memory", "m0");
}
#pragma clang diagnostic pop

__device__ __forceinline__ uint32_t lds_address(const void *p) {
    return uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const uint8_t *)(p)));
}

__device__ uint4_t mx_zeros;

typedef const __attribute__((address_space(1))) uint8_t *global_ptr;

__device__ __forceinline__ uint4_t load_u4(global_ptr p) {
    return *reinterpret_cast<const __attribute__((address_space(1))) uint4_t *>(p);
}

// Sixteen bytes of zeros, as an address of which the compiler knows nothing: a
// load from there or from a row stays one load.
__device__ __forceinline__ global_ptr zero_chunk() {
    uint64_t p = reinterpret_cast<uint64_t>(&mx_zeros);
    asm("" : "+v"(p));
    return reinterpret_cast<global_ptr>(p);
}

// ------------------------------------------------------------- single pairs ---
//
// A workgroup computes 16 outputs of one token-expert pair.  Its wavefronts
// split the reduction axis, four tiles of 128 columns each, whose loads are all
// in flight before the first is used, and their sums meet in LDS.  The
// activations of a wavefront's 512 columns go straight into LDS (one load of 1 KiB,
// 256 bytes of 4-bit codes) and are read by all lanes of a block of 32, so every
// column of the MFMA holds the same slot: 15 of 16 columns are wasted, and free, for
// what bounds it is the weights' way.  48 pairs [4096 x 2048] take 35 us (6.1 TB/s,
// as much as a stream of reads reaches), 6 pairs [2048 x 4096] 6.9 (3.9 TB/s:
// the first loads' latency and the launch).
constexpr int kPairSteps = 4;

template <int ACT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void mx_pair_kernel(MxArgs a) {
    constexpr int XBYTES = act_mx(ACT) ? 256 : 1024;
    __shared__ float part[WAVES][kMxRows];
    __shared__ __attribute__((aligned(16))) uint8_t xlds[WAVES][XBYTES];
    const uint32_t trows = a.rows / kMxRows;
    const uint32_t p = blockIdx.x / trows;
    uint32_t t = blockIdx.x % trows;
    // the four tile rows that share words of scales run on one XCD (workgroups
    // eight apart), so that HBM is read once for them
    if (trows % 32 == 0) t = (t & ~31u) | (t & 7u) << 2 | (t >> 3 & 3u);
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t e = a.ids ? expert_id(a.ids, p, a.wide) : 0u;
    if (e >= a.E) {
        const uint32_t row = kMxRows * t + threadIdx.x;
        if (threadIdx.x < kMxRows && row < a.N) a.y[size_t(p) * a.N + row] = kOutNaN<ACT>;
        return;
    }
    const uint4_t *const tile = a.tiles + (size_t(e) * trows + t) * a.steps * 64 + lane;
    const uint32_t *const ts = a.tscale + (size_t(e) * a.steps * a.quads + t / 4) * 64 + lane;
    const size_t xrow = p / a.per_row;
    const uint32_t xat = lds_address(xlds[wave]), blocks = a.K / kMxBlock;
    float4_t acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    // the row's exponent, needed last, is on its way from the start (rows past N: up to 16, they exist)
    const int32_t ex = a.rexp[size_t(e) * a.rows + kMxRows * t + (threadIdx.x & 15u)];
    for (uint32_t s0 = wave * kPairSteps; s0 < a.steps; s0 += WAVES * kPairSteps) {
        if constexpr (act_mx(ACT)) {  // lane: 8 columns
            const uint32_t c = 64 * s0 + lane * 4;
            to_lds4(xat, c < a.K / 2 ? static_cast<const void *>(a.x + xrow * (a.K / 2) + c) : &mx_zeros);
        } else {
            const uint32_t c = 128 * s0 + lane * 8;
            to_lds16(xat, c < a.K ? static_cast<const void *>(a.x + 2 * (xrow * a.K + c)) : &mx_zeros);
        }
        uint4_t w[kPairSteps];
        uint32_t sc[kPairSteps], xs[kPairSteps];
#pragma unroll
        for (int i = 0; i < kPairSteps; ++i) {
            const uint32_t s = min(s0 + i, a.steps - 1u);  // past the last: its weights again, against zeros
            w[i] = tile[size_t(s) * 64];
            sc[i] = ts[size_t(s) * a.quads * 64];
            if constexpr (act_mx(ACT))
                xs[i] = *reinterpret_cast<const uint32_t *>(a.xscale + xrow * a.xscale_stride + 4 * s);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < kPairSteps; ++i) {
            const uint32_t byte = (sc[i] >> (8 * (t & 3u))) & 255u;
            if constexpr (act_mx(ACT)) {
                const uint32_t sx = 4 * (s0 + i) + g < blocks ? xs[i] >> (8 * g) : 127u;
                acc[i & 1] = mfma4(w[i], byte, load_u4(xlds[wave] + 64 * i + 16 * g), sx, acc[i & 1]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[j & 1] = mfma16<ACT>(eight16<act_bf16(ACT)>(w[i][j], scale_float(byte)),
                                             load_u4(xlds[wave] + 256 * i + 64 * g + 16 * j), acc[j & 1]);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // before the next turn's load into the same place
    }
    if ((lane & 15u) == 0) *reinterpret_cast<float4_t *>(&part[wave][4 * g]) = acc[0] + acc[1];
    __syncthreads();
    const uint32_t row = kMxRows * t + threadIdx.x;
    if (threadIdx.x < kMxRows && row < a.N) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) v += part[k][threadIdx.x];
        a.y[size_t(p) * a.N + row] = uint16_t(out16<ACT>(ldexpf(v, ex)));
    }
}

// ------------------------------------------------------------------- groups ---
//
// Slots sorted by expert; a workgroup of four wavefronts computes 256 outputs
// of up to 64 slots of one expert, a wavefront 64 of the outputs for all the
// slots, so that each weight is loaded and scaled by one wavefront only.  The
// weights go from memory into registers in the MFMA's layout, two steps of 128
// columns (4-bit activations: four) ahead; the slots' rows go through LDS, 256
// bytes a slot and turn (128 columns, or 512 of 4 bits), two buffers.  Two
// workgroups fit a CU, so that one's start, end and waits run under the other's
// products: with one workgroup of 128 slots a CU and both operands in an LDS
// ring, finding the tile, the first loads and the stores took 8 us a tile in
// which the CU did nothing else.
//
// The slots' 16-byte chunks are stored at positions chunk ^ swizzle(slot), so
// that an operand read (16 slots, one chunk each) meets no bank twice in any of
// its four parts of 16 lanes, which are {0-3, 12-15, 20-23, 24-27} and alike.
//
// Work list: the experts' M-tiles in order, an expert's ceil(slots / 64) of them.  A
// wavefront finds its tile from the offsets with two scans in registers: no
// list, and no workgroup without work but past the end.  (Numbers with gaps,
// offs[e] / 64 + e on for expert e, need no scan, but their empty workgroups cost
// more than their run: 256 experts of 64 slots took 451 us, and 286 without.)
// Measured, [2048 x 4096]: 144 pairs of 4-bit slots through 256 experts (117
// named) 86 us (5.7 TB/s: the weights), the 2048-token Zipf prefill (12288
// slots in bf16, 255 experts) 310 us, where 8192 evenly spread take 233 (4.9 TB/s)
// and 32768 530 (1.0 PFLOP/s; the matrix cores are busy for 61% of 1.6 GHz).
//
// The workgroups of an M-tile's outputs run on one XCD, with those of the next
// few M-tiles, so that it reads a slot's activations once for all outputs and a slice
// of the weights once for an expert's M-tiles.  An XCD's workgroups go to its shader
// engines in turn, whatever these still have to do, so consecutive ones are alike:
// eight blocks of outputs of one M-tile.  (One M-tile a shader engine, as heavy as it
// happens to be, left 27% of the wavefronts' places empty: 334 us against 317
// on the 2048-token Zipf prefill.)
constexpr int kMxBM = 64, kMxBN = 256, kMxWaves = 4;
constexpr int kMxRowBytes = 256;          // of a slot and turn in LDS
constexpr uint32_t kMxMaxExperts = 4096;  // 64 x 64, the two scans

template <int ACT>
__device__ __forceinline__ uint32_t swizzle(uint32_t slot) {
    // chunks read together: 4 g + j (16-bit), 4 j + g
    return act_mx(ACT) ? 2u * (slot & 3u) + (slot & 8u) : (slot & 3u) | ((slot & 8u) ? 12u : 0u);
}

struct MxTile {
    uint32_t e, m0, n, n0;  // expert, first slot, slots, first output
};

// The M-tile and the block of outputs of the workgroup: 8 a.set M-tiles at a time,
// a.set on each XCD; there a.run blocks of outputs of each of them, then the next a.run.
template <int BN>
__device__ __forceinline__ uint32_t tile_place(const MxArgs &a, uint32_t &n0) {
    const uint32_t nblocks = (a.N + BN - 1) / BN;
    uint32_t u = blockIdx.x / nblocks, nb = blockIdx.x % nblocks;
    if (a.set) {
        const uint32_t span = 8u * a.set * nblocks, v = blockIdx.x / span, i = blockIdx.x % span, k = i >> 3;
        u = (8u * v + (i & 7u)) * a.set + k / a.run % a.set;
        nb = k / (a.run * a.set) * a.run + k % a.run;
    }
    n0 = nb * BN;
    return u;
}

// The expert that holds M-tile u of all, or a.E past the last; u becomes its place in
// the expert.  tiles_of(from, n): the M-tiles of experts from .. from + n - 1.  Lane l
// counts those of `per` experts from l per on; the lane whose count holds u is
// then taken apart, a lane an expert.
template <class F>
__device__ __forceinline__ uint32_t find_expert(const MxArgs &a, uint32_t &u, F tiles_of) {
    const uint32_t lane = threadIdx.x & 63u, per = (a.E + 63u) / 64u;
    // the first lane whose running total exceeds u; u becomes its place in that lane
    const auto find = [&](uint32_t count) {
        uint32_t total = count;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t before = uint32_t(__shfl_up(int(total), off, 64));
            if (lane >= uint32_t(off)) total += before;
        }
        const uint64_t past = __ballot(total > u);
        if (past == 0) return 64u;
        const int at = __ffsll((unsigned long long)past) - 1;
        u -= uint32_t(__builtin_amdgcn_readlane(int(total - count), at));
        return uint32_t(at);
    };
    const uint32_t at = find(tiles_of(lane * per, per));
    if (at == 64u) return a.E;  // past the last tile
    if (per == 1) return at;
    const uint32_t first = at * per;
    return first + find(lane < per ? tiles_of(first + lane, 1) : 0u);
}

// The workgroup's tile of at most BM slots by BN outputs; false (uniformly) past the last.
template <int BM, int BN>
__device__ __forceinline__ bool find_tile(const MxArgs &a, MxTile &t) {
    uint32_t u = tile_place<BN>(a, t.n0);
    if (!a.offs) {
        t.e = 0;
        if (u >= (a.n_slots + BM - 1) / BM) return false;
        t.m0 = u * BM;
        t.n = min(a.n_slots - t.m0, uint32_t(BM));
        return true;
    }
    t.e = find_expert(a, u, [&](uint32_t from, uint32_t n) {
        uint32_t count = 0, lo = a.offs[min(from, a.E)];
        for (uint32_t i = 1; i <= n; ++i) {
            const uint32_t hi = a.offs[min(from + i, a.E)];
            count += (hi - lo + BM - 1u) / BM;
            lo = hi;
        }
        return count;
    });
    if (t.e >= a.E) return false;
    const uint32_t lo = a.offs[t.e], hi = min(a.offs[t.e + 1], a.n_slots);
    const uint64_t m0 = uint64_t(lo) + uint64_t(u) * BM;
    if (m0 >= hi) return false;
    t.m0 = uint32_t(m0);
    t.n = min(hi - t.m0, uint32_t(BM));
    return true;
}

// Few pairs are grouped by the workgroups themselves, which spares the launch
// that sorts them: each counts the experts' pairs in LDS, finds its tile and the pairs
// of its expert that are in it, in their order.
// The sorting takes 3.5 us; this up to 1 us a workgroup at 1024 pairs, so it has to
// be spared where workgroups are many (ids_pay: a round of 256 ids for 4096 of
// them): 60 experts [1000 x 1440], 596 pairs 14.7 us against 18.3 (0.25 of a
// limit), 256 experts [2048 x 4096], 400 pairs 152 against 157 (1), but 256 of
// [4096 x 2048], 1000 pairs 207 against 205 (4).
constexpr uint32_t kIdsPairs = 1024, kIdsExperts = 512;
constexpr int kIdsRounds = kIdsPairs / 256;

inline bool ids_pay(const MxArgs &a) {
    const uint64_t tiles = uint64_t(min(a.E, a.n_slots)) * ((a.N + kMxBN - 1) / kMxBN);
    return a.n_slots <= kIdsPairs && a.E <= kIdsExperts && tiles * ((a.n_slots + 255) / 256) <= 4096;
}

struct MxIds {
    uint32_t count[kIdsExperts];
    uint32_t hits[kIdsRounds][kMxWaves];
};

// A tile's slots: activation row, and output row, bit 31 where the slot's activations
// are real (~0: no slot).
template <int BM>
struct MxSlots {
    uint32_t row[BM], dst[BM];
};

// find_tile for the pairs a.ids, with the tile's slots.
template <int BM, int BN>
__device__ __forceinline__ bool find_ids(const MxArgs &a, MxTile &t, MxIds &sh, MxSlots<BM> &slots) {
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    uint32_t id[kIdsRounds];
#pragma unroll
    for (int i = 0; i < kIdsRounds; ++i) {
        const uint32_t p = tid + 256 * i;
        if (256u * i < a.n_slots) id[i] = expert_id(a.ids, min(p, a.n_slots - 1u), a.wide);
    }
    for (uint32_t e = tid; e < a.E; e += 256) sh.count[e] = 0;
    if (tid < BM) {
        slots.row[tid] = 0;
        slots.dst[tid] = 0xffffffffu;
    }
    __syncthreads();
    // an id out of range counts as the last expert's
#pragma unroll
    for (int i = 0; i < kIdsRounds; ++i)
        if (tid + 256 * i < a.n_slots) atomicAdd(&sh.count[min(id[i], a.E - 1u)], 1u);
    __syncthreads();
    uint32_t u = tile_place<BN>(a, t.n0);
    t.e = find_expert(a, u, [&](uint32_t from, uint32_t n) {
        uint32_t tiles = 0;
        for (uint32_t e = from; e < min(from + n, a.E); ++e) tiles += (sh.count[e] + BM - 1u) / BM;
        return tiles;
    });
    if (t.e >= a.E) return false;
    t.m0 = u * BM;  // of the expert's pairs
    t.n = min(sh.count[t.e] - t.m0, uint32_t(BM));
    uint64_t hit[kIdsRounds];
#pragma unroll
    for (int i = 0; i < kIdsRounds; ++i) {
        hit[i] = __ballot(tid + 256 * i < a.n_slots && min(id[i], a.E - 1u) == t.e);
        if (lane == 0) sh.hits[i][wave] = uint32_t(__popcll(hit[i]));
    }
    __syncthreads();
    uint32_t before = 0;
#pragma unroll
    for (int i = 0; i < kIdsRounds; ++i) {
        if (256u * i >= a.n_slots) break;
        uint32_t all = 0, mine = 0;
#pragma unroll
        for (uint32_t w = 0; w < kMxWaves; ++w) {
            const uint32_t n = sh.hits[i][w];
            mine += w < wave ? n : 0u;
            all += n;
        }
        const uint32_t at = before + mine + uint32_t(__popcll(hit[i] & ((uint64_t(1) << lane) - 1u))) - t.m0;
        if ((hit[i] >> lane & 1u) && at < BM) {
            const uint32_t p = tid + 256 * i, row = p / a.per_row;
            const bool real = id[i] < a.E && row < a.n_x_rows;
            slots.row[at] = real ? row : 0u;
            slots.dst[at] = p | (real ? 0x80000000u : 0u);
        }
        before += all;
    }
    __syncthreads();
    return true;
}

struct MxShared {
    __attribute__((aligned(16))) uint8_t x[2][kMxBM * kMxRowBytes];
    uint32_t xs[2][256];  // 4-bit slots' scales, a word a step
};

// A word of scales (a step's four blocks) with those of blocks past the row's end made 1.
__device__ __forceinline__ uint32_t clip_scales(uint32_t word, uint32_t step, uint32_t blocks) {
    const int n = int(blocks) - int(4 * step);  // blocks of this step
    const uint32_t keep = n >= 4 ? 0xffffffffu : n <= 0 ? 0u : (1u << (8 * n)) - 1u;
    return (word & keep) | (0x7f7f7f7fu & ~keep);
}

// The weights of a wavefront's 64 outputs: AHEAD steps of four tile rows in
// registers, and their words of scales.
template <int ACT, int AHEAD>
struct MxWeights {
    const uint4_t *src[4];
    const uint32_t *ssrc;
    uint32_t steps, sstep;
    uint4_t w[AHEAD][4];
    uint32_t sw[AHEAD];

    __device__ __forceinline__ void init(const MxArgs &a, uint32_t e, uint32_t row, uint32_t lane) {
        const uint32_t trows = a.rows / kMxRows;
        steps = a.steps;
        sstep = a.quads * 64;
#pragma unroll
        for (int i = 0; i < 4; ++i)  // outputs past the last: its tile row, never stored
            src[i] = a.tiles + (size_t(e) * trows + min(row / kMxRows + i, trows - 1u)) * steps * 64 + lane;
        ssrc = a.tscale + (size_t(e) * steps * a.quads + min(row / 64, a.quads - 1u)) * 64 + lane;
    }
    __device__ __forceinline__ void load(int slot, uint32_t step) {  // past the last: the last again
        const size_t s = min(step, steps - 1u);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[slot][i] = src[i][s * 64];
        sw[slot] = ssrc[s * sstep];
    }
    // four MFMAs of 4-bit operands: the weights' scale is byte i of the word
    __device__ __forceinline__ void multiply4(int slot, uint4_t b, uint32_t sb, float4_t &c0, float4_t &c1,
                                              float4_t &c2, float4_t &c3) const {
        const int8v_t bv = {int(b.x), int(b.y), int(b.z), int(b.w), 0, 0, 0, 0};
        const auto av = [&](int i) {
            const uint4_t v = w[slot][i];
            return int8v_t{int(v.x), int(v.y), int(v.z), int(v.w), 0, 0, 0, 0};
        };
        const int sa = int(sw[slot]);
        c0 = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av(0), bv, c0, 4, 4, 0, sa, 0, int(sb));
        c1 = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av(1), bv, c1, 4, 4, 1, sa, 0, int(sb));
        c2 = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av(2), bv, c2, 4, 4, 2, sa, 0, int(sb));
        c3 = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av(3), bv, c3, 4, 4, 3, sa, 0, int(sb));
    }
    // the j-th eight of each block's values in 16 bits
    __device__ __forceinline__ void scaled(int slot, int j, uint4_t (&wv)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            wv[i] = eight16<act_bf16(ACT)>(w[slot][i][j], scale_float((sw[slot] >> (8 * i)) & 255u));
    }
};

// The activation row of a slot of the tile; of one without activations, any row.
__device__ __forceinline__ uint32_t slot_row(const MxArgs &a, const MxTile &t, uint32_t slot) {
    uint32_t row = 0;
    if (slot < t.n) row = a.xr ? a.xr[t.m0 + slot] : t.m0 + slot;
    return row < a.n_x_rows ? row : 0u;
}
template <bool IDS, int BM>
__device__ __forceinline__ uint32_t slot_row(const MxArgs &a, const MxTile &t, const MxSlots<BM> &slots, uint32_t slot) {
    return IDS ? slots.row[slot] : slot_row(a, t, slot);
}

// A slot's output row, bit 31 set where its activations are real (else it is NaN); ~0: not stored.
__device__ __forceinline__ uint32_t slot_output(const MxArgs &a, const MxTile &t, uint32_t in_tile) {
    if (in_tile >= t.n) return 0xffffffffu;
    const uint32_t slot = t.m0 + in_tile, yrow = a.yr ? a.yr[slot] : slot, xrow = a.xr ? a.xr[slot] : slot;
    return yrow < a.n_slots ? yrow | (xrow < a.n_x_rows ? 0x80000000u : 0u) : 0xffffffffu;
}

// The exponents of rows row .. row + 3 (or, past the last, of any).
__device__ __forceinline__ int4v_t row_exps(const MxArgs &a, uint32_t e, uint32_t row) {
    return *reinterpret_cast<const int4v_t *>(a.rexp + size_t(e) * a.rows + min(row, a.rows - 4u));
}

// Outputs row .. row + 3 of a slot; d: its output row, bit 31 set where its activations are real.
template <int ACT>
__device__ __forceinline__ void store_four(const MxArgs &a, uint32_t d, uint32_t row, float4_t acc, int4v_t ex,
                                           bool whole) {
    uint32_t v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = d >> 31 ? out16<ACT>(ldexpf(acc[k], ex[k])) : uint32_t(kOutNaN<ACT>);
    uint16_t *const y = a.y + size_t(d & 0x7fffffffu) * a.N + row;
    if (whole) {
        *reinterpret_cast<uint2_t *>(y) = uint2_t{v[0] | v[1] << 16, v[2] | v[3] << 16};
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (row + k < a.N) y[k] = uint16_t(v[k]);
    }
}

// The wavefront's outputs: row0 its first, acc[i][c] tile row i, slots 16 c ...
// The exponents are read before the first store: the compiler must take each store
// for one that may change them, and would read them again after it.
template <int ACT, int RT, int NC>
__device__ __forceinline__ void store_outputs(const MxArgs &a, uint32_t e, uint32_t row0, const uint32_t *dst,
                                              const float4_t (&acc)[RT][NC], uint32_t lane) {
    const uint32_t g = lane >> 4, r = lane & 15u;
    const bool whole = a.N % 4 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 7u) == 0;
    int4v_t ex[RT];
    uint32_t d[NC];
#pragma unroll
    for (int i = 0; i < RT; ++i) ex[i] = row_exps(a, e, row0 + i * kMxRows + 4 * g);
#pragma unroll
    for (int c = 0; c < NC; ++c) d[c] = dst[16 * c + r];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        if (d[c] == 0xffffffffu) continue;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const uint32_t row = row0 + i * kMxRows + 4 * g;
            if (row < a.N) store_four<ACT>(a, d[c], row, acc[i][c], ex[i], whole);
        }
    }
}

// The loops below run whole rounds of AHEAD steps without a way out in between,
// and no loaded value is touched before its use: a branch or a select there
// makes the compiler copy the registers that a load in flight will fill, and
// wait for it.  So what lies past the end is read from a zero (activations) or is
// the last step again (weights), and adds nothing.  The loads before a loop are in
// the order in which its rounds leave them: the waits inside count the loads
// behind the awaited one, and take the fewest of the two ways in.  (All weights
// first, then all slots: the loops waited for everything once a round; 8 experts [2048
// x 4096] of 32 slots took 27.0 us against 23.3, 32 of 32 40.3 against 34.3.)

// Up to 16 slots by a wavefront's 64 outputs, over the steps first, first + stride, ..:
// the slots' rows come straight from memory in the MFMA's layout too, so the
// wavefronts run on their own, with AHEAD steps of both operands in flight, and HBM
// is kept busy.  (Eight steps of weights for 16-bit slots too: 220 us against
// 203 over 256 experts of eight slots.)
template <int ACT, bool IDS, int BM>
__device__ __forceinline__ void few_slots(const MxArgs &a, const MxTile &t, const MxSlots<BM> &slots, uint32_t row0,
                                          uint32_t first, uint32_t stride, float4_t (&acc)[4][1]) {
    constexpr bool MX = act_mx(ACT);
    constexpr int AHEAD = MX ? 8 : 4, XN = MX ? 1 : 4, STEP = MX ? 64 : 256;
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, r = lane & 15u;
    const uint32_t steps = row0 < a.N ? a.steps : 0u;
    MxWeights<ACT, AHEAD> w;
    w.init(a, t.e, row0, lane);
    // the lane's bytes of a step stand at [STEP step + STEP / 4 g, ..)
    const size_t row = slot_row<IDS>(a, t, slots, r);
    const uint32_t xbytes = MX ? a.K / 2 : 2 * a.K, end = r < t.n ? xbytes - STEP / 4 * g : 0u;
    const global_ptr xsrc = global_ptr(a.x) + row * xbytes + STEP / 4 * g;
    const uint8_t *const xscale = MX ? a.xscale + row * a.xscale_stride : nullptr;
    const global_ptr zeros = zero_chunk();
    uint4_t x[AHEAD][XN];
    uint32_t xs[AHEAD];
    const auto load_x = [&](int slot, uint32_t step) {
        const uint32_t at = step * STEP;
        const bool in = int(at) < int(end);
#pragma unroll
        for (int j = 0; j < XN; ++j) x[slot][j] = load_u4(in ? xsrc + at + 16 * j : zeros);
        if constexpr (MX) xs[slot] = *reinterpret_cast<const uint32_t *>(xscale + 4 * min(step, a.steps - 1u));
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
        w.load(i, first + i * stride);
        load_x(i, first + i * stride);
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i][0] = float4_t{0, 0, 0, 0};
    for (uint32_t s0 = first; s0 < steps; s0 += AHEAD * stride) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const uint32_t s = s0 + i * stride;
            if constexpr (MX) {
                const uint32_t sx = clip_scales(xs[i], s, a.K / kMxBlock) >> (8 * g);
                w.multiply4(i, x[i][0], sx, acc[0][0], acc[1][0], acc[2][0], acc[3][0]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint4_t wv[4];
                    w.scaled(i, j, wv);
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[k][0] = mfma16<ACT>(wv[k], x[i][j], acc[k][0]);
                }
            }
            w.load(i, s + AHEAD * stride);
            load_x(i, s + AHEAD * stride);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
}

template <int ACT, bool IDS>
__device__ __forceinline__ void few_tile(const MxArgs &a, const MxTile &t, const MxSlots<kMxBM> &slots) {
    const uint32_t row0 = t.n0 + 64 * __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    float4_t acc[4][1];
    few_slots<ACT, IDS>(a, t, slots, row0, 0, 1, acc);
    __syncthreads();  // the slots' outputs
    store_outputs<ACT, 4, 1>(a, t.e, row0, slots.dst, acc, threadIdx.x & 63u);
}

// Where the tiles above would leave CUs without work: tiles of 16 slots, whose
// wavefronts split the reduction axis, in four for 64 outputs or in two for 128, and
// add up in LDS, in their order.  A round of them takes 10 us with 4096 columns and
// 8 with 1440, 4-bit slots as long; one of 64 x 256 tiles as long as its slots: 14
// us for a few, 23 for 16, 30 for 64 (4-bit: 12, 17, 16).  So they serve while every
// CU has one at most, first of 64, then of 128 outputs: 8 experts [2048 x 4096] of 8
// slots 10.0, 11.6 and 17.7 us by 64, 128 and 256 outputs (4-bit 10.6, 10.7, 14.7);
// of 32 slots (past the first limit) 17.1, 15.9 and 19.5; 16 of 24 (past both)
// 31.9, 28.6 and 22.5; 60 [1000 x 1440] of 10 22.4, 17.0 and 14.3.  4-bit slots under
// 24 steps leave four ways out, which are slower below 17 (8 experts x 2048 outputs of 8
// slots, 16 steps 9.0 by four, 8.2 by two, 10.0 by one; 12 steps 8.3, 7.9 and 9.4) and would
// be faster from 18 on (8.9, 9.6 and 11.2; 22 steps 9.2, 9.8 and 11.3); and two where an expert has several such tiles: 8 experts of 32 slots 16.9, 16.2
// and 12.7, but 16 of 16 19.3, 18.1 and 22.3.
constexpr int kSplitBM = 16;

// About how many M-tiles of bm slots a call has: an expert one, or its share of the slots.
inline uint32_t likely_tiles(const MxArgs &a, uint32_t bm) {
    return max(min(a.E, a.n_slots), (a.n_slots + bm - 1) / bm);
}

// Into how many ways its tiles split the reduction axis; 1: 64 x 256 tiles.
template <int ACT>
int split_ways(const MxArgs &a) {
    const uint64_t tiles = likely_tiles(a, kSplitBM);
    const bool mx = act_mx(ACT), once = a.E == 1 || tiles == min(a.E, a.n_slots);
    if (tiles * ((a.N + 63) / 64) <= 256 && (!mx || a.steps >= 24)) return 4;
    if (tiles * ((a.N + 127) / 128) <= 256 && (!mx || once)) return 2;
    return 1;
}

// The workgroup's tile and its slots, from the lists or the pairs' ids; without IDS,
// slots.dst is there after the next barrier.
template <bool IDS, int BM, int BN>
__device__ __forceinline__ bool find(const MxArgs &a, MxTile &t, MxSlots<BM> &slots) {
    if constexpr (IDS) {
        __shared__ MxIds ids;
        return find_ids<BM, BN>(a, t, ids, slots);
    } else {
        if (!find_tile<BM, BN>(a, t)) return false;
        if (threadIdx.x < BM) slots.dst[threadIdx.x] = slot_output(a, t, threadIdx.x);
        return true;
    }
}

// WAYS: the wavefronts that share a block of 64 outputs.
template <int ACT, bool IDS, int WAYS>
__global__ __launch_bounds__(64 * kMxWaves) __attribute__((amdgpu_waves_per_eu(2)))
void mx_split_kernel(MxArgs a) {
    constexpr int ROWS = 4 / WAYS;  // tile rows that a wavefront adds up and stores
    __shared__ __attribute__((aligned(16))) float4_t part[kMxWaves][4][64];
    __shared__ MxSlots<kSplitBM> slots;
    MxTile t;
    if (!find<IDS, kSplitBM, 64 * kMxWaves / WAYS>(a, t, slots)) return;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t way = wave % WAYS, row0 = t.n0 + 64 * (wave / WAYS);
    float4_t acc[4][1];
    few_slots<ACT, IDS>(a, t, slots, row0, way, WAYS, acc);
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][i][lane] = acc[i][0];
    __syncthreads();
    float4_t sum[ROWS][1];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        sum[i][0] = part[wave - way][ROWS * way + i][lane];
#pragma unroll
        for (int k = 1; k < WAYS; ++k) sum[i][0] += part[wave - way + k][ROWS * way + i][lane];
    }
    store_outputs<ACT, ROWS, 1>(a, t.e, row0 + kMxRows * ROWS * way, slots.dst, sum, lane);
}

// A tile of at most 16 NC slots (NC > 1), T steps a turn: 16 KiB of slots, which
// are loaded XR turns before they go into LDS.
template <int ACT, bool IDS, int NC, int T, int AHEAD, int XR>
__device__ __forceinline__ void group_tile(const MxArgs &a, const MxTile &t, const MxSlots<kMxBM> &slots,
                                           MxShared &sh) {
    constexpr bool MX = act_mx(ACT);
    constexpr int STEP = MX ? 64 : 256;             // bytes of a slot and step
    constexpr int ROW = T * STEP, CHUNKS = ROW / 16;  // of a slot and turn
    constexpr int XL = NC * CHUNKS / 16;            // 16-byte loads of a thread and turn
    static_assert(16 * NC * ROW <= kMxBM * kMxRowBytes && (!MX || 16 * NC * T <= 256) && AHEAD % T == 0, "");
    const uint32_t tid = threadIdx.x, lane = tid & 63u, g = lane >> 4, r = lane & 15u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t row0 = t.n0 + 64 * wave, steps = a.steps;
    MxWeights<ACT, AHEAD> w;
    w.init(a, t.e, row0, lane);

    // activations: chunk tid % CHUNKS of slots tid / CHUNKS + (256 / CHUNKS) i
    constexpr int PER = 256 / CHUNKS;
    const uint32_t xbytes = MX ? a.K / 2 : 2 * a.K, chunk = tid % CHUNKS, slot0 = tid / CHUNKS;
    global_ptr xsrc[XL];
    uint32_t put[XL];
#pragma unroll
    for (int i = 0; i < XL; ++i) {
        const uint32_t slot = slot0 + PER * i;
        xsrc[i] = global_ptr(a.x) + size_t(slot_row<IDS>(a, t, slots, slot)) * xbytes + 16 * chunk;
        put[i] = slot * ROW + 16 * ((chunk & ~15u) | ((chunk & 15u) ^ swizzle<ACT>(slot)));
    }
    // 4-bit slots' scales: word tid % T of slot tid / T
    const uint8_t *const xscale =
        MX ? a.xscale + size_t(slot_row<IDS>(a, t, slots, min(tid / T, uint32_t(16 * NC - 1)))) * a.xscale_stride
           : nullptr;
    const global_ptr zeros = zero_chunk();
    uint4_t xv[XR + 1][XL];  // the last for the first turn's
    uint32_t xsv[XR + 1];
    const auto load_x = [&](int reg, uint32_t turn) {
        const bool in = turn * ROW + 16 * chunk < xbytes;
#pragma unroll
        for (int i = 0; i < XL; ++i) xv[reg][i] = load_u4(in ? xsrc[i] + turn * ROW : zeros);
        if constexpr (MX)
            xsv[reg] = *reinterpret_cast<const uint32_t *>(xscale + 4 * min(T * turn + tid % T, steps - 1u));
    };
    const auto store_x = [&](int reg, uint32_t turn, uint32_t buf) {
#pragma unroll
        for (int i = 0; i < XL; ++i) *reinterpret_cast<uint4_t *>(&sh.x[buf][put[i]]) = xv[reg][i];
        if constexpr (MX) sh.xs[buf][tid] = clip_scales(xsv[reg], T * turn + tid % T, a.K / kMxBlock);
    };

    load_x(XR, 0);
    if constexpr (XR == 2) load_x(1, 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < AHEAD - T; ++i) w.load(i, i);
    __builtin_amdgcn_sched_barrier(0);
    load_x(0, XR);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = AHEAD - T; i < AHEAD; ++i) w.load(i, i);
    __builtin_amdgcn_sched_barrier(0);
    float4_t acc[4][NC];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[i][c] = float4_t{0, 0, 0, 0};
    store_x(XR, 0, 0);
    uint4_t wv[2][4];  // 16-bit: a quarter's weights, made while the one before is multiplied
    if constexpr (!MX) w.scaled(0, 0, wv[0]);
    __syncthreads();

    const uint32_t swz = swizzle<ACT>(r);  // slots 16 c + r have the same
    // Turn s contracts buffer s % 2; turn s + 1's rows, loaded XR turns ago, go into
    // the other one, which every wavefront left before the last barrier.
    constexpr int ROUND = AHEAD < 2 * T ? 2 * T : AHEAD;  // steps of two turns at least
    for (uint32_t s0 = 0; s0 < steps; s0 += ROUND) {
#pragma unroll
        for (int u = 0; u < ROUND / T; ++u) {
            const uint32_t first = s0 + u * T, turn = first / T;
            const int buf = u & 1;
            const int reg = XR == 2 ? buf ^ 1 : 0;
            store_x(reg, turn + 1, buf ^ 1);
            load_x(reg, turn + 1 + XR);
            const uint8_t *const xt = sh.x[buf] + r * ROW;
            const uint32_t *const xs = sh.xs[buf] + r * T;
            // a quarter's (4-bit: a step's) operands are read while the one
            // before is multiplied, and no earlier: the scheduler would read
            // the whole turn's and spill
            constexpr int PARTS = MX ? T : 4 * T;
            uint4_t b[2][NC];
            uint32_t bs[2][NC];
            const auto read = [&](int q) {
                const uint32_t at = MX ? 256 * (q / 4) + 16 * ((4 * (q % 4) + g) ^ swz)
                                       : 256 * (q / 4) + 16 * ((4 * g + q % 4) ^ swz);
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    b[q & 1][c] = load_u4(xt + 16 * c * ROW + at);
                    if constexpr (MX) bs[q & 1][c] = xs[16 * c * T + q];
                }
            };
            read(0);
#pragma unroll
            for (int q = 0; q < PARTS; ++q) {
                const int i = (u * T + (MX ? q : q / 4)) % AHEAD;  // the step's registers
                if (q + 1 < PARTS) {
                    read(q + 1);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if constexpr (MX) {
#pragma unroll
                    for (int c = 0; c < NC; ++c)
                        w.multiply4(i, b[q & 1][c], bs[q & 1][c] >> (8 * g), acc[0][c], acc[1][c], acc[2][c],
                                    acc[3][c]);
                } else {
                    w.scaled((u * T + (q + 1) / 4) % AHEAD, (q + 1) % 4, wv[(q + 1) & 1]);
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int k = 0; k < 4; ++k) acc[k][c] = mfma16<ACT>(wv[q & 1][k], b[q & 1][c], acc[k][c]);
#pragma unroll
                    for (int k = 0; k < 4 * NC; ++k) {
                        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x2, 2, 0);
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                if (MX || q % 4 == 3) w.load(i, first + (MX ? q : q / 4) + AHEAD);
            }
            __syncthreads();
        }
    }
    if (row0 < a.N) store_outputs<ACT, 4, NC>(a, t.e, row0, slots.dst, acc, lane);
}

template <int ACT, bool IDS>
__global__ __launch_bounds__(64 * kMxWaves) __attribute__((amdgpu_waves_per_eu(2)))
void mx_group_kernel(MxArgs a) {
    __shared__ MxShared sh;
    __shared__ MxSlots<kMxBM> slots;
    MxTile t;
    if (!find<IDS, kMxBM, kMxBN>(a, t, slots)) return;
    constexpr bool MX = act_mx(ACT);
    if (t.n <= 16)
        few_tile<ACT, IDS>(a, t, slots);
    else if (t.n <= 32)
        group_tile<ACT, IDS, 2, MX ? 4 : 2, MX ? 8 : 4, MX ? 1 : 2>(a, t, slots, sh);
    else if (t.n <= 48)
        group_tile<ACT, IDS, 3, MX ? 4 : 1, MX ? 4 : 2, MX ? 1 : 2>(a, t, slots, sh);
    else
        group_tile<ACT, IDS, 4, MX ? 4 : 1, MX ? 4 : 2, MX ? 1 : 2>(a, t, slots, sh);
}

// ------------------------------------------------------- many 4-bit slots ---
//
// Both operands in 4 bits are bound by what feeds the matrix cores: a 64 x 256
// tile moves 69 bytes a clock and CU at their full rate.  Where there are many
// slots, a workgroup computes 256 slots by 256 outputs (34 bytes a clock), eight
// wavefronts of 64 outputs by 128 slots, two a SIMD.  Both operands go straight into
// LDS, a step of 128 columns at a time, four steps in a ring; a step's weights are
// read into registers while the step before is multiplied, the slots' three
// columns of 16 ahead.  (Four wavefronts of 128 x 128 read a third less from LDS but
// keep their sums in accumulation registers, where the MFMA took 27 clocks
// against 20.)
// Its start and end take 10 us in which the CU does nothing else, so it is used
// where every CU has a tile: 2048 x 8192 (256 tiles), 4096 columns, 45.9 us
// against 51.9 with tiles of 64; 1000 x 8192 (128 tiles) 40.8 against 28.1.  8192
// slots [8192 x 4096], four tiles a CU, take 175 us (3.1 PFLOP/s) at 2.0 GHz, the
// matrix cores busy for 37% of it; random codes hold a loop of nothing but their
// MFMA to 4.8.  Staying in a workgroup for all of a CU's tiles, with the next one's
// loads under the stores, needs more registers than there are (84 spilled: 350 us).
constexpr int kBigBM = 256, kBigBN = 256, kBigWaves = 8, kBigRing = 4;
constexpr uint32_t kBigTiles = 256;
constexpr int kBigX = 16 * kMxTileBytes;        // [256 slots][64 bytes], chunks at chunk ^ big_swizzle(slot)
constexpr int kBigWS = kBigX + kBigBM * 64;     // the outputs' words of scales: [4][64]
constexpr int kBigXS = kBigWS + kBigBN * 4;     // the slots': [2][16][8], slot 128 i + 16 k + j at [i][j][k]
constexpr int kBigStage = kBigXS + kBigBM * 4;

__device__ __forceinline__ uint32_t big_swizzle(uint32_t slot) { return (slot >> 2) & 2u; }

// All but the N loads issued last have landed, and every wavefront is here.
template <int N>
__device__ __forceinline__ void wait_stage() {
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <int ACT>
__global__ __launch_bounds__(64 * kBigWaves) __attribute__((amdgpu_waves_per_eu(2)))
void mx_big_kernel(MxArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lds[kBigRing * kBigStage];
    __shared__ uint32_t dst[kBigBM];
    MxTile t;
    if (!find_tile<kBigBM, kBigBN>(a, t)) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, g = lane >> 4, r = lane & 15u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave >> 1, wc = wave & 1u;
    if (tid < kBigBM) dst[tid] = slot_output(a, t, tid);
    const uint32_t trows = a.rows / kMxRows, steps = a.steps, base = lds_address(lds), blocks = a.K / kMxBlock;

    // this wavefront's loads of a step: two tile rows, 32 slots, and a quarter of
    // the outputs' scales (wavefronts 0 .. 3) or of the slots'
    constexpr int LOADS = 5;
    const uint4_t *wsrc[2];
    global_ptr xsrc[2];
    uint32_t chunk[2];
    const global_ptr zeros = zero_chunk();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        wsrc[i] = a.tiles + (size_t(t.e) * trows + min(t.n0 / kMxRows + 2 * wave + i, trows - 1u)) * steps * 64 + lane;
        const uint32_t slot = 32 * wave + 16 * i + lane / 4;
        chunk[i] = (lane & 3u) ^ big_swizzle(slot);
        xsrc[i] = global_ptr(a.x) + size_t(slot_row(a, t, slot)) * (a.K / 2) + 16 * chunk[i];
    }
    const uint32_t quarter = wave & 3u;
    const uint8_t *scales;
    size_t scales_step;
    if (wave < 4) {
        scales = reinterpret_cast<const uint8_t *>(
            a.tscale + (size_t(t.e) * steps * a.quads + min(t.n0 / 64 + quarter, a.quads - 1u)) * 64 + lane);
        scales_step = size_t(a.quads) * 256;
    } else {
        const uint32_t at = 64 * quarter + lane;  // a lane's eight columns together
        const uint32_t slot = (at & 128u) + 16 * (at & 7u) + (at >> 3 & 15u);
        scales = a.xscale + size_t(slot_row(a, t, slot)) * a.xscale_stride;
        scales_step = 4;
    }
    const uint32_t scales_at = (wave < 4 ? kBigWS : kBigXS) + quarter * 256;
    uint32_t issued = 0, to = base;
    const auto issue = [&]() {  // past the last step: zeros for slots, the last step again for the rest
#pragma unroll
        for (int i = 0; i < 2; ++i) to_lds16(to + (2 * wave + i) * kMxTileBytes, wsrc[i]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            to_lds16(to + kBigX + (2 * wave + i) * 1024,
                     (const void *)(4 * issued + chunk[i] < blocks ? xsrc[i] + size_t(issued) * 64 : zeros));
        to_lds4(to + scales_at, scales);
        to = to == base + (kBigRing - 1) * kBigStage ? base : to + kBigStage;
        if (++issued < steps) {
#pragma unroll
            for (int i = 0; i < 2; ++i) wsrc[i] += 64;
            scales += scales_step;
        }
    };
#pragma unroll
    for (int i = 0; i < kBigRing - 1; ++i) issue();

    float4_t acc[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 8; ++c) acc[i][c] = float4_t{0, 0, 0, 0};
    uint4_t w[2][4], x[4];
    uint32_t sw[2];
    uint4_t sx[2][2];
    const uint32_t wat = 4 * wr * kMxTileBytes + 16 * lane, swat = kBigWS + wr * 256 + 4 * lane;
    const uint32_t xat = kBigX + (128 * wc + r) * 64 + 16 * (g ^ big_swizzle(r)), sxat = kBigXS + (128 * wc + 8 * r) * 4;
    const auto read_w = [&](int buf, int i, const uint8_t *st) {
        w[buf][i] = load_u4(st + wat + i * kMxTileBytes);
        if (i == 0) sw[buf] = *reinterpret_cast<const uint32_t *>(st + swat);
        if (i >= 2) sx[buf][i - 2] = load_u4(st + sxat + 16 * (i - 2));
    };
    const auto read_x = [&](int place, int c, const uint8_t *st) {
        x[place] = load_u4(st + xat + c * 1024);
    };
    wait_stage<(kBigRing - 2) * LOADS>();
    const uint8_t *st = lds;
#pragma unroll
    for (int i = 0; i < 4; ++i) read_w(0, i, st);
#pragma unroll
    for (int c = 0; c < 3; ++c) read_x(c, c, st);
    // In the middle of step s the wavefronts meet: step s + 1 has landed once only the
    // loads of s + 2 are outstanding, and s + 3 goes where s - 1 stood, whose values
    // every wavefront has multiplied.  (s + 4 into the place of s, whose last reads
    // then have to return first: 94.1 us against 92.2, 8192 slots [8192 x 1440].)
    for (uint32_t s0 = 0; s0 < steps; s0 += 2) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint8_t *const next = st == lds + (kBigRing - 1) * kBigStage ? lds : st + kBigStage;
            const bool in = 4 * (s0 + b) + g < blocks;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                if (c == 5) {
                    wait_stage<(kBigRing - 3) * LOADS>();
                    issue();
                    read_w(b ^ 1, 0, next);
                }
                if (c >= 5) read_w(b ^ 1, c - 4, next);
                read_x((c + 3) & 3, (c + 3) & 7, c < 5 ? st : next);
                __builtin_amdgcn_sched_barrier(0);
                const uint4_t bx = x[c & 3];
                const int8v_t bv = {int(bx.x), int(bx.y), int(bx.z), int(bx.w), 0, 0, 0, 0};
                const uint32_t raw = sx[b][c / 4][c % 4] >> (8 * g);
                const int sb = int(in ? raw : 127u), sa = int(sw[b]);
                const auto av = [&](int i) {
                    const uint4_t v = w[b][i];
                    return int8v_t{int(v.x), int(v.y), int(v.z), int(v.w), 0, 0, 0, 0};
                };
                acc[0][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av(0), bv, acc[0][c], 4, 4, 0, sa, 0, sb);
                acc[1][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av(1), bv, acc[1][c], 4, 4, 1, sa, 0, sb);
                acc[2][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av(2), bv, acc[2][c], 4, 4, 2, sa, 0, sb);
                acc[3][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av(3), bv, acc[3][c], 4, 4, 3, sa, 0, sb);
                __builtin_amdgcn_sched_barrier(0);
            }
            st = next;
        }
    }
    // no load into LDS may be in flight when the workgroup's LDS is released
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    store_outputs<ACT, 4, 8>(a, t.e, t.n0 + 64 * wr, dst + 128 * wc, acc, lane);
}

inline int pair_waves(const MxArgs &a) { return a.steps > 4 * kPairSteps ? 8 : 4; }

template <int ACT>
void launch_pairs(const MxArgs &a, hipStream_t stream) {
    const dim3 grid{a.n_slots * (a.rows / kMxRows)};
    if (pair_waves(a) == 8)
        hipLaunchKernelGGL((mx_pair_kernel<ACT, 8>), grid, dim3{512}, 0, stream, a);
    else
        hipLaunchKernelGGL((mx_pair_kernel<ACT, 4>), grid, dim3{256}, 0, stream, a);
}

// The grid of tiles BM x BN, and how they go to the XCDs (find_tile).
template <int ACT, int BM, int BN>
dim3 tile_grid(MxArgs &a) {
    const uint32_t nblocks = (a.N + BN - 1) / BN;
    const bool groups = a.offs || a.ids;
    uint32_t mtiles = groups ? a.n_slots / BM + min(a.E, a.n_slots) : (a.n_slots + BM - 1) / BM;
    // An XCD takes as many M-tiles together as an expert has of them on average.  Sets
    // of 0 (plain order), 1, 2 and 4 with 2048 x 4096: 64 experts of 64 slots 102, 73, 74 and
    // 72 us (4-bit slots 82, 62, 62 and 61), of 128 153, 128, 126 and 123 (103, 99, 82 and
    // 82), of 256 251, 244, 237 and 231 (141, 179, 137 and 130).  Under 8 M-tiles sets cannot
    // fill the XCDs: 4 experts of 64 slots 15, 16, 15 and 25; under 64 larger ones leave some
    // empty: 8 experts of 64 30, 30, 31 and 32 (17, 17, 17 and 23).
    const uint64_t even = groups ? uint64_t(BM) * a.E : 1;
    a.set = likely_tiles(a, BM) < 8 ? 0 : mtiles < 64 || a.n_slots <= even ? 1 : a.n_slots <= 3 * even ? 2 : 4;
    // eight blocks in a run where they divide into such: 8 experts [8192 x 4096] of 512 slots
    // by 8, 16 and 32 219, 224 and 232 us (4-bit 120, 120 and 178), by 1 to 4 as by 8
    a.run = nblocks % 8 == 0 ? 8 : nblocks % 4 == 0 ? 4 : nblocks < 16 ? nblocks : 1;
    // one matrix, fewer bytes of slots than of weights: the weights stay, a
    // block of outputs on one XCD ([8192 x 4096], plain order and sets of 1: 512 slots 32 and
    // 33 us, 2048 109 and 115, 4-bit 1024 28 and 46; past the limit, with sets of 4, 4096
    // slots 206 and 208, 8192 410 and 413)
    if (!groups && uint64_t(a.n_slots) * (act_mx(ACT) ? 1 : 4) <= a.N) a.set = 0;
    if (a.set) mtiles = (mtiles + 8 * a.set - 1) / (8 * a.set) * (8 * a.set);
    return dim3{mtiles * nblocks};
}

template <int ACT, bool IDS>
void launch_tiles(MxArgs a, hipStream_t stream) {
    const uint32_t nblocks = (a.N + kMxBN - 1) / kMxBN;
    if constexpr (act_mx(ACT)) {
        const uint32_t tiles = (a.n_slots + kBigBM - 1) / kBigBM;
        if (!IDS && !a.offs && tiles * nblocks >= kBigTiles) {
            hipLaunchKernelGGL((mx_big_kernel<ACT>), dim3{tiles * nblocks}, dim3{64 * kBigWaves}, 0, stream, a);
            return;
        }
    }
    const int ways = split_ways<ACT>(a);
    if (ways == 4) {
        const dim3 grid = tile_grid<ACT, kSplitBM, 64>(a);
        hipLaunchKernelGGL((mx_split_kernel<ACT, IDS, 4>), grid, dim3{64 * kMxWaves}, 0, stream, a);
        return;
    }
    if (ways == 2) {
        const dim3 grid = tile_grid<ACT, kSplitBM, 128>(a);
        hipLaunchKernelGGL((mx_split_kernel<ACT, IDS, 2>), grid, dim3{64 * kMxWaves}, 0, stream, a);
        return;
    }
    const dim3 grid = tile_grid<ACT, kMxBM, kMxBN>(a);
    hipLaunchKernelGGL((mx_group_kernel<ACT, IDS>), grid, dim3{64 * kMxWaves}, 0, stream, a);
}

template <bool IDS>
int launch_groups(int act, const MxArgs &a, void *stream) {
    switch (act) {
        case ACT_F16: launch_tiles<ACT_F16, IDS>(a, as_stream(stream)); break;
        case ACT_BF16: launch_tiles<ACT_BF16, IDS>(a, as_stream(stream)); break;
        case ACT_MX_F16: launch_tiles<ACT_MX_F16, IDS>(a, as_stream(stream)); break;
        default: launch_tiles<ACT_MX_BF16, IDS>(a, as_stream(stream)); break;
    }
    return record_launch(hipGetLastError());
}

bool at16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// What both entry points refuse, and the arguments they share.
int product_args(MxArgs &a, int act, int64_t in, int64_t out, int64_t experts, const void *x, int64_t n_x_rows,
                 const uint8_t *x_scales, int64_t x_scale_stride, const void *tiles, const uint8_t *tile_scales,
                 const int32_t *row_exps, int64_t n_slots, void *y) {
    constexpr int64_t kLim = int64_t(1) << 31;
    if (act < ACT_F16 || act > ACT_MX_BF16) return IQK_ERR_ARGUMENT;
    if (in <= 0 || in % kMxBlock || in >= (1 << 24) || out <= 0 || out >= (1 << 24)) return IQK_ERR_GEOMETRY;
    if (experts <= 0 || experts > kMxMaxExperts || n_slots < 0 || n_slots >= kLim || n_x_rows < 0 || n_x_rows >= kLim)
        return IQK_ERR_ARGUMENT;
    if (n_slots == 0) return IQK_OK;
    if (n_x_rows == 0 || !x || !tiles || !tile_scales || !row_exps || !y || !at16(x) || !at16(tiles) ||
        !at16(tile_scales))
        return IQK_ERR_ARGUMENT;
    // 4-bit rows' scales are read four at a time
    if (act_mx(act) && (!x_scales || (reinterpret_cast<uintptr_t>(x_scales) & 3u) || x_scale_stride % 4 ||
                        x_scale_stride < (in + kMxStep - 1) / kMxStep * 4))
        return IQK_ERR_ARGUMENT;
    a = MxArgs{};
    a.x = static_cast<const uint8_t *>(x);
    a.xscale = x_scales;
    a.xscale_stride = x_scale_stride;
    a.tiles = static_cast<const uint4_t *>(tiles);
    a.tscale = reinterpret_cast<const uint32_t *>(tile_scales);
    a.rexp = row_exps;
    a.y = static_cast<uint16_t *>(y);
    a.K = uint32_t(in);
    a.N = uint32_t(out);
    a.rows = uint32_t((out + kMxRows - 1) / kMxRows * kMxRows);
    a.steps = uint32_t((in + kMxStep - 1) / kMxStep);
    a.quads = uint32_t((out + 63) / 64);
    a.E = uint32_t(experts);
    a.n_slots = uint32_t(n_slots);
    a.n_x_rows = uint32_t(n_x_rows);
    return IQK_OK;
}

}  // namespace iqk

extern "C" {

int iqk_mx_pairs(int act, int64_t in_features, int64_t out_features, int64_t num_experts, const void *x,
                 int64_t n_x_rows, const uint8_t *x_scales, int64_t x_scale_stride, const void *tiles,
                 const uint8_t *tile_scales, const int32_t *row_exps, const void *ids, int wide_ids,
                 int64_t pairs_per_x_row, int64_t n_pairs, void *y, void *stream) {
    using namespace iqk;
    MxArgs a;
    const int rc = product_args(a, act, in_features, out_features, num_experts, x, n_x_rows, x_scales, x_scale_stride,
                                tiles, tile_scales, row_exps, n_pairs, y);
    if (rc != IQK_OK || n_pairs == 0) return rc;
    if ((!ids && num_experts != 1) || pairs_per_x_row <= 0 || pairs_per_x_row >= (int64_t(1) << 31) ||
        (n_pairs - 1) / pairs_per_x_row >= n_x_rows || !grid_ok(n_pairs * (a.rows / kMxRows), 64 * pair_waves(a)))
        return IQK_ERR_ARGUMENT;
    a.ids = static_cast<const uint32_t *>(ids);
    a.wide = wide_ids != 0;
    a.per_row = uint32_t(pairs_per_x_row);
    switch (act) {
        case ACT_F16: launch_pairs<ACT_F16>(a, as_stream(stream)); break;
        case ACT_BF16: launch_pairs<ACT_BF16>(a, as_stream(stream)); break;
        case ACT_MX_F16: launch_pairs<ACT_MX_F16>(a, as_stream(stream)); break;
        default: launch_pairs<ACT_MX_BF16>(a, as_stream(stream)); break;
    }
    return record_launch(hipGetLastError());
}

int iqk_mx_groups(int act, int64_t in_features, int64_t out_features, int64_t num_experts, const void *x,
                  int64_t n_x_rows, const uint8_t *x_scales, int64_t x_scale_stride, const void *tiles,
                  const uint8_t *tile_scales, const int32_t *row_exps, const uint32_t *group_offsets,
                  const uint32_t *x_rows, const uint32_t *y_rows, int64_t n_slots, void *y, void *stream) {
    using namespace iqk;
    MxArgs a;
    const int rc = product_args(a, act, in_features, out_features, num_experts, x, n_x_rows, x_scales, x_scale_stride,
                                tiles, tile_scales, row_exps, n_slots, y);
    if (rc != IQK_OK || n_slots == 0) return rc;
    if (!group_offsets && num_experts != 1) return IQK_ERR_ARGUMENT;
    // with the M-tiles that make whole sets for the XCDs; larger and smaller tiles make smaller grids
    const int64_t mtiles = (group_offsets ? n_slots / kMxBM + num_experts : (n_slots + kMxBM - 1) / kMxBM) + 31;
    if (!grid_ok(mtiles * ((out_features + kMxBN - 1) / kMxBN), 64 * kMxWaves)) return IQK_ERR_ARGUMENT;
    a.offs = group_offsets;
    a.xr = x_rows;
    a.yr = y_rows;
    return launch_groups<false>(act, a, stream);
}

int iqk_mx_prefill(int act, int64_t in_features, int64_t out_features, int64_t num_experts, const void *x,
                   int64_t n_x_rows, const uint8_t *x_scales, int64_t x_scale_stride, const void *tiles,
                   const uint8_t *tile_scales, const int32_t *row_exps, const void *ids, int wide_ids,
                   int64_t n_pairs, int64_t rows_per_pair, int64_t pairs_per_x_row, uint32_t *work, void *y,
                   void *stream) {
    using namespace iqk;
    constexpr int64_t kLim = int64_t(1) << 31;
    if (n_pairs < 0 || n_pairs >= kLim || rows_per_pair <= 0 || rows_per_pair >= kLim ||
        n_pairs * rows_per_pair >= kLim)
        return IQK_ERR_ARGUMENT;
    const int64_t slots = n_pairs * rows_per_pair;
    MxArgs a;  // what the product refuses is refused before the route runs
    if (const int rc = product_args(a, act, in_features, out_features, num_experts, x, n_x_rows, x_scales,
                                    x_scale_stride, tiles, tile_scales, row_exps, slots, y);
        rc != IQK_OK || slots == 0)
        return rc;
    if (!ids || !work) return IQK_ERR_ARGUMENT;
    if (rows_per_pair == 1 && ids_pay(a)) {
        if (pairs_per_x_row <= 0 || pairs_per_x_row >= kLim || (n_pairs - 1) / pairs_per_x_row >= n_x_rows)
            return IQK_ERR_ARGUMENT;
        const int64_t mtiles = n_pairs / kSplitBM + num_experts;
        if (mtiles * ((out_features + 63) / 64) >= kLim) return IQK_ERR_ARGUMENT;
        a.ids = static_cast<const uint32_t *>(ids);
        a.wide = wide_ids != 0;
        a.per_row = uint32_t(pairs_per_x_row);
        return launch_groups<true>(act, a, stream);
    }
    uint32_t *const x_rows = work, *const y_rows = work + slots, *const offsets = work + 2 * slots;
    const int rc = wide_ids ? iqk_route_ids64(static_cast<const int64_t *>(ids), n_pairs, num_experts, rows_per_pair,
                                              pairs_per_x_row, n_x_rows, offsets, x_rows, y_rows, stream)
                            : iqk_route(static_cast<const uint32_t *>(ids), n_pairs, num_experts, rows_per_pair,
                                        pairs_per_x_row, n_x_rows, offsets, x_rows, y_rows, stream);
    if (rc != IQK_OK) return rc;
    return iqk_mx_groups(act, in_features, out_features, num_experts, x, n_x_rows, x_scales, x_scale_stride, tiles,
                         tile_scales, row_exps, offsets, x_rows, y_rows, slots, y, stream);
}

}  // extern "C"
