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
    const uint32_t *tscale;
    const int32_t *rexp;
    const uint32_t *ids;     // pairs: expert ids, or null: all expert 0
    const uint32_t *offs;    // groups: first slots, or null: one group
    const uint32_t *xr;      // groups: activation rows, or null: the slots'
    const uint32_t *yr;      // groups: output rows, or null: the slots'
    uint16_t *y;
    uint32_t K, N, rows, steps, E, n_slots, n_x_rows, per_row, wide;
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

// ------------------------------------------------------------- single pairs ---
//
// A workgroup computes 16 outputs of one token-expert pair.  Its wavefronts
// split the reduction axis, four tiles of 128 columns each (all loads of the
// four issued before the first is used), and their sums meet in LDS.  Only
// column 0 of the activations' operand is real, so only its four lanes load.
constexpr int kPairSteps = 4;

template <int ACT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void mx_pair_kernel(MxArgs a) {
    __shared__ float part[WAVES][kMxRows];
    const uint32_t trows = a.rows / kMxRows;
    const uint32_t p = blockIdx.x / trows, t = blockIdx.x % trows;
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, r = lane & 15u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t e = a.ids ? expert_id(a.ids, p, a.wide) : 0u;
    if (e >= a.E) {
        const uint32_t row = kMxRows * t + threadIdx.x;
        if (threadIdx.x < kMxRows && row < a.N) a.y[size_t(p) * a.N + row] = kOutNaN<ACT>;
        return;
    }
    const uint4_t *const tile = a.tiles + (size_t(e) * trows + t) * a.steps * 64 + lane;
    const uint32_t *const ts = a.tscale + size_t(e) * a.steps * a.rows + kMxRows * t + r;
    const size_t xrow = p / a.per_row;
    const uint32_t blocks = a.K / kMxBlock;
    float4_t acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    for (uint32_t s0 = wave * kPairSteps; s0 < a.steps; s0 += WAVES * kPairSteps) {
        uint4_t w[kPairSteps];
        uint32_t sc[kPairSteps];
        constexpr int XN = act_mx(ACT) ? 1 : 4;
        uint4_t x[kPairSteps][XN];
        uint32_t xs[kPairSteps];
#pragma unroll
        for (int i = 0; i < kPairSteps; ++i) {
            const uint32_t s = min(s0 + i, a.steps - 1u);  // past the last: its weights again, against zeros
            w[i] = tile[size_t(s) * 64];
            sc[i] = ts[size_t(s) * a.rows];
        }
#pragma unroll
        for (int i = 0; i < kPairSteps; ++i) {
            const uint32_t b = 4 * (s0 + i) + g;
            xs[i] = 127u;
#pragma unroll
            for (int j = 0; j < XN; ++j) x[i][j] = uint4_t{0, 0, 0, 0};
            if (r == 0 && b < blocks) {
                if constexpr (act_mx(ACT)) {
                    x[i][0] = load_u4(a.x + xrow * (a.K / 2) + 16 * size_t(b));
                    xs[i] = a.xscale[xrow * a.xscale_stride + b];
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[i][j] = load_u4(a.x + xrow * a.K * 2 + 64 * size_t(b) + 16 * j);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kPairSteps; ++i) {
            const uint32_t byte = (sc[i] >> (8 * g)) & 255u;
            if constexpr (act_mx(ACT)) {
                acc[i & 1] = mfma4(w[i], byte, x[i][0], xs[i], acc[i & 1]);
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[j & 1] = mfma16<ACT>(eight16<act_bf16(ACT)>(w[i][j], scale_float(byte)), x[i][j], acc[j & 1]);
            }
        }
    }
    if (r == 0) *reinterpret_cast<float4_t *>(&part[wave][4 * g]) = acc[0] + acc[1];
    __syncthreads();
    const uint32_t row = kMxRows * t + threadIdx.x;
    if (threadIdx.x < kMxRows && row < a.N) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) v += part[k][threadIdx.x];
        a.y[size_t(p) * a.N + row] = uint16_t(out16<ACT>(ldexpf(v, a.rexp[size_t(e) * a.rows + row])));
    }
}

// ------------------------------------------------------------------- groups ---
//
// Slots sorted by expert; a workgroup of eight wavefronts computes 256 outputs
// of up to 128 slots of one expert.  Both operands go from memory straight
// into LDS, in three stages of which two are in flight while one is
// contracted; nothing is held in registers on the way.
//
// A stage is 128 columns (16-bit activations: 256 bytes a slot) or 256 (4-bit:
// 128 bytes a slot).  The slots' 16-byte chunks are stored at positions
// chunk ^ f(slot), so that the 16 lanes of an operand read, one chunk of 16
// slots, cover all 64 banks once; the weights' tiles are in lane order already.
//
// Wavefronts stand 4 x 2 (64 outputs, 64 slots each) in a tile of more than 64
// slots, else 8 x 1 (32 outputs, all the slots), and run only the 16-slot
// columns that the tile has.
//
// Work list: group e's M-tiles take the numbers from offs[e] / BM + e on, at
// least as many as it has: a workgroup finds its group from the offsets by
// two ballots, with no scan and no list, and those in the gaps leave.  The
// output blocks of a tile are consecutive workgroups, so with eight of them
// each XCD keeps one slice of an expert's weights in its L2 over the
// expert's tiles.
constexpr int kMxBM = 128, kMxBN = 256, kMxWaves = 8, kMxStages = 3;
constexpr uint32_t kMxMaxExperts = 4096;  // 64 x 64, the two ballots

template <int ACT>
struct Stage {
    static constexpr int STEPS = act_mx(ACT) ? 2 : 1;                // tiles of 128 columns
    static constexpr int XROW = act_mx(ACT) ? 128 : 256;             // bytes of a slot
    static constexpr int CHUNKS = XROW / 16;
    static constexpr int XROWS = 64 / CHUNKS;                        // slots of a load instruction
    static constexpr int W = 0;                                      // [16 tile rows][STEPS][1024]
    static constexpr int X = W + 16 * STEPS * kMxTileBytes;          // [128 slots][XROW]
    static constexpr int WS = X + kMxBM * XROW;                      // [STEPS][256 rows] u32
    static constexpr int XS = WS + STEPS * kMxBN * 4;                // 4-bit: [STEPS][128 slots] u32
    static constexpr int BYTES = XS + (act_mx(ACT) ? STEPS * kMxBM * 4 : 0);
    static constexpr int WLOADS = 16 * STEPS / kMxWaves;             // of a wavefront
    static __device__ __forceinline__ uint32_t swizzle(uint32_t slot) {
        return act_mx(ACT) ? (slot >> 1) & 7u : slot & 15u;
    }
};

__device__ uint4_t mx_zeros;

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

// All but the N loads issued last have landed, this wavefront's LDS reads have
// returned, and every wavefront is here.
template <int N>
__device__ __forceinline__ void wait_stage() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

struct MxTile {
    uint32_t e, m0, n, n0;  // expert, first slot, slots, first output
};

// The workgroup's tile; false (uniformly) in a gap of the list.
__device__ __forceinline__ bool find_tile(const MxArgs &a, MxTile &t) {
    const uint32_t nblocks = (a.N + kMxBN - 1) / kMxBN;
    const uint32_t u = blockIdx.x / nblocks, lane = threadIdx.x & 63u;
    t.n0 = blockIdx.x % nblocks * kMxBN;
    if (!a.offs) {
        t.e = 0;
        t.m0 = u * kMxBM;
        t.n = min(a.n_slots - t.m0, uint32_t(kMxBM));
        return true;
    }
    const uint32_t stride = (a.E + 63u) / 64u;
    uint32_t at = lane * stride;
    const bool first = at < a.E && a.offs[at < a.E ? at : 0u] / kMxBM + at <= u;
    const uint32_t base = (max(uint32_t(__popcll(__ballot(first))), 1u) - 1u) * stride;
    at = base + lane;
    const bool second = lane < stride && at < a.E && a.offs[at < a.E ? at : 0u] / kMxBM + at <= u;
    t.e = base + max(uint32_t(__popcll(__ballot(second))), 1u) - 1u;
    t.e = __builtin_amdgcn_readfirstlane(t.e);
    const uint32_t lo = a.offs[t.e], hi = min(a.offs[t.e + 1], a.n_slots);
    const uint64_t m0 = uint64_t(lo) + uint64_t(u - (lo / kMxBM + t.e)) * kMxBM;
    if (m0 >= hi) return false;
    t.m0 = uint32_t(m0);
    t.n = min(hi - t.m0, uint32_t(kMxBM));
    return true;
}

template <int ACT>
struct MxBlock {
    using S = Stage<ACT>;
    const MxArgs &a;
    const MxTile &t;
    uint8_t *lds;
    const uint32_t *dst;  // per slot: output row, bit 31 where its activations are real
    uint32_t lane, g, r, wave, stages;

    // XL activation loads a wavefront and stage, RT tile rows and NC columns
    // of 16 slots a wavefront.  EXTRA: the wavefront loads scales too.
    template <int XL, int RT, int NC, bool EXTRA>
    __device__ __forceinline__ void run() {
        const uint32_t base = uint32_t(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t *)(lds)));
        const uint32_t trows = a.rows / kMxRows, blocks = a.K / kMxBlock;
        // activation sources: instruction i of the wavefront moves XROWS slots
        const uint8_t *xsrc[XL];
        uint32_t xchunk[XL];
        const size_t xbytes = act_mx(ACT) ? a.K / 2 : 2 * size_t(a.K);
        const auto xrow_of = [&](uint32_t slot) {
            uint32_t row = 0;
            if (slot < t.n) row = a.xr ? a.xr[t.m0 + slot] : t.m0 + slot;
            return row < a.n_x_rows ? row : 0u;
        };
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            const uint32_t slot = (wave * XL + i) * S::XROWS + lane / S::CHUNKS;
            xchunk[i] = (lane % S::CHUNKS) ^ S::swizzle(slot);
            xsrc[i] = a.x + xrow_of(slot) * xbytes + 16 * xchunk[i];
        }
        // weight sources: tile rows 2 wave, 2 wave + 1
        const uint4_t *wsrc[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t tr = min(t.n0 / kMxRows + 2 * wave + i, trows - 1u);
            wsrc[i] = a.tiles + (size_t(t.e) * trows + tr) * a.steps * 64 + lane;
        }
        const uint32_t *const wscale = a.tscale + size_t(t.e) * a.steps * a.rows + min(t.n0 + 4 * lane, a.rows - 4u);
        const uint32_t xs_q = (wave - uint32_t(S::STEPS)) & 3u;  // 4-bit: of the four wavefronts with slots' scales
        const uint8_t *xscale = nullptr;
        if constexpr (act_mx(ACT) && EXTRA)
            xscale = a.xscale + size_t(xrow_of(64 * (xs_q & 1u) + lane)) * a.xscale_stride;

        const auto issue = [&](uint32_t s) {  // stage s; past the last: the last again
            const uint32_t at = base + s % kMxStages * S::BYTES;
            const uint32_t sc = min(s, stages - 1u);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int q = 0; q < S::STEPS; ++q)
                    to_lds16(at + S::W + ((2 * wave + i) * S::STEPS + q) * kMxTileBytes,
                             wsrc[i] + size_t(min(sc * S::STEPS + q, a.steps - 1u)) * 64);
#pragma unroll
            for (int i = 0; i < XL; ++i) {
                // 16-byte chunks hold 8 or 32 columns: those past K read zeros
                const uint32_t per = act_mx(ACT) ? 32u : 8u;
                const bool in = (sc * S::CHUNKS + xchunk[i]) * per < a.K;
                to_lds16(at + S::X + (wave * XL + i) * 1024,
                         in ? static_cast<const void *>(xsrc[i] + size_t(sc) * S::XROW) : &mx_zeros);
            }
            if constexpr (EXTRA) {
                if (wave < uint32_t(S::STEPS))
                    to_lds16(at + S::WS + wave * (kMxBN * 4),
                             wscale + size_t(min(sc * S::STEPS + wave, a.steps - 1u)) * a.rows);
                else
                    to_lds4(at + S::XS + ((xs_q >> 1) * kMxBM + 64 * (xs_q & 1u)) * 4,
                            xscale + 4 * size_t(min(sc * S::STEPS + (xs_q >> 1), a.steps - 1u)));
            }
        };
        constexpr int LOADS = S::WLOADS + XL + (EXTRA ? 1 : 0);
        issue(0);
        issue(1);

        const uint32_t wr = RT == 4 ? wave >> 1 : wave, wc = RT == 4 ? wave & 1u : 0u;
        float4_t acc[RT][NC];
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int c = 0; c < NC; ++c) acc[i][c] = float4_t{0, 0, 0, 0};

        for (uint32_t s = 0; s < stages; ++s) {
            wait_stage<LOADS>();  // stage s is whole; stage s - 1's place is free
            issue(s + 2);
            const uint8_t *const st = lds + s % kMxStages * S::BYTES;
            const uint8_t *const wt = st + S::W + wr * RT * S::STEPS * kMxTileBytes + 16 * lane;
            const uint8_t *const ws = st + S::WS + 4 * (wr * RT * kMxRows + r);
            const uint8_t *const xt = st + S::X + (64 * wc + r) * S::XROW;
            const uint32_t swz = S::swizzle(r);  // slots 16 c + r of the tile have the same
            if constexpr (act_mx(ACT)) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const uint32_t step = 2 * s + q;
                    if (step >= a.steps) break;  // uniform
                    uint4_t w[RT];
                    uint32_t sw[RT];
#pragma unroll
                    for (int i = 0; i < RT; ++i) {
                        w[i] = load_u4(wt + (i * 2 + q) * kMxTileBytes);
                        sw[i] = *reinterpret_cast<const uint32_t *>(ws + q * kMxBN * 4 + i * kMxRows * 4) >> (8 * g);
                    }
                    const bool in = 4 * step + g < blocks;
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        const uint4_t b = load_u4(xt + c * 16 * S::XROW + 16 * ((4 * q + g) ^ swz));
                        const uint32_t raw = *reinterpret_cast<const uint32_t *>(
                            st + S::XS + (q * kMxBM + 64 * wc + 16 * c + r) * 4) >> (8 * g);
                        const uint32_t sx = in ? raw : 127u;
#pragma unroll
                        for (int i = 0; i < RT; ++i) acc[i][c] = mfma4(w[i], sw[i], b, sx, acc[i][c]);
                    }
                }
            } else {
                uint4_t w[RT];
                float sw[RT];
#pragma unroll
                for (int i = 0; i < RT; ++i) {
                    w[i] = load_u4(wt + i * kMxTileBytes);
                    sw[i] = scale_float(
                        (*reinterpret_cast<const uint32_t *>(ws + i * kMxRows * 4) >> (8 * g)) & 255u);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint4_t wv[RT];
#pragma unroll
                    for (int i = 0; i < RT; ++i) wv[i] = eight16<act_bf16(ACT)>(w[i][j], sw[i]);
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        const uint4_t b = load_u4(xt + c * 16 * S::XROW + 16 * ((4 * g + j) ^ swz));
#pragma unroll
                        for (int i = 0; i < RT; ++i) acc[i][c] = mfma16<ACT>(wv[i], b, acc[i][c]);
                    }
                }
            }
        }
        // no load into LDS may be in flight when the workgroup's LDS is released
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

        const bool whole = a.N % 4 == 0 && (reinterpret_cast<uintptr_t>(a.y) & 7u) == 0;
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            const uint32_t row = t.n0 + (wr * RT + i) * kMxRows + 4 * g;
            if (row >= a.N) continue;
            const int32_t *const re = a.rexp + size_t(t.e) * a.rows + row;
            const int32_t ex[4] = {re[0], re[1], re[2], re[3]};  // rows is a multiple of 16
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const uint32_t slot = 64 * wc + 16 * c + r;
                const uint32_t d = dst[slot];
                if (d == 0xffffffffu) continue;
                uint32_t v[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    v[k] = d >> 31 ? out16<ACT>(ldexpf(acc[i][c][k], ex[k])) : uint32_t(kOutNaN<ACT>);
                uint16_t *const y = a.y + size_t(d & 0x7fffffffu) * a.N + row;
                if (whole) {
                    *reinterpret_cast<uint2_t *>(y) = uint2_t{v[0] | v[1] << 16, v[2] | v[3] << 16};
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (row + k < a.N) y[k] = uint16_t(v[k]);
                }
            }
        }
    }

    template <int XL, int RT, int NC>
    __device__ __forceinline__ void go() {
        // scales: 16-bit, wavefront 0; 4-bit, wavefronts 0, 1 and 2 .. 5
        if (wave < (act_mx(ACT) ? 6u : 1u))
            run<XL, RT, NC, true>();
        else
            run<XL, RT, NC, false>();
    }
};

template <int ACT>
__global__ __launch_bounds__(64 * kMxWaves) __attribute__((amdgpu_waves_per_eu(2)))
void mx_group_kernel(MxArgs a) {
    using S = Stage<ACT>;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kMxStages * S::BYTES];
    __shared__ uint32_t dst[kMxBM];
    MxTile t;
    if (!find_tile(a, t)) return;
    if (threadIdx.x < kMxBM) {
        uint32_t d = 0xffffffffu;  // not stored
        if (threadIdx.x < t.n) {
            const uint32_t slot = t.m0 + threadIdx.x;
            const uint32_t yrow = a.yr ? a.yr[slot] : slot, xrow = a.xr ? a.xr[slot] : slot;
            if (yrow < a.n_slots) d = yrow | (xrow < a.n_x_rows ? 0x80000000u : 0u);
        }
        dst[threadIdx.x] = d;
    }
    __syncthreads();
    const uint32_t lane = threadIdx.x & 63u;
    MxBlock<ACT> b{a, t, lds, dst, lane, lane >> 4, lane & 15u,
                   uint32_t(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)),
                   (a.steps + S::STEPS - 1) / S::STEPS};
    // slots of a wavefront's XL loads: 8 XL XROWS
    constexpr int X32 = act_mx(ACT) ? 1 : 1, X64 = act_mx(ACT) ? 1 : 2, X128 = act_mx(ACT) ? 2 : 4;
    if (t.n <= 16)
        b.template go<X32, 2, 1>();
    else if (t.n <= 32)
        b.template go<X32, 2, 2>();
    else if (t.n <= 48)
        b.template go<X64, 2, 3>();
    else if (t.n <= 64)
        b.template go<X64, 2, 4>();
    else
        b.template go<X128, 4, 4>();
}

template <int ACT>
void launch_pairs(const MxArgs &a, hipStream_t stream) {
    const dim3 grid{a.n_slots * (a.rows / kMxRows)};
    if (a.steps > 4 * kPairSteps)
        hipLaunchKernelGGL((mx_pair_kernel<ACT, 8>), grid, dim3{512}, 0, stream, a);
    else
        hipLaunchKernelGGL((mx_pair_kernel<ACT, 4>), grid, dim3{256}, 0, stream, a);
}

template <int ACT>
void launch_groups(const MxArgs &a, hipStream_t stream) {
    const uint32_t nblocks = (a.N + kMxBN - 1) / kMxBN;
    const uint32_t mtiles = a.offs ? a.n_slots / kMxBM + a.E : (a.n_slots + kMxBM - 1) / kMxBM;
    hipLaunchKernelGGL((mx_group_kernel<ACT>), dim3{mtiles * nblocks}, dim3{64 * kMxWaves}, 0, stream, a);
}

bool at16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// What both entry points refuse, and the arguments they share.
int product_args(MxArgs &a, int act, int64_t in, int64_t out, int64_t experts, const void *x, int64_t n_x_rows,
                 const uint8_t *x_scales, int64_t x_scale_stride, const void *tiles, const uint32_t *tile_scales,
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
    a.tscale = tile_scales;
    a.rexp = row_exps;
    a.y = static_cast<uint16_t *>(y);
    a.K = uint32_t(in);
    a.N = uint32_t(out);
    a.rows = uint32_t((out + kMxRows - 1) / kMxRows * kMxRows);
    a.steps = uint32_t((in + kMxStep - 1) / kMxStep);
    a.E = uint32_t(experts);
    a.n_slots = uint32_t(n_slots);
    a.n_x_rows = uint32_t(n_x_rows);
    return IQK_OK;
}

}  // namespace iqk

extern "C" {

int iqk_mx_pairs(int act, int64_t in_features, int64_t out_features, int64_t num_experts, const void *x,
                 int64_t n_x_rows, const uint8_t *x_scales, int64_t x_scale_stride, const void *tiles,
                 const uint32_t *tile_scales, const int32_t *row_exps, const void *ids, int wide_ids,
                 int64_t pairs_per_x_row, int64_t n_pairs, void *y, void *stream) {
    using namespace iqk;
    MxArgs a;
    const int rc = product_args(a, act, in_features, out_features, num_experts, x, n_x_rows, x_scales, x_scale_stride,
                                tiles, tile_scales, row_exps, n_pairs, y);
    if (rc != IQK_OK || n_pairs == 0) return rc;
    if ((!ids && num_experts != 1) || pairs_per_x_row <= 0 || pairs_per_x_row >= (int64_t(1) << 31) ||
        (n_pairs - 1) / pairs_per_x_row >= n_x_rows || n_pairs * (a.rows / kMxRows) >= (int64_t(1) << 31))
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
                  const uint32_t *tile_scales, const int32_t *row_exps, const uint32_t *group_offsets,
                  const uint32_t *x_rows, const uint32_t *y_rows, int64_t n_slots, void *y, void *stream) {
    using namespace iqk;
    MxArgs a;
    const int rc = product_args(a, act, in_features, out_features, num_experts, x, n_x_rows, x_scales, x_scale_stride,
                                tiles, tile_scales, row_exps, n_slots, y);
    if (rc != IQK_OK || n_slots == 0) return rc;
    if (!group_offsets && num_experts != 1) return IQK_ERR_ARGUMENT;
    const int64_t mtiles = group_offsets ? n_slots / kMxBM + num_experts : (n_slots + kMxBM - 1) / kMxBM;
    if (mtiles * ((out_features + kMxBN - 1) / kMxBN) >= (int64_t(1) << 31)) return IQK_ERR_ARGUMENT;
    a.offs = group_offsets;
    a.xr = x_rows;
    a.yr = y_rows;
    switch (act) {
        case ACT_F16: launch_groups<ACT_F16>(a, as_stream(stream)); break;
        case ACT_BF16: launch_groups<ACT_BF16>(a, as_stream(stream)); break;
        case ACT_MX_F16: launch_groups<ACT_MX_F16>(a, as_stream(stream)); break;
        default: launch_groups<ACT_MX_BF16>(a, as_stream(stream)); break;
    }
    return record_launch(hipGetLastError());
}

}  // extern "C"
