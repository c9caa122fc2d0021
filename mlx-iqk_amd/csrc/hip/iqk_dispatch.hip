// Token-expert pairs sorted by expert, their rows moved there and back (gfx950).
//
// Pair p = (token t, choice j) has the key ids[p], E where that is no expert (the pair
// is left out), and the slot
//   slot(p) = #{q: key_q < key_p} + #{q < p: key_q = key_p},
// a stable counting sort; the left-out pairs' slots come last, so slots are a
// permutation whose first offsets[E] have an expert.  Rows move by it:
//   dispatch       rows[slot(t, j)] = x[t], 0 where left out
//   its gradient   dx[t] = sum_j drows[slot(t, j)]
//   combine        out[t] = sum_j w[t, j] y[slot(t, j)] (+ add[t])
//   its gradients  dy[slot(t, j)] = w[t, j] dout[t],  dw[t, j] = dout[t] . y[slot(t, j)]
// with the left-out pairs skipped in sums.  Sums are f32, in the choices' order; each
// output is rounded once.  Nothing is added in memory, so results repeat bit for bit.
//
// Rows are addressed in 16-byte chunks from their start, at whatever element they start
// (loads and stores of 16 bytes need no alignment here), the last of them by elements.

#include <type_traits>

#include "iqk_host.h"
#include "iqk_mx.h"
#include "iqk_sort.h"

namespace iqk {

constexpr int64_t kSortMaxK = 64;
constexpr int kSortKeys = int(kSortMaxExperts) + 1;
constexpr int kSortWaves = 16, kSortThreads = 64 * kSortWaves;
// Pairs up to which every workgroup counts all of them itself, in one launch: 7108 pairs of 60 experts
// 6.6 us, in two launches 8.4; 12288 of 256 8.5 and 8.6; 16200 (64-bit ids) 11.3 and 10.1.
constexpr int64_t kSortOne = 12288;
// Workgroups of a sort, at most: each reads the counts of all.  us with 32, 64 and 128: 98304 pairs of 256 experts 13.5, 12.4,
// 10.8, 786432 pairs 42.0, 26.9, 21.4; 196608 pairs of 1000 experts 21.5, 19.5, 21.9.
constexpr int64_t kSortBlocks = 64;

struct SortArgs {
    const uint32_t *ids;
    uint32_t *hist;  // [blocks][E + 1], or null: every workgroup counts all pairs
    int32_t *offsets, *sorted_ids, *tokens, *slots;
    uint32_t P, E, k, share;  // share: pairs of a workgroup, in order
    uint32_t per_id;          // pairs of an id
    // instead of the lists: each key's pairs in tiles of kSortTile
    uint4_t *tiles;           // key, -, pairs (0: none), -
    uint32_t *tile_pairs;     // [tile][kSortTile]
    uint32_t n_tiles;
};

template <bool WIDE>
__device__ __forceinline__ uint32_t key_of(const SortArgs &a, uint32_t p) {
    const uint32_t i = a.per_id == 1 ? p : p / a.per_id;
    if constexpr (WIDE) {
        const uint2_t id = reinterpret_cast<const uint2_t *>(a.ids)[i];
        return id.y ? a.E : min(id.x, a.E);
    } else {
        return min(a.ids[i], a.E);
    }
}

// The lanes whose key is this lane's (bits: of the largest key), found by a ballot for each bit.
__device__ __forceinline__ uint64_t same_key(uint32_t key, bool live, int bits) {
    uint64_t same = __ballot(live);
    for (int b = 0; b < bits; ++b) {
        const bool bit = (key >> b) & 1u;
        const uint64_t m = __ballot(bit);
        same &= bit ? m : ~m;
    }
    return same;
}

// How many of a set of lanes come before this one.
__device__ __forceinline__ uint32_t rank_in(uint64_t lanes) {
    return __builtin_amdgcn_mbcnt_hi(uint32_t(lanes >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(lanes), 0));
}

// add(key, p, n) for the pairs p .. p + n of one key, which together are those from `base` to
// `end` that a wavefront takes, 64 at every STRIDE-th: a lane each, or where all 64 have one key
// (a request's rows) lane 0 for them, since LDS adds to one address one after the other.  AHEAD
// loads of ids are on their way at once.
template <bool WIDE, uint32_t STRIDE, typename F>
__device__ __forceinline__ void count_keys(const SortArgs &a, uint32_t base, uint32_t end, F &&add) {
    constexpr int AHEAD = 8;
    const uint32_t lane = threadIdx.x & 63u;
    for (; base < end; base += AHEAD * STRIDE) {
        uint32_t key[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) key[i] = key_of<WIDE>(a, min(base + i * STRIDE + lane, end - 1u));
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const uint32_t p = base + i * STRIDE;
            if (p >= end) continue;  // uniform
            if (__ballot(key[i] == uint32_t(__builtin_amdgcn_readfirstlane(key[i]))) == ~uint64_t(0)) {
                if (lane == 0) add(key[i], p, min(end - p, 64u));
            } else if (p + lane < end) {
                add(key[i], p + lane, 1u);
            }
        }
    }
}

__device__ __forceinline__ int key_bits(const SortArgs &a) { return 32 - __clz(int(a.E)); }  // of the largest key, E

// A workgroup's counts of its share of the pairs, by key.
template <bool WIDE>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortArgs a) {
    __shared__ uint32_t count[kSortKeys];
    const uint32_t K = a.E + 1;
    for (uint32_t e = threadIdx.x; e < K; e += kSortThreads) count[e] = 0;
    __syncthreads();
    const uint32_t lo = min(a.P, blockIdx.x * a.share), hi = min(a.P, lo + a.share);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    count_keys<WIDE, kSortThreads>(a, lo + 64 * wave, hi,
                                   [&](uint32_t key, uint32_t, uint32_t n) { atomicAdd(&count[key], n); });
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < K; e += kSortThreads) a.hist[size_t(blockIdx.x) * K + e] = count[e];
}

// Words of K = E + 1 keys each, of which a call uses as many as it has (to clear them is a part of its time).
template <int WAVES>
struct SortShared {
    __attribute__((aligned(16))) uint32_t words[(WAVES + 2) * kSortKeys + 3];
    uint32_t sums[WAVES];
    uint32_t used;  // tiles with pairs
    __device__ __forceinline__ uint32_t *total() { return words; }  // pairs of each key
    // those of the shares before this one, then (tiles) where the key's pairs end
    __device__ __forceinline__ uint32_t *before(uint32_t K) { return words + K; }
    // those of each wavefront's share, then its next slot
    __device__ __forceinline__ uint32_t *wave(uint32_t K, uint32_t w) { return words + (2 + w) * K; }
};

// Exclusive sums over K keys of f(key): given to g(key, sum).  A barrier before and after.
template <int WAVES, typename F, typename G>
__device__ __forceinline__ void scan_keys(SortShared<WAVES> &s, uint32_t K, F &&f, G &&g) {
    constexpr int THREADS = 64 * WAVES, PER = (kSortKeys + THREADS - 1) / THREADS;  // consecutive keys of a thread
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, first = threadIdx.x * PER;
    uint32_t v[PER], sum = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        v[i] = first + i < K ? f(first + i) : 0u;
        sum += v[i];
    }
    uint32_t incl = sum;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t up = __shfl_up(incl, off, 64);
        if (lane >= uint32_t(off)) incl += up;
    }
    if (lane == 63) s.sums[wave] = incl;
    __syncthreads();
    uint32_t at = incl - sum;
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
        if (uint32_t(w) < wave) at += s.sums[w];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (first + i < K) g(first + i, at);
        at += v[i];
    }
    __syncthreads();
}

// What bounds a sort is latency: the ids' way, three barriers, scattered stores.  Back to back 48
// pairs take 4.0 us (an empty kernel 2.2), 12288 of 256 experts 8.5, 196608 with their count 13.6, of which
// the bytes would take 0.8.
//
// place(pair, key, slot) for the pairs lo .. hi of a workgroup, whose `blocks` workgroups' shares
// follow each other.  Its wavefronts take equal parts of the share in order; a wavefront ranks 64
// pairs at a time among those of the same key, and keeps each key's next slot in LDS.  ROUNDS: the
// 64s of pairs of a wavefront whose keys stay in registers from the first load on (0: any
// number, read again where they are placed).
template <bool WIDE, int WAVES, int ROUNDS, typename F>
__device__ __forceinline__ void sort_share(const SortArgs &a, SortShared<WAVES> &s, uint32_t lo, uint32_t hi, uint32_t block,
                                           uint32_t blocks, F &&place) {
    constexpr int THREADS = 64 * WAVES;
    const uint32_t K = a.E + 1, lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t part = ((hi - lo + WAVES - 1) / WAVES + 63u) & ~63u;
    const uint32_t from = min(hi, lo + wave * part), to = min(hi, from + part);
    uint32_t mine[ROUNDS ? ROUNDS : 1];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) mine[r] = from + 64 * r + lane < to ? key_of<WIDE>(a, from + 64 * r + lane) : 0u;
    uint32_t *const totals = s.total(), *const befores = s.before(K), *const next = s.wave(K, wave);
    for (uint32_t i = 4 * threadIdx.x; i < (WAVES + 2) * K; i += 4 * THREADS)
        *reinterpret_cast<uint4_t *>(&s.words[i]) = uint4_t{0, 0, 0, 0};
    __syncthreads();
    const int bits = key_bits(a);
    if (a.hist) {
        // every 64th key a lane, every WAVES-th share's counts a wavefront, AHEAD of them at once
        constexpr uint32_t AHEAD = 4, KEYS = 5;
        for (uint32_t e0 = lane; e0 < K + lane; e0 += 64 * KEYS) {
            uint32_t total[KEYS] = {}, before[KEYS] = {};
            for (uint32_t b0 = wave; b0 < blocks; b0 += AHEAD * WAVES) {
                uint32_t n[AHEAD][KEYS];
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i)
#pragma unroll
                    for (uint32_t k = 0; k < KEYS; ++k)
                        n[i][k] = a.hist[size_t(min(b0 + i * WAVES, blocks - 1u)) * K + min(e0 + 64 * k, K - 1u)];
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i)
#pragma unroll
                    for (uint32_t k = 0; k < KEYS; ++k) {
                        if (b0 + i * WAVES < blocks) total[k] += n[i][k];
                        if (b0 + i * WAVES < block) before[k] += n[i][k];
                    }
            }
#pragma unroll
            for (uint32_t k = 0; k < KEYS; ++k) {
                if (e0 + 64 * k < K) {
                    atomicAdd(&totals[e0 + 64 * k], total[k]);
                    atomicAdd(&befores[e0 + 64 * k], before[k]);
                }
            }
        }
    } else {
        count_keys<WIDE, THREADS>(a, 64 * wave, a.P, [&](uint32_t key, uint32_t p, uint32_t n) {
            atomicAdd(&totals[key], n);
            if (p < lo) atomicAdd(&befores[key], min(n, lo - p));
        });
    }
    uint64_t same[ROUNDS ? ROUNDS : 1];
    if constexpr (ROUNDS > 0) {
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const bool live = from + 64 * r + lane < to;
            same[r] = same_key(mine[r], live, bits);
            if (live && rank_in(same[r]) == 0) atomicAdd(&next[mine[r]], uint32_t(__popcll(same[r])));
        }
    } else {
        count_keys<WIDE, 64>(a, from, to, [&](uint32_t key, uint32_t, uint32_t n) { atomicAdd(&next[key], n); });
    }
    __syncthreads();
    const bool first = block == 0;
    const auto own = [&](uint32_t e, uint32_t at) {  // the next slots of a key in this share, at: its first slot
        at += befores[e];
        uint32_t n[WAVES];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) n[w] = s.wave(K, w)[e];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            s.wave(K, w)[e] = at;
            at += n[w];
        }
    };
    if (a.tiles) {
        // a key's pairs begin at a tile: their slots are places in the tiles
        const auto whole = [](uint32_t n) { return (n + kSortTile - 1) / kSortTile * uint32_t(kSortTile); };
        scan_keys(s, K, [&](uint32_t e) { return whole(totals[e]); }, [&](uint32_t e, uint32_t at) {
            own(e, at);
            befores[e] = at + totals[e];  // where the key's pairs end
            if (e == K - 1) s.used = (at + whole(totals[e])) / uint32_t(kSortTile);
        });
        if (first)
            for (uint32_t i = s.used + threadIdx.x; i < a.n_tiles; i += THREADS) a.tiles[i] = uint4_t{0, 0, 0, 0};
    } else {
        scan_keys(s, K, [&](uint32_t e) { return totals[e]; }, [&](uint32_t e, uint32_t at) {
            if (first) a.offsets[e] = int32_t(at);
            own(e, at);
        });
    }
    volatile uint32_t *const place_of = next;
    const auto put = [&](uint32_t base, uint32_t key, uint64_t same) {
        if (base + lane < to) {
            const uint32_t rank = rank_in(same), slot = place_of[key] + rank;
            __builtin_amdgcn_wave_barrier();  // all lanes have read before the last of each key writes
            if (rank + 1 == uint32_t(__popcll(same))) place_of[key] = slot + 1;
            place(base + lane, key, slot);
        }
        __builtin_amdgcn_wave_barrier();
    };
    if constexpr (ROUNDS > 0) {
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) put(from + 64 * r, mine[r], same[r]);
    } else {
        for (uint32_t base = from; base < to; base += 64) {
            const bool live = base + lane < to;
            const uint32_t key = live ? key_of<WIDE>(a, base + lane) : 0u;
            put(base, key, same_key(key, live, bits));
        }
    }
}

template <bool WIDE, int WAVES, int ROUNDS>
__global__ __launch_bounds__(64 * WAVES) void sort_kernel(SortArgs a) {
    __shared__ SortShared<WAVES> s;
    const uint32_t lo = min(a.P, blockIdx.x * a.share), hi = min(a.P, lo + a.share);
    sort_share<WIDE, WAVES, ROUNDS>(a, s, lo, hi, blockIdx.x, gridDim.x, [&](uint32_t p, uint32_t key, uint32_t slot) {
        if (a.tiles) {
            if (slot >= a.n_tiles * uint32_t(kSortTile)) return;
            a.tile_pairs[slot] = p;
            if (slot % kSortTile == 0)
                a.tiles[slot / kSortTile] = uint4_t{key, 0, uint32_t(min(s.before(a.E + 1)[key] - slot, uint32_t(kSortTile))), 0};
        } else if (slot < a.P) {  // unless another stream changed the ids meanwhile
            a.slots[p] = int32_t(slot);
            a.sorted_ids[slot] = int32_t(key);
            a.tokens[slot] = int32_t(p / a.k);
        }
    });
}

// --------------------------------------------------------------------- rows ---

// 16 bytes at any element.
typedef uint32_t chunk_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint16_t half16_t __attribute__((aligned(2)));

template <int DT>
constexpr int kChunk = DT == MX_F32 ? 4 : 8;  // values of a chunk

template <int DT>
__device__ __forceinline__ void unpack(uint4_t w, float (&v)[kChunk<DT>]) {
    if constexpr (DT == MX_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t word = w[i];  // a bit cast of the vector's element itself reads element 0
            v[i] = __builtin_bit_cast(float, word);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == MX_F16) {
                v[2 * i] = half_bits_to_float(w[i] & 0xffffu);
                v[2 * i + 1] = half_bits_to_float(w[i] >> 16);
            } else {
                v[2 * i] = __builtin_bit_cast(float, w[i] << 16);
                v[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xffff0000u);
            }
        }
    }
}

template <int DT>
__device__ __forceinline__ uint4_t pack(const float (&v)[kChunk<DT>]) {
    uint4_t w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == MX_F32)
            w[i] = __builtin_bit_cast(uint32_t, v[i]);
        else if constexpr (DT == MX_F16)
            w[i] = float_to_half_bits(v[2 * i]) | float_to_half_bits(v[2 * i + 1]) << 16;
        else
            w[i] = bf16_bits(v[2 * i]) | bf16_bits(v[2 * i + 1]) << 16;
    }
    return w;
}

// A chunk, or (not WHOLE) its first `halves` (1 .. 7) 16-bit halves and zeros behind them.  ONCE:
// of the slots' rows, which are many and pass through once, so that they do not stay in the caches in
// place of what does not (16384 tokens, 6 rows of 8 KiB each: their sum 185 us, 161 so; rows and
// gradient of a training step 391, 345).  What reads the rows at once loses by it while the caches hold them: dispatched
// and scaled by a kernel of torch's, 2048 tokens 61.6 us, 69.1 so, 8192 tokens 221, 242; dispatched and combined
// 46.8, 50.3 and 216, 177.
template <bool WHOLE, bool ONCE = false>
__device__ __forceinline__ uint4_t load_chunk(const uint8_t *p, uint32_t halves) {
    if constexpr (WHOLE && ONCE) {
        return __builtin_nontemporal_load(reinterpret_cast<const chunk_t *>(p));
    } else if constexpr (WHOLE) {
        return *reinterpret_cast<const chunk_t *>(p);
    } else {
        uint4_t w = {0, 0, 0, 0};
#pragma unroll
        for (uint32_t i = 0; i < 7; ++i)
            if (i < halves) w[i / 2] |= uint32_t(reinterpret_cast<const half16_t *>(p)[i]) << (16 * (i & 1));
        return w;
    }
}

template <bool WHOLE, bool ONCE = false>
__device__ __forceinline__ void store_chunk(uint8_t *p, uint4_t w, uint32_t halves) {
    if constexpr (WHOLE && ONCE) {
        __builtin_nontemporal_store(chunk_t(w), reinterpret_cast<chunk_t *>(p));
    } else if constexpr (WHOLE) {
        *reinterpret_cast<chunk_t *>(p) = w;
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 7; ++i)
            if (i < halves) reinterpret_cast<half16_t *>(p)[i] = uint16_t(w[i / 2] >> (16 * (i & 1)));
    }
}

struct RowArgs {
    const uint8_t *in;        // a row for each token (dispatch, combine's gradients), or for each slot
    const uint8_t *y;         // combine's gradients: the slots' rows, or null
    const uint8_t *add;       // a row for each token, or null
    const int32_t *slots;     // [T][k], or null: the pairs'
    const int32_t *kept;      // the slots that have an expert, or null: all
    const float *weights;     // [T][k], or null: ones
    uint8_t *out;             // rows of tokens, or of slots, or null
    float *dweights;          // or null
    uint32_t T, k, P;
    uint32_t row, chunks;     // bytes and chunks of a row
    uint32_t log_width, columns;  // threads of a token (a power of two), and workgroups of a row
    uint32_t first;           // the launch's first token
};

// What one thread has of rows: a token and a chunk of them.  UNIFORM: a wavefront's threads have
// one token (at least 64 threads a token), so that its slots and weights are scalars.
template <bool UNIFORM>
struct Place {
    uint32_t t, chunk, halves;
    bool live;
    __device__ __forceinline__ explicit Place(const RowArgs &a) {
        const uint32_t width = 1u << a.log_width;
        t = a.first + (blockIdx.x / a.columns << (8 - a.log_width)) + (threadIdx.x >> a.log_width);
        if constexpr (UNIFORM) t = __builtin_amdgcn_readfirstlane(t);
        chunk = (blockIdx.x % a.columns << a.log_width) + (threadIdx.x & (width - 1u));
        live = t < a.T && chunk < a.chunks;
        halves = min(8u, (a.row - 16u * chunk) / 2u);
    }
};

__device__ __forceinline__ uint32_t slots_kept(const RowArgs &a) { return a.kept ? min(uint32_t(*a.kept), a.P) : a.P; }

constexpr int kAhead = 8;  // choices whose rows are on their way at once

template <bool WHOLE, typename PLACE>
__device__ __forceinline__ void dispatch_chunk(const RowArgs &a, const PLACE &at) {
    const uint32_t kept = slots_kept(a);
    const size_t column = size_t(at.chunk) * 16;
    const uint4_t w = load_chunk<WHOLE>(a.in + size_t(at.t) * a.row + column, at.halves);
    for (uint32_t j = 0; j < a.k; ++j) {
        const uint32_t slot = uint32_t(a.slots[size_t(at.t) * a.k + j]);
        if (slot < a.P)
            store_chunk<WHOLE, true>(a.out + size_t(slot) * a.row + column, slot < kept ? w : uint4_t{0, 0, 0, 0}, at.halves);
    }
}

// Each token's row to its slots, zeros to those left out: a row is read once and written k times.
// Bound by memory: 16384 tokens to 6 slots of 8 KiB each in 173 us, 5.4 TB/s.
template <bool UNIFORM>
__global__ __launch_bounds__(256) void dispatch_kernel(RowArgs a) {
    const Place<UNIFORM> at(a);
    if (!at.live) return;
    if (at.halves == 8)
        dispatch_chunk<true>(a, at);
    else
        dispatch_chunk<false>(a, at);
}

// Few pairs: the rows' workgroups sort for themselves, in one launch.  Each counts all pairs, ranks
// those of its own tokens, and moves its part of their rows; one of a token's workgroups writes
// its lists.  (A launch before costs 3 us of the GPU's time and 2 of the host's.)  us in one launch and in two, 256
// experts: 1020 pairs' rows of 1 KiB 6.1, 8.5, of 8 KiB 7.2, 8.9; 4092 pairs' 7.7, 9.5, of 8 KiB 17.0, 13.7.
constexpr int64_t kDispatchOne = 1024;  // pairs

template <bool WIDE>
__global__ __launch_bounds__(256) void sort_dispatch_kernel(SortArgs sort, RowArgs a) {
    __shared__ SortShared<4> s;
    __shared__ uint32_t slots[kDispatchOne];
    const uint32_t tokens = 256u >> a.log_width, block = blockIdx.x / a.columns;
    const uint32_t lo = min(sort.P, block * tokens * a.k), hi = min(sort.P, lo + tokens * a.k);
    const bool writes = blockIdx.x % a.columns == 0;
    const uint32_t t = block * tokens + (threadIdx.x >> a.log_width);
    const uint32_t chunk = (blockIdx.x % a.columns << a.log_width) + (threadIdx.x & ((1u << a.log_width) - 1u));
    const bool live = t < a.T && chunk < a.chunks;
    const uint32_t halves = min(8u, (a.row - 16u * chunk) / 2u);
    const size_t column = size_t(chunk) * 16;
    uint4_t w = {0, 0, 0, 0};
    if (live) {  // on its way while the pairs are sorted
        const uint8_t *const from = a.in + size_t(t) * a.row + column;
        w = halves == 8 ? load_chunk<true>(from, 8) : load_chunk<false>(from, halves);
    }
    sort_share<WIDE, 4, 0>(sort, s, lo, hi, writes ? block : 1u, 1u, [&](uint32_t p, uint32_t key, uint32_t slot) {
        slots[p - lo] = key < sort.E ? slot : slot | 0x80000000u;  // left out
        if (writes && slot < sort.P) {
            sort.slots[p] = int32_t(slot);
            sort.sorted_ids[slot] = int32_t(key);
            sort.tokens[slot] = int32_t(p / a.k);
        }
    });
    __syncthreads();
    if (!live) return;
    for (uint32_t j = 0; j < a.k; ++j) {
        const uint32_t slot = slots[t * a.k + j - lo], at = slot & 0x7fffffffu;
        if (at >= a.P) continue;
        uint8_t *const to = a.out + size_t(at) * a.row + column;
        const uint4_t v = slot >> 31 ? uint4_t{0, 0, 0, 0} : w;
        if (halves == 8)
            store_chunk<true>(to, v, 8);
        else
            store_chunk<false>(to, v, halves);
    }
}

template <int DT, bool WHOLE, typename PLACE>
__device__ __forceinline__ void combine_chunk(const RowArgs &a, const PLACE &at) {
    constexpr int N = kChunk<DT>;
    const uint32_t kept = slots_kept(a);
    const size_t column = size_t(at.chunk) * 16, pair = size_t(at.t) * a.k;
    float sum[N] = {};
    for (uint32_t j0 = 0; j0 < a.k; j0 += kAhead) {
        uint32_t slot[kAhead];
        uint4_t w[kAhead];
        float weight[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const uint32_t j = min(j0 + i, a.k - 1u);
            slot[i] = a.slots ? uint32_t(a.slots[pair + j]) : uint32_t(pair) + j;
            weight[i] = a.weights ? a.weights[pair + j] : 1.f;
            if (j0 + i >= a.k) slot[i] = a.P;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (slot[i] < kept) w[i] = load_chunk<WHOLE, true>(a.in + size_t(slot[i]) * a.row + column, at.halves);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (slot[i] >= kept) continue;
            float v[N];
            unpack<DT>(w[i], v);
#pragma unroll
            for (int n = 0; n < N; ++n) sum[n] = fmaf(weight[i], v[n], sum[n]);
        }
    }
    const size_t mine = size_t(at.t) * a.row + column;
    if (a.add) {
        float v[N];
        unpack<DT>(load_chunk<WHOLE>(a.add + mine, at.halves), v);
#pragma unroll
        for (int n = 0; n < N; ++n) sum[n] += v[n];
    }
    store_chunk<WHOLE>(a.out + mine, pack<DT>(sum), at.halves);
}

// A token's rows, weighted and summed.  A thread has one chunk and up to kAhead rows of it on their
// way, so that it waits once.  Bound by memory: 16384 sums of 6 rows of 8 KiB in 161 us, 5.8 TB/s;
// 2048 of them with a row added 23.3 us.
template <int DT, bool UNIFORM>
__global__ __launch_bounds__(256) void combine_kernel(RowArgs a) {
    const Place<UNIFORM> at(a);
    if (!at.live) return;
    if (at.halves == 8)
        combine_chunk<DT, true>(a, at);
    else
        combine_chunk<DT, false>(a, at);
}

// What a chunk of a token's dout adds to its choices' dots, and its chunk of their rows' gradients.
template <int DT, bool WHOLE>
__device__ __forceinline__ void grad_chunk(const RowArgs &a, uint32_t t, uint32_t chunk, uint32_t halves, uint32_t kept,
                                           const uint32_t (&slot)[kAhead], const float (&weight)[kAhead], float (&dot)[kAhead]) {
    constexpr int N = kChunk<DT>;
    const size_t column = size_t(chunk) * 16;
    const uint4_t gw = load_chunk<WHOLE>(a.in + size_t(t) * a.row + column, halves);
    uint4_t w[kAhead];
    if (a.dweights) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (slot[i] < kept) w[i] = load_chunk<WHOLE, true>(a.y + size_t(slot[i]) * a.row + column, halves);
    }
    float g[N];
    unpack<DT>(gw, g);
    if (a.out) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (slot[i] >= a.P) continue;
            float v[N];
#pragma unroll
            for (int n = 0; n < N; ++n) v[n] = weight[i] * g[n];
            store_chunk<WHOLE, true>(a.out + size_t(slot[i]) * a.row + column,
                               slot[i] < kept ? pack<DT>(v) : uint4_t{0, 0, 0, 0}, halves);
        }
    }
    if (a.dweights) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (slot[i] >= kept) continue;
            float v[N];
            unpack<DT>(w[i], v);
#pragma unroll
            for (int n = 0; n < N; ++n) dot[i] = fmaf(g[n], v[n], dot[i]);
        }
    }
}

// Both gradients of a token's sum: WAVES wavefronts a token take its row's chunks in turn, so that dout
// and y are read once for both.  One where a row has at most a chunk a lane, else four.  Bound by memory:
// 16384 tokens of 6 rows of 8 KiB in 333 us, 5.2 TB/s.
template <int DT, int WAVES>
__global__ __launch_bounds__(256) void combine_grad_kernel(RowArgs a) {
    __shared__ float part[4][kAhead];
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t t = a.first + (WAVES == 1 ? blockIdx.x * 4 + wave : blockIdx.x);
    if (WAVES == 1 && t >= a.T) return;  // whole wavefronts, and no barrier follows
    const uint32_t kept = slots_kept(a);
    const size_t pair = size_t(t) * a.k;
    for (uint32_t j0 = 0; j0 < a.k; j0 += kAhead) {
        uint32_t slot[kAhead];
        float weight[kAhead], dot[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const uint32_t j = min(j0 + i, a.k - 1u);
            slot[i] = a.slots ? uint32_t(a.slots[pair + j]) : uint32_t(pair) + j;
            weight[i] = a.weights[pair + j];
            if (j0 + i >= a.k) slot[i] = a.P;
            dot[i] = 0.f;
        }
        for (uint32_t c = (WAVES == 1 ? 0 : wave * 64) + lane; c < a.chunks; c += WAVES * 64) {
            const uint32_t halves = min(8u, (a.row - 16u * c) / 2u);
            if (halves == 8)
                grad_chunk<DT, true>(a, t, c, halves, kept, slot, weight, dot);
            else
                grad_chunk<DT, false>(a, t, c, halves, kept, slot, weight, dot);
        }
        if (!a.dweights) continue;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) dot[i] += __shfl_xor(dot[i], off, 64);
        }
        if constexpr (WAVES == 1) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                if (lane == uint32_t(i) && j0 + i < a.k) a.dweights[pair + j0 + i] = dot[i];
        } else {
            if (lane == 0) {
#pragma unroll
                for (int i = 0; i < kAhead; ++i) part[wave][i] = dot[i];
            }
            __syncthreads();
            if (threadIdx.x < kAhead && j0 + threadIdx.x < a.k) {
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) sum += part[w][threadIdx.x];
                a.dweights[pair + j0 + threadIdx.x] = sum;
            }
            __syncthreads();  // before the next choices' parts
        }
    }
}

// dy where the slots are no permutation (a caller's order): a slot's first and last pair, then a wavefront for
// each slot, which looks between them for others and adds them in the pairs' order.  16384 tokens of 6 rows of
// 8 KiB: a fifth of the pairs dropped 257 us (a permutation, by its tokens, 156); six pairs of each row far
// apart 2.2 ms, which the looking takes.
__global__ __launch_bounds__(256) void slot_span_clear_kernel(int32_t *first, int32_t *last, uint32_t n) {
    const uint32_t s = blockIdx.x * 256 + threadIdx.x;
    if (s < n) first[s] = 0x7fffffff, last[s] = -1;
}

__global__ __launch_bounds__(256) void slot_span_kernel(RowArgs a, int32_t *first, int32_t *last) {
    const uint32_t p = blockIdx.x * 256 + threadIdx.x;
    if (p >= a.P) return;
    const uint32_t slot = uint32_t(a.slots[p]);
    if (slot >= slots_kept(a)) return;
    atomicMin(&first[slot], int32_t(p));
    atomicMax(&last[slot], int32_t(p));
}

template <int DT>
__global__ __launch_bounds__(256) void combine_grad_rows_kernel(RowArgs a, const int32_t *first, const int32_t *last) {
    constexpr int N = kChunk<DT>;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t slot = a.first + blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (slot >= a.T) return;  // whole wavefronts
    const uint32_t lo = __builtin_amdgcn_readfirstlane(first[slot]);
    const int32_t hi = __builtin_amdgcn_readfirstlane(last[slot]);  // -1: no pair
    for (uint32_t c0 = 0; c0 < a.chunks; c0 += 64) {
        const uint32_t c = c0 + lane, halves = c < a.chunks ? min(8u, (a.row - 16u * c) / 2u) : 0u;
        const size_t column = size_t(c) * 16;
        uint8_t *const to = a.out + size_t(slot) * a.row + column;
        float sum[N] = {}, g[N];
        const auto load = [&](uint32_t p) __attribute__((always_inline)) {  // p: uniform
            const uint8_t *const from = a.in + size_t(p / a.k) * a.row + column;
            unpack<DT>(halves == 8 ? load_chunk<true>(from, 8) : load_chunk<false>(from, halves), g);
        };
        const auto add = [&](uint32_t p) __attribute__((always_inline)) {
            if (halves == 0) return;
            load(p);
#pragma unroll
            for (int n = 0; n < N; ++n) sum[n] = fmaf(a.weights[p], g[n], sum[n]);
        };
        if (hi >= 0 && uint32_t(hi) == lo) {  // one pair: as combine_grad_kernel has it, bit for bit
            const uint8_t *const from = a.in + size_t(lo / a.k) * a.row + column;
            const auto move = [&](auto whole) __attribute__((always_inline)) {
                constexpr bool WHOLE = decltype(whole)::value;
                unpack<DT>(load_chunk<WHOLE>(from, halves), g);
                float v[N];
#pragma unroll
                for (int n = 0; n < N; ++n) v[n] = a.weights[lo] * g[n];
                store_chunk<WHOLE>(to, pack<DT>(v), halves);
            };
            if (halves == 8)
                move(std::true_type{});
            else if (halves)
                move(std::false_type{});
            continue;
        }
        if (hi >= 0) add(lo);
        for (uint32_t base = lo + 1; hi >= 0 && base <= uint32_t(hi); base += 64) {
            const uint32_t p = base + lane;
            for (uint64_t own = __ballot(p <= uint32_t(hi) && uint32_t(a.slots[min(p, uint32_t(hi))]) == slot); own; own &= own - 1)
                add(base + uint32_t(__builtin_ctzll(own)));
        }
        if (halves == 8)
            store_chunk<true>(to, pack<DT>(sum), 8);
        else if (halves)
            store_chunk<false>(to, pack<DT>(sum), halves);
    }
}

// --------------------------------------------------------------------- host ---

SortPlan sort_plan(int64_t pairs, int64_t experts) {
    const int64_t turns = (pairs + kSortThreads - 1) / kSortThreads;
    const int64_t per = turns ? (turns + kSortBlocks - 1) / kSortBlocks : 1;
    const int64_t blocks = turns ? (turns + per - 1) / per : 1;
    return {blocks, per * kSortThreads, pairs > kSortOne ? blocks * (experts + 1) : 0};
}

namespace {

bool sort_shape_ok(int64_t tokens, int64_t k, int64_t experts) {
    return experts > 0 && experts <= kSortMaxExperts && k > 0 && k <= kSortMaxK && tokens >= 0 &&
           tokens < (int64_t(1) << 31) && tokens * k < (int64_t(1) << 31);
}

}  // namespace

int sort_launch(const SortCall &c, hipStream_t stream) {
    const SortPlan plan = sort_plan(c.pairs, c.experts);
    SortArgs a{};
    a.ids = static_cast<const uint32_t *>(c.ids);
    a.hist = plan.words ? c.work : nullptr;
    a.offsets = c.offsets;
    a.sorted_ids = c.sorted_ids;
    a.tokens = c.tokens;
    a.slots = c.slots;
    a.P = uint32_t(c.pairs);
    a.E = uint32_t(c.experts);
    a.k = uint32_t(c.per_token);
    a.per_id = uint32_t(c.per_id);
    a.share = uint32_t(plan.share);
    a.tiles = static_cast<uint4_t *>(c.tiles);
    a.tile_pairs = c.tile_pairs;
    a.n_tiles = uint32_t(c.n_tiles);
    const auto run = [&](auto kernel, int threads) {
        hipLaunchKernelGGL(kernel, dim3{uint32_t(plan.blocks)}, dim3{uint32_t(threads)}, 0, stream, a);
        return hipGetLastError();
    };
    if (plan.words) {
        const hipError_t err = c.wide ? run(sort_count_kernel<true>, kSortThreads) : run(sort_count_kernel<false>, kSortThreads);
        if (err != hipSuccess) return record_launch(err);
    }
    const auto sized = [&](auto wide) {
        constexpr bool W = decltype(wide)::value;
        // one pair a thread; in 16 wavefronts 48 pairs take 4.5 us, 4.1 so, 252 pairs 4.5, 4.2
        if (c.pairs <= 256) return run(sort_kernel<W, 4, 1>, 256);
        if (plan.share == kSortThreads) return run(sort_kernel<W, kSortWaves, 1>, kSortThreads);
        if (plan.share <= 4 * kSortThreads) return run(sort_kernel<W, kSortWaves, 4>, kSortThreads);
        return run(sort_kernel<W, kSortWaves, 0>, kSortThreads);
    };
    return record_launch(c.wide ? sized(std::true_type{}) : sized(std::false_type{}));
}

namespace {

bool rows_shape_ok(int dtype, int64_t tokens, int64_t k, int64_t cols) {
    return dtype >= MX_F32 && dtype <= MX_BF16 && k > 0 && k <= kSortMaxK && tokens >= 0 && tokens < (int64_t(1) << 31) &&
           tokens * k < (int64_t(1) << 31) && cols > 0 && cols < (int64_t(1) << 28);
}

RowArgs row_args(int dtype, int64_t tokens, int64_t k, int64_t cols) {
    RowArgs a{};
    a.T = uint32_t(tokens);
    a.k = uint32_t(k);
    a.P = uint32_t(tokens * k);
    a.row = uint32_t(cols * (dtype == MX_F32 ? 4 : 2));
    a.chunks = (a.row + 15u) / 16u;
    while (a.log_width < 8 && (1u << a.log_width) < a.chunks) ++a.log_width;
    a.columns = (a.chunks + (1u << a.log_width) - 1u) >> a.log_width;
    return a;
}

// launch(a, workgroups) for each part of the tokens that a grid of under 2^32 threads holds.
template <typename F>
void by_tokens(RowArgs a, int64_t tokens_of_group, int64_t groups_of_tokens, F &&launch) {
    const int64_t T = a.T, most = (int64_t(1) << 23) / groups_of_tokens * tokens_of_group;
    for (int64_t first = 0; first < T; first += most) {
        const int64_t n = T - first < most ? T - first : most;
        a.first = uint32_t(first);
        a.T = uint32_t(first + n);
        launch(a, uint32_t((n + tokens_of_group - 1) / tokens_of_group * groups_of_tokens));
    }
}

template <typename F>
void by_dtype(int dtype, F &&f) {
    if (dtype == MX_F32)
        f(std::integral_constant<int, MX_F32>{});
    else if (dtype == MX_F16)
        f(std::integral_constant<int, MX_F16>{});
    else
        f(std::integral_constant<int, MX_BF16>{});
}

}  // namespace
}  // namespace iqk

extern "C" {

int64_t iqk_sort_work(int64_t n_tokens, int64_t pairs_per_token, int64_t num_experts) {
    using namespace iqk;
    if (!sort_shape_ok(n_tokens, pairs_per_token, num_experts)) return -1;
    return sort_plan(n_tokens * pairs_per_token, num_experts).words;
}

int iqk_sort(const void *ids, int wide_ids, int64_t n_tokens, int64_t pairs_per_token, int64_t num_experts,
             uint32_t *work, int32_t *offsets, int32_t *sorted_ids, int32_t *tokens, int32_t *slots, void *stream) {
    using namespace iqk;
    if (!sort_shape_ok(n_tokens, pairs_per_token, num_experts)) return IQK_ERR_GEOMETRY;
    if (!offsets || (n_tokens && (!ids || !sorted_ids || !tokens || !slots))) return IQK_ERR_ARGUMENT;
    if (sort_plan(n_tokens * pairs_per_token, num_experts).words &&
        (!work || (reinterpret_cast<uintptr_t>(work) & 15u)))
        return IQK_ERR_ARGUMENT;
    SortCall c{};
    c.ids = ids;
    c.wide = wide_ids != 0;
    c.pairs = n_tokens * pairs_per_token;
    c.experts = num_experts;
    c.per_token = pairs_per_token;
    c.per_id = 1;
    c.work = work;
    c.offsets = offsets;
    c.sorted_ids = sorted_ids;
    c.tokens = tokens;
    c.slots = slots;
    return sort_launch(c, as_stream(stream));
}

int iqk_dispatch(int dtype, const void *x, const void *ids, int wide_ids, int64_t n_tokens, int64_t pairs_per_token,
                 int64_t num_experts, int64_t cols, uint32_t *work, int32_t *offsets, int32_t *sorted_ids,
                 int32_t *tokens, int32_t *slots, void *rows, void *stream) {
    using namespace iqk;
    if (!rows_shape_ok(dtype, n_tokens, pairs_per_token, cols) || !sort_shape_ok(n_tokens, pairs_per_token, num_experts))
        return IQK_ERR_GEOMETRY;
    if (n_tokens && (!x || !rows)) return IQK_ERR_ARGUMENT;
    RowArgs a = row_args(dtype, n_tokens, pairs_per_token, cols);
    const int64_t each = 256 >> a.log_width, blocks = (n_tokens + each - 1) / each * a.columns;
    if (n_tokens == 0 || n_tokens * pairs_per_token > kDispatchOne || !grid_ok(blocks, 256)) {
        if (const int rc = iqk_sort(ids, wide_ids, n_tokens, pairs_per_token, num_experts, work, offsets, sorted_ids,
                                    tokens, slots, stream);
            rc != IQK_OK || n_tokens == 0)
            return rc;
        a.in = static_cast<const uint8_t *>(x);
        a.slots = slots;
        a.kept = offsets + num_experts;
        a.out = static_cast<uint8_t *>(rows);
        by_tokens(a, 256 >> a.log_width, a.columns, [&](const RowArgs &part, uint32_t blocks) {
            if (part.log_width >= 6)
                hipLaunchKernelGGL(dispatch_kernel<true>, dim3{blocks}, dim3{256}, 0, as_stream(stream), part);
            else
                hipLaunchKernelGGL(dispatch_kernel<false>, dim3{blocks}, dim3{256}, 0, as_stream(stream), part);
        });
        return record_launch(hipGetLastError());
    }
    if (!ids || !offsets || !sorted_ids || !tokens || !slots) return IQK_ERR_ARGUMENT;
    SortArgs sort{};
    sort.ids = static_cast<const uint32_t *>(ids);
    sort.offsets = offsets;
    sort.sorted_ids = sorted_ids;
    sort.tokens = tokens;
    sort.slots = slots;
    sort.P = a.P;
    sort.E = uint32_t(num_experts);
    sort.k = a.k;
    sort.per_id = 1;
    a.in = static_cast<const uint8_t *>(x);
    a.out = static_cast<uint8_t *>(rows);
    if (wide_ids)
        hipLaunchKernelGGL(sort_dispatch_kernel<true>, dim3{uint32_t(blocks)}, dim3{256}, 0, as_stream(stream), sort, a);
    else
        hipLaunchKernelGGL(sort_dispatch_kernel<false>, dim3{uint32_t(blocks)}, dim3{256}, 0, as_stream(stream), sort, a);
    return record_launch(hipGetLastError());
}

int iqk_combine(int dtype, const void *y, const int32_t *slots, const int32_t *kept, const float *weights,
                const void *add, int64_t n_tokens, int64_t pairs_per_token, int64_t cols, void *out, void *stream) {
    using namespace iqk;
    if (!rows_shape_ok(dtype, n_tokens, pairs_per_token, cols)) return IQK_ERR_GEOMETRY;
    if (n_tokens == 0) return IQK_OK;
    if (!y || !out) return IQK_ERR_ARGUMENT;
    RowArgs a = row_args(dtype, n_tokens, pairs_per_token, cols);
    a.in = static_cast<const uint8_t *>(y);
    a.add = static_cast<const uint8_t *>(add);
    a.slots = slots;
    a.kept = kept;
    a.weights = weights;
    a.out = static_cast<uint8_t *>(out);
    by_dtype(dtype, [&](auto dt) {
        by_tokens(a, 256 >> a.log_width, a.columns, [&](const RowArgs &part, uint32_t blocks) {
            constexpr int DT = decltype(dt)::value;
            if (part.log_width >= 6)
                hipLaunchKernelGGL((combine_kernel<DT, true>), dim3{blocks}, dim3{256}, 0, as_stream(stream), part);
            else
                hipLaunchKernelGGL((combine_kernel<DT, false>), dim3{blocks}, dim3{256}, 0, as_stream(stream), part);
        });
    });
    return record_launch(hipGetLastError());
}

int iqk_combine_grad(int dtype, const void *dout, const void *y, const int32_t *slots, const int32_t *kept,
                     const float *weights, int64_t n_tokens, int64_t pairs_per_token, int64_t cols, void *dy,
                     float *dweights, void *stream) {
    using namespace iqk;
    if (!rows_shape_ok(dtype, n_tokens, pairs_per_token, cols)) return IQK_ERR_GEOMETRY;
    if (n_tokens == 0 || (!dy && !dweights)) return IQK_OK;
    if (!dout || !weights || (dweights && !y)) return IQK_ERR_ARGUMENT;
    RowArgs a = row_args(dtype, n_tokens, pairs_per_token, cols);
    a.in = static_cast<const uint8_t *>(dout);
    a.y = static_cast<const uint8_t *>(y);
    a.slots = slots;
    a.kept = kept;
    a.weights = weights;
    a.out = static_cast<uint8_t *>(dy);
    a.dweights = dweights;
    by_dtype(dtype, [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (a.chunks <= 64)
            by_tokens(a, 4, 1, [&](const RowArgs &part, uint32_t blocks) {
                hipLaunchKernelGGL((combine_grad_kernel<DT, 1>), dim3{blocks}, dim3{256}, 0, as_stream(stream), part);
            });
        else
            by_tokens(a, 1, 1, [&](const RowArgs &part, uint32_t blocks) {
                hipLaunchKernelGGL((combine_grad_kernel<DT, 4>), dim3{blocks}, dim3{256}, 0, as_stream(stream), part);
            });
    });
    return record_launch(hipGetLastError());
}

int iqk_combine_grad_rows(int dtype, const void *dout, const int32_t *slots, const int32_t *kept, const float *weights,
                          int64_t n_tokens, int64_t pairs_per_token, int64_t cols, uint32_t *work, void *dy, void *stream) {
    using namespace iqk;
    if (!rows_shape_ok(dtype, n_tokens, pairs_per_token, cols)) return IQK_ERR_GEOMETRY;
    if (n_tokens == 0) return IQK_OK;
    if (!dout || !slots || !weights || !work || !dy) return IQK_ERR_ARGUMENT;
    RowArgs a = row_args(dtype, n_tokens, pairs_per_token, cols);
    a.in = static_cast<const uint8_t *>(dout);
    a.slots = slots;
    a.kept = kept;
    a.weights = weights;
    a.out = static_cast<uint8_t *>(dy);
    int32_t *const first = reinterpret_cast<int32_t *>(work), *const last = first + a.P;
    const uint32_t blocks = (a.P + 255u) / 256u;  // fewer than 2^31 threads
    hipLaunchKernelGGL(slot_span_clear_kernel, dim3{blocks}, dim3{256}, 0, as_stream(stream), first, last, a.P);
    hipLaunchKernelGGL(slot_span_kernel, dim3{blocks}, dim3{256}, 0, as_stream(stream), a, first, last);
    a.T = a.P;  // a wavefront for each slot
    by_dtype(dtype, [&](auto dt) {
        by_tokens(a, 4, 1, [&](const RowArgs &part, uint32_t groups) {
            hipLaunchKernelGGL((combine_grad_rows_kernel<decltype(dt)::value>), dim3{groups}, dim3{256}, 0, as_stream(stream),
                               part, first, last);
        });
    });
    return record_launch(hipGetLastError());
}

}  // extern "C"
