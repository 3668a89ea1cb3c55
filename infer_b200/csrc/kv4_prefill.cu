// Attention over the 4-bit cache, more than 128 query rows per kv head (prompts, chunks of them).
//
// A tile of 128 query rows (queries x heads of the group, so a group shares every key) against tiles of 128 tokens,
//     S = Q K^T     tcgen05.mma kind::f16, both operands in shared memory, accumulator in tensor memory
//     P = exp2(S - maximum), rounded to FP16, written over S in tensor memory
//     O = O + P V   the probabilities read from tensor memory
// Values enter as numbers, minimum + scale * code rounded once to FP16 (11 bits) after a power of two that brings the
// largest of the tokens so far to 2^14: a scale and a minimum per token would have to be handed to every row of
// probabilities, and what a warp reads from shared memory for all its lanes costs as much as 32 different words.  The
// rounding moves a result by at most 2^-12 of the values it averages, as the rounding of the probabilities does.
// Keys enter the same way with BF16 queries, whose own elements are eight times coarser than the rounding.  With FP16 queries
// they enter as their codes, c * 2^-24 in the low four bits of a half-precision number and 16 c * 2^-24 four bits higher, both
// exact (kv4_attention.cu); q has its elements in the order this gives, and scale and minimum are applied to the scores, two
// reads of shared memory for four of them.
// Four warps unpack, holding the next tile's words in registers while the matrix unit still reads the present one; one warp
// prepares the tokens' parameters.  Four more per tile of rows own a row per thread: scores out of tensor memory 32 at a
// time, an FMA or two on pairs, one exp2, the sum.  A warp per tile of rows issues the matrix instructions.  All operands are
// K-major with the 128-byte swizzle.  The loops are rolled where that costs a few moves: with five kinds of warps at work their code
// together has to stay in the SM's instruction cache (fully unrolled, with keys and values in separate warps, a quarter of
// the fetches missed it and the prompts below took 1.97 ms).
//
// Scores of half a tile and probabilities of the other half lie side by side: the matrix unit multiplies one while the other
// becomes probabilities (1.10 ms without, 1.06 ms with).
//
// A block of threads has two tiles of query rows (one for 256-wide heads, whose results fill tensor memory) that share the
// unpacked tokens: while one's scores become probabilities the matrix unit works for the other.  Unpacked tiles are
// double-buffered (not for 256-wide heads, where shared memory holds one).
//
// Work is dealt out as in the decode kernel: the flat list of (request, kv head, 128 query rows, tile of tokens the
// rows see) in equal contiguous shares, cut units joined by the part that arrives last.
//
// Bound: 4 * rows * tokens * head_dim operations on the matrix units; one exponential per score (16 a clock and SM) takes as
// long as the products of 128-wide heads do.  Three prompts of up to 4000 rows over up to 8100 tokens, 32 heads of 128 on 8,
// BF16: 1.02 ms, 0.71 PFLOP/s, 44 % of what a large product reaches (FP16: 1.27 ms; heads of 64: 0.87 and 1.15 ms, of 256: 3.15 and
// 3.25 ms).  Neither unit is full (34 % each): the softmax warps, two to a scheduler, need four to five cycles an instruction, one
// result waiting for the last.
#include "kv4_attention.cuh"
#include "kv4_prefill.h"
#include "tcgen05.cuh"

namespace fth {
namespace kv4 {

namespace {

constexpr int kRows = 128;          // query rows of a tile
constexpr int kTokens = 128;        // tokens of a tile
constexpr int kSite = kSiteAttentionWait;
constexpr int kNoExponent = 1000;
constexpr int kUnitCost = 4, kLongShare = 64;
constexpr float kProbabilityUp = 7.0f;  // probabilities are kept times 2^7: up to 2^15 with a lagging maximum, FP16's normal range down to 2^-21

template <int D>
struct Tiles {
    static constexpr int kQueryTiles = D == 256 ? 1 : 2;
    static constexpr int kUnitRows = kQueryTiles * kRows;
    static constexpr int kStages = D == 256 ? 1 : 2;               // unpacked tiles of tokens
    static constexpr int kSoftmax = kQueryTiles * 128;             // threads: softmax, then unpacking, then a warp for parameters
    static constexpr int kThreads = kSoftmax + 128 + 32 + kQueryTiles * 32;   // and one per tile of rows that issues products
    static constexpr int kBlocks64 = D / 64;                       // 128-byte wide pieces of a row
    static constexpr int kPieceBytes = 128 * 128;
    static constexpr int kOperandBytes = kBlocks64 * kPieceBytes;  // Q, K or V of one tile
    static constexpr int kKeys = kQueryTiles * kOperandBytes;      // stages of K, then of V
    static constexpr int kParams = kKeys + 2 * kStages * kOperandBytes;
    static constexpr int kParamStages = 4;                         // tiles whose parameters are prepared: two ahead of the operands
    static constexpr int kParamBytes = 2 * kTokens * 4;            // of one tile's keys
    static constexpr size_t kBytes = kParams + kParamStages * kParamBytes + 1024;  // 1024: alignment
    static constexpr uint32_t kTmemColumns = 512;
};
__device__ __forceinline__ void MmaShared(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void MmaTensor(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// One lane of the warp, the same at every call.
__device__ __forceinline__ bool ElectOne() {
    uint32_t chosen;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}" : "=r"(chosen));
    return chosen != 0;
}
__device__ __forceinline__ void TmemLoad32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
        "%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
          "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr)
        : "memory");
    umma::TmemLoadWait();
}
__device__ __forceinline__ void TmemStore16(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                   "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void TmemStoreWait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Two tokens' values of one element: codes in bits 0 .. 3 of both halves of x (HIGH: bits 4 .. 7), times scale, plus minimum.
// 1024 + c and 1024 + 16 c are half-precision numbers made by an OR, c = (1024 + c) - 1024 = (1024 + 16 c) / 16 - 64 exactly.
template <int HIGH>
__device__ __forceinline__ uint32_t ValuePair(uint32_t x, uint32_t scale, uint32_t minimum) {
    const uint32_t bits = (x & (HIGH ? 0x00f000f0u : 0x000f000fu)) | 0x64006400u;
    const __half2 n = *reinterpret_cast<const __half2*>(&bits);
    const __half2 c = HIGH ? __hfma2(n, __half2half2(__ushort_as_half(0x2c00)), __half2half2(__ushort_as_half(0xd400)))
                           : __hsub2(n, __half2half2(__ushort_as_half(0x6400)));
    const __half2 v = __hfma2(c, *reinterpret_cast<const __half2*>(&scale), *reinterpret_cast<const __half2*>(&minimum));
    return *reinterpret_cast<const uint32_t*>(&v);
}
// A barrier of some warps.  Not the aligned form: one thread of a warp may come to it later than the others (it has been
// at work for its group), and the compiler may place the instruction on both paths.
__device__ __forceinline__ void WarpsSync(int barrier, int threads) {
    __syncwarp();
    asm volatile("barrier.cta.sync %0, %1;" ::"r"(barrier), "r"(threads) : "memory");
}

// The rows' results so far times `factor`, by the warp that owns them.
template <int D>
__device__ __forceinline__ void ScaleResults(uint32_t o_tmem, float factor) {
    __syncwarp();
#pragma unroll 1
    for (int b = 0; b < D / 16; ++b) {
        uint32_t w[16];
        umma::TmemLoad16(o_tmem + b * 16, w);
        umma::TmemLoadWait();
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(__uint_as_float(w[i]) * factor);
        TmemStore16(o_tmem + b * 16, w);
    }
    TmemStoreWait();
}
// Token tiles of all units of one kv head of a request, by a whole warp.
template <int UNIT>
__device__ __forceinline__ int64_t RequestTiles(const AttentionParams& p, const Request& r) {
    int64_t sum = 0;
    for (int row = (threadIdx.x & 31) * UNIT; row < r.rows; row += 32 * UNIT) {
        int a, b;
        UnitTiles<kTokens>(p, r, row, UNIT, &a, &b);
        sum += b - a;
    }
    return WarpSum(sum);
}

// What a block of threads works on: a place in the list of units.  Every group of warps keeps its own in shared memory (the
// groups run ahead of each other), so that it costs no registers in the loops over tokens.
struct Place {
    int b, head, row;
    int tile_first, tile_last;  // of the unit
    int t0, steps;              // this block's tiles of it
    int low, high;              // tokens that some row of the unit sees
    int more;                   // a unit, not the end of the share
    int64_t into;               // tiles of the unit that other blocks take
    int64_t at;                 // in the flat list: of the first of this block's tiles
    Request req;
};
template <int UNIT>
__device__ __forceinline__ void Settle(const AttentionParams& p, int64_t share_end, Place& u) {
    const int64_t left = share_end - u.at, tiles = u.tile_last - u.tile_first - u.into;
    u.t0 = u.tile_first + static_cast<int>(u.into);
    u.steps = static_cast<int>(tiles < left ? tiles : left);
    int unused;
    Visible(p, u.req, QueryOf(p, u.row), &u.low, &unused);
    Visible(p, u.req, QueryOf(p, (u.row + UNIT < u.req.rows ? u.row + UNIT : u.req.rows) - 1), &unused, &u.high);
    u.more = 1;
}
// To the next unit.
template <int UNIT>
__device__ __forceinline__ void Advance(const AttentionParams& p, int64_t share_end, int cost, Place& u) {
    u.at += u.tile_last - u.tile_first - u.into + cost;
    u.into = 0;
    if (u.at >= share_end) {
        u.more = 0;
        return;
    }
    u.row += UNIT;
    if (u.row >= u.req.rows) {
        u.row = 0;
        if (++u.head == p.kv_heads) {
            u.head = 0;
            do {
                ++u.b;
                u.req = LoadRequest(p, u.b);
            } while (u.req.rows == 0);
        }
    }
    UnitTiles<kTokens>(p, u.req, u.row, UNIT, &u.tile_first, &u.tile_last);
    Settle<UNIT>(p, share_end, u);
}
// By one thread of the group.
template <int UNIT>
__device__ __forceinline__ void Advance(const AttentionParams& p, int64_t share_end, int cost, Place* place) {
    Place u = *place;
    Advance<UNIT>(p, share_end, cost, u);
    *place = u;
}

// Bounded like MbarWait, in little code.  The lanes of a warp may leave it one after another: a __syncwarp comes before the
// next tensor-memory instruction, which the whole warp executes together.
__device__ __forceinline__ bool WaitFor(uint64_t* bar, uint32_t parity, int* status, int detail) {
    uint64_t since = 0;
#pragma unroll 1
    for (int i = 1; !MbarTryWait(bar, parity); ++i) {
        if ((i & 255) != 0) continue;
        const uint64_t now = GlobalTimerNs();
        if (since == 0) since = now;
        else if (now - since > kWaitBudgetNs) {
            ReportTimeout(status, kSite, detail);
            return false;
        }
    }
    return true;
}
// Sixteen bytes of codes, not kept in L1.  Not by the read-only path: the kernel in front may still store the step's tokens when
// this one has started (it waits for it before the first of these loads).
__device__ __forceinline__ uint4 LoadCodes(const uint8_t* from) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(from) : "memory");
    return v;
}
// Whether some row sees one of the sixteen tokens around `token`.
__device__ __forceinline__ bool SomeSeen(const Place& u, int token) { return (token & ~15) < u.high && (token & ~15) + 16 > u.low; }
// What the table names as the block of `token` if any of its sixteen neighbours is seen by a row, else -1.
__device__ __forceinline__ int BlockOf(const AttentionParams& p, const Place& u, int token) {
    return SomeSeen(u, token) ? p.table[static_cast<int64_t>(u.b) * p.max_blocks + (token >> p.cache.block_shift)] : -1;
}
__device__ __forceinline__ bool IsBlock(const AttentionParams& p, int id) { return id >= 0 && id < p.cache.blocks; }
__device__ __forceinline__ int64_t TokenIndex(const AttentionParams& p, int block, int head, int token) {
    return HeadBase(p.cache, block, head) + (token & ((1 << p.cache.block_shift) - 1));
}

template <int D, int DTYPE>
__global__ void __launch_bounds__(Tiles<D>::kThreads, 1) PrefillKernel(const __grid_constant__ AttentionParams p) {
    using T = Tiles<D>;
    constexpr int kThreads = T::kThreads, G = T::kQueryTiles, S = T::kStages, P = T::kParamStages, kUnit = T::kUnitRows;
    constexpr bool kKeyCodes = DTYPE == FTH_B200_FP16;   // keys as codes, else as numbers
    extern __shared__ uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    __shared__ uint32_t tmem_slot;
    __shared__ __align__(8) uint64_t q_full[G], s_full[G][2], p_full[G][2], o_done[G][2], k_full[S], k_empty[S], v_full[S], v_empty[S], params_full[P], tile_done[P], back_full;
    __shared__ int64_t unit_work[kThreads];   // of a request, per kv head: tiles of its units
    __shared__ int unit_count_of[kThreads];   // and units
    __shared__ int64_t work_total, units_total;
    constexpr int kUnpackPlace = G, kParamPlace = G + 1, kIssuePlace = G + 2, kPlaces = 2 * G + 2;
    __shared__ Place places[kPlaces];      // one per tile of rows (softmax), unpacking, parameters, one per tile of rows (products)
    // of a tile
    __shared__ uint32_t present[P][4];     // a bit per token that some row may see
    __shared__ uint32_t spoiled[P][4];     // a bit per token whose parameters are no numbers
    __shared__ float4 about[P];            // power of two on the values; 1 / that on the keys; 1: all present, none spoiled
    __shared__ int64_t place_of[P][kTokens / 16];   // offset of the codes of sixteen tokens, -1: no block
    __shared__ __align__(16) __half value_scale[P][kTokens], value_min[P][kTokens], key_scale[P][kTokens], key_min[P][kTokens];
    __shared__ float q_big[2][4 * G], unit_back;
    __shared__ int join_last[G];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kUnpackWarp = T::kSoftmax / 32, kParamWarp = kUnpackWarp + 4, kIssueWarp = kParamWarp + 1;
    if (threadIdx.x == 0) {
        for (int g = 0; g < G; ++g) {
            MbarInit(&q_full[g], 128);
            for (int h = 0; h < 2; ++h) {
                MbarInit(&s_full[g][h], 1);
                MbarInit(&p_full[g][h], 128);
                MbarInit(&o_done[g][h], 1);
            }
        }
        for (int s = 0; s < S; ++s) {
            MbarInit(&k_full[s], 128);
            MbarInit(&k_empty[s], G);
            MbarInit(&v_full[s], 128);
            MbarInit(&v_empty[s], G);
        }
        for (int i = 0; i < P; ++i) {
            MbarInit(&params_full[i], 32);
            MbarInit(&tile_done[i], G);
        }
        MbarInit(&back_full, 1);
        FenceBarrierInit();
    }
    // tensor memory is taken before the next kernel of the stream may start on this SM and take it
    if (warp == kIssueWarp) umma::TmemAlloc(&tmem_slot, T::kTmemColumns);
    umma::FenceBeforeThreadSync();
    __syncthreads();
    umma::FenceAfterThreadSync();
    const uint32_t tmem = tmem_slot;
    WaitForPrevious();

    // ---- this block's share ----------------------------------------------------------------------------------------------
    // A warp takes a request at a time; thread 0 adds.  Few requests have many rows.
    if (threadIdx.x == 0) work_total = units_total = 0;
    __syncthreads();
    const auto count_tiles = [&](int base, int count) {
        for (int i = warp; i < count; i += kThreads / 32) {
            const Request r = LoadRequest(p, base + i);
            const int64_t sum = RequestTiles<kUnit>(p, r);
            if (lane == 0) {
                unit_work[i] = sum;
                unit_count_of[i] = (r.rows + kUnit - 1) / kUnit;
            }
        }
    };
    for (int base = 0; base < p.requests; base += kThreads) {
        const int count = p.requests - base < kThreads ? p.requests - base : kThreads;
        if (p.few_units) {
            if (threadIdx.x < count) {
                const Request r = LoadRequest(p, base + threadIdx.x);
                int64_t sum = 0;
                for (int row = 0; row < r.rows; row += kUnit) {
                    int a, b;
                    UnitTiles<kTokens>(p, r, row, kUnit, &a, &b);
                    sum += b - a;
                }
                unit_work[threadIdx.x] = sum;
                unit_count_of[threadIdx.x] = (r.rows + kUnit - 1) / kUnit;
            }
        } else {
            count_tiles(base, count);
        }
        __syncthreads();
        if (warp == 0) {
            int64_t sum = 0, units = 0;
            for (int i = lane; i < count; i += 32) {
                sum += unit_work[i];
                units += unit_count_of[i];
            }
            sum = WarpSum(sum);
            units = WarpSum(units);
            if (lane == 0) {
                work_total += sum * p.kv_heads;
                units_total += units * p.kv_heads;
            }
        }
        __syncthreads();
    }
    // Starting and ending a unit takes about as long as kUnitCost tiles (25 thousand cycles): with long shares it is counted as
    // such, behind the unit's tiles, so that shares of many short units are not the last to end (three prompts of 4000 rows over
    // 8100 tokens: 1059 us without, 1008, 998 and 1006 us with 2, 4 and 8).  Short shares are rather cut evenly.
    const int cost = work_total >= kLongShare * gridDim.x ? kUnitCost : 0;
    const int64_t work = work_total + cost * units_total;
    const int64_t per = work > 0 ? Divide(work + gridDim.x - 1, gridDim.x) : 1;
    const int64_t share_begin = blockIdx.x * per;
    const int64_t share_end = share_begin + per < work ? share_begin + per : work;
    bool busy = share_begin < share_end;
    if (busy) {
        // the request, then the head, then the rows that share_begin falls into
        int64_t passed = 0;
        for (int base = 0; base < p.requests; base += kThreads) {
            const int count = p.requests - base < kThreads ? p.requests - base : kThreads;
            if (p.requests > kThreads) {
                __syncthreads();
                count_tiles(base, count);
                __syncthreads();
            }
            bool found = false;
            if (warp == 0) {
                for (int i = 0; i < count && !found; i += 32) {
                    int64_t mine = i + lane < count ? (unit_work[i + lane] + cost * unit_count_of[i + lane]) * p.kv_heads : 0, sum = mine;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int64_t n = __shfl_up_sync(0xffffffffu, sum, o);
                        if (lane >= o) sum += n;
                    }
                    const int64_t all = __shfl_sync(0xffffffffu, sum, 31);
                    const int64_t before = passed + sum - mine;
                    const uint32_t who = __ballot_sync(0xffffffffu, share_begin >= before && share_begin < before + mine);
                    if (who != 0) {
                        found = true;
                        const int src = __ffs(who) - 1;
                        int64_t off = share_begin - __shfl_sync(0xffffffffu, before, src);
                        const int64_t per_head = unit_work[i + src] + cost * unit_count_of[i + src];
                        Place u;
                        u.b = base + i + src;
                        u.req = LoadRequest(p, u.b);
                        u.head = static_cast<int>(Divide(off, per_head));
                        off -= u.head * per_head;
                        // rows, 32 units at a time
                        for (int row = 0;; row += 32 * kUnit) {
                            const int my_row = row + lane * kUnit;
                            int a = 0, c = 0;
                            if (my_row < u.req.rows) UnitTiles<kTokens>(p, u.req, my_row, kUnit, &a, &c);
                            const int64_t own = c - a + (c > a ? cost : 0);
                            int64_t upto = own;
#pragma unroll
                            for (int o = 1; o < 32; o <<= 1) {
                                const int64_t n = __shfl_up_sync(0xffffffffu, upto, o);
                                if (lane >= o) upto += n;
                            }
                            const uint32_t here = __ballot_sync(0xffffffffu, off < upto);
                            if (here != 0) {
                                if (lane == __ffs(here) - 1) {
                                    u.row = my_row;
                                    u.tile_first = a;
                                    u.tile_last = c;
                                    u.into = off - (upto - own);
                                    u.at = share_begin;
                                    u.more = 1;
                                    if (u.into < c - a) Settle<kUnit>(p, share_end, u);
                                    else Advance<kUnit>(p, share_end, cost, u);   // the share begins behind its last tile
                                    for (int i = 0; i < kPlaces; ++i) places[i] = u;
                                }
                                break;
                            }
                            off -= __shfl_sync(0xffffffffu, upto, 31);
                        }
                    }
                    passed += all;
                }
            }
            if (__syncthreads_or(found ? 1 : 0)) break;
        }
        __syncthreads();
        busy = places[0].more != 0;
        __syncthreads();   // before a group moves on
    }

    float* const params = reinterpret_cast<float*>(smem + T::kParams);
    bool failed = false;
    const auto wait = [&](uint64_t* bar, uint32_t parity, int detail) {
        if (!failed && !WaitFor(bar, parity, p.status, 16 + detail)) failed = true;
    };

    if (warp < kUnpackWarp) {
        if (busy) {
        // ================================================ softmax ====================================================
        const int g = warp >> 2;                   // tile of rows
        const int r = threadIdx.x & 127;           // row of the tile, lane of tensor memory
        const uint32_t s_tmem = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + g * 256, o_tmem = s_tmem + 128;
        uint8_t* const q_smem = smem + g * T::kOperandBytes;
        const Place& u = places[g];
        uint32_t tile_count = 0, unit_count = 0, used = 0;
        for (;;) {
            // ---- the unit's queries, as operands: copied as they are, measured by the thread that owns the row, rewritten in place
            const int tile_row = u.row + g * kRows, row = tile_row + r;
            const bool active = g == 0 || u.req.rows - u.row > kRows;
            const bool valid = row < u.req.rows;
            const int query = valid ? QueryOf(p, row) : 0;
            const auto piece = [&](int of, int w) { return reinterpret_cast<uint4*>(q_smem + (w >> 3) * T::kPieceBytes + of * 128 + (((w & 7) ^ (of & 7)) << 4)); };
            const int64_t own = (u.req.first_row + static_cast<int64_t>(query)) * p.ldq + (static_cast<int64_t>(u.head) * p.group + (row - query * p.group)) * D;
            if (active) {   // the 32 rows of a warp, neighbouring lanes neighbouring pieces of a row
                constexpr int kLanes = D / 8 < 32 ? D / 8 : 32, kRowsAtOnce = 32 / kLanes;
                const int w = lane % kLanes;
                const auto copy = [&](int i, auto fetch) {
                    const int lane_of = i * kRowsAtOnce + lane / kLanes, of = (warp & 3) * 32 + lane_of;
                    const int64_t from = __shfl_sync(0xffffffffu, own, lane_of);
                    *piece(of, w) = tile_row + of < u.req.rows ? fetch(static_cast<const uint16_t*>(p.q) + from + w * 8) : make_uint4(0, 0, 0, 0);
                };
                if (p.q_vec) {
#pragma unroll 8
                    for (int i = 0; i < 32 / kRowsAtOnce; ++i) copy(i, [](const uint16_t* from) { return *reinterpret_cast<const uint4*>(from); });
                } else {
#pragma unroll 1
                    for (int i = 0; i < 32 / kRowsAtOnce; ++i) copy(i, [](const uint16_t* from) { return LoadUnaligned8(from); });
                }
                __syncwarp();
            }
            float big = 0.0f, qsum = 0.0f;
#pragma unroll 2
            for (int w = 0; active && w < D / 8; ++w) {
                const uint4 x = *piece(r, w);
                const uint32_t raw[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 v = HalfPair<DTYPE>(raw[i]);
                    big = Max3(big, FiniteAbs(v.x), FiniteAbs(v.y));
                    if constexpr (kKeyCodes) qsum += v.x + v.y;
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
            float* const bigs = q_big[unit_count & 1u];   // one of the groups may be a unit ahead
            if (lane == 0) bigs[warp] = big;
            // one power of two for the unit where it goes into the keys' parameters, else one for the tile of rows
            WarpsSync(kKeyCodes ? 3 : 1 + g, kKeyCodes ? T::kSoftmax : 128);
#pragma unroll
            for (int w = 0; w < (kKeyCodes ? 4 * G : 4); ++w) big = fmaxf(big, bigs[kKeyCodes ? w : 4 * g + w]);
            const int e = QueryExponent(big);
            const float up = PowerOfTwo(e), back = p.scale_log2 * PowerOfTwo((kKeyCodes ? 24 : 0) - e);
            if (kKeyCodes && threadIdx.x == 0) {
                unit_back = back;
                MbarArrive(&back_full);
            }
            qsum *= p.scale_log2;
#pragma unroll 2
            for (int w = 0; active && w < D / 8; ++w) {
                const uint4 x = *piece(r, w);
                const uint32_t raw[4] = {x.x, x.y, x.z, x.w};
                uint32_t f[4];
                QueryOperands<DTYPE>(raw, up, kKeyCodes ? 0.0625f : 1.0f, f);
                *piece(r, w) = make_uint4(f[0], f[1], f[2], f[3]);
            }
            FenceProxyAsync();
            if (active) MbarArrive(&q_full[g]);
            int low = 0, high = 0;
            if (valid) Visible(p, u.req, query, &low, &high);

            // ---- tiles.  Scores are kept relative to ref = maximum - 7.
            float ref = 0.0f, limit = kNotStarted, up_now = 1.0f;
            float2 mass = make_float2(0.0f, 0.0f);
            const int steps = u.steps, first_token = u.t0 * kTokens;
            if (!active) tile_count += steps;   // no rows
            for (int step = 0; active && step < steps; ++step, ++tile_count, ++used) {
                const uint32_t par = tile_count % P;
                // The scores' barrier counts this tile of rows' own tiles.  The parameters' counts all tiles, of which it may have passed
                // over many (units in which it has no rows): only with the scores there is it known to be at this one.
                wait(&s_full[g][0], used & 1u, 6);
                wait(&params_full[par], (tile_count / P) & 1u, 10);
                const float4 tile = about[par];
                const int token0 = first_token + step * kTokens;
                const bool inside = __all_sync(0xffffffffu, tile.z != 0.0f && (!valid || (token0 >= low && token0 + kTokens <= high)));
                const float tile_up = tile.x;
                if (tile_up != up_now) {   // the same for every row
                    if (step > 0) {
                        wait(&o_done[g][1], (used - 1) & 1u, 7);
                        __syncwarp();
                        umma::FenceAfterThreadSync();
                        ScaleResults<D>(o_tmem, tile_up / up_now);
                    }
                    up_now = tile_up;
                }
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    const int h = c >> 1;
                    const uint32_t p_tmem = s_tmem + h * 64;   // the half's probabilities, over its scores
                    uint32_t s[32];
                    if ((c & 1) == 0) {
                        if (h != 0) wait(&s_full[g][h], used & 1u, 6);
                        __syncwarp();
                        umma::FenceAfterThreadSync();
                    }
                    __syncwarp();
                    TmemLoad32(s_tmem + c * 32, s);
                    float2 z[16];
                    const float2 rr = make_float2(-ref, -ref);
                    if constexpr (kKeyCodes) {
                        const float4* ks = reinterpret_cast<const float4*>(params + par * (T::kParamBytes / 4) + c * 32);
                        const float4* km = ks + kTokens / 4;
                        const float2 qq = make_float2(qsum, qsum);
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float4 s4 = ks[i], m4 = km[i];
                            z[2 * i] = Fma2(make_float2(s4.x, s4.y), make_float2(__uint_as_float(s[4 * i]), __uint_as_float(s[4 * i + 1])), Fma2(make_float2(m4.x, m4.y), qq, rr));
                            z[2 * i + 1] = Fma2(make_float2(s4.z, s4.w), make_float2(__uint_as_float(s[4 * i + 2]), __uint_as_float(s[4 * i + 3])), Fma2(make_float2(m4.z, m4.w), qq, rr));
                        }
                    } else {
                        const float2 bb = make_float2(back * tile.y, back * tile.y);
#pragma unroll
                        for (int i = 0; i < 16; ++i) z[i] = Fma2(make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), bb, rr);
                    }
                    if (__builtin_expect(!inside, 0)) {
                        // bits of the tokens of this chunk that the row sees
                        const int from = low - token0 - c * 32, to = high - token0 - c * 32;
                        uint32_t seen = present[par][c];
                        if (from > 0) seen = from < 32 ? seen & (0xffffffffu << from) : 0u;
                        if (to < 32) seen = to > 0 ? seen & (0xffffffffu >> (32 - to)) : 0u;
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            if (((seen >> (2 * i)) & 1u) == 0) z[i].x = -INFINITY;
                            if (((seen >> (2 * i + 1)) & 1u) == 0) z[i].y = -INFINITY;
                        }
                        const uint32_t bad = spoiled[par][c] & seen;
                        if (bad != 0) z[0].x = NAN;   // the row is NaN, whichever token makes it
                    }
                    float bests[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < 16; ++i) bests[i & 3] = Max3(bests[i & 3], z[i].x, z[i].y);
                    const float best = Max3(fmaxf(bests[0], bests[1]), bests[2], bests[3]);
                    if (__builtin_expect(__any_sync(0xffffffffu, best > limit), 0)) {
                        // move the maximum: scores of this chunk, the probabilities of the half's first one, sums and results
                        const bool first = limit == kNotStarted;
                        const float over = first ? best : best - kProbabilityUp;   // above the old maximum
                        float shift = 0.0f;
                        if (first ? over > kNotStarted : over > 0.0f) {
                            // a whole number of doublings keeps earlier probabilities' bits
                            shift = first ? over - kProbabilityUp : ceilf(over);
                            limit = kLazy + kProbabilityUp;
                        }
                        const float alpha = first ? 0.0f : Exp2(-shift);
                        ref += shift;
                        mass = Mul2(mass, make_float2(alpha, alpha));
#pragma unroll
                        for (int i = 0; i < 16; ++i) z[i] = make_float2(z[i].x - shift, z[i].y - shift);
                        TmemStoreWait();
                        if ((c & 1) != 0) {
                            uint32_t w[16];
                            umma::TmemLoad16(p_tmem, w);
                            umma::TmemLoadWait();
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float2 v = HalfPair<FTH_B200_FP16>(w[i]);
                                w[i] = PackHalf(v.x * alpha, v.y * alpha);
                            }
                            TmemStore16(p_tmem, w);
                        }
                        if (step > 0 || h > 0) {   // after the products of the half before
                            wait(&o_done[g][h ^ 1], (h == 0 ? used - 1 : used) & 1u, 7);
                            __syncwarp();
                            umma::FenceAfterThreadSync();
                            ScaleResults<D>(o_tmem, alpha);
                        }
                        TmemStoreWait();
                    }
                    uint32_t packed[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 prob = make_float2(Exp2(z[i].x), Exp2(z[i].y));
                        mass = Add2(mass, prob);
                        packed[i] = PackHalf(prob.x, prob.y);
                    }
                    __syncwarp();
                    TmemStore16(p_tmem + (c & 1) * 16, packed);
                    if ((c & 1) != 0) {
                        TmemStoreWait();
                        umma::FenceBeforeThreadSync();
                        MbarArrive(&p_full[g][h]);
                    }
                }
            }

            // ---- the unit's results
            if (active) wait(&o_done[g][1], (used - 1) & 1u, 7);
            __syncwarp();
            umma::FenceAfterThreadSync();
            const float total = mass.x + mass.y;
            const int64_t unit_begin = u.at - u.into, unit_end = unit_begin + (u.tile_last - u.tile_first);
            const int64_t part_first = unit_begin >= share_begin ? blockIdx.x : Divide(unit_begin, per);
            const int64_t part_last = unit_end <= share_end ? blockIdx.x : Divide(unit_end - 1, per);
            const bool whole = part_first == part_last;
            const int64_t slot_floats = static_cast<int64_t>(kUnit) * kRow<D>;
            float* const tile_partials = p.partials + g * kRows * kRow<D>;
            float* partial = tile_partials + (static_cast<int64_t>(blockIdx.x) * 2 + (blockIdx.x == part_first ? 1 : 0)) * slot_floats + r * kRow<D>;
            const float best = limit == kNotStarted ? kNoMax : ref;
            const int q_head = u.head * p.group + row - query * p.group;
            const int64_t q_row = u.req.first_row + static_cast<int64_t>(query);
            uint16_t* const out = static_cast<uint16_t*>(p.out) + q_row * p.ldo + static_cast<int64_t>(q_head) * D;
            const float scale = total == 0.0f ? 0.0f : __fdiv_rn(1.0f, total);
            const float down = 1.0f / up_now;   // a power of two
#pragma unroll 1
            for (int c = 0; active && c < D / 16; ++c) {
                uint32_t w[16];
                __syncwarp();
                umma::TmemLoad16(o_tmem + c * 16, w);
                umma::TmemLoadWait();
                if (!valid || failed) continue;   // a wait that gave up is in the status word; nothing is stored then
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(w[i]) * down;
                if (whole) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) v[i] = total == 0.0f ? 0.0f : v[i] * scale;
                    if (p.out_vec) {
#pragma unroll
                        for (int i = 0; i < 16; i += 8)
                            *reinterpret_cast<uint4*>(out + c * 16 + i) = make_uint4(PackTo<DTYPE>(v[i], v[i + 1]), PackTo<DTYPE>(v[i + 2], v[i + 3]),
                                                                                     PackTo<DTYPE>(v[i + 4], v[i + 5]), PackTo<DTYPE>(v[i + 6], v[i + 7]));
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            const uint32_t two = PackTo<DTYPE>(v[i], v[i + 1]);
                            out[c * 16 + i] = static_cast<uint16_t>(two);
                            out[c * 16 + i + 1] = static_cast<uint16_t>(two >> 16);
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(partial + c * 16 + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                }
            }
            if (active && whole && valid && !failed && p.lse != nullptr)
                p.lse[q_row * p.kv_heads * p.group + q_head] = total == 0.0f ? -INFINITY : (best + log2f(total)) * 0.6931471805599453f;
            if (active && !whole) {
                if (valid) *reinterpret_cast<float4*>(partial + D) = make_float4(best, 0.0f, total, total);
                const int parts = static_cast<int>(part_last - part_first) + 1;
                const auto sync = [&] { WarpsSync(1 + g, 128); };
                __threadfence();
                sync();
                if (r == 0) {
                    int* const counter = &p.counters[part_first * G + g];
                    join_last[g] = atomicAdd(counter, 1) == parts - 1;
                    if (join_last[g]) *counter = 0;
                }
                sync();
                if (join_last[g]) {
                    __threadfence();
                    const int rows = u.req.rows - u.row - g * kRows < kRows ? u.req.rows - u.row - g * kRows : kRows;
                    // the query operands' memory: every product that read it is done
                    JoinParts<D, DTYPE, 128>(p, u.req, u.head, u.row + g * kRows, rows, tile_partials, static_cast<int>(part_first), parts, slot_floats,
                                             reinterpret_cast<float*>(q_smem), T::kOperandBytes / 4, r, sync);
                }
            }
            ++unit_count;
            umma::FenceBeforeThreadSync();
            WarpsSync(1 + g, 128);
            if (r == 0) Advance<kUnit>(p, share_end, cost, &places[g]);
            WarpsSync(1 + g, 128);
            if (!u.more) break;
        }
        }
    } else if (warp < kParamWarp) {
        if (busy) {
        // ================================================ unpacking ==================================================
        // K: this thread's 16-byte pieces, 32 elements of a token each: neighbouring lanes take the halves of 64 bytes of four
        // tokens, then further 64-byte pieces.  V: eight tokens (four pairs) by kWords words of four elements: neighbouring
        // lanes take neighbouring eights of tokens.  Either way the eight lanes of a store phase hit eight different 16-byte
        // columns.
        const int tid = threadIdx.x & 127, octet = tid & 15;
        constexpr int kPieces = D / 32, kWords = D == 64 ? 2 : 4, kTasks = D / (32 * kWords);
        const auto token_of = [&](int j) { return ((tid + 128 * j) >> 1 & 3) | ((tid + 128 * j) / (4 * kPieces) << 2); };
        const auto piece_of = [&](int j) { return ((tid + 128 * j) & 1) | (((tid + 128 * j) >> 3) % (kPieces / 2) << 1); };
        const Place& u = places[kUnpackPlace];
        uint32_t tile_count = 0;
        uint4 keys[kPieces];
        uint32_t values[kTasks][4][kWords];
        do {
            const int steps = u.steps;
            const auto load_keys = [&](uint32_t tile) {
#pragma unroll
                for (int j = 0; j < kPieces; ++j) {
                    const int64_t from = place_of[tile % P][token_of(j) >> 4];
                    keys[j] = make_uint4(0, 0, 0, 0);
                    if (from >= 0) keys[j] = LoadCodes(p.cache.k_codes + from + (token_of(j) & 15) * (D / 2) + piece_of(j) * 16);
                }
            };
            const auto load_values = [&](uint32_t tile) {
                const int64_t from = place_of[tile % P][octet >> 1];
                const uint8_t* codes = p.cache.v_codes + from + (octet & 1) * (8 * D / 2) + (tid >> 4) * (kWords * 4);
#pragma unroll
                for (int t = 0; t < kTasks; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint8_t* row = codes + j * D + 8 * t * (kWords * 4);
                        if constexpr (kWords == 4) {
                            const uint4 x = from >= 0 ? LoadCodes(row) : make_uint4(0, 0, 0, 0);
                            values[t][j][0] = x.x;
                            values[t][j][1] = x.y;
                            values[t][j][2] = x.z;
                            values[t][j][3] = x.w;
                        } else {
                            const uint2 x = from >= 0 ? *reinterpret_cast<const uint2*>(row) : make_uint2(0, 0);
                            values[t][j][0] = x.x;
                            values[t][j][1] = x.y;
                        }
                    }
            };
            wait(&params_full[tile_count % P], (tile_count / P) & 1u, 10);
            load_keys(tile_count);
            load_values(tile_count);
            for (int step = 0; step < steps; ++step, ++tile_count) {
                const uint32_t stage = tile_count % S, turn = (tile_count / S) & 1u, par = tile_count % P, next = tile_count + 1;
                uint8_t* const k_smem = smem + T::kKeys + stage * T::kOperandBytes;
                uint8_t* const v_smem = smem + T::kKeys + (S + stage) * T::kOperandBytes + (octet >> 3) * (D * 128);
                if (tile_count >= S) wait(&k_empty[stage], turn ^ 1u, 0);
#pragma unroll 1
                for (int j = 0; j < kPieces; ++j) {
                    const int token = token_of(j), piece = piece_of(j);
                    uint8_t* row = k_smem + (piece >> 1) * T::kPieceBytes + token * 128;
                    const uint32_t w[4] = {keys[0].x, keys[0].y, keys[0].z, keys[0].w};
                    uint32_t scale = 0, minimum = 0;
                    if constexpr (!kKeyCodes) {
                        scale = *reinterpret_cast<const uint16_t*>(&key_scale[par][token]) * 0x10001u;
                        minimum = *reinterpret_cast<const uint16_t*>(&key_min[par][token]) * 0x10001u;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t x = w[i], y = x >> 8;
                        uint4 o;
                        if constexpr (kKeyCodes) o = make_uint4(x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u);
                        else o = make_uint4(ValuePair<0>(x, scale, minimum), ValuePair<1>(x, scale, minimum), ValuePair<0>(y, scale, minimum), ValuePair<1>(y, scale, minimum));
                        *reinterpret_cast<uint4*>(row + ((((piece & 1) * 4 + i) ^ (token & 7)) << 4)) = o;
                    }
#pragma unroll
                    for (int i = 0; i + 1 < kPieces; ++i) keys[i] = keys[i + 1];   // the next one to the front
                }
                FenceProxyAsync();
                MbarArrive(&k_full[stage]);
                if (step + 1 < steps) {
                    wait(&params_full[next % P], (next / P) & 1u, 10);
                    load_keys(next);
                }
                if (tile_count >= S) wait(&v_empty[stage], turn ^ 1u, 1);
                const uint4 s4 = *reinterpret_cast<const uint4*>(&value_scale[par][octet * 8]), m4 = *reinterpret_cast<const uint4*>(&value_min[par][octet * 8]);
                const uint32_t sp[4] = {s4.x, s4.y, s4.z, s4.w}, mp[4] = {m4.x, m4.y, m4.z, m4.w};
#pragma unroll 1
                for (int w = 0; w < kTasks * kWords; ++w) {
                    uint32_t v[4][4];   // element, pair
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t x = values[0][j][0], y = x >> 8;
                        v[0][j] = ValuePair<0>(x, sp[j], mp[j]);
                        v[1][j] = ValuePair<1>(x, sp[j], mp[j]);
                        v[2][j] = ValuePair<0>(y, sp[j], mp[j]);
                        v[3][j] = ValuePair<1>(y, sp[j], mp[j]);
#pragma unroll
                        for (int i = 0; i + 1 < kTasks * kWords; ++i) values[i / kWords][j][i % kWords] = values[(i + 1) / kWords][j][(i + 1) % kWords];
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int element = (((tid >> 4) + 8 * (w / kWords)) * kWords + w % kWords) * 4 + i;
                        *reinterpret_cast<uint4*>(v_smem + element * 128 + (((octet & 7) ^ (element & 7)) << 4)) = make_uint4(v[i][0], v[i][1], v[i][2], v[i][3]);
                    }
                }
                FenceProxyAsync();
                MbarArrive(&v_full[stage]);
                if (step + 1 < steps) load_values(next);
            }
            WarpsSync(4, 128);
            if (tid == 0) Advance<kUnit>(p, share_end, cost, &places[kUnpackPlace]);
            WarpsSync(4, 128);
        } while (u.more);
        }
    } else {
        if (busy && warp == kParamWarp) {
        // ================================================ parameters =================================================
        // A lane has four neighbouring tokens of a tile.
        const Place& u = places[kParamPlace];
        uint32_t tile_count = 0, unit_count = 0;
        do {
            const int steps = u.steps, first_token = u.t0 * kTokens;
            int id;
            bool has;     // this lane's tokens are in a block
            int64_t at;
            uint4 kp, vp;
            const auto lookup = [&](int step) { id = step < steps ? BlockOf(p, u, first_token + step * kTokens + lane * 4) : -1; };
            const auto load = [&](int step) {
                has = IsBlock(p, id);
                kp = vp = make_uint4(0, 0, 0, 0);
                if (has) {
                    at = TokenIndex(p, id, u.head, first_token + step * kTokens + lane * 4);
                    kp = *reinterpret_cast<const uint4*>(p.cache.k_params + at);
                    vp = *reinterpret_cast<const uint4*>(p.cache.v_params + at);
                } else if (step < steps && SomeSeen(u, first_token + step * kTokens + lane * 4)) {
                    ReportTimeout(p.status, kSiteAttention, u.b);
                }
            };
            int up_exponent = kNoExponent;   // of the values, largest so far in the unit
            lookup(0);
            load(0);
            if (kKeyCodes) wait(&back_full, unit_count & 1u, 9);
            const float back = kKeyCodes ? unit_back : 1.0f;
            for (int step = 0; step < steps; ++step, ++tile_count) {
                const uint32_t par = tile_count % P;
                const int token = first_token + step * kTokens + lane * 4;
                lookup(step + 1);
                const uint32_t k4[4] = {kp.x, kp.y, kp.z, kp.w}, v4[4] = {vp.x, vp.y, vp.z, vp.w};
                uint32_t there = 0, bad = 0;
                float big_k = 0.0f, big_v = 0.0f, ks[4], km[4], vs[4], vm[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    // a token with parameters that are no numbers spoils the rows that see it through its score; as an operand it
                    // must not reach the others (0 * NaN is no zero)
                    const bool here = has && token + i >= u.low && token + i < u.high;
                    ks[i] = ParamScale(k4[i]);
                    km[i] = ParamMin(k4[i]);
                    vs[i] = ParamScale(v4[i]);
                    vm[i] = ParamMin(v4[i]);
                    const bool finite = ks[i] < INFINITY && fabsf(km[i]) < INFINITY && vs[i] < INFINITY && fabsf(vm[i]) < INFINITY;
                    there |= (here ? 1u : 0u) << i;
                    bad |= (here && !finite ? 1u : 0u) << i;
                    if (!here || !finite) ks[i] = km[i] = vs[i] = vm[i] = 0.0f;
                    big_k = fmaxf(big_k, fmaxf(fabsf(km[i]), fabsf(fmaf(15.0f, ks[i], km[i]))));
                    big_v = fmaxf(big_v, fmaxf(fabsf(vm[i]), fabsf(fmaf(15.0f, vs[i], vm[i]))));
                }
                const uint32_t eight = 0xffu << (lane & 24);   // lanes of the same word
                there = __reduce_or_sync(eight, there << (4 * (lane & 7)));
                bad = __reduce_or_sync(eight, bad << (4 * (lane & 7)));
                __syncwarp();
                big_v = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big_v)));
                if (big_v > 0.0f) {
                    const int e = QueryExponent(big_v);
                    if (up_exponent == kNoExponent || e < up_exponent) up_exponent = e;
                }
                const float up = PowerOfTwo(up_exponent == kNoExponent ? 0 : up_exponent);
                if (tile_count >= P) wait(&tile_done[par], ((tile_count / P) & 1u) ^ 1u, 11);
                if ((lane & 7) == 0) {
                    present[par][lane >> 3] = there;
                    spoiled[par][lane >> 3] = bad;
                }
                *reinterpret_cast<uint2*>(&value_scale[par][lane * 4]) = make_uint2(PackHalf(vs[0] * up, vs[1] * up), PackHalf(vs[2] * up, vs[3] * up));
                *reinterpret_cast<uint2*>(&value_min[par][lane * 4]) = make_uint2(PackHalf(vm[0] * up, vm[1] * up), PackHalf(vm[2] * up, vm[3] * up));
                if ((lane & 3) == 0) place_of[par][lane >> 2] = has ? at * (D / 2) : -1;   // this lane's first token is the sixteen's first
                const bool plain = __all_sync(0xffffffffu, there == 0xffffffffu && bad == 0);
                float down = 1.0f;   // of the keys
                if constexpr (kKeyCodes) {
                    float4* a = reinterpret_cast<float4*>(params + par * (T::kParamBytes / 4)) + lane;
                    a[0] = make_float4(ks[0] * back, ks[1] * back, ks[2] * back, ks[3] * back);
                    a[kTokens / 4] = make_float4(km[0], km[1], km[2], km[3]);
                } else {
                    big_k = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(big_k)));
                    const int e = QueryExponent(big_k);
                    const float ku = PowerOfTwo(e);
                    *reinterpret_cast<uint2*>(&key_scale[par][lane * 4]) = make_uint2(PackHalf(ks[0] * ku, ks[1] * ku), PackHalf(ks[2] * ku, ks[3] * ku));
                    *reinterpret_cast<uint2*>(&key_min[par][lane * 4]) = make_uint2(PackHalf(km[0] * ku, km[1] * ku), PackHalf(km[2] * ku, km[3] * ku));
                    down = PowerOfTwo(-e);
                }
                if (lane == 0) about[par] = make_float4(up, down, plain ? 1.0f : 0.0f, 0.0f);
                MbarArrive(&params_full[par]);
                load(step + 1);
            }
            ++unit_count;
            __syncwarp();
            if (lane == 0) Advance<kUnit>(p, share_end, cost, &places[kParamPlace]);
            __syncwarp();
        } while (u.more);
        } else if (busy) {
        // ================================================ products ===================================================
        // The whole warp runs the loops, so that descriptors are computed once for the warp and not gathered from a lane
        // (82 .. 93 cycles per product when one lane did); one lane issues.
        const int g = __shfl_sync(0xffffffffu, warp - kIssueWarp, 0);   // tile of rows
        Place* const place = &places[kIssuePlace + g];
        const uint32_t s_desc = umma::InstrDesc(1, 0, 0, false, false, kRows, kTokens / 2), o_desc = umma::InstrDesc(1, 0, 0, false, false, kRows, D);
        const uint32_t q_addr = SmemAddr(smem) + g * T::kOperandBytes, k_addr = SmemAddr(smem) + T::kKeys, v_addr = k_addr + S * T::kOperandBytes;
        const uint32_t s_tmem = __shfl_sync(0xffffffffu, tmem, 0) + g * 256, o_tmem = s_tmem + 128;
        const uint64_t qd = umma::SmemDesc(q_addr, 0, 1024);
        uint32_t tile_count = 0, active_units = 0, used = 0;   // tiles of tokens; units and tiles that this tile of rows took part in
        const auto wait_all = [&](uint64_t* bar, uint32_t parity, int detail) {
            if (!failed && !WaitFor(bar, parity, p.status, 16 + detail)) failed = true;
            failed = __any_sync(0xffffffffu, failed);
        };
        // S against half a tile.  It is written where an earlier tile's P was read, whose products are done.
        const auto scores = [&](int h, uint32_t tile) {
            umma::FenceAfterThreadSync();
            if (failed) return;
            const uint64_t kd = umma::SmemDesc(k_addr + (tile % S) * T::kOperandBytes + h * (64 * 128), 0, 1024);
            if (ElectOne()) {
#pragma unroll
                for (int i = 0; i < T::kBlocks64 * 4; ++i) {   // 32 bytes on, then the next piece
                    const uint64_t at = (i >> 2) * (T::kPieceBytes >> 4) + (i & 3) * 2;
                    MmaShared(s_tmem + h * 64, qd + at, kd + at, s_desc, i > 0);
                }
                umma::Commit(&s_full[g][h]);
                if (h == 1) umma::Commit(&k_empty[tile % S]);
            }
            __syncwarp();
        };
        const auto values = [&](int h, uint32_t tile, bool first) {
            wait_all(&p_full[g][h], used & 1u, 4);
            umma::FenceAfterThreadSync();
            if (failed) return;
            const uint64_t vd = umma::SmemDesc(v_addr + (tile % S) * T::kOperandBytes + h * (D * 128), 0, 1024);
            if (ElectOne()) {
#pragma unroll
                for (int i = 0; i < 4; ++i) MmaTensor(o_tmem, s_tmem + h * 64 + i * 8, vd + i * 2, o_desc, !first || i > 0);
                umma::Commit(&o_done[g][h]);
                if (h == 1) {
                    umma::Commit(&v_empty[tile % S]);
                    umma::Commit(&tile_done[tile % P]);
                }
            }
            __syncwarp();
        };
        bool more_units = true;
        do {
            const int steps = __shfl_sync(0xffffffffu, place->steps, 0);
            const bool active = g == 0 || __shfl_sync(0xffffffffu, place->req.rows - place->row, 0) > kRows;   // has rows
            if (active) {
                wait_all(&q_full[g], active_units++ & 1u, 2);
                wait_all(&k_full[tile_count % S], (tile_count / S) & 1u, 3);
                if (used > 0) wait_all(&o_done[g][1], (used - 1) & 1u, 8);   // and with it the other half's
                scores(0, tile_count);
                scores(1, tile_count);
                for (int step = 0; step < steps && !failed; ++step, ++tile_count, ++used) {
                    const uint32_t next = tile_count + 1;
                    wait_all(&v_full[tile_count % S], (tile_count / S) & 1u, 5);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        values(h, tile_count, step == 0 && h == 0);
                        if (step + 1 < steps) {
                            if (h == 0) wait_all(&k_full[next % S], (next / S) & 1u, 3);
                            wait_all(&o_done[g][h], used & 1u, 8);
                            scores(h, next);
                        }
                    }
                }
            } else {
                for (int step = 0; step < steps && !failed; ++step, ++tile_count) {
                    wait_all(&k_full[tile_count % S], (tile_count / S) & 1u, 3);
                    if (lane == 0) MbarArrive(&k_empty[tile_count % S]);
                    wait_all(&v_full[tile_count % S], (tile_count / S) & 1u, 5);
                    if (lane == 0) {
                        MbarArrive(&v_empty[tile_count % S]);
                        MbarArrive(&tile_done[tile_count % P]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) Advance<kUnit>(p, share_end, cost, place);
            __syncwarp();
            more_units = __shfl_sync(0xffffffffu, place->more, 0) != 0;
        } while (!failed && more_units);
        }
    }
    __syncwarp();
    umma::FenceBeforeThreadSync();
    __syncthreads();
    umma::FenceAfterThreadSync();
    if (warp == kIssueWarp) umma::TmemDealloc(tmem, T::kTmemColumns);
}

template <int D, int DTYPE>
int LaunchTyped(const AttentionParams& p, int grid, cudaStream_t s) {
    const auto kernel = PrefillKernel<D, DTYPE>;
    if (EnsureDynamicSmem(reinterpret_cast<const void*>(kernel), Tiles<D>::kBytes) != FTH_B200_OK) return FTH_B200_ERR_CUDA;
    return Launch(kernel, dim3(static_cast<unsigned>(grid)), Tiles<D>::kThreads, Tiles<D>::kBytes, s, p);
}

}  // namespace

int PrefillGrid() { return SmCount(); }

int64_t PrefillPartialFloats(int head_dim) { return static_cast<int64_t>(PrefillGrid()) * 2 * (head_dim == 256 ? 1 : 2) * kRows * (head_dim + 4); }

int LaunchPrefill(const AttentionParams& p, int head_dim, int dtype, cudaStream_t s) {
    const int grid = PrefillGrid();
    if (dtype == FTH_B200_BF16) {
        if (head_dim == 64) return LaunchTyped<64, FTH_B200_BF16>(p, grid, s);
        if (head_dim == 128) return LaunchTyped<128, FTH_B200_BF16>(p, grid, s);
        return LaunchTyped<256, FTH_B200_BF16>(p, grid, s);
    }
    if (head_dim == 64) return LaunchTyped<64, FTH_B200_FP16>(p, grid, s);
    if (head_dim == 128) return LaunchTyped<128, FTH_B200_FP16>(p, grid, s);
    return LaunchTyped<256, FTH_B200_FP16>(p, grid, s);
}

}  // namespace kv4
}  // namespace fth
