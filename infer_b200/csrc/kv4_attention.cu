// Attention over the 4-bit cache, up to 128 query rows per kv head (single tokens, drafts).
//
// The codes go into the matrix instructions as they are.  With value = m + s c per token (one scale and minimum for a
// whole head),
//     q . k = s_k (q . c) + m_k sum(q),      sum_t p_t v_t = sum_t (p_t s_v,t) c_t + sum_t p_t m_v,t
// so scales touch scores and probabilities, never elements.  A four-bit code in the low bits of a half-precision number is
// the number c * 2^-24 (a subnormal, exact in the matrix units), and four bits higher 16 c * 2^-24: one AND makes two
// operands out of a packed word, and eight codes take five operations.  The factors go into q (1/16 on the elements in
// the higher places, a power of two that puts the largest element of the rows at 2^14) and into the results; all are exact.
//
// S^T = K q^T: tokens are the 16 rows of the instruction, query rows its 8 columns, so a group of up to eight query
// heads fills it and the products of one K word serve all of them (up to four take every other column, and what a lane
// would do for the other ones is left out).  O^T = V^T P^T likewise: head elements are its rows.
// P^T comes from S^T by transposing 8 x 8 tiles within the warp.  One warp of a block of threads streams the tokens of its
// share through a ring in shared memory with bulk copies (a block's codes of one head are contiguous), also across units,
// so that the next unit's tokens fly while this one's results are joined; four warps compute, each on its 32 or 64 tokens
// of every tile, and every lane finds the words it multiplies 16 bytes apart from its neighbours'.
//
// A weight p s rounded to FP16 (11 bits) stands for the probability in all three sums of the result: the weighted codes, the
// sum of minima and the sum that divides them (weight / s gives the probability back), so a rounding moves the result by
// a rounding of that token's share of (v - out), not by one of its code, which is far larger than the value when minimum
// and code cancel.  The lse is taken from the probabilities before the rounding.
//
// Work is the flat list of (request, kv head, block of 4, 8 or 16 query rows, tile of tokens); every block of threads
// takes an equal, contiguous share, found from the lengths on the device.  A unit cut by shares leaves partial results
// (maximum, sum, weighted values, FP32) in the workspace; the part that arrives last joins them in order.
//
// Bound: cache bytes, tokens * (head_dim + 8) per kv head.  64 tokens over up to 6000 tokens each, 64 heads of 128 on 8: 75 us,
// 3.6 TB/s; one over 200 thousand, 32 heads on 8: 66 us.  Both are 15 us (set-up, the cut units' joining) and 5 TB/s, at
// which the instructions that unpack and weigh the codes keep up; the same copies without them run at 6.6 TB/s.
#include "kv4_attention.cuh"
#include "kv4_prefill.h"

namespace fth {
namespace kv4 {

namespace {

using namespace rowops;

constexpr int kWarps = 4;                         // that compute; one more copies
constexpr int kCompute = kWarps * 32;
constexpr int kThreads = kCompute + 32;
constexpr int kMinShare = 4;                      // tiles; below, cutting a unit costs more than it saves

template <int D>
struct Shape {
    static constexpr int kWords = D / 32;                 // packed words a lane holds of a token (K) or of a pair of tokens (V)
    static constexpr int kStep = D == 64 ? 64 : 32;       // tokens of a warp
    static constexpr int kSubs = kStep / 16;
    static constexpr int kStages = D == 256 ? 2 : 3;
    static constexpr int kTile = kWarps * kStep;          // tokens of a stage: K codes, V codes, K parameters, V parameters
    static constexpr int kCodeBytes = kTile * D / 2;
    static constexpr int kStageBytes = 2 * kCodeBytes + 2 * kTile * 4;
};
// Blocks of threads that share an SM; registers per thread follow from it.
template <int D, int NT>
constexpr int kBlocksPerSm = D == 256 || NT == 2 ? 2 : 3;

// Dynamic shared memory: the ring, then the place where the warps' results are joined.
template <int D, int NT>
struct Layout {
    static constexpr size_t kJoin = static_cast<size_t>(Shape<D>::kStages) * Shape<D>::kStageBytes;
    static constexpr size_t kJoinFloats = static_cast<size_t>(kWarps) * 8 * NT * kRow<D>;
    static constexpr size_t kBytes = kJoin + kJoinFloats * sizeof(float);
};

// Barrier of the warps that compute.
__device__ __forceinline__ void ComputeSync() {
    __syncwarp();
    asm volatile("barrier.cta.sync 1, %0;" ::"n"(kCompute) : "memory");   // not the aligned form: lanes may come one after another
}

// Tiles of a unit in the list: a multiple of `whole`.
__device__ __forceinline__ int64_t Rounded(int tiles, int64_t whole) { return whole == 1 ? tiles : Divide(tiles + whole - 1, whole) * whole; }
// A kv head of request b in the list: its units (blocks of `unit_rows` rows).
template <int TILE>
__device__ __forceinline__ int64_t RequestTiles(const AttentionParams& p, int b, int unit_rows, int64_t whole) {
    const Request r = LoadRequest(p, b);
    int64_t sum = 0;
    for (int row = 0; row < r.rows; row += unit_rows) {
        int first, last;
        UnitTiles<TILE>(p, r, row, unit_rows, &first, &last);
        sum += Rounded(last - first, whole);
    }
    return sum;
}

// A lane's packed words of one token row (or row of a pair of tokens): four words every 64 (K) or 128 (V) bytes.
template <int W, int SPACING>
__device__ __forceinline__ void LoadChunk(const uint8_t* row, int place, int chunk, uint32_t (&w)[4]) {
    if constexpr (W == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(row + place * 8);
        w[0] = x.x;
        w[1] = x.y;
    } else {
        const uint4 x = *reinterpret_cast<const uint4*>(row + chunk * SPACING + place * 16);
        w[0] = x.x;
        w[1] = x.y;
        w[2] = x.z;
        w[3] = x.w;
    }
}

struct Shares {
    int64_t begin, end;   // this block's share of the list
    int64_t per, whole;   // the length of a share, of which a unit's length in the list is a multiple
};

// C: columns of the score tile that a lane works on.  1: up to four rows, in the columns 2 * quad; the odd ones are zeros and nothing
// is computed for them.
template <int D, int DTYPE, int NT, int C>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm<D, NT>) DecodeKernel(const __grid_constant__ AttentionParams p) {
    using T = Shape<D>;
    constexpr int W = T::kWords;
    constexpr int CW = W == 2 ? 2 : 4;        // words of a chunk
    constexpr int S = T::kStages;
    constexpr int R = 4 * NT * C;             // rows of a unit
    static_assert(C == 2 || NT == 1, "");
    constexpr int I = 2;   // sixteens of tokens worked on together
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Shares share;    // not held in registers over the tokens
    __shared__ int join_last;
    __shared__ __align__(8) uint64_t full[S], empty[S];
    __shared__ uint32_t stage_present[S];   // a bit for every 16 tokens of the stage that are there
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, quad = lane & 3;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            MbarInit(&full[i], 1);
            MbarInit(&empty[i], kWarps);
        }
        FenceBarrierInit();
    }
    __syncthreads();
    WaitForPrevious();

    // ---- this block's share of the tiles: every warp finds it by itself, a lane per request --------------------------------
    int64_t work = 0;
#pragma unroll 4
    for (int i = lane; i < p.requests; i += 32) work += RequestTiles<T::kTile>(p, i, R, 1);
    work = WarpSum(work) * p.kv_heads;
    int64_t per = Divide(work + gridDim.x - 1, gridDim.x), whole = 1;
    if (per < kMinShare) per = kMinShare;
    // With fewer units than blocks of threads a share ends with its unit, if there are blocks enough: units up to `per` tiles
    // are not cut then (one request of 333 tokens, 2 kv heads: 13.9 us when the second unit was).  In the list such a unit
    // is as long as its shares.
    if (static_cast<int64_t>(p.requests) * p.kv_heads <= gridDim.x) {
        int64_t length = 0;
        for (int i = lane; i < p.requests; i += 32) length += RequestTiles<T::kTile>(p, i, R, per);
        length = WarpSum(length) * p.kv_heads;
        if (length <= per * gridDim.x) {
            whole = per;
            work = length;
        }
    }
    const int64_t share_begin = blockIdx.x * per;
    const int64_t share_end = share_begin + per < work ? share_begin + per : work;
    if (share_begin >= share_end) return;
    if (threadIdx.x == 0) share = Shares{share_begin, share_end, per, whole};
    __syncthreads();

    // ---- the first unit: request, head, tiles -----------------------------------------------------------------------------
    int b = 0;
    int64_t offset_in = 0, per_head = 1;   // of share_begin in the request; the request's length in the list per head
    int64_t passed = 0;
    for (int base = 0; base < p.requests; base += 32) {
        const int64_t length = base + lane < p.requests ? RequestTiles<T::kTile>(p, base + lane, R, whole) : 0;
        const int64_t mine = length * p.kv_heads;
        int64_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t n = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += n;
        }
        const uint32_t who = __ballot_sync(0xffffffffu, share_begin < passed + upto);
        if (who != 0) {
            const int src = __ffs(who) - 1;
            b = base + src;
            offset_in = share_begin - passed - __shfl_sync(0xffffffffu, upto - mine, src);
            per_head = __shfl_sync(0xffffffffu, length, src);
            break;
        }
        passed += __shfl_sync(0xffffffffu, upto, 31);
    }
    Request req = LoadRequest(p, b);
    int head = static_cast<int>(Divide(offset_in, per_head));
    int row = 0;
    int64_t into = offset_in - head * per_head;  // tiles of the unit that other blocks take
    int tile_first, tile_last;
    for (;;) {
        UnitTiles<T::kTile>(p, req, row, R, &tile_first, &tile_last);
        const int64_t length = Rounded(tile_last - tile_first, whole);
        if (into < length || row + R >= req.rows) break;
        into -= length;
        row += R;
    }
    int64_t at = share_begin;
    int t0, steps, first_low, last_high;   // of this block's part of the unit
    const auto place = [&] {
        const int64_t left = share.end - at, tiles = tile_last - tile_first - into;
        t0 = tile_first + static_cast<int>(into);
        steps = static_cast<int>(tiles < left ? tiles : left);
        int unused;
        Visible(p, req, QueryOf(p, row), &first_low, &unused);
        Visible(p, req, QueryOf(p, (row + R < req.rows ? row + R : req.rows) - 1), &unused, &last_high);
    };
    const auto next_unit = [&] {   // false: the share is done
        at += Rounded(tile_last - tile_first, share.whole) - into;
        if (at >= share.end) return false;
        into = 0;
        row += R;
        if (row >= req.rows) {
            row = 0;
            if (++head == p.kv_heads) {
                head = 0;
                do {
                    ++b;
                    req = LoadRequest(p, b);
                } while (req.rows == 0);
            }
        }
        UnitTiles<T::kTile>(p, req, row, R, &tile_first, &tile_last);
        place();
        return true;
    };
    place();
    int stage = 0;
    uint32_t phase = 0;
    bool failed = false;

    if (warp == kWarps) {
        // ---- copies: lane = 4 * (16 tokens) + (K codes, V codes, K parameters, V parameters) ----------------------------------
        // Blocks of more than 16 tokens are copied by the lanes of their first 16, up to a whole tile at once.
        constexpr int kRounds = T::kTile / 128;
        constexpr int kTileShift = T::kTile == 256 ? 8 : 7;
        const int span_shift = p.cache.block_shift < kTileShift ? p.cache.block_shift : kTileShift;
        const int span = 1 << span_shift;
        int id[kRounds];
        int64_t issued = 0;
        do {
            const int32_t* table = p.table + static_cast<int64_t>(b) * p.max_blocks;
            const auto lookup = [&](int step) {
#pragma unroll
                for (int r = 0; r < kRounds; ++r) {
                    const int in_tile = r * 128 + (lane >> 2) * 16;
                    const int token = (t0 + step) * T::kTile + in_tile;
                    id[r] = -2;
                    if (step < steps && (in_tile & (span - 1)) == 0 && token < last_high && token + span > first_low)
                        id[r] = table[token >> p.cache.block_shift];
                }
            };
            lookup(0);
            for (int step = 0; step < steps; ++step) {
                if (issued >= S && !failed && !MbarWait(&empty[stage], phase ^ 1u, p.status, kSiteAttentionWait, stage)) failed = true;
                uint32_t there = 0;
                int copies = 0;
                bool good[kRounds];
#pragma unroll
                for (int r = 0; r < kRounds; ++r) {
                    good[r] = id[r] >= 0 && id[r] < p.cache.blocks;
                    if (id[r] != -2 && !good[r] && quad == 0) ReportTimeout(p.status, kSiteAttention, b);
                    const uint32_t who = __ballot_sync(0xffffffffu, good[r]);
                    copies += __popc(who & 0x11111111u);
#pragma unroll
                    for (int i = 0; i < 8; ++i) there |= ((who >> (4 * i)) & 1u) << (r * 8 + i);
                }
                for (int sh = 1; sh < (span >> 4); sh <<= 1) there |= there << sh;   // a span's later sixteens
                if (lane == 0) {
                    stage_present[stage] = there;
                    MbarExpectTx(&full[stage], static_cast<uint32_t>(copies) * span * (D + 8));
                }
                __syncwarp();
                uint8_t* dst = smem + stage * T::kStageBytes;
#pragma unroll
                for (int r = 0; r < kRounds; ++r) {
                    if (good[r] && !failed) {
                        const int in_tile = r * 128 + (lane >> 2) * 16;
                        const int64_t from = HeadBase(p.cache, id[r], head) + (((t0 + step) * T::kTile + in_tile) & ((1 << p.cache.block_shift) - 1));
                        if (quad < 2) {
                            BulkLoad(dst + quad * T::kCodeBytes + in_tile * (D / 2), (quad == 0 ? p.cache.k_codes : p.cache.v_codes) + from * (D / 2),
                                     span * (D / 2), &full[stage]);
                        } else {
                            BulkLoad(dst + 2 * T::kCodeBytes + (quad - 2) * (T::kTile * 4) + in_tile * 4,
                                     (quad == 2 ? p.cache.k_params : p.cache.v_params) + from, span * 4, &full[stage]);
                        }
                    }
                }
                lookup(step + 1);
                ++issued;
                if (++stage == S) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        } while (next_unit());
        return;
    }

    for (;;) {
        const int64_t unit_begin = at - into;
        const int64_t unit_end = unit_begin + (tile_last - tile_first);

        // ---- query rows ----------------------------------------------------------------------------------------------------
        uint32_t qf[NT][2 * W][2];
        float qsum[NT][2];   // of the columns 2 * quad, 2 * quad + 1
        int row_low[NT][2], row_high[NT][2];
        int all_low = 0, all_high = 0x7fffffff;
        float back;
        {
            uint32_t raw[NT][W][4];   // eight 16-bit elements per word of codes
            float big = 0.0f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int r = row + n * 8 + (C == 1 ? g >> 1 : g);   // in column g
                const bool valid = r < req.rows && (C == 2 || (g & 1) == 0);
                const int query = valid ? QueryOf(p, r) : 0;
                const uint16_t* from = static_cast<const uint16_t*>(p.q) + (req.first_row + static_cast<int64_t>(query)) * p.ldq +
                                       (static_cast<int64_t>(head) * p.group + r - query * p.group) * D;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const int word = W == 2 ? quad * 2 + w : (w >> 2) * 16 + quad * 4 + (w & 3);
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (valid) {
                        if (p.q_vec) x = *reinterpret_cast<const uint4*>(from + word * 8);
                        else x = LoadUnaligned8(from + word * 8);
                    }
                    raw[n][w][0] = x.x;
                    raw[n][w][1] = x.y;
                    raw[n][w][2] = x.z;
                    raw[n][w][3] = x.w;
                }
                int low = 0, high = 0;
                if (valid) {
                    Visible(p, req, query, &low, &high);
                    all_low = low > all_low ? low : all_low;
                    all_high = high < all_high ? high : all_high;
                }
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 v = HalfPair<DTYPE>(raw[n][w][i]);
                        big = fmaxf(big, fmaxf(FiniteAbs(v.x), FiniteAbs(v.y)));
                        sum += v.x + v.y;
                    }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                qsum[n][0] = p.scale_log2 * __shfl_sync(0xffffffffu, sum, quad * 8);
                qsum[n][1] = p.scale_log2 * __shfl_sync(0xffffffffu, sum, quad * 8 + 4);
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    row_low[n][c] = __shfl_sync(0xffffffffu, low, quad * 8 + c * 4);
                    row_high[n][c] = __shfl_sync(0xffffffffu, high, quad * 8 + c * 4);
                }
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                const int l = __shfl_xor_sync(0xffffffffu, all_low, o), h = __shfl_xor_sync(0xffffffffu, all_high, o);
                all_low = l > all_low ? l : all_low;
                all_high = h < all_high ? h : all_high;
            }
            // one power of two for all rows, the largest element to 2^14: odd elements, with their 1/16, keep FP16's 11 bits down to 2^-24
            // of it (its normal numbers end at 2^-14) and BF16's 8 down to 2^-27, even ones 16 times farther
            const int e = QueryExponent(big);
            back = p.scale_log2 * PowerOfTwo(24 - e);
            const float up = PowerOfTwo(e);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    uint32_t f[4];
                    QueryOperands<DTYPE>(raw[n][w], up, 0.0625f, f);
                    qf[n][2 * w][0] = f[0];
                    qf[n][2 * w][1] = f[1];
                    qf[n][2 * w + 1][0] = f[2];
                    qf[n][2 * w + 1][1] = f[3];
                }
            }
        }

        // ---- tokens -----------------------------------------------------------------------------------------------------------
        float acc[NT][2 * W][4];
        float top[NT][2], sum[NT][2], mass[NT][2], offset[NT][2];   // top: the running maximum; scores are kept relative to it
        float limit[NT][2];                    // a relative score above it moves the maximum
        float shrink = 1.0f;                   // value scales are multiplied by this power of two before they become FP16
        float scale_limit = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int m = 0; m < 2 * W; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[n][m][i] = 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                top[n][c] = sum[n][c] = mass[n][c] = offset[n][c] = 0.0f;
                limit[n][c] = kNotStarted;
            }
        }
        for (int step = 0; step < steps; ++step) {
            if (!failed && !MbarWait(&full[stage], phase, p.status, kSiteAttentionWait, S + stage)) failed = true;
            const uint8_t* data = smem + stage * T::kStageBytes + warp * (T::kStep * D / 2);
            const uint32_t* k_params = reinterpret_cast<const uint32_t*>(smem + stage * T::kStageBytes + 2 * T::kCodeBytes) + warp * T::kStep;
            const uint32_t* v_params = k_params + T::kTile;
            const uint32_t present_all = failed ? 0u : stage_present[stage] >> (T::kSubs * warp);
#pragma unroll 1
            for (int part = 0; part < T::kSubs / I; ++part) {   // 16 * I tokens
                const uint32_t present = (present_all >> (I * part)) & ((1u << I) - 1);
                if (present == 0) continue;
                const int place0 = part * (16 * I);
                const int token0 = (t0 + step) * T::kTile + warp * T::kStep + place0;
                const uint8_t* k_rows = data + place0 * (D / 2);
                const uint8_t* v_rows = k_rows + T::kCodeBytes;

                // q . c
                float z[I][NT][4];
#pragma unroll
                for (int c = 0; c < W / CW; ++c) {
#pragma unroll
                    for (int s = 0; s < I; ++s) {
                        uint32_t k0[4], k1[4];
                        LoadChunk<W, 64>(k_rows + (s * 16 + g) * (D / 2), quad, c, k0);
                        LoadChunk<W, 64>(k_rows + (s * 16 + 8 + g) * (D / 2), quad, c, k1);
#pragma unroll
                        for (int i = 0; i < CW; ++i) {
                            const int w = c * CW + i;
                            const uint32_t x0 = k0[i], x1 = k1[i], y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const uint4 f = make_uint4(qf[n][2 * w][0], qf[n][2 * w][1], qf[n][2 * w + 1][0], qf[n][2 * w + 1][1]);
                                if (w == 0) MmaF16First(z[s][n], x0 & 0x000f000fu, x1 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x00f000f0u, f.x, f.y);
                                else MmaF16(z[s][n], x0 & 0x000f000fu, x1 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x00f000f0u, f.x, f.y);
                                MmaF16(z[s][n], y0 & 0x000f000fu, y1 & 0x000f000fu, y0 & 0x00f000f0u, y1 & 0x00f000f0u, f.z, f.w);
                            }
                        }
                    }
                }
                // scores, exponents of two, relative to the running maximum
                const bool inside = token0 >= all_low && token0 + 16 * I <= all_high && present == (1u << I) - 1;
                float best[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) best[n][0] = best[n][1] = -INFINITY;
#pragma unroll
                for (int s = 0; s < I; ++s) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t kp = k_params[place0 + s * 16 + h * 8 + g];
                        const float ks = ParamScale(kp) * back, km = ParamMin(kp);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
#pragma unroll
                            for (int c = 0; c < C; ++c) {
                                float& score = z[s][n][2 * h + c];
                                score = fmaf(ks, score, fmaf(km, qsum[n][c], -top[n][c]));
                            }
                        }
                    }
                }
                // value scales of these tokens, as bits (positive numbers order like their bits; NaN comes out as the largest)
                uint32_t scale_bits = v_params[place0 + lane] << 16;
                if (!inside) {
                    bool lane_seen = false;   // of the token whose scale this lane holds
#pragma unroll
                    for (int s = 0; s < I; ++s) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int token = token0 + s * 16 + h * 8 + g;
                            const bool there = ((present >> s) & 1u) != 0;
                            bool any = false;
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
#pragma unroll
                                for (int c = 0; c < C; ++c) {
                                    const bool seen = there && token >= row_low[n][c] && token < row_high[n][c];
                                    if (!seen) z[s][n][2 * h + c] = -INFINITY;
                                    any = any || seen;
                                }
                            }
                            // columns of all four lanes of a token, then bit = token within these 32
                            const uint32_t who = __ballot_sync(0xffffffffu, any);
                            const int mine_at = lane - (s * 16 + h * 8);
                            if (mine_at >= 0 && mine_at < 8) lane_seen = ((who >> (4 * mine_at)) & 15u) != 0;
                        }
                    }
                    if (!lane_seen) scale_bits = 0;
                }
                const uint32_t scale_top = __reduce_max_sync(0xffffffffu, scale_bits), scale_low = __reduce_min_sync(0xffffffffu, scale_bits);
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < C; ++c)
#pragma unroll
                        for (int s = 0; s < I; ++s) best[n][c] = fmaxf(best[n][c], fmaxf(z[s][n][c], z[s][n][2 + c]));
                float biggest = __uint_as_float(scale_top);
                // a scale that is no number spoils the rows that see its token, through their weights; the others' weights need the
                // largest scale beside it
                if (!(biggest < INFINITY)) biggest = __uint_as_float(__reduce_max_sync(0xffffffffu, scale_bits < 0x7f800000u ? scale_bits : 0u));
                bool rescale = biggest > scale_limit;
#pragma unroll
                for (int n = 0; n < NT; ++n) rescale = rescale || best[n][0] > limit[n][0] || (C == 2 && best[n][1] > limit[n][1]);
                if (__any_sync(0xffffffffu, rescale)) {
                    float change = 1.0f;
                    if (biggest > scale_limit) {
                        const int e = ScaleExponent(biggest);
                        const float next = PowerOfTwo(7 - e);
                        change = scale_limit == 0.0f ? 0.0f : next / shrink;
                        shrink = next;
                        scale_limit = PowerOfTwo(e);
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float moved[2], factor[2];
#pragma unroll
                        for (int c = 0; c < C; ++c) {
                            float m = best[n][c];
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                            const bool first = limit[n][c] == kNotStarted;
                            const bool move = first ? m > kNotStarted : m > 0.0f;
                            moved[c] = move ? m : 0.0f;
                            if (move) limit[n][c] = kLazy;
                            // before the first score the sums are zeros (or NaN, which stay)
                            const float alpha = first ? 0.0f : Exp2(-moved[c]);
                            factor[c] = alpha * change;
                            top[n][c] += moved[c];
                            sum[n][c] *= alpha;
                            mass[n][c] *= alpha;
                            offset[n][c] *= alpha;
                        }
#pragma unroll
                        for (int m = 0; m < 2 * W; ++m) {
                            acc[n][m][0] *= factor[0];
                            acc[n][m][2] *= factor[0];
                            if constexpr (C == 2) {
                                acc[n][m][1] *= factor[1];
                                acc[n][m][3] *= factor[1];
                            }
                        }
#pragma unroll
                        for (int s = 0; s < I; ++s)
#pragma unroll
                            for (int i = 0; i < 4; i += 3 - C) z[s][n][i] -= moved[i & 1];
                    }
                }
                // probabilities, weights, weighted values
                const bool plain = !inside || !(__uint_as_float(scale_low) * shrink >= 1.0f) || !(__uint_as_float(scale_top) < INFINITY);
#pragma unroll
                for (int s = 0; s < I; ++s) {
                    uint32_t pt[NT][2];
                    float vs[2], vm[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t vp = v_params[place0 + s * 16 + h * 8 + g];
                        vs[h] = ParamScale(vp) * shrink;
                        vm[h] = ParamMin(vp);
                    }
                    if (!plain) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float inverse = Reciprocal(vs[h]), ratio = vm[h] * inverse;
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                const float p0 = Exp2(z[s][n][2 * h]), p1 = C == 2 ? Exp2(z[s][n][2 * h + 1]) : 0.0f;
                                mass[n][0] += p0;
                                const uint32_t packed = PackHalf(p0 * vs[h], C == 2 ? p1 * vs[h] : 0.0f);
                                const float2 w = HalfPair<FTH_B200_FP16>(packed);
                                sum[n][0] = fmaf(w.x, inverse, sum[n][0]);
                                offset[n][0] = fmaf(w.x, ratio, offset[n][0]);
                                if constexpr (C == 2) {
                                    mass[n][1] += p1;
                                    sum[n][1] = fmaf(w.y, inverse, sum[n][1]);
                                    offset[n][1] = fmaf(w.y, ratio, offset[n][1]);
                                }
                                pt[n][h] = Transpose8x8(packed);
                            }
                        }
                    } else {
                        // hidden tokens (whatever stands there: 0 * NaN is no zero), and value scales too small beside the
                        // largest for a weight to give the probability back
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                float w[2] = {};
#pragma unroll
                                for (int c = 0; c < C; ++c) {
                                    const float score = z[s][n][2 * h + c];
                                    const bool hidden = score == -INFINITY;
                                    const float prob = Exp2(score);
                                    w[c] = hidden ? 0.0f : __half2float(__float2half_rn(prob * vs[h]));
                                    const float kept = vs[h] >= 1.0f ? w[c] * Reciprocal(vs[h]) : prob;
                                    if (!hidden) {
                                        mass[n][c] += prob;
                                        sum[n][c] += kept;
                                        offset[n][c] = fmaf(kept, vm[h], offset[n][c]);
                                    }
                                }
                                pt[n][h] = Transpose8x8(PackHalf(w[0], w[1]));
                            }
                        }
                    }
#pragma unroll
                    for (int c = 0; c < W / CW; ++c) {
                        uint32_t v0[4], v1[4];
                        LoadChunk<W, 128>(v_rows + (s * 8 + quad) * D, g, c, v0);
                        LoadChunk<W, 128>(v_rows + (s * 8 + 4 + quad) * D, g, c, v1);
#pragma unroll
                        for (int i = 0; i < CW; ++i) {
                            const int w = c * CW + i;
                            const uint32_t x0 = v0[i], x1 = v1[i], y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                MmaF16(acc[n][2 * w], x0 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x000f000fu, x1 & 0x00f000f0u, pt[n][0], pt[n][1]);
                                MmaF16(acc[n][2 * w + 1], y0 & 0x000f000fu, y0 & 0x00f000f0u, y1 & 0x000f000fu, y1 & 0x00f000f0u, pt[n][0], pt[n][1]);
                            }
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) MbarArrive(&empty[stage]);
            if (++stage == S) {
                stage = 0;
                phase ^= 1u;
            }
        }

        // ---- the four warps' results together: [warp][row][D values, maximum, unused, sum, sum for the lse] ---------------------------
        float* join = reinterpret_cast<float*>(smem + Layout<D, NT>::kJoin);
        ComputeSync();
        {
            const float unit = PowerOfTwo(24) / shrink;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int c = 0; c < C; ++c) {
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) {
                        sum[n][c] += __shfl_xor_sync(0xffffffffu, sum[n][c], o);
                        mass[n][c] += __shfl_xor_sync(0xffffffffu, mass[n][c], o);
                        offset[n][c] += __shfl_xor_sync(0xffffffffu, offset[n][c], o);
                    }
                    float* out = join + static_cast<size_t>(warp * R + n * 8 + quad * C + c) * kRow<D>;
                    const float shift = offset[n][c];
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        const int word = W == 2 ? g * 2 + w : (w >> 2) * 32 + g * 4 + (w & 3);
                        out[word * 4] = fmaf(acc[n][2 * w][c], unit, shift);
                        out[word * 4 + 1] = fmaf(acc[n][2 * w][2 + c], unit * 0.0625f, shift);
                        out[word * 4 + 2] = fmaf(acc[n][2 * w + 1][c], unit, shift);
                        out[word * 4 + 3] = fmaf(acc[n][2 * w + 1][2 + c], unit * 0.0625f, shift);
                    }
                    if (g == 0) {
                        out[D] = limit[n][c] == kNotStarted ? kNoMax : top[n][c];
                        out[D + 2] = sum[n][c];
                        out[D + 3] = mass[n][c];
                    }
                }
            }
        }
        ComputeSync();
        // blocks of threads that hold the first and the last part of the unit
        const int64_t part_first = unit_begin >= share.begin ? blockIdx.x : Divide(unit_begin, share.per);
        const int64_t part_last = unit_end <= share.end ? blockIdx.x : Divide(unit_end - 1, share.per);
        const bool whole = part_first == part_last;
        const int valid_rows = req.rows - row < R ? req.rows - row : R;
        const int64_t slot_floats = static_cast<int64_t>(R) * kRow<D>;
        float* partial = p.partials + (static_cast<int64_t>(blockIdx.x) * 2 + (blockIdx.x == part_first ? 1 : 0)) * slot_floats;
        for (int i = threadIdx.x; i < valid_rows * (D / 4); i += kCompute) {
            const int r = i / (D / 4), d = (i - r * (D / 4)) * 4;
            float best = kNoMax;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) best = fmaxf(best, join[(w * R + r) * kRow<D> + D]);
            float total = 0.0f, all = 0.0f;
            float4 value = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float* from = join + (w * R + r) * kRow<D>;
                const float weight = Exp2(from[D] - best);
                total = fmaf(weight, from[D + 2], total);
                all = fmaf(weight, from[D + 3], all);
                FmaFour(value, weight, *reinterpret_cast<const float4*>(from + d));
            }
            if (whole) {
                StoreFour<D, DTYPE>(p, req, head, row + r, d, value, total, best, all);
            } else {
                *reinterpret_cast<float4*>(partial + r * kRow<D> + d) = value;
                if (d == 0) *reinterpret_cast<float4*>(partial + r * kRow<D> + D) = make_float4(best, 0.0f, total, all);
            }
        }
        if (!whole) {
            const int parts = static_cast<int>(part_last - part_first) + 1;
            __threadfence();
            ComputeSync();
            if (threadIdx.x == 0) {
                join_last = atomicAdd(&p.counters[part_first], 1) == parts - 1;
                if (join_last) p.counters[part_first] = 0;
            }
            ComputeSync();
            if (join_last) {
                __threadfence();
                JoinParts<D, DTYPE, kCompute>(p, req, head, row, valid_rows, p.partials, static_cast<int>(part_first), parts, slot_floats, join,
                                              static_cast<int>(Layout<D, NT>::kJoinFloats), threadIdx.x, ComputeSync);
            }
        }
        if (!next_unit()) break;
    }
}

int CheckAttention(const fth_b200_kv4_attention_desc* d) {
    if (d == nullptr) return FTH_B200_ERR_INVALID;
    const int rc = CheckCache(d->cache);
    if (rc != FTH_B200_OK) return rc;
    if (d->requests <= 0 || d->tokens < 0 || d->q_heads <= 0 || d->max_blocks <= 0 || d->max_query <= 0 || d->window < 0) return FTH_B200_ERR_INVALID;
    if (d->q_heads % d->cache.kv_heads != 0 || !std::isfinite(d->scale)) return FTH_B200_ERR_INVALID;
    if (d->query_start == nullptr && (d->max_query != 1 || d->tokens != d->requests)) return FTH_B200_ERR_INVALID;
    if (d->block_table == nullptr || d->total_lens == nullptr) return FTH_B200_ERR_INVALID;
    if (d->tokens > 0 && (d->q == nullptr || d->out == nullptr)) return FTH_B200_ERR_INVALID;
    const int64_t row = static_cast<int64_t>(d->q_heads) * d->cache.head_dim;
    if ((d->ldq != 0 && d->ldq < row) || (d->ldo != 0 && d->ldo < row)) return FTH_B200_ERR_INVALID;
    if (d->dtype != FTH_B200_BF16 && d->dtype != FTH_B200_FP16) return FTH_B200_ERR_UNSUPPORTED;
    if (!AlignedTo(d->q, 2) || !AlignedTo(d->out, 2) || !WordAligned(d->lse, d->block_table, d->total_lens, d->query_start)) return FTH_B200_ERR_INVALID;
    if (d->tokens > 0x7fffffff || d->q_heads > 65536 || static_cast<int64_t>(d->max_query) * (d->q_heads / d->cache.kv_heads) > 0x7fffffff)
        return FTH_B200_ERR_UNSUPPORTED;
    // places of tokens are 31 bits, also one tile (of up to 256) behind the last
    if (static_cast<int64_t>(d->max_blocks) * d->cache.block_size > 0x7fffffff - 511) return FTH_B200_ERR_UNSUPPORTED;
    return FTH_B200_OK;
}

constexpr int kMaxGrid = 1024;
constexpr size_t kCounterBytes = kMaxGrid * sizeof(int);

// Rows of a kv head that a request may have.
int64_t MostRows(const fth_b200_kv4_attention_desc& d) { return static_cast<int64_t>(d.max_query) * (d.q_heads / d.cache.kv_heads); }
// Query rows of a unit, in eights.  Sixteen share what unpacking costs (12 requests of 3500 .. 9000 tokens, 2 kv heads of 128, 32 rows:
// 27.5 us, 32.4 us in eights), unless half of the last ones would be missing (32 requests, 8 kv heads, 20 rows: 123 us, 113 us in eights); 256-wide
// heads leave no registers for them (20 rows: 69 us, 42 us in eights).  With 9 to 16 rows, one unit of sixteen, two of eight would be as
// fast or faster: 12 rows of those 12 requests 29 us, 23 us in eights; one request of 8000 tokens, 8 heads of 128, 23 and 20 us.
int DecodeTiles(const fth_b200_kv4_attention_desc& d) { return d.cache.head_dim != 256 && (MostRows(d) + 7) / 8 % 2 == 0 ? 2 : 1; }
// Blocks of threads that are resident together.
int DecodeGrid(int head_dim, int tiles) {
    const int per_sm = head_dim == 256 || tiles == 2 ? kBlocksPerSm<256, 1> : kBlocksPerSm<128, 1>;
    const int grid = SmCount() * per_sm;
    return grid < kMaxGrid ? grid : kMaxGrid;
}

// The kernel with 128-row tiles.  It unpacks as much for a row as for 256, and its tiles start late.  Where the two cross depends on the
// lengths, which the host does not know: heads of 128 take the kernel for few rows (let on to more) and that for many
//   12 requests of 3500 .. 9000 tokens, 2 kv heads    132 rows  97 and 136 us   256 rows 135 and 146 us   384 rows 195 and 125 us
//   one request of 8000 tokens, 8 kv heads            132 rows  57 and 181 us   384 rows  99 and 121 us   768 rows 180 and 135 us
//   40 requests of 1000 tokens, 4 kv heads            128 rows 106 us           132 rows 129 and  84 us   256 rows 195 and  91 us
// 64-wide heads cross at the same places, 256-wide ones at 132, 256 and below 128 rows.  128 costs the long requests and spares the short.
bool ManyRows(const fth_b200_kv4_attention_desc& d) { return MostRows(d) > 128; }

// What a call with these or fewer rows needs, so that the largest step's workspace serves all: units of sixteen rows, in fewer blocks of
// threads, need more than the units of eight that some larger steps have.
size_t WorkspaceBytes(const fth_b200_kv4_attention_desc& d) {
    if (ManyRows(d)) return kCounterBytes + static_cast<size_t>(PrefillPartialFloats(d.cache.head_dim)) * sizeof(float);
    const auto need = [&](int tiles) { return static_cast<size_t>(DecodeGrid(d.cache.head_dim, tiles)) * 2 * 8 * tiles * (d.cache.head_dim + 4) * sizeof(float); };
    const size_t eights = need(1), sixteens = d.cache.head_dim != 256 && MostRows(d) > 8 ? need(2) : 0;
    return kCounterBytes + (eights > sixteens ? eights : sixteens);
}

template <int D, int DTYPE>
int LaunchDecode(const AttentionParams& p, int tiles, bool four, int grid, cudaStream_t s) {
    const auto run = [&](auto kernel, size_t smem) {
        if (EnsureDynamicSmem(reinterpret_cast<const void*>(kernel), smem) != FTH_B200_OK) return static_cast<int>(FTH_B200_ERR_CUDA);
        return Launch(kernel, dim3(static_cast<unsigned>(grid)), kThreads, smem, s, p);
    };
    if constexpr (D != 256) {
        if (tiles == 2) return run(DecodeKernel<D, DTYPE, 2, 2>, Layout<D, 2>::kBytes);
    }
    return four ? run(DecodeKernel<D, DTYPE, 1, 1>, Layout<D, 1>::kBytes) : run(DecodeKernel<D, DTYPE, 1, 2>, Layout<D, 1>::kBytes);
}

}  // namespace
}  // namespace kv4
}  // namespace fth

using namespace fth;

extern "C" int fth_b200_kv4_attention_supported(const fth_b200_kv4_attention_desc* d) { return kv4::CheckAttention(d); }

extern "C" size_t fth_b200_kv4_attention_workspace_bytes(const fth_b200_kv4_attention_desc* d) {
    return kv4::CheckAttention(d) == FTH_B200_OK ? kv4::WorkspaceBytes(*d) : 0;
}

extern "C" int fth_b200_kv4_attention(const fth_b200_kv4_attention_desc* d, fth_b200_stream_t stream) {
    ClearStaleError();
    const int rc = kv4::CheckAttention(d);
    if (rc != FTH_B200_OK) return rc;
    if (d->tokens == 0) return FTH_B200_OK;
    if (d->workspace == nullptr || !kv4::AlignedTo(d->workspace, 256) || d->workspace_bytes < kv4::WorkspaceBytes(*d)) return FTH_B200_ERR_INVALID;
    kv4::AttentionParams p = {};
    const int64_t row = static_cast<int64_t>(d->q_heads) * d->cache.head_dim;
    p.cache = kv4::MakeCache(d->cache);
    p.q = d->q;
    p.out = d->out;
    p.lse = d->lse;
    p.ldq = d->ldq ? d->ldq : row;
    p.ldo = d->ldo ? d->ldo : row;
    p.tokens = d->tokens;
    p.table = d->block_table;
    p.total_lens = d->total_lens;
    p.query_start = d->query_start;
    p.requests = d->requests;
    p.max_blocks = d->max_blocks;
    p.max_query = d->max_query;
    p.kv_heads = d->cache.kv_heads;
    p.group = d->q_heads / d->cache.kv_heads;
    p.group_inverse = 0xffffffffu / static_cast<uint32_t>(p.group);
    p.causal = d->causal != 0;
    p.window = d->window;
    p.q_vec = kv4::AlignedTo(d->q, 16) && p.ldq % 8 == 0;
    p.out_vec = kv4::AlignedTo(d->out, 16) && p.ldo % 8 == 0;
    p.scale_log2 = d->scale * 1.4426950408889634f;
    p.status = DeviceStatusPtr();
    p.counters = static_cast<int*>(d->workspace);
    p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(d->workspace) + kv4::kCounterBytes);
    auto s = static_cast<cudaStream_t>(stream);
    int status;
    if (kv4::ManyRows(*d)) {
        p.few_units = static_cast<int64_t>(d->max_query) * p.group <= 512;
        status = kv4::LaunchPrefill(p, d->cache.head_dim, d->dtype, s);
        if (status == FTH_B200_OK) NoteLaunch("kv4_attention_rows");
        return status;
    }
    // units of four rows where no request has more: half of a score tile is left out then (40 requests of 3000 tokens, one row to a head,
    // 16 heads of 64: 48.7 us, 45.3 us with four; 4 heads of 256: 43.1 and 39.9 us; one request of 200 thousand tokens: 64.4 and 66.5 us)
    const bool four = kv4::MostRows(*d) <= 4;
    const int tiles = kv4::DecodeTiles(*d), grid = kv4::DecodeGrid(d->cache.head_dim, tiles);
    if (d->dtype == FTH_B200_BF16) {
        if (d->cache.head_dim == 64) status = kv4::LaunchDecode<64, FTH_B200_BF16>(p, tiles, four, grid, s);
        else if (d->cache.head_dim == 128) status = kv4::LaunchDecode<128, FTH_B200_BF16>(p, tiles, four, grid, s);
        else status = kv4::LaunchDecode<256, FTH_B200_BF16>(p, tiles, four, grid, s);
    } else {
        if (d->cache.head_dim == 64) status = kv4::LaunchDecode<64, FTH_B200_FP16>(p, tiles, four, grid, s);
        else if (d->cache.head_dim == 128) status = kv4::LaunchDecode<128, FTH_B200_FP16>(p, tiles, four, grid, s);
        else status = kv4::LaunchDecode<256, FTH_B200_FP16>(p, tiles, four, grid, s);
    }
    if (status == FTH_B200_OK) NoteLaunch("kv4_attention");
    return status;
}
