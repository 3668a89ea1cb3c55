// Attention over the 4-bit cache.
//
// The codes go into the matrix instructions as they are.  With value = m + s c per token (one scale and minimum for a
// whole head),
//     q . k = s_k (q . c) + m_k sum(q),      sum_t p_t v_t = sum_t (p_t s_v,t) c_t + sum_t p_t m_v,t
// so scales touch scores and probabilities, never elements.  A four-bit code in the low bits of a half-precision number is
// the number c * 2^-24 (a subnormal, exact in the matrix units), and four bits higher 16 c * 2^-24: one AND makes two
// operands out of a packed word, and eight codes take five operations.  The factors go into q (1/16 on the elements in
// the higher places, a power of two per row that puts its largest element at 2^14) and into the results; all are exact.
//
// S^T = K q^T: tokens are the 16 rows of the instruction, query rows its 8 columns, so a group of up to eight query
// heads fills it and the products of one K word serve all of them.  O^T = V^T P^T likewise: head elements are its rows.
// P^T comes from S^T by transposing 8 x 8 tiles within the warp.  Every lane loads exactly the words it multiplies (16
// bytes, neighbouring lanes neighbouring addresses) through a ring of its own in shared memory: no exchange, no barrier.
//
// Work is the flat list of (request, kv head, block of 8 or 16 query rows, tile of 128 tokens); every block of threads
// takes an equal, contiguous share, found from the lengths on the device.  A unit cut by shares leaves partial results
// (maximum, sum, weighted values, FP32) in the workspace; the part that arrives last joins them in order.
//
// Bound: cache bytes, tokens * (head_dim + 8) per kv head.
#include "kv4_attention.cuh"

namespace fth {
namespace kv4 {

namespace {

using namespace rowops;

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kWarpTokens = 32;
constexpr int kTile = kWarps * kWarpTokens;
constexpr float kNoMax = -1e30f;      // below every score, and finite: differences stay numbers
constexpr float kLazy = 8.0f;         // a running maximum may lag by 2^8 before sums are rescaled

__device__ __forceinline__ void CopyAsync16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void CopyAsync8(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void CopyAsync4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void CopyCommit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void CopyWait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void MmaF16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t Transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float Exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t PackHalf(float low, float high) {
    const __half2 h = __floats2half2_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float PowerOfTwo(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

template <int D>
struct Shape {
    static constexpr int kWords = D / 32;            // packed words a lane holds of a token (K) or of a pair of tokens (V)
    static constexpr int kStages = D == 256 ? 3 : 4;
    // a stage of a warp's ring: per 16 tokens two K rows and two V rows of kWords words for each lane, then 32 parameters
    static constexpr int kSubBytes = 4 * kWords * 4 * 32;
    static constexpr int kStageBytes = 2 * kSubBytes + 2 * 128;
    static constexpr int kRingBytes = kStages * kStageBytes;
};

template <int D, int NT>
constexpr size_t DecodeSmem() {
    const size_t ring = static_cast<size_t>(kWarps) * Shape<D>::kRingBytes;
    const size_t join = static_cast<size_t>(kWarps) * 8 * NT * (D + 2) * sizeof(float);
    return ring > join ? ring : join;
}

// Sum of v over the block, and the sum over the threads before this one.
__device__ __forceinline__ int64_t ScanWork(int64_t v, int64_t* shared, int64_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t n = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += n;
    }
    __syncthreads();
    if (lane == 31) shared[warp] = s;
    __syncthreads();
    int64_t before = 0, all = 0;
    for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {
        if (w < warp) before += shared[w];
        all += shared[w];
    }
    *total = all;
    return before + s - v;
}

// Tiles of all units of one kv head of a request.
template <int TILE>
__device__ __forceinline__ int64_t RequestTiles(const AttentionParams& p, const Request& r, int unit_rows) {
    int64_t sum = 0;
    for (int row = 0; row < r.rows; row += unit_rows) {
        int a, b;
        UnitTiles<TILE>(p, r, row, unit_rows, &a, &b);
        sum += b - a;
    }
    return sum;
}

// One lane's place in the cache for the 16 tokens that start at `token` (a multiple of 16 within a block).
template <int D>
__device__ __forceinline__ void IssueSub(const AttentionParams& p, uint32_t ring, int64_t base, int offset, int lane) {
    constexpr int W = Shape<D>::kWords;
    const int g = lane >> 2, quad = lane & 3;
    const uint8_t* k = p.cache.k_codes + (base + offset) * (D / 2);
    const uint8_t* v = p.cache.v_codes + (base + offset) * (D / 2);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const uint8_t* krow = k + (g + 8 * half) * (D / 2);
        const uint8_t* vrow = v + (quad + 4 * half) * D;
        const uint32_t dk = ring + half * (W * 128), dv = ring + (2 + half) * (W * 128);
        if constexpr (W == 2) {
            CopyAsync8(dk + lane * 8, krow + quad * 8);
            CopyAsync8(dv + lane * 8, vrow + g * 8);
        } else {
#pragma unroll
            for (int c = 0; c < W / 4; ++c) {
                CopyAsync16(dk + c * 512 + lane * 16, krow + c * 64 + quad * 16);
                CopyAsync16(dv + c * 512 + lane * 16, vrow + c * 128 + g * 16);
            }
        }
    }
}
template <int W>
__device__ __forceinline__ void LoadWords(const uint8_t* at, int lane, uint32_t (&w)[W]) {
    if constexpr (W == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(at + lane * 8);
        w[0] = x.x;
        w[1] = x.y;
    } else {
#pragma unroll
        for (int c = 0; c < W / 4; ++c) {
            const uint4 x = *reinterpret_cast<const uint4*>(at + c * 512 + lane * 16);
            w[4 * c] = x.x;
            w[4 * c + 1] = x.y;
            w[4 * c + 2] = x.z;
            w[4 * c + 3] = x.w;
        }
    }
}

template <int D, int DTYPE, int NT>
__global__ void __launch_bounds__(kThreads) DecodeKernel(const __grid_constant__ AttentionParams p) {
    constexpr int W = Shape<D>::kWords;
    constexpr int S = Shape<D>::kStages;
    constexpr int R = 8 * NT;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int64_t scan[kWarps];
    __shared__ int start_request;
    __shared__ int64_t start_offset;
    __shared__ int join_last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, quad = lane & 3;
    WaitForPrevious();

    // ---- this block's share of the tiles --------------------------------------------------------------------------------
    int64_t work = 0, mine = 0, before = 0;
    for (int base = 0; base < p.requests; base += kThreads) {
        const int b = base + threadIdx.x;
        mine = 0;
        if (b < p.requests) mine = RequestTiles<kTile>(p, LoadRequest(p, b), R) * p.kv_heads;
        int64_t total;
        before = ScanWork(mine, scan, &total);
        work += total;
    }
    int64_t per = (work + gridDim.x - 1) / gridDim.x;
    if (per < 2) per = 2;
    const int64_t share_begin = blockIdx.x * per;
    const int64_t share_end = share_begin + per < work ? share_begin + per : work;
    if (share_begin >= share_end) return;
    int64_t passed = 0;
    for (int base = 0; base < p.requests; base += kThreads) {
        int64_t total = work;
        if (p.requests > kThreads) {
            const int b = base + threadIdx.x;
            mine = 0;
            if (b < p.requests) mine = RequestTiles<kTile>(p, LoadRequest(p, b), R) * p.kv_heads;
            before = ScanWork(mine, scan, &total);
        }
        if (share_begin >= passed + before && share_begin < passed + before + mine) {
            start_request = base + threadIdx.x;
            start_offset = share_begin - passed - before;
        }
        passed += total;
        if (passed > share_begin) break;
    }
    __syncthreads();

    // ---- the first unit: request, head, rows, tiles ---------------------------------------------------------------------
    int b = start_request;
    Request req = LoadRequest(p, b);
    const int64_t per_head = RequestTiles<kTile>(p, req, R);
    int head = static_cast<int>(start_offset / per_head);
    int row = 0;
    int64_t into = start_offset % per_head;  // tiles of the unit that other blocks take
    int tile_first, tile_last;
    for (;;) {
        UnitTiles<kTile>(p, req, row, R, &tile_first, &tile_last);
        if (into < tile_last - tile_first) break;
        into -= tile_last - tile_first;
        row += R;
    }
    int64_t at = share_begin;
    const uint32_t ring = SmemAddr(smem) + warp * Shape<D>::kRingBytes;
    uint8_t* ring_ptr = smem + warp * Shape<D>::kRingBytes;

    for (;;) {
        const int64_t unit_begin = at - into;
        const int64_t unit_end = unit_begin + (tile_last - tile_first);
        const int t0 = tile_first + static_cast<int>(into);
        const int64_t here = (unit_end < share_end ? unit_end : share_end) - at;
        const int t1 = t0 + static_cast<int>(here);

        // ---- query rows ----------------------------------------------------------------------------------------------------
        uint32_t qf[NT][2 * W][2];
        float f[NT][2], qsum[NT][2];   // of the columns 2 * quad, 2 * quad + 1
        int row_low[NT][2], row_high[NT][2];
        int all_low = 0, all_high = 0x7fffffff;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int r = row + n * 8 + g;
            const bool valid = r < req.rows;
            const int query = valid ? r / p.group : 0;
            const int64_t from = valid ? (req.first_row + static_cast<int64_t>(query)) * p.ldq + (static_cast<int64_t>(head) * p.group + r % p.group) * D : 0;
            float x[W][8];
            float big = 0.0f, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const int word = W == 2 ? quad * 2 + w : (w >> 2) * 16 + quad * 4 + (w & 3);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    x[w][i] = valid ? ReadFloat<DTYPE>(p.q, from + word * 8 + i) : 0.0f;
                    big = fmaxf(big, fabsf(x[w][i]));
                    sum += x[w][i];
                }
            }
#pragma unroll
            for (int o = 1; o < 4; o <<= 1) {
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                sum += __shfl_xor_sync(0xffffffffu, sum, o);
            }
            int e = 14 - (static_cast<int>((__float_as_uint(big) >> 23) & 0xffu) - 127);
            if (big == 0.0f) e = 0;
            e = e > 120 ? 120 : e < -86 ? -86 : e;
            const float up = PowerOfTwo(e);
#pragma unroll
            for (int w = 0; w < W; ++w) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[w][i] *= (i & 1) ? up * 0.0625f : up;
                qf[n][2 * w][0] = PackHalf(x[w][0], x[w][4]);
                qf[n][2 * w][1] = PackHalf(x[w][1], x[w][5]);
                qf[n][2 * w + 1][0] = PackHalf(x[w][2], x[w][6]);
                qf[n][2 * w + 1][1] = PackHalf(x[w][3], x[w][7]);
            }
            const float back = p.scale_log2 * PowerOfTwo(24 - e), weighted = p.scale_log2 * sum;
            int low = 0, high = 0;
            if (valid) Visible(p, req, query, &low, &high);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int from_lane = (quad * 2 + c) * 4;
                f[n][c] = __shfl_sync(0xffffffffu, back, from_lane);
                qsum[n][c] = __shfl_sync(0xffffffffu, weighted, from_lane);
                row_low[n][c] = __shfl_sync(0xffffffffu, low, from_lane);
                row_high[n][c] = __shfl_sync(0xffffffffu, high, from_lane);
            }
            if (valid) {
                all_low = low > all_low ? low : all_low;
                all_high = high < all_high ? high : all_high;
            }
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            const int l = __shfl_xor_sync(0xffffffffu, all_low, o), h = __shfl_xor_sync(0xffffffffu, all_high, o);
            all_low = l > all_low ? l : all_low;
            all_high = h < all_high ? h : all_high;
        }
        int first_low, last_high, unused;
        Visible(p, req, row / p.group, &first_low, &unused);
        Visible(p, req, ((row + R < req.rows ? row + R : req.rows) - 1) / p.group, &unused, &last_high);

        // ---- tokens -----------------------------------------------------------------------------------------------------------
        float acc[NT][2 * W][4];
        float top[NT][2], sum[NT][2], offset[NT][2];
        float shrink = 1.0f;   // value scales are multiplied by this power of two before they become FP16
        float scale_limit = 0.0f;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int m = 0; m < 2 * W; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[n][m][i] = 0.0f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                top[n][c] = kNoMax;
                sum[n][c] = offset[n][c] = 0.0f;
            }
        }
        const int steps = t1 - t0;
        const int32_t* table = p.table + static_cast<int64_t>(b) * p.max_blocks;
        uint32_t have = 0;   // two bits per stage: the block of these 16 tokens exists
        int id[2];
        const auto lookup = [&](int step) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int token = (t0 + step) * kTile + warp * kWarpTokens + s * 16;
                id[s] = -2;
                if (step < steps && token < last_high && token + 16 > first_low) id[s] = table[token >> p.cache.block_shift];
            }
        };
        const auto issue = [&](int step) {
            const int stage = step % S;
            have &= ~(3u << (2 * stage));
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int token = (t0 + step) * kTile + warp * kWarpTokens + s * 16;
                if (id[s] >= 0 && id[s] < p.cache.blocks) {
                    have |= 1u << (2 * stage + s);
                    const int64_t base = HeadBase(p.cache, id[s], head);
                    const int off = token & ((1 << p.cache.block_shift) - 1);
                    const uint32_t dst = ring + stage * Shape<D>::kStageBytes;
                    IssueSub<D>(p, dst + s * Shape<D>::kSubBytes, base, off, lane);
                    const uint32_t* params = (lane < 16 ? p.cache.k_params : p.cache.v_params) + base + off + (lane & 15);
                    CopyAsync4(dst + 2 * Shape<D>::kSubBytes + s * 128 + lane * 4, params);
                } else if (id[s] != -2 && lane == 0) {
                    ReportTimeout(p.status, kSiteAttention, b);
                }
            }
            CopyCommit();
        };
        lookup(0);
#pragma unroll
        for (int s = 0; s < S - 1; ++s) {
            issue(s);
            lookup(s + 1);
        }
        for (int step = 0; step < steps; ++step) {
            CopyWait<S - 2>();
            __syncwarp();
            issue(step + S - 1);
            lookup(step + S);
            const int stage = step % S;
            const uint8_t* data = ring_ptr + stage * Shape<D>::kStageBytes;
            const uint32_t* params = reinterpret_cast<const uint32_t*>(data + 2 * Shape<D>::kSubBytes);
            const uint32_t present = (have >> (2 * stage)) & 3u;
            if (present == 0) continue;
            const int token0 = (t0 + step) * kTile + warp * kWarpTokens;

            // scores, as exponents of two
            float z[2][NT][4];
            uint32_t kp[2][2], vp[2][2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                uint32_t k0[W], k1[W];
                LoadWords<W>(data + s * Shape<D>::kSubBytes, lane, k0);
                LoadWords<W>(data + s * Shape<D>::kSubBytes + W * 128, lane, k1);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    kp[s][h] = params[s * 32 + g + 8 * h];
                    vp[s][h] = params[s * 32 + 16 + g + 8 * h];
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[s][n][i] = 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint32_t x0 = k0[w], x1 = k1[w], y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        MmaF16(z[s][n], x0 & 0x000f000fu, x1 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x00f000f0u, qf[n][2 * w][0], qf[n][2 * w][1]);
                        MmaF16(z[s][n], y0 & 0x000f000fu, y1 & 0x000f000fu, y0 & 0x00f000f0u, y1 & 0x00f000f0u, qf[n][2 * w + 1][0], qf[n][2 * w + 1][1]);
                    }
                }
            }
            const bool inside = token0 >= all_low && token0 + kWarpTokens <= all_high && present == 3u;
            bool rescale = false;
            float vs[2][2], vm[2][2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float ks = ParamScale(kp[s][h]), km = ParamMin(kp[s][h]);
                    vs[s][h] = ParamScale(vp[s][h]);
                    vm[s][h] = ParamMin(vp[s][h]);
                    bool seen_by_any = inside;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float& score = z[s][n][2 * h + c];
                            score = fmaf(ks, score * f[n][c], km * qsum[n][c]);
                            if (!inside) {
                                const int token = token0 + s * 16 + h * 8 + g;
                                const bool seen = ((present >> s) & 1u) != 0 && token >= row_low[n][c] && token < row_high[n][c];
                                if (!seen) score = -INFINITY;
                                seen_by_any = seen_by_any || seen;
                            }
                            rescale = rescale || score > top[n][c] + kLazy;
                        }
                    }
                    if (!seen_by_any) vs[s][h] = vm[s][h] = 0.0f;  // whatever stands there: 0 * NaN is no zero
                    rescale = rescale || vs[s][h] > scale_limit;
                }
            }
            if (__any_sync(0xffffffffu, rescale)) {
                float biggest = scale_limit * 0.5f;
#pragma unroll
                for (int s = 0; s < 2; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (vs[s][h] > biggest) biggest = vs[s][h];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) biggest = fmaxf(biggest, __shfl_xor_sync(0xffffffffu, biggest, o));
                float change = 1.0f;
                if (biggest > scale_limit) {
                    // 2^e > biggest: with probabilities up to 2^8 the products stay below 2^15
                    int e = static_cast<int>((__float_as_uint(biggest) >> 23) & 0xffu) - 126;
                    e = e > 120 ? 120 : e < -100 ? -100 : e;
                    const float next = PowerOfTwo(7 - e);
                    change = scale_limit == 0.0f ? 0.0f : next / shrink;
                    shrink = next;
                    scale_limit = PowerOfTwo(e);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float factor[2];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float best = top[n][c];
#pragma unroll
                        for (int s = 0; s < 2; ++s) best = fmaxf(best, fmaxf(z[s][n][c], z[s][n][2 + c]));
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
                        const float alpha = Exp2(top[n][c] - best);
                        top[n][c] = best;
                        sum[n][c] *= alpha;
                        offset[n][c] *= alpha;
                        factor[c] = alpha * change;
                    }
#pragma unroll
                    for (int m = 0; m < 2 * W; ++m) {
                        acc[n][m][0] *= factor[0];
                        acc[n][m][1] *= factor[1];
                        acc[n][m][2] *= factor[0];
                        acc[n][m][3] *= factor[1];
                    }
                }
            }
            // probabilities and weighted values
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                uint32_t pt[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float weight[2];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const float prob = Exp2(z[s][n][2 * h + c] - top[n][c]);
                            sum[n][c] += prob;
                            offset[n][c] = fmaf(prob, vm[s][h], offset[n][c]);
                            weight[c] = prob * (vs[s][h] * shrink);
                        }
                        pt[n][h] = Transpose8x8(PackHalf(weight[0], weight[1]));
                    }
                }
                uint32_t v0[W], v1[W];
                LoadWords<W>(data + s * Shape<D>::kSubBytes + 2 * W * 128, lane, v0);
                LoadWords<W>(data + s * Shape<D>::kSubBytes + 3 * W * 128, lane, v1);
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const uint32_t x0 = v0[w], x1 = v1[w], y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        MmaF16(acc[n][2 * w], x0 & 0x000f000fu, x0 & 0x00f000f0u, x1 & 0x000f000fu, x1 & 0x00f000f0u, pt[n][0], pt[n][1]);
                        MmaF16(acc[n][2 * w + 1], y0 & 0x000f000fu, y0 & 0x00f000f0u, y1 & 0x000f000fu, y1 & 0x00f000f0u, pt[n][0], pt[n][1]);
                    }
                }
            }
        }
        CopyWait<0>();

        // ---- the four warps' results together ---------------------------------------------------------------------------------
        // [warp][row][D values, maximum, sum], in the rings' memory
        float* join = reinterpret_cast<float*>(smem);
        __syncthreads();
        {
            const float unit = PowerOfTwo(24) / shrink;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) {
                        sum[n][c] += __shfl_xor_sync(0xffffffffu, sum[n][c], o);
                        offset[n][c] += __shfl_xor_sync(0xffffffffu, offset[n][c], o);
                    }
                    float* out = join + static_cast<size_t>(warp * R + n * 8 + quad * 2 + c) * (D + 2);
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        const int word = W == 2 ? g * 2 + w : (w >> 2) * 32 + g * 4 + (w & 3);
                        out[word * 4] = fmaf(acc[n][2 * w][c], unit, offset[n][c]);
                        out[word * 4 + 1] = fmaf(acc[n][2 * w][2 + c], unit * 0.0625f, offset[n][c]);
                        out[word * 4 + 2] = fmaf(acc[n][2 * w + 1][c], unit, offset[n][c]);
                        out[word * 4 + 3] = fmaf(acc[n][2 * w + 1][2 + c], unit * 0.0625f, offset[n][c]);
                    }
                    if (g == 0) {
                        out[D] = top[n][c];
                        out[D + 1] = sum[n][c];
                    }
                }
            }
        }
        __syncthreads();
        const int64_t part_first = unit_begin / per, part_last = (unit_end - 1) / per;
        const bool whole = part_first == part_last;
        const int valid_rows = req.rows - row < R ? req.rows - row : R;
        const int64_t slot_floats = static_cast<int64_t>(R) * (D + 2);
        float* partial = p.partials + (static_cast<int64_t>(blockIdx.x) * 2 + (blockIdx.x == part_first ? 1 : 0)) * slot_floats;
        for (int i = threadIdx.x; i < valid_rows * D; i += kThreads) {
            const int r = i / D, d = i - r * D;
            float best = kNoMax;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) best = fmaxf(best, join[(w * R + r) * (D + 2) + D]);
            float total = 0.0f, value = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float* from = join + (w * R + r) * (D + 2);
                const float weight = Exp2(from[D] - best);
                total = fmaf(weight, from[D + 1], total);
                value = fmaf(weight, from[d], value);
            }
            if (whole) {
                const int query = (row + r) / p.group;
                const int64_t q_row = req.first_row + static_cast<int64_t>(query);
                const int q_head = head * p.group + (row + r) % p.group;
                WriteFloat<DTYPE>(p.out, q_row * p.ldo + static_cast<int64_t>(q_head) * D + d, total == 0.0f ? 0.0f : value / total);
                if (d == 0 && p.lse != nullptr)
                    p.lse[q_row * p.kv_heads * p.group + q_head] = total == 0.0f ? -INFINITY : (best + log2f(total)) * 0.6931471805599453f;
            } else {
                partial[r * (D + 2) + d] = value;
                if (d == 0) {
                    partial[r * (D + 2) + D] = best;
                    partial[r * (D + 2) + D + 1] = total;
                }
            }
        }
        if (!whole) {
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                const int parts = static_cast<int>(part_last - part_first) + 1;
                join_last = atomicAdd(&p.counters[part_first], 1) == parts - 1;
                if (join_last) p.counters[part_first] = 0;
            }
            __syncthreads();
            if (join_last) {
                __threadfence();
                for (int i = threadIdx.x; i < valid_rows * D; i += kThreads) {
                    const int r = i / D, d = i - r * D;
                    float best = kNoMax, total = 0.0f, value = 0.0f;
                    for (int64_t c = part_first; c <= part_last; ++c) {
                        const float* from = p.partials + (c * 2 + (c == part_first ? 1 : 0)) * slot_floats + r * (D + 2);
                        const float m = __ldcg(from + D), next = fmaxf(best, m);
                        const float old = Exp2(best - next), now = Exp2(m - next);
                        total = fmaf(now, __ldcg(from + D + 1), total * old);
                        value = fmaf(now, __ldcg(from + d), value * old);
                        best = next;
                    }
                    const int query = (row + r) / p.group;
                    const int64_t q_row = req.first_row + static_cast<int64_t>(query);
                    const int q_head = head * p.group + (row + r) % p.group;
                    WriteFloat<DTYPE>(p.out, q_row * p.ldo + static_cast<int64_t>(q_head) * D + d, total == 0.0f ? 0.0f : value / total);
                    if (d == 0 && p.lse != nullptr)
                        p.lse[q_row * p.kv_heads * p.group + q_head] = total == 0.0f ? -INFINITY : (best + log2f(total)) * 0.6931471805599453f;
                }
            }
        }
        __syncthreads();  // the rings are free again

        at += here;
        if (at >= share_end) break;
        // the next unit
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
        UnitTiles<kTile>(p, req, row, R, &tile_first, &tile_last);
    }
}

bool Aligned16Strided(const void* p, int64_t ld) { return AlignedTo(p, 16) && ld % 8 == 0; }

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
    if (!AlignedTo(d->q, 2) || !AlignedTo(d->out, 2) || !AlignedTo(d->lse, 4)) return FTH_B200_ERR_INVALID;
    if (d->tokens > 0x7fffffff || d->q_heads > 65536 || static_cast<int64_t>(d->max_query) * (d->q_heads / d->cache.kv_heads) > 0x7fffffff)
        return FTH_B200_ERR_UNSUPPORTED;
    if (static_cast<int64_t>(d->max_blocks) * d->cache.block_size > 0x7fffffff) return FTH_B200_ERR_UNSUPPORTED;
    return FTH_B200_OK;
}

// Query rows of a unit, in eights: 8 when no request has more.
int DecodeTiles(const fth_b200_kv4_attention_desc& d) {
    return static_cast<int64_t>(d.max_query) * (d.q_heads / d.cache.kv_heads) <= 8 ? 1 : 2;
}
// Blocks of threads that are resident together.
int DecodeGrid(const fth_b200_kv4_attention_desc& d) { return SmCount() * (d.cache.head_dim == 256 ? 2 : 3); }

constexpr size_t kCounterBytes = 4096;

size_t WorkspaceBytes(const fth_b200_kv4_attention_desc& d) {
    return kCounterBytes + static_cast<size_t>(DecodeGrid(d)) * 2 * 8 * DecodeTiles(d) * (d.cache.head_dim + 2) * sizeof(float);
}

template <int D, int DTYPE>
int LaunchDecode(const AttentionParams& p, int tiles, int grid, cudaStream_t s) {
    const auto run = [&](auto kernel, size_t smem) {
        if (EnsureDynamicSmem(reinterpret_cast<const void*>(kernel), smem) != FTH_B200_OK) return static_cast<int>(FTH_B200_ERR_CUDA);
        return Launch(kernel, dim3(static_cast<unsigned>(grid)), kThreads, smem, s, p);
    };
    return tiles == 1 ? run(DecodeKernel<D, DTYPE, 1>, DecodeSmem<D, 1>()) : run(DecodeKernel<D, DTYPE, 2>, DecodeSmem<D, 2>());
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
    p.causal = d->causal != 0;
    p.window = d->window;
    p.scale_log2 = d->scale * 1.4426950408889634f;
    p.status = DeviceStatusPtr();
    p.counters = static_cast<int*>(d->workspace);
    p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(d->workspace) + kv4::kCounterBytes);
    auto s = static_cast<cudaStream_t>(stream);
    const int tiles = kv4::DecodeTiles(*d), grid = kv4::DecodeGrid(*d);
    int status;
    if (d->dtype == FTH_B200_BF16) {
        if (d->cache.head_dim == 64) status = kv4::LaunchDecode<64, FTH_B200_BF16>(p, tiles, grid, s);
        else if (d->cache.head_dim == 128) status = kv4::LaunchDecode<128, FTH_B200_BF16>(p, tiles, grid, s);
        else status = kv4::LaunchDecode<256, FTH_B200_BF16>(p, tiles, grid, s);
    } else {
        if (d->cache.head_dim == 64) status = kv4::LaunchDecode<64, FTH_B200_FP16>(p, tiles, grid, s);
        else if (d->cache.head_dim == 128) status = kv4::LaunchDecode<128, FTH_B200_FP16>(p, tiles, grid, s);
        else status = kv4::LaunchDecode<256, FTH_B200_FP16>(p, tiles, grid, s);
    }
    if (status == FTH_B200_OK) NoteLaunch("kv4_attention");
    return status;
}
