// What the two attention kernels over the 4-bit cache share: their parameters, the rows and tokens of a request, the flat
// list of work that is dealt out in equal shares, and the joining of partial results.
#pragma once

#include "kv4.cuh"

namespace fth {
namespace kv4 {

constexpr int kSiteAttention = 42, kSiteAttentionWait = 43;
constexpr float kLazy = 8.0f;     // a running maximum may lag by 2^8 before sums are rescaled
constexpr float kNotStarted = -INFINITY;
constexpr float kNoMax = -3.402823466e38f;  // the maximum of no scores: not above any, and finite, so that kNoMax - kNoMax is 0

struct AttentionParams {
    Cache cache;
    const void* q;
    void* out;
    float* lse;
    int64_t ldq, ldo, tokens;
    const int32_t* table;
    const int32_t* total_lens;
    const int32_t* query_start;
    int requests, max_blocks, max_query, kv_heads, group, causal, window, q_vec, out_vec;
    uint32_t group_inverse;  // floor((2^32 - 1) / group)
    int few_units;     // no request has more than a few units of rows
    float scale_log2;  // scale * log2(e): scores are kept as exponents of two
    int* status;
    int* counters;     // one per block of threads: arrivals of the parts of the unit that begins in it
    float* partials;   // [block of threads][2][rows of a unit][head_dim values, maximum, unused, sum, sum for the lse]
};

// row / group.  The product is at most one short: row / group - row * inverse / 2^32 < (row / 2^32) * 2 <= 1.
__device__ __forceinline__ int QueryOf(const AttentionParams& p, int row) {
    const uint32_t q = __umulhi(static_cast<uint32_t>(row), p.group_inverse);
    return static_cast<int>(q + (static_cast<uint32_t>(row) - q * static_cast<uint32_t>(p.group) >= static_cast<uint32_t>(p.group) ? 1u : 0u));
}
// The rows of one request and what they see.  Row i of n stands at position total - n + i.
struct Request {
    int first_row;  // row of its first query in q
    int queries;
    int rows;       // queries * group: (query, head of the group), heads innermost
    int length;     // tokens that the table can hold
    int total;
};
__device__ __forceinline__ Request LoadRequest(const AttentionParams& p, int b) {
    Request r;
    r.first_row = b;
    int end = b + 1;
    if (p.query_start != nullptr) {
        r.first_row = p.query_start[b];
        end = p.query_start[b + 1];
    }
    const int limit = static_cast<int>(p.tokens);
    if (r.first_row < 0 || r.first_row >= limit) r.first_row = end = 0;
    // rows are the request's last tokens: those beyond max_query or behind `tokens` are not computed, the others keep their positions
    const int given = end > r.first_row ? end - r.first_row : 0;
    int n = given > p.max_query ? p.max_query : given;
    if (n > limit - r.first_row) n = limit - r.first_row;
    r.total = p.total_lens[b] - (given - n);
    r.queries = n;
    r.rows = n * p.group;
    const int64_t room = static_cast<int64_t>(p.max_blocks) << p.cache.block_shift;
    r.length = p.total_lens[b] < 0 ? 0 : p.total_lens[b] > room ? static_cast<int>(room) : p.total_lens[b];
    return r;
}
// Tokens [low, high) that query i of the request sees (high <= low: none).
__device__ __forceinline__ void Visible(const AttentionParams& p, const Request& r, int query, int* low, int* high) {
    const int position = r.total - r.queries + query;
    int h = r.length;
    if (p.causal && position + 1 < h) h = position + 1;
    int l = 0;
    if (p.window > 0 && position + 1 > p.window) l = position + 1 - p.window;
    *low = l;
    *high = h;
}
// Token tiles [first, last) of the unit that holds rows [row, row + count) of a request; at least one, so that a unit
// whose rows see nothing is still somebody's to write.
template <int TILE>
__device__ __forceinline__ void UnitTiles(const AttentionParams& p, const Request& r, int row, int count, int* first, int* last) {
    int end = row + count;
    if (end > r.rows) end = r.rows;
    int l0, h0, l1, h1;
    Visible(p, r, QueryOf(p, row), &l0, &h0);
    Visible(p, r, QueryOf(p, end - 1), &l1, &h1);
    *first = l0 / TILE;
    *last = h1 > 0 ? (h1 + TILE - 1) / TILE : 0;
    if (*last <= *first) *last = *first + 1;
}

// a / b of numbers that are not negative; most fit 32 bits, whose division is much shorter.
__device__ __forceinline__ int64_t Divide(int64_t a, int64_t b) {
    return ((a | b) >> 31) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}

// Sum of v over the warp.
__device__ __forceinline__ int64_t WarpSum(int64_t v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// ---- arithmetic -----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void MmaF16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The first of a sum: c is written, not read.
__device__ __forceinline__ void MmaF16First(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t Transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float Exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float PowerOfTwo(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// |x|, 0 for what is not finite: an infinity spoils its own row, and must not take the others' bits by the power of two.
__device__ __forceinline__ float FiniteAbs(float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.0f; }
// Power of two that brings the largest query element to [2^14, 2^15); 24 - e stays an FP32 exponent.
__device__ __forceinline__ int QueryExponent(float biggest) {
    if (biggest == 0.0f) return 0;
    const int e = 14 - (static_cast<int>((__float_as_uint(biggest) >> 23) & 0xffu) - 127);
    return e > 120 ? 120 : e < -86 ? -86 : e;
}
// 2^e > biggest: shrunk by 2^(7 - e), value scales stay below 2^7 and weights with probabilities up to 2^8 below 2^15.
__device__ __forceinline__ int ScaleExponent(float biggest) {
    const int e = static_cast<int>((__float_as_uint(biggest) >> 23) & 0xffu) - 126;
    return e > 120 ? 120 : e < -100 ? -100 : e;
}
// Eight query elements in the order a word of eight codes gives its operands: (0, 4), (1, 5) * odd, (2, 6), (3, 7) * odd.
template <int DTYPE>
__device__ __forceinline__ void QueryOperands(const uint32_t (&raw)[4], float up, float odd, uint32_t (&f)[4]) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = HalfPair<DTYPE>(raw[i]);
        x[2 * i] = v.x * up;
        x[2 * i + 1] = v.y * (up * odd);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = PackHalf(x[i], x[i + 4]);
}
__device__ __forceinline__ uint4 LoadUnaligned8(const uint16_t* from) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = from[2 * i] | (static_cast<uint32_t>(from[2 * i + 1]) << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// Copy of `bytes` (a multiple of 16) contiguous bytes, both addresses 16-byte aligned; the bytes are reported to `bar`.
__device__ __forceinline__ void BulkLoad(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(SmemAddr(dst)), "l"(src), "r"(bytes), "r"(SmemAddr(bar)) : "memory");
}

// Floats of a row of partial results.
template <int D>
constexpr int kRow = D + 4;

// ---- results ---------------------------------------------------------------------------------------------------------------
// Elements d .. d + 3 of row `row` of the request: value / total, and the row's lse (mass: the sum of its probabilities)
// with its first elements.
template <int D, int DTYPE>
__device__ __forceinline__ void StoreFour(const AttentionParams& p, const Request& req, int head, int row, int d, float4 v, float total, float best, float mass) {
    const int query = QueryOf(p, row);
    const int64_t q_row = req.first_row + static_cast<int64_t>(query);
    const int q_head = head * p.group + row - query * p.group;
    const float scale = total == 0.0f ? 0.0f : __fdiv_rn(1.0f, total);
    const float x[4] = {v.x * scale, v.y * scale, v.z * scale, v.w * scale};
    const int64_t at = q_row * p.ldo + static_cast<int64_t>(q_head) * D + d;
    if (p.out_vec) {
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = make_uint2(PackTo<DTYPE>(x[0], x[1]), PackTo<DTYPE>(x[2], x[3]));
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) rowops::WriteFloat<DTYPE>(p.out, at + i, x[i]);
    }
    if (d == 0 && p.lse != nullptr)
        p.lse[q_row * p.kv_heads * p.group + q_head] = total == 0.0f ? -INFINITY : (best + log2f(mass)) * 0.6931471805599453f;
}
__device__ __forceinline__ void FmaFour(float4& a, float w, float4 x) {
    a.x = fmaf(w, x.x, a.x);
    a.y = fmaf(w, x.y, a.y);
    a.z = fmaf(w, x.z, a.z);
    a.w = fmaf(w, x.w, a.w);
}
// Joins the parts of a unit, in order: part i is slot 1 of block `first` for i = 0 and slot 0 of block first + i behind it.
// Every part's weight is computed once into shared memory, by as many lanes per row as there are parts; the values are then
// read sixteen bytes at a time, four pieces by four parts in flight together.  `sync` is a barrier of the THREADS threads (thread = 0 .. THREADS - 1) that call this.
template <int D, int DTYPE, int THREADS, typename Sync>
__device__ __forceinline__ void JoinParts(const AttentionParams& p, const Request& req, int head, int row, int rows, const float* partials, int first, int parts,
                                          int64_t slot_floats, float* shared, int shared_floats, int thread, Sync sync) {
    const float* base = partials + (static_cast<int64_t>(first) * 2 + 1) * slot_floats;  // part i > 0 lies 2 i - 1 slots behind
    const auto slot = [&](int i) { return base + (i == 0 ? 0 : 2 * static_cast<int64_t>(i) - 1) * slot_floats; };
    int at_once = shared_floats / (parts + 3);   // rows
    if (at_once > rows) at_once = rows;
    if (at_once < 1) return;                     // cannot be: shared memory is sized for it
    float* best_of = shared;                     // [at_once] maximum, sum, sum for the lse
    float* weights = shared + 3 * at_once;       // [at_once][parts]
    int lanes = 1;                               // that share a row
    while (lanes < parts && lanes < 32) lanes <<= 1;
    const int i0 = thread & (lanes - 1);
    for (int r0 = 0; r0 < rows; r0 += at_once) {
        const int count = rows - r0 < at_once ? rows - r0 : at_once;
        sync();
        for (int first_row = 0; first_row < count; first_row += THREADS / lanes) {
            const int r = first_row + thread / lanes;
            float best = kNoMax, total = 0.0f, mass = 0.0f;
            if (r < count) {
#pragma unroll 4
                for (int i = i0; i < parts; i += lanes) {
                    const float4 v = __ldcg(reinterpret_cast<const float4*>(slot(i) + (r0 + r) * kRow<D> + D));
                    weights[r * parts + i] = v.x;
                    const float next = fmaxf(best, v.x), old = Exp2(best - next), now = Exp2(v.x - next);
                    total = fmaf(now, v.z, total * old);
                    mass = fmaf(now, v.w, mass * old);
                    best = next;
                }
            }
            __syncwarp();
            for (int o = lanes >> 1; o > 0; o >>= 1) {
                const float b = __shfl_xor_sync(0xffffffffu, best, o), t = __shfl_xor_sync(0xffffffffu, total, o), m = __shfl_xor_sync(0xffffffffu, mass, o);
                const float next = fmaxf(best, b), old = Exp2(best - next), now = Exp2(b - next);
                total = fmaf(now, t, total * old);
                mass = fmaf(now, m, mass * old);
                best = next;
            }
            if (r < count) {
                for (int i = i0; i < parts; i += lanes) weights[r * parts + i] = Exp2(weights[r * parts + i] - best);
                if (i0 == 0) {
                    best_of[r] = best;
                    best_of[at_once + r] = total;
                    best_of[2 * at_once + r] = mass;
                }
            }
        }
        sync();
        constexpr int kFours = 4;                // of a thread at a time
        for (int i = thread; i < count * (D / 4); i += kFours * THREADS) {
            float4 value[kFours];
            int r[kFours], d[kFours];
#pragma unroll
            for (int j = 0; j < kFours; ++j) {
                r[j] = (i + j * THREADS) / (D / 4);
                d[j] = (i + j * THREADS - r[j] * (D / 4)) * 4;
                if (r[j] >= count) r[j] = -1;
                value[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll 4
            for (int c = 0; c < parts; ++c) {
                const float* from = slot(c);
#pragma unroll
                for (int j = 0; j < kFours; ++j)
                    if (r[j] >= 0) FmaFour(value[j], weights[r[j] * parts + c], __ldcg(reinterpret_cast<const float4*>(from + (r0 + r[j]) * kRow<D> + d[j])));
            }
#pragma unroll
            for (int j = 0; j < kFours; ++j)
                if (r[j] >= 0) StoreFour<D, DTYPE>(p, req, head, row + r0 + r[j], d[j], value[j], best_of[at_once + r[j]], best_of[r[j]], best_of[2 * at_once + r[j]]);
        }
    }
}

}  // namespace kv4
}  // namespace fth
