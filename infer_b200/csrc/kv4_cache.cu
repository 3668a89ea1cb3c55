// Storing keys and values in the 4-bit cache (with the rotary positions of q and k in the same launch, if asked for) and
// reading them back.
//
// A vector x of head_dim elements becomes codes c in 0 .. 15 with value m + s * c:
//   m = largest BF16 <= min(x),  s = smallest BF16 >= (max(x) - m) / 15,  c = nearest((x - m) / s), ties to even.
// m is never above min(x) and 15 s reaches max(x), so no code is clamped by more than rounding; for BF16 input m is min(x)
// itself.  Every border is decided exactly: an FP32 estimate of (x - m) / s is off by less than 2^-21 * 15 < 10^-5, so
// eight elements are looked at again, in 64 bits, only if one's estimate is within 10^-4 of a half.
// One pass over the data: 2 * tokens * kv_heads * head_dim * size bytes in, head_dim + 8 bytes per token and head out;
// a launch for single tokens.  Prompts, 16384 tokens of 8 heads of 128 in BF16: storing takes 36 us, 2.4 TB/s, 104 warp instructions a
// vector in 72 % of the issue slots.  Reading back takes 23 us, 3.6 TB/s, half of what memory gives: 62 % of the issue
// slots, and warps that wait for a lane's four bytes of codes, whose address stands behind a load of the slot.  With rope and 32 query
// heads 200 us (64 tokens: 5.0 us), more than fth_b200_rope and storing apart (69 + 36 us): 96 registers leave two blocks of threads
// on an SM and 41 % of the issue slots used.  A vector belongs to head_dim / 8 neighbouring lanes, eight elements each, so minimum
// and maximum are three to five shuffles (both in one word for 16-bit types) and a lane's codes are one 32-bit word.
#include <type_traits>

#include "kv4.cuh"

namespace fth {
namespace kv4 {

namespace {

using namespace rowops;

constexpr int kThreads = 256;
constexpr int kAppendBlocks = 4, kGatherBlocks = 6;   // on an SM at once
// Waits for a rank report under the same two sites; kBadSlot in the detail, which no rank reaches, tells a slot beyond the cache.
constexpr int kSiteAppend = 40, kSiteGather = 41, kBadSlot = 0x8000;
__device__ __forceinline__ void ReportSlot(int* status, int site, int64_t token) {
    ReportTimeout(status, site, kBadSlot | static_cast<int>(token & (kBadSlot - 1)));
}

struct AppendParams {
    Cache cache;
    int64_t slots_limit;
    int64_t tokens;
    const void* k;
    const void* v;
    int64_t ldk, ldv;
    const int32_t* slots;
    int* status;
    int block_tokens;  // tokens of one block of threads (with rope)
    int vec_k, vec_v, vec_q;
    int two;           // 1: two tokens at a time
    Rope rope;
};

__device__ __forceinline__ float Bf16At(uint32_t bits) { return __uint_as_float(bits << 16); }

// Largest BF16 <= x (x finite); -infinity below the range.
__device__ __forceinline__ uint32_t Bf16Floor(float x) {
    const uint32_t b = __float_as_uint(x);
    uint32_t h = b >> 16;
    if ((b & 0xffffu) != 0 && (b >> 31) != 0) ++h;  // toward -infinity grows the magnitude of a negative number
    return h;
}

// Smallest BF16 s with 15 s >= spread, at least 2^-126; 0 for spread = 0.  `spread` is the difference rounded up: 15 s has
// 12 bits, so it is an FP32 number and not below the difference exactly when it is not below that.  The estimate is off by
// less than 2^-22 of itself, so cut off to BF16 it is s or the one before.
__device__ __forceinline__ uint32_t ScaleBits(float spread) {
    if (!(spread > 0.0f)) return 0;
    uint32_t b = __float_as_uint(__fmul_rn(spread, 1.0f / 15.0f)) >> 16;
    if (b < 0x0080u) b = 0x0080u;
    return __fmul_rn(15.0f, Bf16At(b)) < spread ? b + 1 : b;
}

// One code, decided in 64 bits: nearest((x - minimum) / scale), ties to even.
__device__ __forceinline__ uint32_t ExactCode(float x, float minimum, float scale, float estimate) {
    const float fl = floorf(estimate);
    const double d = static_cast<double>(x) - static_cast<double>(minimum);
    const double border = (static_cast<double>(fl) + 0.5) * static_cast<double>(scale);
    const bool odd = (static_cast<int>(fl) & 1) != 0;
    return static_cast<uint32_t>(d > border || (d == border && odd) ? fl + 1.0f : fl);
}

// Smallest and largest of a vector whose elements LANES lanes hold, eight each; false if one is an infinity or a NaN.
template <int LANES>
__device__ __forceinline__ bool Range(const float (&x)[8], float* low, float* high) {
    float a = x[0], b = x[0], zero = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        a = fminf(a, x[i]);
        b = fmaxf(b, x[i]);
        zero = __fmaf_rn(x[i], 0.0f, zero);   // NaN after an infinity or a NaN
    }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
        a = fminf(a, __shfl_xor_sync(0xffffffffu, a, o));
        b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, o));
    }
    *low = a;
    *high = b;
    const uint32_t group = LANES == 32 ? 0xffffffffu : ((1u << (LANES & 31)) - 1u) << ((threadIdx.x & 31) / LANES * LANES);
    return (__ballot_sync(0xffffffffu, zero != 0.0f) & group) == 0;
}
// The same for 16-bit elements, two to a word: smallest and negated largest side by side, one shuffle for both.
template <int DTYPE>
__device__ __forceinline__ uint32_t Min2(uint32_t a, uint32_t b) {
    uint32_t d;
    if constexpr (DTYPE == FTH_B200_BF16) asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    else asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
template <int DTYPE, int LANES>
__device__ __forceinline__ bool Range(const uint32_t (&w)[4], float* low, float* high) {
    constexpr uint32_t kSigns = 0x80008000u, kExponent = DTYPE == FTH_B200_BF16 ? 0x7f80u : 0x7c00u;
    const uint32_t a = Min2<DTYPE>(Min2<DTYPE>(w[0], w[1]), Min2<DTYPE>(w[2], w[3]));
    const uint32_t b = Min2<DTYPE>(Min2<DTYPE>(w[0] ^ kSigns, w[1] ^ kSigns), Min2<DTYPE>(w[2] ^ kSigns, w[3] ^ kSigns));
    uint32_t r = Min2<DTYPE>(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) r = Min2<DTYPE>(r, __shfl_xor_sync(0xffffffffu, r, o));
    const float2 v = HalfPair<DTYPE>(r);
    *low = v.x;
    *high = -v.y;
    return (r & kExponent) != kExponent && (r >> 16 & kExponent) != kExponent;
}

// Eight elements of a lane as they were loaded: words of two for 16-bit types.
template <int DTYPE>
struct Eight {
    uint32_t w[DTYPE == FTH_B200_FP32 ? 8 : 4];
    __device__ __forceinline__ void Load(const void* from, int64_t at, bool vec) {
        if constexpr (DTYPE == FTH_B200_FP32) {
            float v[8];
            ReadEight<DTYPE>(from, at, vec, v);
            Set(v);
        } else if (vec) {
            const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(from) + at);
            w[0] = x.x;
            w[1] = x.y;
            w[2] = x.z;
            w[3] = x.w;
        } else {
            const uint16_t* e = static_cast<const uint16_t*>(from) + at;
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = e[2 * i] | (static_cast<uint32_t>(e[2 * i + 1]) << 16);
        }
    }
    __device__ __forceinline__ void Set(const float (&v)[8]) {   // rounded to the type
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (DTYPE == FTH_B200_FP32) w[i] = __float_as_uint(v[i]);
            else if ((i & 1) == 0) w[i / 2] = PackTo<DTYPE>(v[i], v[i + 1]);
        }
    }
    __device__ __forceinline__ float2 Pair(int i) const {
        if constexpr (DTYPE == FTH_B200_FP32) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
        else return HalfPair<DTYPE>(w[i]);
    }
};

// Eight elements of each lane of a group of LANES lanes that share a vector -> eight codes and the vector's parameters.
template <int DTYPE, int LANES>
__device__ __forceinline__ uint32_t QuantiseEight(const Eight<DTYPE>& e, uint32_t* params) {
    float2 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = e.Pair(i);
    float low, high;
    bool finite;
    if constexpr (DTYPE == FTH_B200_FP32) {
        const float all[8] = {x[0].x, x[0].y, x[1].x, x[1].y, x[2].x, x[2].y, x[3].x, x[3].y};
        finite = Range<LANES>(all, &low, &high);
    } else {
        finite = Range<DTYPE, LANES>(e.w, &low, &high);
    }
    const uint32_t min_bits = Bf16Floor(low);
    const float minimum = Bf16At(min_bits);
    if (!finite || (min_bits & 0x7f80u) == 0x7f80u || !(__fsub_rn(high, minimum) < INFINITY)) {
        *params = 0x7fc0u;
        return 0;
    }
    const uint32_t scale_bits = ScaleBits(fminf(__fsub_ru(high, minimum), 3.402823466e38f));   // the largest scale reaches past 2^128
    const float scale = Bf16At(scale_bits);
    const float inverse = scale_bits == 0 ? 0.0f : Reciprocal(scale);   // scale < 2^125, so it is no subnormal
    *params = scale_bits | (min_bits << 16);
    // estimates are in [0, 15.0001]; added to 1.5 * 2^23 their nearest integers are the sum's last bits
    constexpr float kMagic = 12582912.0f;
    float2 est[4], nearest[4];
    float unsure = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        est[i] = Mul2(Add2(x[i], make_float2(-minimum, -minimum)), make_float2(inverse, inverse));
        nearest[i] = Add2(Add2(est[i], make_float2(kMagic, kMagic)), make_float2(-kMagic, -kMagic));
        const float2 off = Fma2(nearest[i], make_float2(-1.0f, -1.0f), est[i]);
        unsure = Max3(unsure, fabsf(off.x), fabsf(off.y));
    }
    if (unsure > 0.4999f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (fabsf(__fsub_rn(est[i].x, nearest[i].x)) > 0.4999f) nearest[i].x = static_cast<float>(ExactCode(x[i].x, minimum, scale, est[i].x));
            if (fabsf(__fsub_rn(est[i].y, nearest[i].y)) > 0.4999f) nearest[i].y = static_cast<float>(ExactCode(x[i].y, minimum, scale, est[i].y));
        }
    }
    // four codes are a sum of up to 16 bits, exact
    const float four0 = __fmaf_rn(nearest[1].y, 4096.0f, __fmaf_rn(nearest[1].x, 256.0f, __fmaf_rn(nearest[0].y, 16.0f, nearest[0].x)));
    const float four1 = __fmaf_rn(nearest[3].y, 4096.0f, __fmaf_rn(nearest[3].x, 256.0f, __fmaf_rn(nearest[2].y, 16.0f, nearest[2].x)));
    return (__float_as_uint(__fadd_rn(four0, 8388608.0f)) & 0xffffu) | (__float_as_uint(__fadd_rn(four1, 8388608.0f)) << 16);
}

// Lane `lane` of the vector's group stores its eight codes; the first one the parameters.
template <int LANES>
__device__ __forceinline__ void StoreKey(const Cache& c, int slot, int head, int lane, uint32_t codes, uint32_t params) {
    const int64_t at = HeadBase(c, slot >> c.block_shift, head) + (slot & ((1 << c.block_shift) - 1));
    *reinterpret_cast<uint32_t*>(c.k_codes + at * (LANES * 4) + lane * 4) = codes;
    if (lane == 0) c.k_params[at] = params;
}
template <int LANES>
__device__ __forceinline__ void StoreValue(const Cache& c, int slot, int head, int lane, uint32_t codes, uint32_t params) {
    const int64_t base = HeadBase(c, slot >> c.block_shift, head);
    const int offset = slot & ((1 << c.block_shift) - 1);
    // the pair's row of LANES * 2 words; this token's half of two of them
    uint16_t* row = reinterpret_cast<uint16_t*>(c.v_codes + (base + (offset & ~1)) * (LANES * 4)) + (offset & 1);
    row[lane * 4] = static_cast<uint16_t>(codes);
    row[lane * 4 + 2] = static_cast<uint16_t>(codes >> 16);
    if (lane == 0) c.v_params[base + offset] = params;
}

// A walk over (one token or a pair of neighbours, head of the keys, then of the values): one division, then additions.
struct PairWalk {
    int64_t pair, pairs;   // of tokens
    int h2, heads2;        // head, twice the number of heads
    int64_t pair_step;
    int h2_step;
    __device__ __forceinline__ PairWalk(int64_t tokens, int two, int heads, int first, int step) : pairs((tokens + two) >> two), heads2(2 * heads) {
        pair = first / heads2;
        h2 = first - static_cast<int>(pair) * heads2;
        pair_step = step / heads2;
        h2_step = step - static_cast<int>(pair_step) * heads2;
    }
    __device__ __forceinline__ void Next() {
        pair += pair_step;
        h2 += h2_step;
        if (h2 >= heads2) {
            h2 -= heads2;
            ++pair;
        }
    }
};
// Whether two tokens share a row of value words: neighbours in a block, the first at an even place.
__device__ __forceinline__ bool SharePairs(int slot0, int slot1) { return slot0 >= 0 && (slot0 & 1) == 0 && slot1 == slot0 + 1; }

// A group of lanes takes two neighbouring tokens' vectors at a time: twice the loads in flight, and the words of values, which
// hold two tokens, are written whole when the tokens are neighbours in the cache too.
template <int DTYPE, int LANES, bool TURN>
__device__ __forceinline__ void AppendVectors(const AppendParams& p, int64_t first, int tokens, int start, int stride, const float2* angles) {
    const int lane = (threadIdx.x & 31) % LANES;
    const int heads = p.cache.kv_heads;
    PairWalk walk(tokens, p.two, heads, start / LANES, stride / LANES);
    for (; __any_sync(0xffffffffu, walk.pair < walk.pairs); walk.Next()) {   // the loop is the warp's
        const int64_t row = walk.pair << p.two;
        const bool has0 = row < tokens, has1 = p.two != 0 && row + 1 < tokens;
        const bool is_key = walk.h2 < heads;
        const int head = is_key ? walk.h2 : walk.h2 - heads;
        const int64_t token = first + row;
        const int slots[2] = {has0 ? p.slots[token] : -1, has1 ? p.slots[token + 1] : -1};
        // a negative position: the row is not turned, its key is stored as it is
        const bool turned[2] = {TURN && is_key && has0 && p.rope.positions[token] >= 0, TURN && is_key && has1 && p.rope.positions[token + 1] >= 0};
        Eight<DTYPE> x[2] = {};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (!(j == 0 ? has0 : has1)) continue;
            const int64_t at = (token + j) * (is_key ? p.ldk : p.ldv) + static_cast<int64_t>(head) * (LANES * 8);
            if (turned[j]) {
                float v[8];
                RopeEight<DTYPE>(p.rope, p.k, at, lane * 8, angles + (row + j) * (p.rope.rotary_dim >> 1), p.vec_k != 0, v);
                x[j].Set(v);
            } else {
                x[j].Load(is_key ? p.k : p.v, at + lane * 8, (is_key ? p.vec_k : p.vec_v) != 0);
            }
        }
        uint32_t codes[2] = {}, params[2] = {};
        codes[0] = QuantiseEight<DTYPE, LANES>(x[0], &params[0]);
        if (p.two) codes[1] = QuantiseEight<DTYPE, LANES>(x[1], &params[1]);
        bool good[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            good[j] = slots[j] >= 0 && slots[j] < p.slots_limit;
            if (slots[j] >= p.slots_limit && lane == 0) ReportSlot(p.status, kSiteAppend, token + j);
        }
        if (good[0] && good[1] && SharePairs(slots[0], slots[1])) {
            const int64_t at = HeadBase(p.cache, slots[0] >> p.cache.block_shift, head) + (slots[0] & ((1 << p.cache.block_shift) - 1));
            uint8_t* const to = (is_key ? p.cache.k_codes : p.cache.v_codes) + at * (LANES * 4);
            if (is_key) {
                *reinterpret_cast<uint32_t*>(to + lane * 4) = codes[0];
                *reinterpret_cast<uint32_t*>(to + (LANES + lane) * 4) = codes[1];
            } else {
                *reinterpret_cast<uint2*>(to + lane * 8) = make_uint2(__byte_perm(codes[0], codes[1], 0x5410), __byte_perm(codes[0], codes[1], 0x7632));
            }
            if (lane == 0) *reinterpret_cast<uint2*>((is_key ? p.cache.k_params : p.cache.v_params) + at) = make_uint2(params[0], params[1]);
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (!good[j]) continue;
                if (is_key) StoreKey<LANES>(p.cache, slots[j], head, lane, codes[j], params[j]);
                else StoreValue<LANES>(p.cache, slots[j], head, lane, codes[j], params[j]);
            }
        }
    }
}

template <int DTYPE, int LANES>
__global__ void __launch_bounds__(kThreads, kAppendBlocks) AppendKernel(const __grid_constant__ AppendParams p) {
    WaitForPrevious();
    AppendVectors<DTYPE, LANES, false>(p, 0, static_cast<int>(p.tokens), blockIdx.x * kThreads + threadIdx.x, gridDim.x * kThreads, nullptr);
}

// With rope: a block of threads takes a few tokens (blockIdx.x) and a share of their vectors (blockIdx.y).
template <int DTYPE, int LANES>
__global__ void __launch_bounds__(kThreads) RopeAppendKernel(const __grid_constant__ AppendParams p) {
    extern __shared__ float2 angles[];
    WaitForPrevious();
    const Rope& r = p.rope;
    const int pairs = r.rotary_dim >> 1;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * p.block_tokens;
    const int mine = static_cast<int>(p.tokens - first < p.block_tokens ? p.tokens - first : p.block_tokens);
    for (int i = threadIdx.x; i < mine * pairs; i += kThreads) {
        const int t = i / pairs;
        angles[i] = RopeAngle(r.positions[first + t], r.turns[i - t * pairs], r.amplitude);
    }
    __syncthreads();
    const int start = blockIdx.y * kThreads + threadIdx.x, stride = gridDim.y * kThreads;
    AppendVectors<DTYPE, LANES, true>(p, first, mine, start, stride, angles);
    // q: both members of a pair are read before either is written (the rows may be turned in place)
    const int half = pairs;
    const int items = p.vec_q ? r.head_dim >> 4 : r.head_dim - pairs;
    const int total = mine * r.q_heads * items;
    for (int i = start; i < total; i += stride) {
        const int head_row = i / items, item = i - head_row * items;
        const int t = head_row / r.q_heads, h = head_row - t * r.q_heads;
        const int64_t token = first + t;
        if (r.positions[token] < 0) continue;
        const int64_t in = token * r.ldq + static_cast<int64_t>(h) * r.head_dim, out = token * r.ldq_out + static_cast<int64_t>(h) * r.head_dim;
        const float2* cs = angles + t * pairs;
        if (p.vec_q) {
            const bool turned = item < (r.rotary_dim >> 4);
            const int j1 = turned ? (r.half_layout ? item * 8 : item * 16) : r.rotary_dim + (item - (r.rotary_dim >> 4)) * 16;
            const int j2 = turned && r.half_layout ? j1 + half : j1 + 8;
            float a[8], b[8];
            RopeEight<DTYPE>(r, r.q, in, j1, cs, true, a);
            RopeEight<DTYPE>(r, r.q, in, j2, cs, true, b);
            WriteEight<DTYPE>(r.q_out, out + j1, true, a);
            WriteEight<DTYPE>(r.q_out, out + j2, true, b);
        } else if (item < half) {
            const int j1 = r.half_layout ? item : 2 * item, j2 = r.half_layout ? item + half : 2 * item + 1;
            const float2 y = RopeTurn(ReadFloat<DTYPE>(r.q, in + j1), ReadFloat<DTYPE>(r.q, in + j2), cs[item]);
            WriteFloat<DTYPE>(r.q_out, out + j1, y.x);
            WriteFloat<DTYPE>(r.q_out, out + j2, y.y);
        } else {
            const int j = r.rotary_dim + item - half;
            WriteFloat<DTYPE>(r.q_out, out + j, ReadFloat<DTYPE>(r.q, in + j));
        }
    }
}

struct GatherParams {
    Cache cache;
    int64_t slots_limit;
    int64_t tokens;
    const int32_t* slots;
    void* k_out;
    void* v_out;
    int64_t ldk, ldv;
    int* status;
    int vec_k, vec_v;
    int two;
};

template <int DTYPE, int LANES>
__global__ void __launch_bounds__(kThreads, kGatherBlocks) GatherKernel(const __grid_constant__ GatherParams p) {
    WaitForPrevious();
    const int heads = p.cache.kv_heads;
    const int lane = threadIdx.x % LANES;
    constexpr int kGroups = kThreads / LANES;
    for (PairWalk walk(p.tokens, p.two, heads, blockIdx.x * kGroups + threadIdx.x / LANES, gridDim.x * kGroups); walk.pair < walk.pairs; walk.Next()) {
        const int64_t token = walk.pair << p.two;
        const bool is_key = walk.h2 < heads;
        const int head = is_key ? walk.h2 : walk.h2 - heads;
        void* out = is_key ? p.k_out : p.v_out;
        if (out == nullptr) continue;
        const int slots[2] = {p.slots[token], p.two != 0 && token + 1 < p.tokens ? p.slots[token + 1] : -1};
        uint32_t codes[2], params[2];
        bool good[2];
        int64_t base[2];
        int offset[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            good[j] = slots[j] >= 0 && slots[j] < p.slots_limit;
            if (slots[j] >= p.slots_limit && lane == 0) ReportSlot(p.status, kSiteGather, token + j);
            base[j] = good[j] ? HeadBase(p.cache, slots[j] >> p.cache.block_shift, head) : 0;
            offset[j] = good[j] ? slots[j] & ((1 << p.cache.block_shift) - 1) : 0;
            codes[j] = params[j] = 0;
        }
        if (is_key) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (!good[j]) continue;
                codes[j] = *reinterpret_cast<const uint32_t*>(p.cache.k_codes + (base[j] + offset[j]) * (LANES * 4) + lane * 4);
                params[j] = p.cache.k_params[base[j] + offset[j]];
            }
        } else if (good[0] && good[1] && SharePairs(slots[0], slots[1])) {
            const uint2 words = *reinterpret_cast<const uint2*>(p.cache.v_codes + (base[0] + offset[0]) * (LANES * 4) + lane * 8);
            const uint2 both = *reinterpret_cast<const uint2*>(p.cache.v_params + base[0] + offset[0]);
            codes[0] = __byte_perm(words.x, words.y, 0x5410);
            codes[1] = __byte_perm(words.x, words.y, 0x7632);
            params[0] = both.x;
            params[1] = both.y;
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                if (!good[j]) continue;
                const uint16_t* row = reinterpret_cast<const uint16_t*>(p.cache.v_codes + (base[j] + (offset[j] & ~1)) * (LANES * 4)) + (offset[j] & 1);
                codes[j] = row[lane * 4] | (static_cast<uint32_t>(row[lane * 4 + 2]) << 16);
                params[j] = p.cache.v_params[base[j] + offset[j]];
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            if (!good[j]) continue;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __fmaf_rn(ParamScale(params[j]), __fsub_rn(__uint_as_float(((codes[j] >> (4 * i)) & 15u) | 0x4b000000u), 8388608.0f), ParamMin(params[j]));
            const int64_t at = (token + j) * (is_key ? p.ldk : p.ldv) + static_cast<int64_t>(head) * (LANES * 8) + lane * 8;
            const bool vec = (is_key ? p.vec_k : p.vec_v) != 0;
            if (DTYPE != FTH_B200_FP32 && vec)
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + at) =
                    make_uint4(PackTo<DTYPE>(v[0], v[1]), PackTo<DTYPE>(v[2], v[3]), PackTo<DTYPE>(v[4], v[5]), PackTo<DTYPE>(v[6], v[7]));
            else
                WriteEight<DTYPE>(out, at, vec, v);
        }
    }
}

template <template <int, int> class F, typename... Args>
int ByTypeAndDim(int dtype, int head_dim, Args... args) {
    const auto dim = [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (head_dim == 64) return F<D, 8>::Run(args...);
        if (head_dim == 128) return F<D, 16>::Run(args...);
        return F<D, 32>::Run(args...);
    };
    if (dtype == FTH_B200_FP32) return dim(std::integral_constant<int, FTH_B200_FP32>{});
    if (dtype == FTH_B200_BF16) return dim(std::integral_constant<int, FTH_B200_BF16>{});
    return dim(std::integral_constant<int, FTH_B200_FP16>{});
}
template <int D, int L> struct RunAppend {
    static int Run(const AppendParams& p, dim3 grid, cudaStream_t s) { return Launch(AppendKernel<D, L>, grid, kThreads, 0, s, p); }
};
template <int D, int L> struct RunRopeAppend {
    static int Run(const AppendParams& p, dim3 grid, size_t smem, cudaStream_t s) { return Launch(RopeAppendKernel<D, L>, grid, kThreads, smem, s, p); }
};
template <int D, int L> struct RunGather {
    static int Run(const GatherParams& p, dim3 grid, cudaStream_t s) { return Launch(GatherKernel<D, L>, grid, kThreads, 0, s, p); }
};

// Two tokens at a time once one at a time would fill every SM twice over: 64 tokens of 8 heads of 128 are stored in 2.5 us one
// at a time and 3.3 us in pairs, 16384 of them in 52 and 43 us (36 us in pairs by now), and read back in 35 and 23 us.
int TwoAtATime(int64_t threads) { return threads >= static_cast<int64_t>(SmCount()) * 2048 * 2 ? 1 : 0; }
// No more blocks than run at once, `per_sm` on each SM: every thread walks on.
unsigned SpreadBlocks(int64_t threads, int per_sm) {
    const int64_t blocks = (threads + kThreads - 1) / kThreads, cap = static_cast<int64_t>(SmCount()) * per_sm;
    return static_cast<unsigned>(blocks < 1 ? 1 : blocks > cap ? cap : blocks);
}

}  // namespace
}  // namespace kv4
}  // namespace fth

using namespace fth;

extern "C" int fth_b200_kv4_append(const fth_b200_kv4_append_desc* d, fth_b200_stream_t stream_) {
    ClearStaleError();
    if (d == nullptr || d->tokens < 0) return FTH_B200_ERR_INVALID;
    int rc = kv4::CheckCache(d->cache);
    if (rc != FTH_B200_OK) return rc;
    const int64_t row = static_cast<int64_t>(d->cache.kv_heads) * d->cache.head_dim;
    if ((d->ldk != 0 && d->ldk < row) || (d->ldv != 0 && d->ldv < row)) return FTH_B200_ERR_INVALID;
    if (!kv4::FloatType(d->dtype)) return FTH_B200_ERR_UNSUPPORTED;
    if (d->tokens > 0x7fffffff) return FTH_B200_ERR_UNSUPPORTED;
    if (d->tokens > 0 && (d->k == nullptr || d->v == nullptr || d->slots == nullptr)) return FTH_B200_ERR_INVALID;
    const int size = kv4::ElementBytes(d->dtype);
    if (!kv4::AlignedTo(d->k, size) || !kv4::AlignedTo(d->v, size) || !kv4::WordAligned(d->slots)) return FTH_B200_ERR_INVALID;
    if (d->rope != nullptr) {
        rc = kv4::CheckRope(d->rope, true);
        if (rc != FTH_B200_OK) return rc;
        const fth_b200_rope_desc& r = *d->rope;
        if (r.k != d->k || r.k_heads != d->cache.kv_heads || r.head_dim != d->cache.head_dim || r.dtype != d->dtype || r.tokens != d->tokens)
            return FTH_B200_ERR_INVALID;
        if ((r.ldk ? r.ldk : row) != (d->ldk ? d->ldk : row)) return FTH_B200_ERR_INVALID;
    }
    if (d->tokens == 0) return FTH_B200_OK;
    kv4::AppendParams p = {};
    p.cache = kv4::MakeCache(d->cache);
    p.slots_limit = d->cache.blocks * d->cache.block_size;
    p.tokens = d->tokens;
    p.k = d->k;
    p.v = d->v;
    p.ldk = d->ldk ? d->ldk : row;
    p.ldv = d->ldv ? d->ldv : row;
    p.slots = d->slots;
    p.status = DeviceStatusPtr();
    const int per16 = 16 / size;
    p.vec_k = kv4::AlignedTo(d->k, 16) && p.ldk % per16 == 0;
    p.vec_v = kv4::AlignedTo(d->v, 16) && p.ldv % per16 == 0;
    auto s = static_cast<cudaStream_t>(stream_);
    const int64_t lanes = row / 4;  // threads of one token's keys and values, eight elements each
    int status;
    if (d->rope == nullptr) {
        p.two = kv4::TwoAtATime(d->tokens * lanes);
        status = kv4::ByTypeAndDim<kv4::RunAppend>(d->dtype, d->cache.head_dim, p, dim3(kv4::SpreadBlocks(((d->tokens + p.two) >> p.two) * lanes, kv4::kAppendBlocks)), s);
        if (status == FTH_B200_OK) NoteLaunch("kv4_append");
        return status;
    }
    p.rope = kv4::MakeRope(*d->rope);
    p.rope.k_out = nullptr;
    const bool whole = p.rope.rotary_dim % 16 == 0;
    p.vec_k = p.vec_k && whole;
    p.vec_q = whole && kv4::AlignedTo(p.rope.q, 16) && kv4::AlignedTo(p.rope.q_out, 16) && p.rope.ldq % per16 == 0 && p.rope.ldq_out % per16 == 0;
    // one token a block while there are few, so that every SM has some; up to four (one set-up for more work) otherwise
    const int64_t spread = d->tokens / (4 * SmCount());
    p.block_tokens = static_cast<int>(spread < 1 ? 1 : spread > 4 ? 4 : spread);
    p.two = p.block_tokens > 1;
    const int64_t blocks = (d->tokens + p.block_tokens - 1) / p.block_tokens;
    const int64_t work = p.block_tokens * (lanes + static_cast<int64_t>(p.rope.q_heads) * d->cache.head_dim / 16);
    int64_t share = blocks >= 2 * SmCount() ? 1 : (work + kv4::kThreads - 1) / kv4::kThreads;
    if (share > 16) share = 16;
    const size_t smem = static_cast<size_t>(p.block_tokens) * (p.rope.rotary_dim / 2) * sizeof(float2);
    status = kv4::ByTypeAndDim<kv4::RunRopeAppend>(d->dtype, d->cache.head_dim, p, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(share)), smem, s);
    if (status == FTH_B200_OK) NoteLaunch("rope_kv4_append");
    return status;
}

extern "C" int fth_b200_kv4_gather(const fth_b200_kv4_gather_desc* d, fth_b200_stream_t stream_) {
    ClearStaleError();
    if (d == nullptr || d->tokens < 0) return FTH_B200_ERR_INVALID;
    const int rc = kv4::CheckCache(d->cache);
    if (rc != FTH_B200_OK) return rc;
    const int64_t row = static_cast<int64_t>(d->cache.kv_heads) * d->cache.head_dim;
    if ((d->ldk != 0 && d->ldk < row) || (d->ldv != 0 && d->ldv < row)) return FTH_B200_ERR_INVALID;
    if (!kv4::FloatType(d->dtype)) return FTH_B200_ERR_UNSUPPORTED;
    if (d->tokens > 0x7fffffff) return FTH_B200_ERR_UNSUPPORTED;
    if (d->k_out == nullptr && d->v_out == nullptr) return FTH_B200_ERR_INVALID;
    const int size = kv4::ElementBytes(d->dtype);
    if (!kv4::AlignedTo(d->k_out, size) || !kv4::AlignedTo(d->v_out, size) || !kv4::WordAligned(d->slots)) return FTH_B200_ERR_INVALID;
    if (d->tokens == 0) return FTH_B200_OK;
    if (d->slots == nullptr) return FTH_B200_ERR_INVALID;
    const int per16 = 16 / size;
    const int64_t ldk = d->ldk ? d->ldk : row, ldv = d->ldv ? d->ldv : row;
    const kv4::GatherParams p{kv4::MakeCache(d->cache), d->cache.blocks * d->cache.block_size, d->tokens, d->slots, d->k_out, d->v_out, ldk, ldv,
                              DeviceStatusPtr(), kv4::AlignedTo(d->k_out, 16) && ldk % per16 == 0, kv4::AlignedTo(d->v_out, 16) && ldv % per16 == 0, kv4::TwoAtATime(d->tokens * row / 4)};
    const int status = kv4::ByTypeAndDim<kv4::RunGather>(d->dtype, d->cache.head_dim, p, dim3(kv4::SpreadBlocks(((d->tokens + p.two) >> p.two) * row / 4, kv4::kGatherBlocks)),
                                                         static_cast<cudaStream_t>(stream_));
    if (status == FTH_B200_OK) NoteLaunch("kv4_gather");
    return status;
}
