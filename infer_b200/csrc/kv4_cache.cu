// Storing keys and values in the 4-bit cache (with the rotary positions of q and k in the same launch, if asked for) and
// reading them back.
//
// A vector x of head_dim elements becomes codes c in 0 .. 15 with value m + s * c:
//   m = largest BF16 <= min(x),  s = smallest BF16 >= (max(x) - m) / 15,  c = nearest((x - m) / s), ties to even.
// m is never above min(x) and 15 s reaches max(x), so no code is clamped by more than rounding; for BF16 input m is min(x)
// itself.  Every border is decided exactly: an FP32 estimate of (x - m) / s is off by less than 2^-21 * 15 < 10^-5, so
// only estimates within 10^-4 of a half are looked at again, in 64 bits.
// One pass over the data: 2 * tokens * kv_heads * head_dim * size bytes in, head_dim + 8 bytes per token and head out;
// memory bound for prompts, a launch for single tokens.  A vector belongs to head_dim / 8 neighbouring lanes, eight
// elements each, so minimum and maximum are three to five shuffles and a lane's codes are one 32-bit word.
#include <type_traits>

#include "kv4.cuh"

namespace fth {
namespace kv4 {

namespace {

using namespace rowops;

constexpr int kThreads = 256;
constexpr int kSiteAppend = 40, kSiteGather = 41;

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
    int turn;
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

// Smallest BF16 s with 15 s >= spread, at least 2^-126; 0 for spread = 0.  15 s has 12 bits, so the comparison is exact.
__device__ __forceinline__ uint32_t ScaleBits(double spread) {
    if (!(spread > 0.0)) return 0;
    uint32_t b = __float_as_uint(static_cast<float>(spread) * (1.0f / 15.0f)) >> 16;
    if (b < 0x0080u) b = 0x0080u;
    while (b > 0x0080u && 15.0 * static_cast<double>(Bf16At(b - 1)) >= spread) --b;
    while (15.0 * static_cast<double>(Bf16At(b)) < spread) ++b;
    return b;
}

// One code.  `inverse` = 1 / scale (0 when the scale is 0).
__device__ __forceinline__ uint32_t Code(float x, float minimum, float scale, float inverse) {
    const float est = __fmul_rn(__fsub_rn(x, minimum), inverse);
    float r = rintf(est);
    const float fl = floorf(est);
    if (fabsf(est - fl - 0.5f) < 1e-4f) {
        const double d = static_cast<double>(x) - static_cast<double>(minimum);
        const double border = (static_cast<double>(fl) + 0.5) * static_cast<double>(scale);
        const bool odd = (static_cast<int>(fl) & 1) != 0;
        r = d > border || (d == border && odd) ? fl + 1.0f : fl;
    }
    return static_cast<uint32_t>(fminf(fmaxf(r, 0.0f), 15.0f));
}

// Eight elements of each lane of a group of LANES lanes that share a vector -> eight codes and the vector's parameters.
template <int LANES>
__device__ __forceinline__ uint32_t QuantiseEight(const float (&x)[8], uint32_t* params) {
    float low = x[0], high = x[0];
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        low = fminf(low, x[i]);
        high = fmaxf(high, x[i]);
        finite = finite && (__float_as_uint(x[i]) & 0x7f800000u) != 0x7f800000u;
    }
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) {
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
        finite = __shfl_xor_sync(0xffffffffu, finite ? 1 : 0, o) != 0 && finite;
    }
    const uint32_t min_bits = Bf16Floor(low);
    if (!finite || (min_bits & 0x7f80u) == 0x7f80u || !(__fsub_rn(high, Bf16At(min_bits)) < INFINITY)) {
        *params = 0x7fc0u;
        return 0;
    }
    const float minimum = Bf16At(min_bits);
    const uint32_t scale_bits = ScaleBits(static_cast<double>(high) - static_cast<double>(minimum));
    const float scale = Bf16At(scale_bits);
    const float inverse = scale_bits == 0 ? 0.0f : __fdiv_rn(1.0f, scale);
    *params = scale_bits | (min_bits << 16);
    uint32_t codes = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) codes |= Code(x[i], minimum, scale, inverse) << (4 * i);
    return codes;
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

// A work item is one vector: for every token kv_heads keys, then kv_heads values.
template <int DTYPE, int LANES>
__device__ __forceinline__ void AppendVectors(const AppendParams& p, int64_t first, int tokens, int start, int stride, const float2* angles) {
    constexpr int kGroups = 32 / LANES;  // vectors a warp works on side by side
    const int warp = start >> 5, warps = stride >> 5;
    const int lane = (threadIdx.x & 31) % LANES, group = (threadIdx.x & 31) / LANES;
    const int heads = p.cache.kv_heads;
    const int64_t total = static_cast<int64_t>(tokens) * heads * 2;
    for (int64_t base = static_cast<int64_t>(warp) * kGroups; base < total; base += static_cast<int64_t>(warps) * kGroups) {
        const int64_t item = base + group;
        const bool valid = item < total;
        const int64_t row = valid ? item / (2 * heads) : 0;
        const int h2 = valid ? static_cast<int>(item - row * (2 * heads)) : 0;
        const bool is_key = h2 < heads;
        const int head = is_key ? h2 : h2 - heads;
        const int64_t token = first + row;
        const int slot = valid ? p.slots[token] : -1;
        float x[8] = {};
        if (slot >= 0) {
            const int64_t at = token * (is_key ? p.ldk : p.ldv) + static_cast<int64_t>(head) * (LANES * 8);
            if (is_key && p.turn) {
                RopeEight<DTYPE>(p.rope, p.k, at, lane * 8, angles + row * (p.rope.rotary_dim >> 1), p.vec_k != 0, x);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = Rounded<DTYPE>(x[i]);
            } else {
                ReadEight<DTYPE>(is_key ? p.k : p.v, at + lane * 8, (is_key ? p.vec_k : p.vec_v) != 0, x);
            }
        }
        uint32_t params;
        const uint32_t codes = QuantiseEight<LANES>(x, &params);
        if (slot < 0) continue;
        if (slot >= p.slots_limit) {
            if (lane == 0) ReportTimeout(p.status, kSiteAppend, static_cast<int>(token));
            continue;
        }
        if (is_key) StoreKey<LANES>(p.cache, slot, head, lane, codes, params);
        else StoreValue<LANES>(p.cache, slot, head, lane, codes, params);
    }
}

template <int DTYPE, int LANES>
__global__ void __launch_bounds__(kThreads) AppendKernel(const __grid_constant__ AppendParams p) {
    WaitForPrevious();
    AppendVectors<DTYPE, LANES>(p, 0, static_cast<int>(p.tokens), blockIdx.x * kThreads + threadIdx.x, gridDim.x * kThreads, nullptr);
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
    AppendVectors<DTYPE, LANES>(p, first, mine, start, stride, angles);
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
};

template <int DTYPE, int LANES>
__global__ void __launch_bounds__(kThreads) GatherKernel(const __grid_constant__ GatherParams p) {
    WaitForPrevious();
    const int heads = p.cache.kv_heads;
    const int64_t total = p.tokens * heads * 2 * LANES;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total; i += static_cast<int64_t>(gridDim.x) * kThreads) {
        const int lane = static_cast<int>(i % LANES);
        const int64_t item = i / LANES;
        const int64_t token = item / (2 * heads);
        const int h2 = static_cast<int>(item - token * (2 * heads));
        const bool is_key = h2 < heads;
        const int head = is_key ? h2 : h2 - heads;
        void* out = is_key ? p.k_out : p.v_out;
        const int slot = p.slots[token];
        if (out == nullptr || slot < 0) continue;
        if (slot >= p.slots_limit) {
            if (lane == 0) ReportTimeout(p.status, kSiteGather, static_cast<int>(token));
            continue;
        }
        const int64_t base = HeadBase(p.cache, slot >> p.cache.block_shift, head);
        const int offset = slot & ((1 << p.cache.block_shift) - 1);
        uint32_t codes, params;
        if (is_key) {
            codes = *reinterpret_cast<const uint32_t*>(p.cache.k_codes + (base + offset) * (LANES * 4) + lane * 4);
            params = p.cache.k_params[base + offset];
        } else {
            const uint16_t* row = reinterpret_cast<const uint16_t*>(p.cache.v_codes + (base + (offset & ~1)) * (LANES * 4)) + (offset & 1);
            codes = row[lane * 4] | (static_cast<uint32_t>(row[lane * 4 + 2]) << 16);
            params = p.cache.v_params[base + offset];
        }
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fmaf_rn(ParamScale(params), static_cast<float>((codes >> (4 * j)) & 15u), ParamMin(params));
        WriteEight<DTYPE>(out, token * (is_key ? p.ldk : p.ldv) + static_cast<int64_t>(head) * (LANES * 8) + lane * 8, (is_key ? p.vec_k : p.vec_v) != 0, v);
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

unsigned SpreadBlocks(int64_t threads) {
    const int64_t blocks = (threads + kThreads - 1) / kThreads, cap = static_cast<int64_t>(SmCount()) * 8;
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
    if (!kv4::AlignedTo(d->k, size) || !kv4::AlignedTo(d->v, size)) return FTH_B200_ERR_INVALID;
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
        status = kv4::ByTypeAndDim<kv4::RunAppend>(d->dtype, d->cache.head_dim, p, dim3(kv4::SpreadBlocks(d->tokens * lanes)), s);
        if (status == FTH_B200_OK) NoteLaunch("kv4_append");
        return status;
    }
    p.turn = 1;
    p.rope = kv4::MakeRope(*d->rope);
    p.rope.k_out = nullptr;
    const bool whole = p.rope.rotary_dim % 16 == 0;
    p.vec_k = p.vec_k && whole;
    p.vec_q = whole && kv4::AlignedTo(p.rope.q, 16) && kv4::AlignedTo(p.rope.q_out, 16) && p.rope.ldq % per16 == 0 && p.rope.ldq_out % per16 == 0;
    // one token a block while there are few, so that every SM has some; up to four (one set-up for more work) otherwise
    const int64_t spread = d->tokens / (4 * SmCount());
    p.block_tokens = static_cast<int>(spread < 1 ? 1 : spread > 4 ? 4 : spread);
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
    if (!kv4::AlignedTo(d->k_out, size) || !kv4::AlignedTo(d->v_out, size)) return FTH_B200_ERR_INVALID;
    if (d->tokens == 0) return FTH_B200_OK;
    if (d->slots == nullptr) return FTH_B200_ERR_INVALID;
    const int per16 = 16 / size;
    const int64_t ldk = d->ldk ? d->ldk : row, ldv = d->ldv ? d->ldv : row;
    const kv4::GatherParams p{kv4::MakeCache(d->cache), d->cache.blocks * d->cache.block_size, d->tokens, d->slots, d->k_out, d->v_out, ldk, ldv,
                              DeviceStatusPtr(), kv4::AlignedTo(d->k_out, 16) && ldk % per16 == 0, kv4::AlignedTo(d->v_out, 16) && ldv % per16 == 0};
    const int status = kv4::ByTypeAndDim<kv4::RunGather>(d->dtype, d->cache.head_dim, p, dim3(kv4::SpreadBlocks(d->tokens * row / 4)),
                                                         static_cast<cudaStream_t>(stream_));
    if (status == FTH_B200_OK) NoteLaunch("kv4_gather");
    return status;
}
