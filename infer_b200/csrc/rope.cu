// Rotary positions of q and k in one launch, and the host-side table of turns.
//
// y1 = x1 cos - x2 sin, y2 = x2 cos + x1 sin per pair, FP32, one rounding to the output type.  Every element is read and
// written once (2 * tokens * heads * head_dim * size bytes), three operations each: memory bound, and a launch at decode
// size.  A block takes a few tokens and all or some of their heads; the cosines and sines of a token are the same for all
// its heads, so they are computed once per block (64-bit reduction, sincospif) into shared memory.  16383 tokens, 16 + 4 heads of
// 256 in FP16: 61 us, 5.5 TB/s; 16 tokens, 32 + 8 heads of 128: 2.2 us.
#include "kv4.cuh"

namespace fth {
namespace kv4 {

namespace {

using namespace rowops;

constexpr int kThreads = 256;
constexpr int kMaxPairs = 256;

struct RopeParams {
    Rope rope;
    int64_t tokens;
    int block_tokens;  // tokens of one block
    int vec;           // elements in eights with 16-byte accesses
};

// Work item: eight elements of one head (vec), or all head_dim elements one by one.  In the half layout an eight and
// its partner eight are written by one thread after both have been read, so a row can be turned in place.
template <int DTYPE>
__device__ __forceinline__ void TurnHeadVec(const Rope& r, const void* x, int64_t row_in, void* out, int64_t row_out, int item, const float2* angles) {
    const int half_items = r.rotary_dim >> 4;
    const int half = r.rotary_dim >> 1;
    float a[8], b[8];
    if (item < half_items) {
        if (r.half_layout) {
            const int j = item * 8;
            ReadEight<DTYPE>(x, row_in + j, true, a);
            ReadEight<DTYPE>(x, row_in + j + half, true, b);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 y = RopeTurn(a[i], b[i], angles[j + i]);
                a[i] = y.x;
                b[i] = y.y;
            }
            WriteEight<DTYPE>(out, row_out + j, true, a);
            WriteEight<DTYPE>(out, row_out + j + half, true, b);
        } else {
            const int j = item * 16;
            ReadEight<DTYPE>(x, row_in + j, true, a);
            ReadEight<DTYPE>(x, row_in + j + 8, true, b);
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float2 y = RopeTurn(a[i], a[i + 1], angles[(j + i) >> 1]);
                const float2 z = RopeTurn(b[i], b[i + 1], angles[(j + 8 + i) >> 1]);
                a[i] = y.x;
                a[i + 1] = y.y;
                b[i] = z.x;
                b[i + 1] = z.y;
            }
            WriteEight<DTYPE>(out, row_out + j, true, a);
            WriteEight<DTYPE>(out, row_out + j + 8, true, b);
        }
    } else {  // behind the rotated part
        const int j = r.rotary_dim + (item - half_items) * 16;
        ReadEight<DTYPE>(x, row_in + j, true, a);
        ReadEight<DTYPE>(x, row_in + j + 8, true, b);
        WriteEight<DTYPE>(out, row_out + j, true, a);
        WriteEight<DTYPE>(out, row_out + j + 8, true, b);
    }
}

template <int DTYPE>
__device__ __forceinline__ void TurnHeadPair(const Rope& r, const void* x, int64_t row_in, void* out, int64_t row_out, int item, const float2* angles) {
    const int half = r.rotary_dim >> 1;
    if (item < half) {
        const int j1 = r.half_layout ? item : 2 * item;
        const int j2 = r.half_layout ? item + half : 2 * item + 1;
        const float2 y = RopeTurn(ReadFloat<DTYPE>(x, row_in + j1), ReadFloat<DTYPE>(x, row_in + j2), angles[item]);
        WriteFloat<DTYPE>(out, row_out + j1, y.x);
        WriteFloat<DTYPE>(out, row_out + j2, y.y);
    } else {
        const int j = r.rotary_dim + item - half;
        WriteFloat<DTYPE>(out, row_out + j, ReadFloat<DTYPE>(x, row_in + j));
    }
}

template <int DTYPE>
__global__ void __launch_bounds__(kThreads) RopeKernel(const __grid_constant__ RopeParams p) {
    extern __shared__ float2 angles[];  // [block_tokens][pairs]
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
    const int items = p.vec ? r.head_dim >> 4 : r.head_dim - pairs;
    const int heads = r.q_heads + r.k_heads;
    const int total = mine * heads * items;
    for (int i = threadIdx.x + blockIdx.y * kThreads; i < total; i += kThreads * gridDim.y) {
        const int head_row = i / items;
        const int item = i - head_row * items;
        const int t = head_row / heads;
        const int h = head_row - t * heads;
        const int64_t token = first + t;
        if (r.positions[token] < 0) continue;  // a row behind the last
        const bool is_q = h < r.q_heads;
        const void* x = is_q ? r.q : r.k;
        void* out = is_q ? r.q_out : r.k_out;
        const int64_t column = static_cast<int64_t>(is_q ? h : h - r.q_heads) * r.head_dim;
        const int64_t row_in = token * (is_q ? r.ldq : r.ldk) + column;
        const int64_t row_out = token * (is_q ? r.ldq_out : r.ldk_out) + column;
        if (p.vec) TurnHeadVec<DTYPE>(r, x, row_in, out, row_out, item, angles + t * pairs);
        else TurnHeadPair<DTYPE>(r, x, row_in, out, row_out, item, angles + t * pairs);
    }
}

}  // namespace

int CheckRope(const fth_b200_rope_desc* d, bool keys_stay) {
    if (d == nullptr || d->tokens < 0 || d->head_dim <= 0 || d->rotary_dim <= 0 || d->q_heads < 0 || d->k_heads < 0) return FTH_B200_ERR_INVALID;
    if (d->q_heads + static_cast<int64_t>(d->k_heads) <= 0) return FTH_B200_ERR_INVALID;
    if (d->layout != FTH_B200_ROPE_HALF && d->layout != FTH_B200_ROPE_INTERLEAVED) return FTH_B200_ERR_INVALID;
    if (d->rotary_dim % 2 != 0 || d->rotary_dim > d->head_dim) return FTH_B200_ERR_INVALID;
    if (d->positions == nullptr || d->turns == nullptr || !std::isfinite(d->amplitude)) return FTH_B200_ERR_INVALID;
    if (!WordAligned(d->positions) || !AlignedTo(d->turns, alignof(double))) return FTH_B200_ERR_INVALID;
    if (d->q_heads > 0 && (d->q == nullptr || d->q_out == nullptr)) return FTH_B200_ERR_INVALID;
    if (d->k_heads > 0 && (d->k == nullptr || (d->k_out == nullptr) != keys_stay)) return FTH_B200_ERR_INVALID;
    const int64_t q_row = static_cast<int64_t>(d->q_heads) * d->head_dim, k_row = static_cast<int64_t>(d->k_heads) * d->head_dim;
    if ((d->ldq != 0 && d->ldq < q_row) || (d->ldq_out != 0 && d->ldq_out < q_row)) return FTH_B200_ERR_INVALID;
    if ((d->ldk != 0 && d->ldk < k_row) || (d->ldk_out != 0 && d->ldk_out < k_row)) return FTH_B200_ERR_INVALID;
    // in place means the same rows: another stride would write over rows that are still to be read
    if (d->q_heads > 0 && d->q == d->q_out && (d->ldq ? d->ldq : q_row) != (d->ldq_out ? d->ldq_out : q_row)) return FTH_B200_ERR_INVALID;
    if (d->k_heads > 0 && d->k == d->k_out && (d->ldk ? d->ldk : k_row) != (d->ldk_out ? d->ldk_out : k_row)) return FTH_B200_ERR_INVALID;
    if (!FloatType(d->dtype)) return FTH_B200_ERR_UNSUPPORTED;
    if (d->rotary_dim > 2 * kMaxPairs || d->head_dim > 4096 || d->q_heads > 4096 || d->k_heads > 4096) return FTH_B200_ERR_UNSUPPORTED;
    if (d->tokens > 0x7fffffff) return FTH_B200_ERR_UNSUPPORTED;
    const int size = ElementBytes(d->dtype);
    for (const void* ptr : {d->q, static_cast<const void*>(d->q_out), d->k, static_cast<const void*>(d->k_out)})
        if (!AlignedTo(ptr, size)) return FTH_B200_ERR_INVALID;
    return FTH_B200_OK;
}

Rope MakeRope(const fth_b200_rope_desc& d) {
    const int64_t q_row = static_cast<int64_t>(d.q_heads) * d.head_dim, k_row = static_cast<int64_t>(d.k_heads) * d.head_dim;
    return Rope{d.layout == FTH_B200_ROPE_HALF, d.head_dim, d.rotary_dim, d.q_heads, d.k_heads, d.q, d.q_out, d.k, d.k_out,
                d.ldq ? d.ldq : q_row, d.ldq_out ? d.ldq_out : q_row, d.ldk ? d.ldk : k_row, d.ldk_out ? d.ldk_out : k_row,
                d.positions, d.turns, d.amplitude};
}

}  // namespace kv4
}  // namespace fth

using namespace fth;

extern "C" int fth_b200_rope_turns(const fth_b200_rope_scaling* s, double* turns, float* amplitude) {
    if (s == nullptr || turns == nullptr || amplitude == nullptr) return FTH_B200_ERR_INVALID;
    if (s->rotary_dim <= 0 || s->rotary_dim % 2 != 0 || !(s->base > 1.0) || !std::isfinite(s->base)) return FTH_B200_ERR_INVALID;
    if (s->scaling < FTH_B200_ROPE_SCALE_NONE || s->scaling > FTH_B200_ROPE_SCALE_BANDED) return FTH_B200_ERR_INVALID;
    const bool by_turns = s->scaling == FTH_B200_ROPE_SCALE_YARN || s->scaling == FTH_B200_ROPE_SCALE_BANDED;
    if (s->scaling != FTH_B200_ROPE_SCALE_NONE && (!(s->factor >= 1.0) || !std::isfinite(s->factor))) return FTH_B200_ERR_INVALID;
    if (by_turns && (!(s->original > 0.0) || !(s->slow > 0.0) || !(s->fast > s->slow) || !std::isfinite(s->original) || !std::isfinite(s->fast)))
        return FTH_B200_ERR_INVALID;
    if (s->scaling == FTH_B200_ROPE_SCALE_NTK && s->rotary_dim <= 2) return FTH_B200_ERR_INVALID;
    const double pi2 = 2.0 * std::acos(-1.0), dim = s->rotary_dim;
    const double base = s->scaling == FTH_B200_ROPE_SCALE_NTK ? s->base * std::pow(s->factor, dim / (dim - 2.0)) : s->base;
    double low = 0.0, high = 0.0;
    if (s->scaling == FTH_B200_ROPE_SCALE_YARN) {
        // the pair (a real number) that makes n turns in `original` positions
        const auto pair = [&](double n) { return dim * std::log(s->original / (n * pi2)) / (2.0 * std::log(base)); };
        low = std::fmax(std::floor(pair(s->fast)), 0.0);
        high = std::fmin(std::ceil(pair(s->slow)), dim - 1.0);
    }
    for (int i = 0; i < s->rotary_dim / 2; ++i) {
        const double plain = std::pow(base, -2.0 * i / dim) / pi2;
        double keep = 1.0;  // share of the unscaled frequency
        if (s->scaling == FTH_B200_ROPE_SCALE_LINEAR) keep = 0.0;
        else if (s->scaling == FTH_B200_ROPE_SCALE_YARN) keep = 1.0 - std::fmin(1.0, std::fmax(0.0, (i - low) / std::fmax(high - low, 0.001)));
        else if (s->scaling == FTH_B200_ROPE_SCALE_BANDED) keep = std::fmin(1.0, std::fmax(0.0, (plain * s->original - s->slow) / (s->fast - s->slow)));
        turns[i] = keep == 1.0 ? plain : plain * keep + plain / s->factor * (1.0 - keep);
    }
    *amplitude = s->scaling == FTH_B200_ROPE_SCALE_YARN ? static_cast<float>(0.1 * std::log(s->factor) + 1.0) : 1.0f;
    return FTH_B200_OK;
}

extern "C" int fth_b200_rope(const fth_b200_rope_desc* d, fth_b200_stream_t stream_) {
    ClearStaleError();
    const int rc = kv4::CheckRope(d, false);
    if (rc != FTH_B200_OK || d->tokens == 0) return rc;
    kv4::RopeParams p;
    p.rope = kv4::MakeRope(*d);
    p.tokens = d->tokens;
    const kv4::Rope& r = p.rope;
    bool vec = d->rotary_dim % 16 == 0 && d->head_dim % 16 == 0;
    const int per16 = 16 / kv4::ElementBytes(d->dtype);
    if (r.q_heads > 0) vec = vec && kv4::AlignedTo(r.q, 16) && kv4::AlignedTo(r.q_out, 16) && r.ldq % per16 == 0 && r.ldq_out % per16 == 0;
    if (r.k_heads > 0) vec = vec && kv4::AlignedTo(r.k, 16) && kv4::AlignedTo(r.k_out, 16) && r.ldk % per16 == 0 && r.ldk_out % per16 == 0;
    p.vec = vec ? 1 : 0;
    // About five items a thread: enough tokens per block for that; when there are few tokens, several blocks share one.
    const int64_t items = static_cast<int64_t>(r.q_heads + r.k_heads) * (vec ? r.head_dim / 16 : r.head_dim - r.rotary_dim / 2);
    int64_t tokens = (4 * kv4::kThreads + items - 1) / items;
    const int64_t spread = (d->tokens + 2 * SmCount() - 1) / (2 * SmCount());  // tokens per block that still fill the chip twice
    if (tokens > spread) tokens = spread;
    if (tokens > 8) tokens = 8;
    p.block_tokens = static_cast<int>(tokens);
    const int64_t blocks = (d->tokens + tokens - 1) / tokens;
    int64_t share = (tokens * items + 4 * kv4::kThreads - 1) / (4 * kv4::kThreads);
    if (blocks < SmCount()) {
        const int64_t most = (tokens * items + kv4::kThreads - 1) / kv4::kThreads, want = SmCount() / blocks;
        share = want < most ? (want > share ? want : share) : most;
    }
    if (share > 64) share = 64;
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(share < 1 ? 1 : share));
    const size_t smem = static_cast<size_t>(tokens) * (r.rotary_dim / 2) * sizeof(float2);
    auto s = static_cast<cudaStream_t>(stream_);
    int status;
    if (d->dtype == FTH_B200_FP32) status = kv4::Launch(kv4::RopeKernel<FTH_B200_FP32>, grid, kv4::kThreads, smem, s, p);
    else if (d->dtype == FTH_B200_BF16) status = kv4::Launch(kv4::RopeKernel<FTH_B200_BF16>, grid, kv4::kThreads, smem, s, p);
    else status = kv4::Launch(kv4::RopeKernel<FTH_B200_FP16>, grid, kv4::kThreads, smem, s, p);
    if (status == FTH_B200_OK) NoteLaunch("rope");
    return status;
}
