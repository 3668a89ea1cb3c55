// What the operators around the 4-bit cache share: launch as a programmatic dependent, checks of the cache descriptor,
// addresses inside the cache, the rotation of a pair.
#pragma once

#include <cmath>

#include "common.cuh"
#include "rowops.cuh"
#include "tma.cuh"

namespace fth {
namespace kv4 {

template <typename... Params, typename... Args>
int Launch(void (*kernel)(Params...), dim3 grid, unsigned block, size_t smem, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
        ClearStaleError();
        return FTH_B200_ERR_CUDA;
    }
    return CheckLaunch();
}

// Every thread of every block runs this before it touches memory that an earlier kernel of the stream may have written
// or may still read, also threads without work: a kernel that ended early would let the next one pass its own wait.
__device__ __forceinline__ void WaitForPrevious() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

inline bool AlignedTo(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
// Arrays of 32-bit numbers; null is aligned.
template <typename... Pointers>
bool WordAligned(Pointers... p) { return (AlignedTo(p, 4) && ...); }
inline int ElementBytes(int dtype) { return dtype == FTH_B200_FP32 ? 4 : 2; }
inline bool FloatType(int dtype) { return dtype == FTH_B200_FP32 || dtype == FTH_B200_BF16 || dtype == FTH_B200_FP16; }
inline int Log2(int v) { int s = 0; while ((1 << s) < v) ++s; return s; }

inline int CheckBlockSize(int block_size) {
    if (block_size <= 0) return FTH_B200_ERR_INVALID;
    return block_size >= 16 && block_size <= 256 && (block_size & (block_size - 1)) == 0 ? FTH_B200_OK : FTH_B200_ERR_UNSUPPORTED;
}
inline int CheckPool(int64_t blocks, int block_size) {
    if (blocks <= 0) return FTH_B200_ERR_INVALID;
    const int rc = CheckBlockSize(block_size);
    if (rc != FTH_B200_OK) return rc;
    return blocks <= 0x7fffffff / block_size ? FTH_B200_OK : FTH_B200_ERR_UNSUPPORTED;
}
inline int CheckCache(const fth_b200_kv4_cache& c) {
    if (c.k_codes == nullptr || c.v_codes == nullptr || c.k_params == nullptr || c.v_params == nullptr) return FTH_B200_ERR_INVALID;
    if (c.kv_heads <= 0 || c.head_dim <= 0) return FTH_B200_ERR_INVALID;
    const int rc = CheckPool(c.blocks, c.block_size);
    if (rc != FTH_B200_OK) return rc;
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return FTH_B200_ERR_UNSUPPORTED;
    if (c.kv_heads > 4096) return FTH_B200_ERR_UNSUPPORTED;
    if (!AlignedTo(c.k_codes, 16) || !AlignedTo(c.v_codes, 16) || !AlignedTo(c.k_params, 16) || !AlignedTo(c.v_params, 16)) return FTH_B200_ERR_INVALID;
    return FTH_B200_OK;
}

// The cache as the kernels see it.  A token's index within a head is (block * kv_heads + head) * block_size + offset; it
// and every byte offset made of it are 64-bit: a cache passes 4 GB long before its slots pass 31 bits.
struct Cache {
    uint8_t* k_codes;
    uint8_t* v_codes;
    uint32_t* k_params;
    uint32_t* v_params;
    int blocks, kv_heads, block_shift;
};
inline Cache MakeCache(const fth_b200_kv4_cache& c) {
    return Cache{static_cast<uint8_t*>(c.k_codes), static_cast<uint8_t*>(c.v_codes), static_cast<uint32_t*>(c.k_params),
                 static_cast<uint32_t*>(c.v_params), static_cast<int>(c.blocks), c.kv_heads, Log2(c.block_size)};
}
__device__ __forceinline__ int64_t HeadBase(const Cache& c, int block, int head) {
    return (static_cast<int64_t>(block) * c.kv_heads + head) << c.block_shift;
}
__device__ __forceinline__ float ParamScale(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float ParamMin(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// ---- arithmetic ----------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float Reciprocal(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two FP32 operations per instruction.
__device__ __forceinline__ float2 Fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n .reg .b64 x, y, z, r;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n fma.rn.f32x2 r, x, y, z;\n mov.b64 {%0, %1}, r;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 Mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 x, y, r;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mul.rn.f32x2 r, x, y;\n mov.b64 {%0, %1}, r;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 Add2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 x, y, r;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n add.rn.f32x2 r, x, y;\n mov.b64 {%0, %1}, r;\n}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ uint32_t PackHalf(float low, float high) {
    const __half2 h = __floats2half2_rn(low, high);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <int DTYPE>
__device__ __forceinline__ uint32_t PackTo(float low, float high) {
    if constexpr (DTYPE == FTH_B200_FP16) return PackHalf(low, high);
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(high), "f"(low));
    return d;
}
template <int DTYPE>
__device__ __forceinline__ float2 HalfPair(uint32_t x) {
    if constexpr (DTYPE == FTH_B200_BF16) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
    else return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
__device__ __forceinline__ float Max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// ---- rotary positions --------------------------------------------------------------------------------------------------
struct Rope {
    int half_layout, head_dim, rotary_dim, q_heads, k_heads;
    const void* q;
    void* q_out;
    const void* k;
    void* k_out;
    int64_t ldq, ldq_out, ldk, ldk_out;
    const int32_t* positions;
    const double* turns;
    float amplitude;
};
int CheckRope(const fth_b200_rope_desc* d, bool keys_stay);  // rope.cu; keys_stay: k_out is not written
Rope MakeRope(const fth_b200_rope_desc& d);

// Cosine and sine of position * turns full turns.  The product and its reduction to half a turn are 64-bit: at position
// 10^6 an FP32 product is off by 0.06 rad, this one by 10^-10.  What is left is below pi and FP32 serves it.
__device__ __forceinline__ float2 RopeAngle(int position, double turns, float amplitude) {
    const double t = static_cast<double>(position) * turns;
    float s, c;
    sincospif(static_cast<float>(2.0 * (t - rint(t))), &s, &c);
    return make_float2(__fmul_rn(c, amplitude), __fmul_rn(s, amplitude));
}
// One order of operations for every kernel that turns a pair, so that they give the same bits.
__device__ __forceinline__ float2 RopeTurn(float x1, float x2, float2 cs) {
    return make_float2(__fmaf_rn(x1, cs.x, -__fmul_rn(x2, cs.y)), __fmaf_rn(x2, cs.x, __fmul_rn(x1, cs.y)));
}
// Element j of the turned row that starts at element `row` of x; `angles` holds the row's rotary_dim / 2 pairs.
template <int DTYPE>
__device__ __forceinline__ float RopeElement(const Rope& r, const void* x, int64_t row, int j, const float2* angles) {
    const float own = rowops::ReadFloat<DTYPE>(x, row + j);
    if (j >= r.rotary_dim) return own;
    const int half = r.rotary_dim >> 1;
    const int pair = r.half_layout ? (j < half ? j : j - half) : j >> 1;
    const bool first = r.half_layout ? j < half : (j & 1) == 0;
    const int other = r.half_layout ? (first ? j + half : j - half) : j ^ 1;
    const float o = rowops::ReadFloat<DTYPE>(x, row + other);
    const float2 y = first ? RopeTurn(own, o, angles[pair]) : RopeTurn(o, own, angles[pair]);
    return first ? y.x : y.y;
}
// Elements j .. j + 7 of the turned row, j a multiple of 8; `vec`: 16-byte loads are aligned and half the rotary part is
// a multiple of 8, so that the eight lie in one part and their partners in another eight.
template <int DTYPE>
__device__ __forceinline__ void RopeEight(const Rope& r, const void* x, int64_t row, int j, const float2* angles, bool vec, float (&v)[8]) {
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = RopeElement<DTYPE>(r, x, row, j + i, angles);
        return;
    }
    rowops::ReadEight<DTYPE>(x, row + j, true, v);
    if (j >= r.rotary_dim) return;
    if (r.half_layout) {
        const int half = r.rotary_dim >> 1;
        const bool first = j < half;
        const int pair = first ? j : j - half;
        float o[8];
        rowops::ReadEight<DTYPE>(x, row + (first ? j + half : j - half), true, o);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 y = first ? RopeTurn(v[i], o[i], angles[pair + i]) : RopeTurn(o[i], v[i], angles[pair + i]);
            v[i] = first ? y.x : y.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            const float2 y = RopeTurn(v[i], v[i + 1], angles[(j + i) >> 1]);
            v[i] = y.x;
            v[i + 1] = y.y;
        }
    }
}

}  // namespace kv4
}  // namespace fth
