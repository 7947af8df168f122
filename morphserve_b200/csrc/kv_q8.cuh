// The 8-bit KV pool: device view, number format, and the conversions between codes and values.
//
// One scale for each (block, layer, kv head), K and V apart; a code q of the block stands for q * s.
//   int8: s = fl32(amax / 127), q = rne(x * fl32(1 / s)).
//   e4m3: s = 2^e, the smallest power of two with amax <= 448 s, q = e4m3(x / s).  A power of two costs nothing here -
//         e4m3's steps are relative - and makes x / s exact, so a value is rounded once, and an appended token that
//         raises the scale re-rounds the older codes only where they become subnormal.
// A scale that would not be a normal 32-bit number is 0 and its codes are 0.  If a block's values are not all finite its
// scale is NaN and the codes of the tokens that were not are 0: what is read back is NaN, for that block and head alone.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace mkv {

// Device-side view of mkv_pool_q8, by value as a kernel parameter.
struct PoolViewQ8 {
    int32_t num_segments;
    int32_t code;
    int32_t num_layers;
    int32_t num_kv_heads;
    int32_t block_size;
    int32_t head_dim;
    int64_t num_blocks_org;
    int64_t chunk_blocks;
    int64_t total_blocks;
    int64_t tile_bytes;  // codes of one (block, layer, head): block_size * head_dim
    uint8_t *k_base[MKV_MAX_SEGMENTS];
    uint8_t *v_base[MKV_MAX_SEGMENTS];
    float *k_scale[MKV_MAX_SEGMENTS];
    float *v_scale[MKV_MAX_SEGMENTS];
};

int validate_pool_q8(const mkv_pool_q8 *pool, PoolViewQ8 *out);

// Segment of block `blk` and its row there: the id -> address rule of locate_block (common.cuh).
__device__ __forceinline__ void locate_block(const PoolViewQ8 &p, int64_t blk, int &seg, int64_t &row) {
    if (blk < p.num_blocks_org) {
        seg = 0;
        row = blk;
    } else {
        const int64_t rel = blk - p.num_blocks_org;
        const int64_t j = rel / p.chunk_blocks;
        seg = 1 + (int)j;
        row = rel - j * p.chunk_blocks;
    }
}

// (block row, layer, head) counted through a segment: times tile_bytes it is the tile's offset in the codes, as it
// stands the offset in the scales.
__device__ __forceinline__ int64_t tile_index(const PoolViewQ8 &p, int64_t row, int layer, int head) {
    return (row * p.num_layers + layer) * p.num_kv_heads + head;
}

// ---- scales ---------------------------------------------------------------------------------------------------
// From the bits of the largest absolute value, as fp32 (an ordinary number, infinity or NaN; the sign bit is clear).
template <int CODE>
__device__ __forceinline__ float scale_of(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fffffffu);
    if (CODE == MKV_Q8_INT8) {
        const float s = __fdiv_rn(__uint_as_float(amax_bits), 127.f);
        return s < 1.17549435e-38f ? 0.f : s;
    }
    // amax = (1 + f) 2^k, 448 = 1.75 * 2^8: e = k - 8, one more if f > 0.75
    const int e = (int)(amax_bits >> 23) - 8 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e <= 0 ? 0.f : __uint_as_float((uint32_t)e << 23);
}
// 0 for the scale 0 and for NaN: every code becomes 0.  Exact for the powers of two of e4m3.
__device__ __forceinline__ float inverse_of(float s) { return s > 0.f ? __frcp_rn(s) : 0.f; }
// Scale of a block that gains a token: NaN once either is NaN.
__device__ __forceinline__ float larger_scale(float held, float fresh) {
    return (held > fresh || held != held) ? held : fresh;
}

// ---- values to codes ------------------------------------------------------------------------------------------
// Four codes, the first in the lowest byte.  int8: 1.5 * 2^23 + x * inv is rounded once, to an integer, half to even, by
// the fused multiply-add; its low byte is the code in two's complement.  |x * inv| <= 127 (1 + 2^-22), so nothing needs
// clamping.  e4m3: x * inv is exact.
template <int CODE>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float inv) {
    if (CODE == MKV_Q8_INT8) {
        constexpr float kMagic23 = 12582912.f;
        const uint32_t x = __float_as_uint(__fmaf_rn(a, inv, kMagic23)), y = __float_as_uint(__fmaf_rn(b, inv, kMagic23));
        const uint32_t z = __float_as_uint(__fmaf_rn(c, inv, kMagic23)), w = __float_as_uint(__fmaf_rn(d, inv, kMagic23));
        return __byte_perm(__byte_perm(x, y, 0x0040), __byte_perm(z, w, 0x0040), 0x5410);
    }
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(a, inv), __fmul_rn(b, inv)), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__fmul_rn(c, inv), __fmul_rn(d, inv)), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
template <int CODE>
__device__ __forceinline__ uint8_t encode1(float a, float inv) {
    return (uint8_t)encode4<CODE>(a, 0.f, 0.f, 0.f, inv);
}

// ---- codes to numbers -----------------------------------------------------------------------------------------
// Four e4m3 codes as fp16: exact.
__device__ __forceinline__ void e4m3x4_to_half2(uint32_t w, uint32_t &lo, uint32_t &hi) {
    asm("{\n.reg .b16 l, h;\nmov.b32 {l, h}, %2;\ncvt.rn.f16x2.e4m3x2 %0, l;\ncvt.rn.f16x2.e4m3x2 %1, h;\n}\n" : "=r"(lo), "=r"(hi) : "r"(w));
}
template <int CODE>
__device__ __forceinline__ float decode1(uint32_t byte) {
    if (CODE == MKV_Q8_INT8) return (float)(int8_t)byte;
    return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)byte, __NV_E4M3)));
}
template <int CODE>
__device__ __forceinline__ float4 decode4(uint32_t w) {
    uint32_t lo, hi;
    if (CODE == MKV_Q8_INT8) {  // behind the byte 0x64 a code with its sign bit flipped is the fp16 number 1024 + 128 + q
        const uint32_t x = w ^ 0x80808080u, y = __byte_perm(x, 0x64646464u, 0x4140), z = __byte_perm(x, 0x64646464u, 0x4342);
        const __half2 off = __float2half2_rn(-1152.f), l = __hadd2(*reinterpret_cast<const __half2 *>(&y), off),
                      h = __hadd2(*reinterpret_cast<const __half2 *>(&z), off);
        lo = *reinterpret_cast<const uint32_t *>(&l);
        hi = *reinterpret_cast<const uint32_t *>(&h);
    } else {
        e4m3x4_to_half2(w, lo, hi);
    }
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&lo)), b = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
    return make_float4(a.x, a.y, b.x, b.y);
}

// ---- the model's types ----------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float value_of(T x);
template <> __device__ __forceinline__ float value_of<float>(float x) { return x; }
template <> __device__ __forceinline__ float value_of<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float value_of<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T rounded(float x);
template <> __device__ __forceinline__ float rounded<float>(float x) { return x; }
template <> __device__ __forceinline__ __half rounded<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 rounded<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

static inline int dtype_bytes(int dtype) { return dtype == MKV_F32 ? 4 : 2; }
static inline bool dtype_ok(int dtype) { return dtype == MKV_F16 || dtype == MKV_BF16 || dtype == MKV_F32; }

}  // namespace mkv
