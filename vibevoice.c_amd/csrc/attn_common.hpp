// What the attention kernels and the kernels that fill a KV cache share: the softmax's exponential, lane exchanges,
// the page size, and the FP8 codec.
#pragma once

#include "vv_common.hpp"

namespace vv {

typedef h16 h16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kPage = 64;            // positions per page (include/vibevoice/kv_quant.h:52)
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// A value and its partner's, 32 (or 16) lanes away, combined in the vector ALU: the gfx950 lane swaps exchange
// the odd rows of one register with the even rows of another (rows of 32 or 16 lanes), so from two copies of v
// one register ends up with the lower row's values in both rows of a pair and the other with the upper row's.
// No trip through the LDS crossbar and no counter to wait for; max and + commute, so every lane gets the bits
// that v (op) shuffle-xor(v) gave it. (As instructions: the compiler's builtin for them hands back the first
// register twice. The two wait states are what it puts between a vector write and a swap that reads it.)
__device__ __forceinline__ void swap_rows32(float& a, float& b) {
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}
__device__ __forceinline__ void swap_rows16(float& a, float& b) {
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(a), "+v"(b));
}
__device__ __forceinline__ float max_xor32(float v) {
    float a = v, b = v;
    swap_rows32(a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float sum_xor32(float v) {
    float a = v, b = v;
    swap_rows32(a, b);
    return a + b;
}
__device__ __forceinline__ float max_xor16(float v) {
    float a = v, b = v;
    swap_rows16(a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float sum_xor16(float v) {
    float a = v, b = v;
    swap_rows16(a, b);
    return a + b;
}

// Cache formats the matrix-core kernels read (include/vibevoice/kv_quant.h:34-36).
// The FP8 ones are widened to FP16 on their way into the registers: every
// E4M3 / E5M2 value is an FP16 value, so from there on the tile is the tile of
// an FP16 cache that holds the decoded values.
constexpr int kFmtFp16 = 0, kFmtE4M3 = 1, kFmtE5M2 = 2;

// Four FP8 codes (the bytes of `codes`) as two half2 words, lanes in byte order.
template <int kFmt>
__device__ __forceinline__ void widen4(uint32_t codes, uint32_t& lo, uint32_t& hi) {
    // byte b -> 16-bit lane b << 8: an E5M2 code IS the top byte of the FP16 value
    lo = __builtin_amdgcn_perm(0u, codes, 0x010C000Cu);
    hi = __builtin_amdgcn_perm(0u, codes, 0x030C020Cu);
    if constexpr (kFmt == kFmtE4M3) {
        // sign stays, exponent and mantissa move down one bit (FP16 has five exponent bits):
        // that reads 2^-8 too small (bias 15 against 7), subnormals included, so scale by 256
        typedef h16 h16x2v __attribute__((ext_vector_type(2)));
        const h16x2v k256 = {(h16)256.0f, (h16)256.0f};
        const uint32_t l = ((lo >> 1) & 0x3F803F80u) | (lo & 0x80008000u);
        const uint32_t h = ((hi >> 1) & 0x3F803F80u) | (hi & 0x80008000u);
        lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h16x2v, l) * k256);
        hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h16x2v, h) * k256);
    }
}

// The FP8 store (src/cuda/kv_codec.cuh:66-128): one value to E4M3 (bias 7, largest finite 448 = 0x7E) or E5M2 (bias 15,
// largest finite 57344 = 0x7B) in integer arithmetic: zero and NaN give a signed
// zero, magnitudes from half a step above the largest finite value saturate to
// it, below the smallest normal the value is a count of subnormal steps rounded
// half up, else round to nearest even on the FP32 mantissa with the carry going
// into the exponent.
template <bool kE5M2>
__device__ __forceinline__ uint32_t fp8_encode(float f) {
    constexpr int kMant = kE5M2 ? 2 : 3, kBias = kE5M2 ? 15 : 7, kDrop = 23 - kMant;
    constexpr uint32_t kMaxCode = kE5M2 ? 0x7Bu : 0x7Eu;
    const uint32_t b = __builtin_bit_cast(uint32_t, f);
    const uint32_t sign = (b >> 24) & 0x80u;
    const float a = fabsf(f);
    if (!(a > 0.0f)) return sign;
    if (a >= (kE5M2 ? 61440.0f : 464.0f)) return sign | kMaxCode;
    int e = (int)((b >> 23) & 0xFFu) - 127;
    if (e < 1 - kBias) {
        int q = (int)(a * (kE5M2 ? 65536.0f : 512.0f) + 0.5f);
        q = min(q, 1 << kMant);                       // rolls into the smallest normal
        return sign | (uint32_t)q;
    }
    const uint32_t m = b & 0x7FFFFFu;
    uint32_t mm = m >> kDrop;
    const uint32_t rem = m & ((1u << kDrop) - 1u), half_way = 1u << (kDrop - 1);
    if (rem > half_way || (rem == half_way && (mm & 1u))) {
        if (++mm == (1u << kMant)) { mm = 0; ++e; }
    }
    if (e > (kE5M2 ? 15 : 8)) return sign | kMaxCode;
    return sign | ((uint32_t)(e + kBias) << kMant) | mm;
}

}  // namespace vv
