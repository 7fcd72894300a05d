// stratametal_amd/csrc/smoe_types.hpp - rows of f32, fp16 or bf16 values for the dense operators round the block: the
// element types, four values from registers, and the exponential their activations take.
#pragma once

#include "smoe_device.hpp"

namespace smoe {

// smoe.h's SMOE_F32, SMOE_F16, SMOE_BF16 (GGUF's type numbers)
enum ElemType : int { kF32 = 0, kF16 = 1, kBf16 = 30 };
__host__ __device__ constexpr int elem_bytes(int type) { return type == kF32 ? 4 : 2; }

// One value to and from f32; the conversion instructions round to nearest even, as the hardware's fp16 does.
__device__ __forceinline__ float elem_to_f32(uint32_t bits, int type) {
    return type == kF32 ? u2f(bits)
                        : type == kBf16 ? bf16_to_f32(bits) : (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}
__device__ __forceinline__ uint16_t f32_to_half_bits(float v, int type) {
    return type == kBf16 ? (uint16_t)f32_to_bf16(v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b, int type) {
    return (uint32_t)f32_to_half_bits(a, type) | (uint32_t)f32_to_half_bits(b, type) << 16;
}

// Four values to `p` (aligned to them), one store: vector types, as the compiler takes stores of structs in two branches
// apart and joins their words again into other widths (a 256 x 256 tile of bf16 was stored at 1.4 TB/s).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void store4(void* p, const float (&v)[4], int type) {
    if (type == kF32) {
        *static_cast<u32x4*>(p) = u32x4{f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])};
    } else if (type == kBf16) {
        *static_cast<u32x2*>(p) = u32x2{pack_half2(v[0], v[1], kBf16), pack_half2(v[2], v[3], kBf16)};
    } else {
        *static_cast<u32x2*>(p) = u32x2{pack_half2(v[0], v[1], kF16), pack_half2(v[2], v[3], kF16)};
    }
}
__device__ __forceinline__ void store1(void* p, int64_t i, float v, int type) {
    if (type == kF32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = f32_to_half_bits(v, type);
}

// e^x = 2^t, t = x log2 e with the product's rounding error and log2 e's low part carried as a first-order factor
// 1 + ln2 * rest, so that the error stays at the hardware exponential's own rounding for every |x| (t alone would be off
// by |x| 2^-24).  x past the range gives 0 or inf.
__device__ __forceinline__ float exp_fast(float x) {
    constexpr float kLog2e = 1.44269502f, kLog2eLow = 1.92596300e-8f;
    const float xc = __builtin_fminf(__builtin_fmaxf(x, -150.0f), 150.0f);  // (the rest of an infinite product is NaN)
    const float t = xc * kLog2e;
    const float rest = __builtin_fmaf(xc, kLog2eLow, __builtin_fmaf(xc, kLog2e, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    const float r = __builtin_fmaf(e, rest * 0.693147181f, e);
    return e == __builtin_inff() ? e : x != x ? x : r;
}
// (the quotient by the hardware's reciprocal: 1 ulp)
__device__ __forceinline__ float sigmoid_fast(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_fast(-x)); }

}  // namespace smoe
