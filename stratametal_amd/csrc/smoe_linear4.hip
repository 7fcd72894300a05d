// stratametal_amd/csrc/smoe_linear4.hip - the product with 4-bit weights and group scales (gfx950, wave64): as the dense
// product, W[o][i] = scale[g][o] (code[o][i] - zero[g][o]), g = i / group.
//
// A group's part of a sum is scale (sum code x - zero sum x): the codes enter the matrix instructions as whole numbers of x's
// type, so that every product is exact and a weight is never rounded, and sum x comes from the same instructions with a
// matrix of ones.
#include "smoe_linear.hpp"

namespace smoe {

namespace {

// The codes of a dword (k = 0 .. 7, k's at bits 4 k) as eight whole numbers of bf16 or fp16.  bf16: a code in a byte is the
// e4m3 number code 2^-9 (its subnormals and first binade are one linear range), converted with a scale of 2^9; fp16: 1024 +
// code by its bits, less 1024.
template <bool F16>
__device__ __forceinline__ u32x4 expand8(uint32_t w) {
    const uint32_t lo = w & 0x0F0F0F0Fu, hi = (w >> 4) & 0x0F0F0F0Fu;
    const uint32_t a = __builtin_amdgcn_perm(hi, lo, 0x05010400u), b = __builtin_amdgcn_perm(hi, lo, 0x07030602u);
    u32x4 r;
    if constexpr (F16) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        const auto two = [](uint32_t c) {
            const f16x2 v = __builtin_bit_cast(f16x2, c | 0x64006400u) - f16x2{(_Float16)1024.0f, (_Float16)1024.0f};
            return __builtin_bit_cast(uint32_t, v);
        };
        r[0] = two(__builtin_amdgcn_perm(0u, a, 0x0C010C00u)), r[1] = two(__builtin_amdgcn_perm(0u, a, 0x0C030C02u));
        r[2] = two(__builtin_amdgcn_perm(0u, b, 0x0C010C00u)), r[3] = two(__builtin_amdgcn_perm(0u, b, 0x0C030C02u));
    } else {
        r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 512.0f, false));
        r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 512.0f, true));
        r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 512.0f, false));
        r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 512.0f, true));
    }
    return r;
}

__device__ __forceinline__ float scale_at(const void* p, int64_t i, int type) {
    return type == kF32 ? static_cast<const float*>(p)[i] : elem_to_f32(static_cast<const uint16_t*>(p)[i], type);
}

}  // namespace

// 16 outputs by 16 tokens to a work-group of eight waves, each every eighth 32 of K.
template <bool PAIR, bool F16>
__global__ __launch_bounds__(512) void k_linear4_few(const Linear4Args a) {
    constexpr int SETS = PAIR ? 2 : 1, WAVES = 8;
    __shared__ f32x4 sum_s[WAVES][SETS][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int o0 = blockIdx.x * 16, t0 = blockIdx.y * 16, q = lane >> 4;
    const uint8_t* w[2] = {static_cast<const uint8_t*>(a.w), static_cast<const uint8_t*>(a.w2)};
    const void* sc[2] = {a.scales, a.scales2};
    const uint8_t* zr[2] = {a.zeros, a.zeros2};
    const int64_t row = min(o0 + (lane & 15), a.n_out - 1), tok = min(t0 + (lane & 15), a.n_tokens - 1);
    const uint16_t* x = static_cast<const uint16_t*>(a.x) + tok * a.x_ld;
    const uint32_t one = F16 ? 0x3C003C00u : 0x3F803F80u;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    f32x4 acc[SETS];
#pragma unroll
    for (int i = 0; i < SETS; ++i) acc[i] = zero;
    for (int u = wave; u < a.n_in / 32; u += WAVES) {
        const int k = u * 32 + 8 * q;
        const uint4 xv = *reinterpret_cast<const uint4*>(x + k);
        const f32x4 sx = mfma16<F16>(make_uint4(one, one, one, one), xv, zero);
        const int64_t g = u * 32 / a.group;
#pragma unroll
        for (int i = 0; i < SETS; ++i) {
            const uint32_t c = *reinterpret_cast<const uint32_t*>(w[i] + row * (a.n_in / 2) + k / 2);
            const f32x4 s = mfma16<F16>(__builtin_bit_cast(uint4, expand8<F16>(c)), xv, zero);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t at = g * a.n_out + min(o0 + 4 * q + j, a.n_out - 1);
                const float z = zr[i] ? (float)zr[i][at] : 8.0f;
                acc[i][j] = __builtin_fmaf(scale_at(sc[i], at, a.s_type), __builtin_fmaf(-z, sx[j], s[j]), acc[i][j]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < SETS; ++i) sum_s[wave][i][lane] = acc[i];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int i = 0; i < SETS; ++i)
#pragma unroll
        for (int v = 1; v < WAVES; ++v) acc[i] = acc[i] + sum_s[v][i][lane];
    const int t = t0 + (lane & 15), o = o0 + 4 * q;
    if (t >= a.n_tokens || o >= a.n_out) return;
    const f32x4 g = acc[0], u = acc[SETS - 1];
    finish4<PAIR>(a, rows_vec(a), t, o, {g[0], g[1], g[2], g[3]}, {u[0], u[1], u[2], u[3]});
}

size_t linear4_part_bytes(int64_t, int, int, bool, int) { return 0; }

hipError_t launch_linear4(const Linear4Args& a, hipStream_t s) {
    const dim3 grid((a.n_out + 15) / 16, (a.n_tokens + 15) / 16);
    const bool f16 = a.w_type == kF16;
    if (a.w2 && f16) hipLaunchKernelGGL((k_linear4_few<true, true>), grid, dim3(512), 0, s, a);
    else if (a.w2) hipLaunchKernelGGL((k_linear4_few<true, false>), grid, dim3(512), 0, s, a);
    else if (f16) hipLaunchKernelGGL((k_linear4_few<false, true>), grid, dim3(512), 0, s, a);
    else hipLaunchKernelGGL((k_linear4_few<false, false>), grid, dim3(512), 0, s, a);
    return hipGetLastError();
}

}  // namespace smoe
