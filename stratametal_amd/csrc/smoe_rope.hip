// stratametal_amd/csrc/smoe_rope.hip - rotary positions, and the write of keys and values into a paged cache (gfx950, wave64).
//
// A pair (a, b) of a head's first `rot` values at position p turns by p t_i revolutions: s (a c - b d, b c + a d), c and d
// the cosine and sine.  p t_i is formed and reduced to an eighth of a turn either side of a quarter in 64 bits (in 32 the
// angle of position 10^6 would be off by 0.03), the polynomials are in 32; the pair's products are fused, one rounding to the
// output's type.
#include "smoe_launch.hpp"
#include "smoe_rules.hpp"
#include "smoe_types.hpp"

namespace smoe {

namespace {

// (cos, sin) of r turns: r = q / 4 + g, |g| <= 1/8; Taylor to the 10th and 9th degree of 2 pi g <= pi / 4, whose next terms are at
// most 2^-32.5 of the cosine and 2^-28.6 of the sine (a 24th of its half step).
__device__ __forceinline__ float2 cos_sin_turns(double r) {
    r -= __builtin_rint(r);
    const double q = __builtin_rint(4.0 * r);
    const float a = 6.28318531f * (float)(r - 0.25 * q);
    const float z = a * a;
    float s = 2.75573192e-6f;
    s = __builtin_fmaf(s, z, -1.98412698e-4f);
    s = __builtin_fmaf(s, z, 8.33333333e-3f);
    s = __builtin_fmaf(s, z, -1.66666667e-1f);
    s = __builtin_fmaf(s * z, a, a);
    float c = -2.75573192e-7f;
    c = __builtin_fmaf(c, z, 2.48015873e-5f);
    c = __builtin_fmaf(c, z, -1.38888889e-3f);
    c = __builtin_fmaf(c, z, 4.16666667e-2f);
    c = __builtin_fmaf(c, z, -0.5f);
    c = __builtin_fmaf(c, z, 1.0f);
    const int k = (int)q & 3;
    const float x = k & 1 ? s : c, y = k & 1 ? c : s;
    return make_float2(k == 1 || k == 2 ? -x : x, k == 2 || k == 3 ? -y : y);
}

// N neighbouring values, aligned to as many bytes as `vec` says (N * size at most 16 a piece).
template <int N>
__device__ __forceinline__ void load_values(const void* p, int64_t i, int type, float (&v)[N]) {
    if (type == kF32) {
        const float* f = static_cast<const float*>(p) + i;
        if constexpr (N % 4 == 0) {
#pragma unroll
            for (int j = 0; j < N; j += 4) {
                const u32x4 q = *reinterpret_cast<const u32x4*>(f + j);
#pragma unroll
                for (int l = 0; l < 4; ++l) v[j + l] = u2f(q[l]);
            }
        } else if constexpr (N == 2) {
            const u32x2 q = *reinterpret_cast<const u32x2*>(f);
            v[0] = u2f(q[0]), v[1] = u2f(q[1]);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] = f[j];
        }
        return;
    }
    uint32_t w[(N + 1) / 2];
    const uint16_t* h = static_cast<const uint16_t*>(p) + i;
    if constexpr (N == 8) {
        const u32x4 q = *reinterpret_cast<const u32x4*>(h);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = q[j];
    } else if constexpr (N == 4) {
        const u32x2 q = *reinterpret_cast<const u32x2*>(h);
        w[0] = q[0], w[1] = q[1];
    } else if constexpr (N == 2) {
        w[0] = *reinterpret_cast<const uint32_t*>(h);
    } else {
        w[0] = h[0];
    }
    const auto each = [&](auto f16) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = elem_to_f32(j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xFFFFu, decltype(f16)::value);
    };
    if (type == kBf16) each(std::integral_constant<int, kBf16>{});
    else each(std::integral_constant<int, kF16>{});
}
template <int N>
__device__ __forceinline__ void store_values(void* p, int64_t i, int type, const float (&v)[N]) {
    if (type == kF32) {
        float* f = static_cast<float*>(p) + i;
        if constexpr (N % 4 == 0) {
#pragma unroll
            for (int j = 0; j < N; j += 4)
                *reinterpret_cast<u32x4*>(f + j) = u32x4{f2u(v[j]), f2u(v[j + 1]), f2u(v[j + 2]), f2u(v[j + 3])};
        } else if constexpr (N == 2) {
            *reinterpret_cast<u32x2*>(f) = u32x2{f2u(v[0]), f2u(v[1])};
        } else {
            f[0] = v[0];
        }
        return;
    }
    uint16_t* h = static_cast<uint16_t*>(p) + i;
    if constexpr (N == 1) {
        h[0] = f32_to_half_bits(v[0], type);
    } else {
        uint32_t w[N / 2];
        const auto each = [&](auto f16) {
#pragma unroll
            for (int j = 0; j < N / 2; ++j) w[j] = pack_half2(v[2 * j], v[2 * j + 1], decltype(f16)::value);
        };
        if (type == kBf16) each(std::integral_constant<int, kBf16>{});
        else each(std::integral_constant<int, kF16>{});
        if constexpr (N == 8) *reinterpret_cast<u32x4*>(h) = u32x4{w[0], w[1], w[2], w[3]};
        else if constexpr (N == 4) *reinterpret_cast<u32x2*>(h) = u32x2{w[0], w[1]};
        else *reinterpret_cast<uint32_t*>(h) = w[0];
    }
}

}  // namespace

// A work-group of 256 threads takes `per` tokens: their cosines and sines once into LDS, then units of 2 W values in turn,
// queries, keys and values alike: W pairs of a head's turned part (HALF: two runs of W values, else one of 2 W), or 2 W of its
// other values.  Bound by the values' bytes; one token by a launch and two memory round trips.  8192 tokens, 32 and 8 heads of 128,
// bf16: 49 us, 4.1 TB/s; one token 4.2 us; per: 4 of many tokens, so that a work-group's sines serve enough values.
template <int W, bool HALF>
__global__ __launch_bounds__(256) void k_rope(const RopeArgs a, int per) {
    extern __shared__ float2 cs[];  // [per][rot / 2]
    const int t0 = blockIdx.x * per, n_t = min(per, a.n_tokens - t0);
    const int half = a.rot / 2;
    for (int i = threadIdx.x; i < n_t * half; i += 256) {
        const int t = i / half;
        float2 v = cos_sin_turns((double)a.positions[t0 + t] * a.turns[i - t * half]);
        cs[i] = make_float2(v.x * a.scale, v.y * a.scale);
    }
    __syncthreads();
    const int of_head = a.head_dim / (2 * W), turned = half / W;
    const int q_units = a.n_heads * of_head, k_units = a.n_kv * of_head, units = q_units + 2 * k_units;
    for (int i = threadIdx.x; i < n_t * units; i += 256) {
        const int t = i / units, tok = t0 + t;
        int u = i - t * units;
        const void* src;
        void* dst;
        int64_t from, to;
        int to_type;
        bool turn = true;
        if (u < q_units) {
            const int h = u / of_head;
            u -= h * of_head;
            src = a.q, dst = a.q_out, to_type = a.q_type;
            from = tok * a.q_ld + h * a.head_dim, to = tok * a.q_out_ld + h * a.head_dim;
        } else {
            u -= q_units;
            turn = u < k_units;
            if (!turn) u -= k_units;
            const int h = u / of_head;
            u -= h * of_head;
            const int64_t slot = a.slots[tok];
            if (slot < 0 || slot >= a.n_slots) continue;
            const int64_t page = slot / a.page_size;
            src = turn ? a.k : a.v, dst = turn ? a.k_pages : a.v_pages, to_type = a.t_type;
            from = tok * (turn ? a.k_ld : a.v_ld) + h * a.head_dim;
            to = ((page * a.n_kv + h) * a.page_size + (slot - page * a.page_size)) * a.head_dim;
        }
        turn = turn && u < turned;
        // the unit's two runs of W values
        const int first = HALF && turn ? u * W : u * 2 * W, second = HALF && turn ? first + half : first + W;
        float x[W], y[W];
        load_values(src, from + first, a.x_type, x);
        load_values(src, from + second, a.x_type, y);
        if (turn) {
            const float2* c = cs + t * half + u * W;
            if constexpr (HALF) {
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    const float2 r = c[j];
                    const float p = x[j], q = y[j];
                    x[j] = __builtin_fmaf(p, r.x, -(q * r.y));
                    y[j] = __builtin_fmaf(q, r.x, p * r.y);
                }
            } else if constexpr (W > 1) {
#pragma unroll
                for (int j = 0; j < W; ++j) {
                    const float2 r = c[j];
                    float(&v)[W] = j < W / 2 ? x : y;
                    const int at = 2 * j % W;
                    const float p = v[at], q = v[at + 1];
                    v[at] = __builtin_fmaf(p, r.x, -(q * r.y));
                    v[at + 1] = __builtin_fmaf(q, r.x, p * r.y);
                }
            } else {
                const float2 r = c[0];
                const float p = x[0], q = y[0];
                x[0] = __builtin_fmaf(p, r.x, -(q * r.y));
                y[0] = __builtin_fmaf(q, r.x, p * r.y);
            }
        }
        store_values(dst, to + first, to_type, x);
        store_values(dst, to + second, to_type, y);
    }
}

namespace {
template <int W>
hipError_t launch_rope_as(const RopeArgs& a, int per, hipStream_t s) {
    const dim3 grid((unsigned)rope_groups(a.n_tokens));
    const size_t lds = (size_t)per * (a.rot / 2) * sizeof(float2);
    if (a.half) hipLaunchKernelGGL((k_rope<W, true>), grid, dim3(256), lds, s, a, per);
    else hipLaunchKernelGGL((k_rope<W, false>), grid, dim3(256), lds, s, a, per);
    return hipGetLastError();
}
}  // namespace

hipError_t launch_rope(const RopeArgs& a, hipStream_t s) {
    // the widest runs that the head, its turned part and the rows' alignment allow
    const auto fits = [&](int w) {
        const auto rows = [&](const void* p, int64_t ld, int type) {
            const int64_t bytes = w * elem_bytes(type) < 16 ? w * elem_bytes(type) : 16;
            return !p || ((reinterpret_cast<uintptr_t>(p) | (uintptr_t)(ld * elem_bytes(type))) & (bytes - 1)) == 0;
        };
        return a.rot % (2 * w) == 0 && a.head_dim % (2 * w) == 0 && rows(a.q, a.q_ld, a.x_type) && rows(a.q_out, a.q_out_ld, a.q_type) &&
               rows(a.k, a.k_ld, a.x_type) && rows(a.v, a.v_ld, a.x_type) && rows(a.k_pages, 0, a.t_type) && rows(a.v_pages, 0, a.t_type);
    };
    const int per = rope_tokens(a.n_tokens);
    if (fits(8)) return launch_rope_as<8>(a, per, s);
    if (fits(4)) return launch_rope_as<4>(a, per, s);
    if (fits(2)) return launch_rope_as<2>(a, per, s);
    return launch_rope_as<1>(a, per, s);
}

}  // namespace smoe
