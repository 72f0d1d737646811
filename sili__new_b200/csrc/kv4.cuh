// The 4-bit key/value cache's format, shared by the kernels that write, read
// and attend over it.
//
// A head vector of `dim` values is cut into groups of 32 along the head.  A
// group holds e2m1 codes (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives; the
// layers' FP4 codes, element 2i in the low nibble of byte i) and one scale
// byte: the eight bits below the sign of an IEEE half (5 exponent and 3
// mantissa bits), so byte << 7 is the scale as a half.  A value is code *
// scale: at most 2 + 4 significant bits, exact in fp16 (|value| <= 61440) and
// bf16.  A group that held an infinity or NaN has the scale byte 0xFF (NaN),
// which poisons exactly that group.
//
//   codes  [pages][2][kv heads][page][dim / 2]    (second axis: 0 K, 1 V)
//   scales [pages][2][kv heads][page][dim / 32]
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace sili {

constexpr int kKvGroup = 32;
// the largest scale on the byte's grid whose 6 * scale is still a finite half
constexpr float kKvScaleMost = 10240.f;
constexpr uint32_t kKvScaleNaN = 0xFFu;

// Where one (page, K or V, kv head) block of the cache starts, in units of
// token rows (a row: dim/2 code bytes, dim/32 scale bytes).  64 bits: a long
// cache's offsets pass 2^32.
__host__ __device__ __forceinline__ int64_t kv4_row(int64_t page_id, int w, int kv_head, int kv_heads, int page) {
    return ((page_id * 2 + w) * kv_heads + kv_head) * (int64_t)page;
}

// the scale byte of a group whose largest |value| has the bits `amax_bits`:
// amax / 6 rounded to a half, its mantissa to three bits, ties to even
__device__ __forceinline__ uint32_t kv4_scale_byte(uint32_t amax_bits) {
    if (amax_bits >= 0x7F800000u) return kKvScaleNaN;
    const float s = fminf(__fdiv_rn(__uint_as_float(amax_bits), 6.f), kKvScaleMost);
    const uint32_t h = __half_as_ushort(__float2half_rn(s));
    return (h + 0x3Fu + ((h >> 7) & 1u)) >> 7;
}
__device__ __forceinline__ float kv4_scale(uint32_t byte) {
    return __half2float(__ushort_as_half((unsigned short)(byte << 7)));
}

// e2m1 code of x under the group scale s: nearest, midpoints up in magnitude,
// at most 6, never a negative zero.  The thresholds t * s are exact in fp32
// (t has at most 3 significant bits, s 4), so no rounded quotient decides;
// s == 0 gives 0 (and so does the NaN scale: every comparison fails).
struct Kv4Thresholds {
    float t[7];
    __device__ __forceinline__ explicit Kv4Thresholds(float s) {
        const float f[7] = {0.25f, 0.75f, 1.25f, 1.75f, 2.5f, 3.5f, 5.f};
#pragma unroll
        for (int i = 0; i < 7; ++i) t[i] = s > 0.f ? f[i] * s : __int_as_float(0x7FC00000);
    }
    // three comparisons: which half of the codes, which quarter, which one
    __device__ __forceinline__ uint32_t code(float x) const {
        const float a = fabsf(x);
        const bool b2 = a >= t[3];
        const bool b1 = a >= (b2 ? t[5] : t[1]);
        const bool b0 = a >= (b1 ? (b2 ? t[6] : t[2]) : (b2 ? t[4] : t[0]));
        const uint32_t m = (b2 ? 4u : 0u) + (b1 ? 2u : 0u) + (b0 ? 1u : 0u);
        return m && x < 0.f ? m + 8u : m;
    }
};

// Four bytes of codes -> four half2 (low nibble first), unscaled.
__device__ __forceinline__ void kv4_decode4(uint32_t w, uint32_t out[4]) {
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(out[0]), "=r"(out[1]), "=r"(out[2]), "=r"(out[3]) : "r"(w));
}

__device__ __forceinline__ float2 half2_bits_to_float2(uint32_t u) {
    __half2_raw r;
    r.x = (unsigned short)(u & 0xFFFFu);
    r.y = (unsigned short)(u >> 16);
    return __half22float2(__half2(r));
}

// element types of the activations
template <typename T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements, one access of N * sizeof(T) bytes (aligned to it)
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

}  // namespace sili
