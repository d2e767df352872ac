// What the kernels that make, read and multiply rows in 8 and 4 bits share.
#pragma once
#include "tv_ops.h"

namespace tv {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

// Four values from p, those of them past `left` zero.
template <typename T>
__device__ __forceinline__ void load4(float (&v)[4], const T *p, int left) {
    typedef T T4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
    if (left >= 4) {
        const T4 x = *reinterpret_cast<const T4 *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = float(x[i]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? float(p[i]) : 0.0f;
}
__device__ __forceinline__ float finite_abs(float x) {
    const float a = fabsf(x);
    return a < __int_as_float(0x7f800000) ? a : 0.0f;      // (a comparison with NaN is false)
}
// Largest over the half wave.
template <int CTRL>
__device__ __forceinline__ float max_moved(float v) {
    return fmaxf(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true)));
}
__device__ __forceinline__ float half_wave_max(float v) {
    v = max_moved<0xb1>(v);       // quad_perm: the neighbour, the pair beside
    v = max_moved<0x4e>(v);
    v = max_moved<0x141>(v);      // row_half_mirror, row_mirror: the other half of 8 and of 16
    v = max_moved<0x140>(v);
    return fmaxf(v, __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(v), 0x401f)));      // lane ^ 16
}
// The scale of a block whose largest finite magnitude is `most`; `stored` is what goes to memory.
template <bool E8>
__device__ __forceinline__ float scale_of(float most, uint32_t &stored) {
    if (!E8) {
        const float s = fmaxf(most / 448.0f, 0x1p-126f);
        stored = __float_as_uint(s);
        return s;
    }
    // most = f * 2^e with 1 <= f < 2, 448 = 1.75 * 2^8: the power is e - 8, one more where f > 1.75
    const uint32_t b = __float_as_uint(most);
    const int e = int(b >> 23) - 127 - 8 + int((b & 0x7fffffu) > 0x600000u);
    const int power = e < -126 ? -126 : e;                 // (denormal maxima, zero among them, end here)
    stored = uint32_t(power + 127);
    return __uint_as_float(stored << 23);
}
template <bool E8>
__device__ __forceinline__ uint32_t codes_of(const float (&v)[4], float s) {
    // (the inverse of a power of two from 2^-126 to 2^120 is one, so that the product is the quotient)
    const float inverse = E8 ? __uint_as_float((254u << 23) - __float_as_uint(s)) : 0.0f;
    float q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = fabsf(v[i]) < __int_as_float(0x7f800000) ? (E8 ? v[i] * inverse : v[i] / s) : __int_as_float(0x7fc00000);
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], r, true));
}
__device__ __forceinline__ void store4(uint8_t *p, uint32_t c, int left) {
    typedef uint32_t Four __attribute__((aligned(1)));
    if (left >= 4) {
        *reinterpret_cast<Four *>(p) = c;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < left) p[i] = uint8_t(c >> (8 * i));
}
template <bool E8>
__device__ __forceinline__ void store_scale(void *scales, size_t at, uint32_t stored) {
    if (E8) static_cast<uint8_t *>(scales)[at] = uint8_t(stored);
    else static_cast<uint32_t *>(scales)[at] = stored;
}

// An e8m0 byte as a float; 255 is NaN, and 0 the denormal 2^-127.
__device__ __forceinline__ float e8_value(uint32_t e) {
    return __uint_as_float(e == 255u ? 0x7fc00000u : e == 0u ? 0x00400000u : e << 23);
}

// Eight values from p, those of them past `left` zero.
template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T *p, int left) {
    typedef T T8 __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    if (left >= 8) {
        const T8 x = *reinterpret_cast<const T8 *>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = float(x[i]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? float(p[i]) : 0.0f;
}

// ---- 4-bit rows: a lane holds eight coordinates, four neighbouring lanes a block ----

// The largest magnitude of eight values as its bits: those of an infinity or a NaN are the largest of all.
__device__ __forceinline__ uint32_t magnitude8(const float (&v)[8]) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
    return most;
}
// Largest over four neighbouring lanes.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
    v = max(v, uint32_t(__builtin_amdgcn_mov_dpp(int(v), 0xb1, 0xf, 0xf, true)));
    return max(v, uint32_t(__builtin_amdgcn_mov_dpp(int(v), 0x4e, 0xf, 0xf, true)));
}
constexpr uint32_t kInfBits = 0x7f800000u;
// The scale of a block whose largest magnitude has the bits `most`; `stored` is what goes to memory, NaN where there is no number for it.
__device__ __forceinline__ float scale4_of(uint32_t most, uint32_t &stored) {
    // most = f * 2^e with 1 <= f < 2, 7 = 1.75 * 2^2: the power is e - 2, one more from f = 1.75 on
    const int e = int(most >> 23) - 127 - 2 + int((most & 0x7fffffu) >= 0x600000u);
    const uint32_t power = uint32_t((e < -126 ? -126 : e) + 127);
    stored = most >= kInfBits ? 255u : power;
    return __uint_as_float(power << 23);
}
// Eight codes, the first in the lowest bits.  (A value divided by its power of two is exact, and what is rounded to 0 may be a denormal: the instruction's
// division by the scale takes both.)
__device__ __forceinline__ uint32_t codes4_of(const float (&v)[8], float s, uint32_t most) {
    uint32_t c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], s, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], s, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], s, 3);
    return most >= kInfBits ? 0u : c;
}
// Those of them that are left, two a byte; values past the end are zeros, and so is the half byte behind an odd one.
__device__ __forceinline__ void store_nibbles(uint8_t *p, uint32_t c, int left) {
    typedef uint32_t Four __attribute__((aligned(1)));
    if (left >= 7) {
        *reinterpret_cast<Four *>(p) = c;
        return;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (2 * i < left) p[i] = uint8_t(c >> (8 * i));
}
__device__ __forceinline__ void values_of4(float (&v)[8], uint32_t c, float s) {
    typedef float v2f __attribute__((ext_vector_type(2)));
    const v2f a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
    const v2f d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2), e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
    v[0] = a[0] * s; v[1] = a[1] * s; v[2] = b[0] * s; v[3] = b[1] * s;
    v[4] = d[0] * s; v[5] = d[1] * s; v[6] = e[0] * s; v[7] = e[1] * s;
}

}  // namespace tv
