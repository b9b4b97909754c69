// Device helpers of the MXFP4 kernels.
#pragma once
#include "mx_numerics.h"
#include "nh_device.h"

namespace nh {

typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));

// Maximum over each quad of lanes.
__device__ __forceinline__ uint32_t quad_max_u32(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0xb1, 0xf, 0xf, false));  // quad_perm 1,0,3,2
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp((int)v, (int)v, 0x4e, 0xf, 0xf, false));  // quad_perm 2,3,0,1
    return v;
}

// Eight consecutive values (the first `count` of them; zeros behind) of x from
// element i: bf16 in v[0], f32 in v[0] and v[1].  Vector loads of global memory
// take any alignment, so rows may start anywhere.  ONCE: values that nobody
// reads again, past the caches (16384 x 4096 f32 to codes and back: 134 us
// without, 109).
template <bool ONCE = false>
__device__ __forceinline__ void mx_load8(const void* x, int64_t i, int count, int dtype, v4i (&v)[2]) {
    typedef int v4i_any __attribute__((ext_vector_type(4), aligned(2)));
    auto load = [](const void* p) {
        if constexpr (ONCE) return (v4i)__builtin_nontemporal_load((const v4i_any*)p);
        else return (v4i)(*(const v4i_any*)p);
    };
    v[0] = v[1] = v4i{0, 0, 0, 0};
    if (count == 8) {
        if (dtype == DT_BF16) {
            v[0] = load((const uint16_t*)x + i);
        } else {
            v[0] = load((const float*)x + i);
            v[1] = load((const float*)x + i + 4);
        }
    } else if (count > 0) {
        uint32_t t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            t[j] = 0;
            if (j < count) t[j] = dtype == DT_BF16 ? (uint32_t)((const uint16_t*)x)[i + j] : f32_bits(((const float*)x)[i + j]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[0][j] = (int)(dtype == DT_BF16 ? t[2 * j] | (t[2 * j + 1] << 16) : t[j]);
            v[1][j] = (int)(dtype == DT_BF16 ? 0u : t[4 + j]);
        }
    }
}

// Bits of the largest magnitude of eight values (infinities and NaNs order above).
__device__ __forceinline__ uint32_t mx_amax8(const v4i (&v)[2], int dtype) {
    if (dtype == DT_BF16) return bf16x8_absmax_bits(v[0]) << 16;
    return absbits_f32x4(v[1], absbits_f32x4(v[0], 0));
}

// Eight codes under scale byte e (255: zeros).
__device__ __forceinline__ uint32_t mx_encode_bf16x8(v4i v, uint32_t e) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const float s = f32_from_bits(e << 23);
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, (uint32_t)v[0]), s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, (uint32_t)v[1]), s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, (uint32_t)v[2]), s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, (uint32_t)v[3]), s, 3);
    return e == kMxNan ? 0u : q;
}

__device__ __forceinline__ uint32_t mx_encode_f32x8(const float (&v)[8], uint32_t e) {
    const float s = f32_from_bits(e << 23);
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], s, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], s, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], s, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], s, 3);
    return e == kMxNan ? 0u : q;
}

__device__ __forceinline__ uint32_t mx_encode8(const v4i (&v)[2], uint32_t e, int dtype) {
    if (dtype == DT_BF16) return mx_encode_bf16x8(v[0], e);
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = f32_from_bits((uint32_t)v[j >> 2][j & 3]);
    return mx_encode_f32x8(f, e);
}

// The first non-finite of eight values (element i on) into the caller's word.
__device__ __forceinline__ void mx_report8(uint64_t* word, int stage, int64_t i, int count, int dtype, const v4i (&v)[2]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float f = dtype == DT_BF16 ? f32_from_bits(((uint32_t)v[0][j >> 1] >> (16 * (j & 1))) << 16)
                                         : f32_from_bits((uint32_t)v[j >> 2][j & 3]);
        if (j < count && !is_finite_f32(f)) {
            report_nonfinite(word, stage, i + j, f);
            return;
        }
    }
}

// Eight codes to values: the sign and twice the magnitude come out of a byte
// table (two v_perm per four codes), the factor 2^(e - 128) is a power of two.
__device__ __forceinline__ void mx_decode8(uint32_t q, uint32_t e, float (&v)[8]) {
    // 2^(e - 128): subnormal for e <= 1, exact in f32 for every e
    const float s = f32_from_bits(e == kMxNan ? 0x7fc00000u : e > 1 ? (e - 1) << 23 : 0x00200000u << e);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t n = h ? q >> 4 : q;  // codes h, h + 2, h + 4, h + 6
        const uint32_t m = __builtin_amdgcn_perm(0x0c080604u, 0x03020100u, n & 0x07070707u);
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const float f = (float)((m >> (8 * b)) & 0xffu) * s;
            v[2 * b + h] = f32_from_bits(f32_bits(f) | (((n >> (8 * b + 3)) & 1u) << 31));
        }
    }
}

// One MFMA K step of 128: weights first, so lane l = 16 g + m holds output
// columns 4 g .. 4 g + 3 of row m.  SW / SA pick the scale byte.
template <int SW, int SA>
__device__ __forceinline__ v4f mx_mfma(v4i w, v4i a, v4f c, int sw, int sa) {
    const v8i w8 = {w[0], w[1], w[2], w[3], 0, 0, 0, 0}, a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, a8, c, 4, 4, SW, sw, SA, sa);
}

}  // namespace nh
