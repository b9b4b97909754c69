// MXFP4 (OCP microscaling) numerics shared by the gfx950 kernels and the host
// twins: e2m1 elements in blocks of 32 consecutive values of a row, each block
// with one e8m0 scale byte E standing for 2^(E - 127) (255: NaN).
//
// Quantization of a block with largest magnitude a: the scale is the power of
// two 2^(floor(log2 a) - 2), 2 being the exponent of the largest element, so
// a / scale lies in [4, 8) and values past 6 saturate there; elements are
// rounded to nearest, ties to the even mantissa.  Every step but that rounding
// is exact.  A block that holds a NaN or an infinity gets E = 255 and codes 0:
// it reads back as NaN and makes every product with it NaN.
#pragma once
#include "nh_numerics.h"

namespace nh {

constexpr int kMxBlock = 32;
constexpr uint32_t kMxNan = 255;

NH_HD uint64_t mx_row_codes(uint64_t cols) { return (cols + 1) / 2; }               // bytes of a row's codes
NH_HD uint64_t mx_row_blocks(uint64_t cols) { return (cols + kMxBlock - 1) / kMxBlock; }  // and of its scales

// The scale byte from the bits of the block's largest magnitude.  The exponent
// field of a subnormal is 0, and so is what 2 less would clamp to: 2^-127, on
// which such values round to zero or a few steps.
NH_HD uint32_t mx_scale_byte(uint32_t amax_bits) {
    const int e = (int)(amax_bits >> 23);
    return amax_bits >= 0x7f800000u ? kMxNan : (uint32_t)(e > 2 ? e - 2 : 0);
}

// 2^(e - 127) of a scale byte (255: NaN; 0 is the subnormal 2^-127).
NH_HD float mx_scale(uint32_t e) {
    return f32_from_bits(e == kMxNan ? 0x7fc00000u : e ? e << 23 : 0x00400000u);
}

// The code of a finite v under scale byte e < 255: sign in bit 3, then the
// index of the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  v * 2^(127 - e) is exact
// (e <= 252: the factor is normal, and a quotient below the grid's first
// midpoint is a zero however it rounds).
NH_HD uint32_t mx_code(float v, uint32_t e) {
    const float a = fabsf(v) * f32_from_bits((254u - e) << 23);
    const uint32_t i = (uint32_t)(a > 0.25f) + (uint32_t)(a >= 0.75f) + (uint32_t)(a > 1.25f) + (uint32_t)(a >= 1.75f) +
                       (uint32_t)(a > 2.5f) + (uint32_t)(a >= 3.5f) + (uint32_t)(a > 5.0f);
    return i | ((f32_bits(v) >> 31) << 3);
}

// Twice the magnitude of a code's element: a whole number.
NH_HD int mx_twice(uint32_t code) {
    const int i = (int)(code & 7);
    return i < 4 ? i : i == 4 ? 4 : i == 5 ? 6 : i == 6 ? 8 : 12;
}

NH_HD float mx_value(uint32_t code, uint32_t e) {
    const float v = 0.5f * (float)mx_twice(code) * mx_scale(e);
    return code & 8 ? -v : v;
}

// Tiled form (weights, and the GEMM's activations): the operand order of
// v_mfma_scale_f32_16x16x128_f8f6f4.  Per 16 rows a region of KT = ceil(K / 128)
// tiles of 1 KiB, then KQ = ceil(KT / 4) pieces of 256 scale bytes.  Lane
// l = 16 g + r of a tile owns bytes [16 l, 16 l + 16): the 32 values (one block)
// 32 g .. 32 g + 31 of row r, low nibble first.  Byte 4 l + j of piece q is the
// scale of lane l's block in tile 4 q + j, so one dword per lane holds the
// scales of four MFMA K steps (the instruction picks its byte).  Codes and
// scales outside the matrix are zero.
NH_HD uint64_t mx_k_tiles(uint64_t k) { return (k + 127) / 128; }
NH_HD uint64_t mx_k_pieces(uint64_t k) { return (mx_k_tiles(k) + 3) / 4; }
NH_HD uint64_t mx_region_bytes(uint64_t k) { return mx_k_tiles(k) * 1024 + mx_k_pieces(k) * 256; }
NH_HD uint64_t mx_tiled_bytes(uint64_t n, uint64_t k) { return (n + 15) / 16 * mx_region_bytes(k); }

// Token form (rows that are gathered): codes [rows][64 KT] in row order,
// scales [rows][KQ][4 g][4 j] of block 4 (4 q + j) + g.
NH_HD uint64_t mx_token_codes(uint64_t k) { return mx_k_tiles(k) * 64; }
NH_HD uint64_t mx_token_scales(uint64_t k) { return mx_k_pieces(k) * 16; }

}  // namespace nh
