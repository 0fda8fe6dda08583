// mx4.hpp -- microscaled 4-bit floating point: e2m1 codes (0, 0.5, 1, 1.5, 2, 3,
// 4, 6 and their negatives) with a power of two for each 32 values along k, kept
// as the byte e + 127 of 2^e (0xff is NaN). Weights and activations have one
// native layout, of a [rows x k] matrix cut into kbs = ceil(k/128) blocks:
//   codes  [ceil(rows/16)][kbs][64 lanes][16 bytes]   (1 KiB per chunk)
//   scales [ceil(rows/64)][kbs][64 lanes][4 bytes]
// Lane l = 16 g + j of chunk (t, kb) holds row 16 t + j, k = 128 kb + 32 g + 0..31,
// two codes a byte, the even k in the low half: a lane's operand of a
// v_mfma_scale_f32_16x16x128_f8f6f4 in one 16-byte load, and exactly one block.
// Byte u of a lane's scale word belongs to tile 4 R + u of row panel R: the
// instruction picks the byte, so that one word serves four tiles of 16 rows.
// Codes past k are 0 and the scales of whole blocks past it 0 (2^-127). Rows past
// the last one up to the tile's 16 (the panel's 64) may hold anything: a row of an
// operand meets no other row's results.
#pragma once

#include "fp8.hpp"

namespace dz {

constexpr int kMicro = 32;  // values with one scale
constexpr size_t kMx4MostCols = (size_t)1 << 20, kMx4MostRows = (size_t)1 << 24;

inline size_t mx4_code_bytes(size_t rows, size_t k) { return (rows + 15) / 16 * ((k + 127) / 128) * 1024; }
inline size_t mx4_scale_bytes(size_t rows, size_t k) { return (rows + 63) / 64 * ((k + 127) / 128) * 256; }

namespace {

// Where chunk (row / 16, kb) keeps the 4-byte piece `part` of block g of a row, and the byte of its scale.
__device__ __forceinline__ size_t mx4_code_at(size_t row, int kb, int g, int part, int kbs) {
    return (row / 16 * kbs + kb) * 1024 + (16 * g + row % 16) * 16 + 4 * part;
}
__device__ __forceinline__ size_t mx4_scale_at(size_t row, int kb, int g, int kbs) {
    return ((row / 64 * kbs + kb) * 64 + 16 * g + row % 16) * 4 + row / 16 % 4;
}

// 2^(byte - 127); byte 0 is 2^-127, a subnormal.
__device__ __forceinline__ float mx4_scale_value(uint32_t byte) {
    return word_as_float(byte == 0 ? 0x00400000u : byte == 255 ? 0x7fc00000u : byte << 23);
}

// Eight codes of v / s, s a power of two given as the exponent field of a float (0: 2^-127).
__device__ __forceinline__ uint32_t mx4_codes8(const float v[8], float s) {
    uint32_t codes = 0;
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[0], v[1], s, 0);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[2], v[3], s, 1);
    codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[4], v[5], s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v[6], v[7], s, 3);
}

// One block of 32 values over a quad of lanes, eight a lane: the scale 2^e, e =
// floor(log2 max|v|) - 2 (at least -127), as its byte, and the lane's eight codes,
// v / 2^e to nearest even and at most 6 (what v_cvt_scalef32_pk_fp4_f32 gives; it
// takes the scale as the exponent field of a float, 0 for 2^-127). A block that holds
// a NaN or an infinity gets the NaN scale and codes 0: it makes its row's outputs NaN.
__device__ __forceinline__ uint32_t mx4_quantize8(const float v[8], uint32_t &scale) {
    uint32_t most = 0;  // |v| as bits: integers order as the values do, NaN above infinity
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const uint32_t b = __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu;
        most = most > b ? most : b;
    }
    most = dpp_max_u32<0xB1>(most);  // quad_perm [1,0,3,2]
    most = dpp_max_u32<0x4E>(most);  // quad_perm [2,3,0,1]
    const uint32_t exponent = most >> 23;
    const uint32_t byte = (exponent > 2 ? exponent : 2u) - 2;
    const float s = word_as_float(byte << 23);
    const uint32_t codes = mx4_codes8(v, s);
    const bool finite = exponent < 255;
    scale = finite ? byte : 255u;
    return finite ? codes : 0u;
}

}  // namespace

}  // namespace dz
