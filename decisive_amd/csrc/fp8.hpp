// fp8.hpp -- weights in 8-bit floating point with a scale for each 128 x 128
// block, and what the kernels on them share.
//
// A code is an e4m3 value (the OCP form: bias 7, largest 448, no infinities,
// 0x7f and 0xff are NaN). Native layout of the codes of a [rows x cols] matrix
// (N x K below), "tile16x128": N padded to 16, K to 128 with zero codes,
//   [N/16][K/128][2 halves][64 lanes][16 bytes]     (2 KiB per chunk)
// Lane l = 16 g + j of half h of a chunk (t, kb) holds row n = 16 t + j,
// k = 128 kb + 64 h + 16 g + 0..15. The two halves of a lane are its 32 bytes
// of a v_mfma_f32_16x16x128_f8f6f4, and 8 bytes of them, as f16 or bf16, are
// its operand of a v_mfma_f32_16x16x32 (which k go together is free as long as
// both operands agree). Each half is 1 KiB that a wave loads with one 16-byte
// load per lane. Scales stay [ceil(N/128)][ceil(K/128)] f32.
#pragma once

#include <new>

#include "kernels.hpp"

namespace dz {

constexpr int kFp8Block = 128;
// A panel of 256 rows stays within 32-bit byte offsets, a grid within its limits.
constexpr size_t kFp8MostCols = (size_t)1 << 20, kFp8MostRows = (size_t)1 << 24;

// What a quantized product reads of a weight.
struct Fp8Weight {
    int rows = 0, cols = 0;
    int np = 0, kbs = 0;        // rows padded to 16, 128-wide blocks of cols
    uint8_t *codes = nullptr;   // device, tile16x128
    float *scales = nullptr;    // device, [ceil(rows/128)][kbs], behind the codes in the same allocation
    size_t code_bytes() const { return (size_t)np * kbs * kFp8Block; }
    size_t scale_bytes() const { return (size_t)((rows + kFp8Block - 1) / kFp8Block) * kbs * sizeof(float); }
};

typedef int int8v_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16_t;
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

namespace {

// The dot of 128 codes of 16 x 16 pairs of rows in one instruction. Products of
// codes are exact, but the unit adds eight neighbouring products on a common
// exponent with 14 bits: what is 2^-14 of the largest is cut off. On normal
// values a dot is 1.5e-5 off (relative, in the 2-norm), a sixteenth of f16's
// rounding; outputs kept in f32 go through fp8_mfma_wide.
__device__ __forceinline__ float4_t fp8_mfma(uint4_t a0, uint4_t a1, uint4_t b0, uint4_t b1) {
    const int8v_t a = {(int)a0[0], (int)a0[1], (int)a0[2], (int)a0[3], (int)a1[0], (int)a1[1], (int)a1[2], (int)a1[3]};
    const int8v_t b = {(int)b0[0], (int)b0[1], (int)b0[2], (int)b0[3], (int)b1[0], (int)b1[1], (int)b1[2], (int)b1[3]};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, float4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

// Eight codes (two words) as f16, exactly: e4m3's exponents lie inside f16's.
__device__ __forceinline__ half8_t fp8_to_half8(uint32_t lo, uint32_t hi) {
    const half2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
    const half2_t b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const half2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
    const half2_t d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return half8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// One lane's 32 codes as the operands of four 16x16x32 products.
struct Fp8Wide {
    half8_t h[4];
};
__device__ __forceinline__ Fp8Wide fp8_widen(uint4_t lo, uint4_t hi) {
    return {{fp8_to_half8(lo[0], lo[1]), fp8_to_half8(lo[2], lo[3]), fp8_to_half8(hi[0], hi[1]),
             fp8_to_half8(hi[2], hi[3])}};
}
// The same dot with f32's accuracy (7.6e-9 off on normal values), at half the rate.
__device__ __forceinline__ float4_t fp8_mfma_wide(const Fp8Wide &a, const Fp8Wide &b) {
    float4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; s++) d = mfma_f16(a.h[s], b.h[s], d);
    return d;
}

// Vectors at any address their elements may have: rows of odd lengths start
// anywhere, and the memory takes whole vectors there.
typedef float float4_any_t __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned int uint4_any_t __attribute__((ext_vector_type(4), aligned(2)));
typedef unsigned int uint2_any_t __attribute__((ext_vector_type(2), aligned(2)));
typedef unsigned int uint4_bytes_t __attribute__((ext_vector_type(4), aligned(1)));

// Eight consecutive values of a row from k0 on as they lie in memory, past k zero. Nothing here waits for whole
// vectors, so that several of these are under way together.
template <class T>
struct Fp8Raw {
    uint4_t w[sizeof(T) / 2 > 1 ? 2 : 1];

    __device__ __forceinline__ void load(const T *__restrict__ row, int k0, int k) {
        if (k0 + 8 <= k) {
            if constexpr (sizeof(T) == 4) {
                w[0] = __builtin_bit_cast(uint4_t, *(const float4_any_t *)(row + k0));
                w[1] = __builtin_bit_cast(uint4_t, *(const float4_any_t *)(row + k0 + 4));
            } else {
                w[0] = *(const uint4_any_t *)(row + k0);
            }
            return;
        }
        w[0] = uint4_t{0, 0, 0, 0};
        if constexpr (sizeof(T) == 4) w[1] = w[0];
        if (k0 >= k) return;
        T some[8];  // all loads together: past the row its last value again, and not used
#pragma unroll
        for (int e = 0; e < 8; e++) some[e] = row[k0 + e < k ? k0 + e : k - 1];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if constexpr (sizeof(T) == 4)
                w[e / 4][e % 4] = k0 + e < k ? __builtin_bit_cast(uint32_t, some[e]) : 0u;
            else
                w[0][e / 2] |= k0 + e < k ? (uint32_t)__builtin_bit_cast(uint16_t, some[e]) << (16 * (e % 2)) : 0u;
        }
    }
    __device__ __forceinline__ void values(float v[8]) const {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if constexpr (sizeof(T) == 4) {
                v[e] = word_as_float(w[0][e]), v[4 + e] = word_as_float(w[1][e]);
            } else if constexpr (__is_same(T, half_t)) {
                const half2_t p = word_as_half2(w[0][e]);
                v[2 * e] = (float)p[0], v[2 * e + 1] = (float)p[1];
            } else {
                v[2 * e] = word_as_float(w[0][e] << 16), v[2 * e + 1] = word_as_float(w[0][e] & 0xffff0000u);
            }
        }
    }
};

// Eight consecutive values of a row from k0 on, as f32; past k zero.
template <class T>
__device__ __forceinline__ void fp8_load8(const T *__restrict__ row, int k0, int k, float v[8]) {
    Fp8Raw<T> raw;
    raw.load(row, k0, k);
    raw.values(v);
}

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max_u32(uint32_t v) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xF, 0xF, true);
    return v > o ? v : o;
}

// One block of 128 values over the 16 lanes of a DPP row, eight a lane: the
// scale max(max|v| / 448, 2^-126) and the codes e4m3(v / scale), nearest even,
// both quotients correctly rounded in f32. A block that holds a NaN or an
// infinity gets a NaN scale (and codes 0): it makes its row's outputs NaN.
__device__ __forceinline__ float fp8_quantize8(const float v[8], uint2_t &codes) {
    uint32_t most = 0;  // |v| as bits: integers order as the values do, NaN above infinity
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const uint32_t b = __builtin_bit_cast(uint32_t, v[e]) & 0x7fffffffu;
        most = most > b ? most : b;
    }
    most = dpp_max_u32<0xB1>(most);   // quad_perm [1,0,3,2]
    most = dpp_max_u32<0x4E>(most);   // quad_perm [2,3,0,1]
    most = dpp_max_u32<0x124>(most);  // row_ror:4
    most = dpp_max_u32<0x128>(most);  // row_ror:8
    const bool finite = most < 0x7f800000u;
    const float s = fmaxf(__fdiv_rn(word_as_float(most), 448.0f), 1.17549435e-38f);
    float q[8];
    if (s > 0x1p-60f) {
        // v / s, correctly rounded, in half a division's instructions: q = v r with
        // r = 1 / s to nearest, then twice q -= r (q s - v), whose residual is exact
        // (the first leaves q within an ulp, the second is Markstein's theorem, IBM
        // J. Res. Dev. 34, 1990). Where a residual underflows q is below 2^-40 and
        // its code 0 all the same. With the residual this way round -0 stays -0: its
        // residual is +0 and -0 - (+0) = -0, where -0 + (+0) would be +0.
        const float r = __frcp_rn(s);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float t = v[e] * r;
            t = __builtin_fmaf(-__builtin_fmaf(t, s, -v[e]), r, t);
            q[e] = __builtin_fmaf(-__builtin_fmaf(t, s, -v[e]), r, t);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) q[e] = __fdiv_rn(v[e], s);
    }
    if (!finite) {
#pragma unroll
        for (int e = 0; e < 8; e++) q[e] = 0.0f;
    }
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
    codes = uint2_t{(uint32_t)lo, (uint32_t)hi};
    return finite ? s : __builtin_nanf("");
}

// v rounded once to the output's type (0 f32, 1 f16, 2 bf16).
__device__ __forceinline__ void fp8_store(void *__restrict__ y, int dtype, size_t at, float v) {
    if (dtype == 0) ((float *)y)[at] = v;
    else if (dtype == 1) ((half_t *)y)[at] = (half_t)v;
    else ((bf16_t *)y)[at] = (bf16_t)v;
}

// Four consecutive outputs at element `at`, `left` of them inside the row.
__device__ __forceinline__ void fp8_store4(void *__restrict__ y, int dtype, size_t at, float4_t v, int left) {
    if (left < 4) {
#pragma unroll
        for (int e = 0; e < 3; e++)
            if (e < left) fp8_store(y, dtype, at + e, v[e]);
    } else if (dtype == 0) {
        *(float4_any_t *)((float *)y + at) = v;
    } else if (dtype == 1) {
        const half2_t a = {(half_t)v[0], (half_t)v[1]}, b = {(half_t)v[2], (half_t)v[3]};
        *(uint2_any_t *)((half_t *)y + at) = uint2_t{half2_as_word(a), half2_as_word(b)};
    } else {
        const bf16x2_t a = {(bf16_t)v[0], (bf16_t)v[1]}, b = {(bf16_t)v[2], (bf16_t)v[3]};
        *(uint2_any_t *)((bf16_t *)y + at) = uint2_t{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
    }
}

}  // namespace

// ---- launchers (fp8.hip) -----------------------------------------------------
// Row-major codes of `count` matrices [rows x cols] (one after the other) into the
// native layout: matrix i at dst + i * matrix_bytes, its tile t tile_bytes and
// k-block kb kb_bytes further; sets *bad on a NaN code.
void launch_fp8_retile(const uint8_t *codes, int count, int rows, int cols, uint8_t *dst, size_t matrix_bytes,
                       size_t tile_bytes, size_t kb_bytes, int *bad, hipStream_t s);
// Copies block scales; sets *bad where one is not finite or is negative.
void launch_fp8_scales(const float *src, float *dst, size_t n, int *bad, hipStream_t s);

}  // namespace dz
