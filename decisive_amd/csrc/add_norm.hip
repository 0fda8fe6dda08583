// add_norm.hip -- the residual's addition, the RMS norm, and the normed rows as
// codes with scales for the products on 8-bit and 4-bit floating point weights.
//
//   h = T(f32(x + r)),  i = f32(1 / sqrt(sum h^2 / d + eps)),  y = f32(f32(h i) w)
//
// The sum of squares is held in 64 bits, where each square is exact: its rounding
// (d 2^-53 of it at most) is far below i's own, so that i, and with it every code,
// does not depend on the order of the sum but for one row in some 10^7. Bound by
// memory: x, r and h move once each and the codes once.
#include "../../include/decisive_rocm.h"
#include "mx4.hpp"
#include "tiles.hpp"

namespace dz {

int32_t ctx_fail(dz_ctx *ctx, int32_t code, const std::string &msg);
hipStream_t ctx_stream(dz_ctx *ctx);
int32_t ctx_launched(dz_ctx *ctx, const char *what);

namespace {

constexpr int kNormThreads = 256;

// What a row's kernel reads and writes; r, h and y may be null.
struct AddNorm {
    const void *x, *r;
    void *h, *y;
    const float *w;
    uint8_t *q;
    void *s;
    int m, d, kbs;
    float eps;
    int zero_centered;
};

// Eight consecutive values from k0 on, those inside the row.
template <class T>
__device__ __forceinline__ void norm_store8(T *row, int k0, int d, const float v[8]) {
    if (k0 + 8 <= d) {
        if constexpr (sizeof(T) == 4) {
            *(float4_any_t *)(row + k0) = float4_t{v[0], v[1], v[2], v[3]};
            *(float4_any_t *)(row + k0 + 4) = float4_t{v[4], v[5], v[6], v[7]};
        } else {
            typedef T pair_t __attribute__((ext_vector_type(2)));
            uint4_t w;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const pair_t p = {(T)v[2 * e], (T)v[2 * e + 1]};
                w[e] = __builtin_bit_cast(uint32_t, p);
            }
            *(uint4_any_t *)(row + k0) = w;
        }
    } else {
        for (int e = 0; e < 8; e++)
            if (k0 + e < d) row[k0 + e] = (T)v[e];
    }
}

// Eight values of h = T(x + r) in f32, stored where the caller keeps them.
template <class T>
__device__ __forceinline__ void norm_sum8(const AddNorm &a, size_t row, int k0, float v[8]) {
    fp8_load8((const T *)a.x + row * a.d, k0, a.d, v);
    if (a.r) {
        float r[8];
        fp8_load8((const T *)a.r + row * a.d, k0, a.d, r);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (float)(T)f32_rounded(v[e] + r[e]);
        if (a.h) norm_store8((T *)a.h + row * a.d, k0, a.d, v);
    }
}

// The normed values of eight, y where it is kept, and their codes.
template <class T, bool MX>
__device__ __forceinline__ void norm_codes8(const AddNorm &a, size_t row, int k0, float inverse, float v[8]) {
    float w[8];
    fp8_load8(a.w, k0, a.d, w);
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = (v[e] * inverse) * (a.zero_centered ? 1.0f + w[e] : w[e]);
    if (k0 + 8 > a.d)  // an infinite or NaN norm makes no values past the row
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = k0 + e < a.d ? v[e] : 0.0f;
    if (a.y) norm_store8((T *)a.y + row * a.d, k0, a.d, v);
    const int kb = k0 / 128;
    if constexpr (MX) {
        uint32_t scale;
        const uint32_t codes = mx4_quantize8(v, scale);
        const int g = k0 / 32 % 4, part = k0 / 8 % 4;
        *(uint32_t *)(a.q + mx4_code_at(row, kb, g, part, a.kbs)) = codes;
        if (part == 0) ((uint8_t *)a.s)[mx4_scale_at(row, kb, g, a.kbs)] = (uint8_t)scale;
    } else {
        uint2_t codes;
        const float scale = fp8_quantize8(v, codes);
        *(uint2_t *)(a.q + (row * a.kbs + kb) * 128 + k0 % 128) = codes;
        if (k0 % 128 == 0) ((float *)a.s)[(size_t)kb * a.m + row] = scale;
    }
}

__device__ __forceinline__ double norm_block_sum(double v) {
    __shared__ double part[kNormThreads / 64];
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    double all = 0.0;
    for (int i = 0; i < kNormThreads / 64; i++) all += part[i];
    return all;
}

// A workgroup takes a row, eight values a thread and piece: PIECES of them stay in
// registers between the sum and the norm; with PIECES = 0, for longer rows, h is
// read again (x and r where it is not kept).
template <class T, bool MX, int PIECES>
__global__ __launch_bounds__(kNormThreads) void add_norm_kernel(const AddNorm a) {
    const size_t row = blockIdx.x;
    const int end = a.kbs * 128;
    constexpr int kStep = kNormThreads * 8;
    double sum = 0.0;
    float v[PIECES > 0 ? PIECES : 1][8];
    if constexpr (PIECES > 0) {
#pragma unroll
        for (int i = 0; i < PIECES; i++) norm_sum8<T>(a, row, threadIdx.x * 8 + i * kStep, v[i]);
#pragma unroll
        for (int i = 0; i < PIECES; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) sum += (double)v[i][e] * (double)v[i][e];
    } else {
        for (int k0 = threadIdx.x * 8; k0 < a.d; k0 += kStep) {
            norm_sum8<T>(a, row, k0, v[0]);
#pragma unroll
            for (int e = 0; e < 8; e++) sum += (double)v[0][e] * (double)v[0][e];
        }
    }
    sum = norm_block_sum(sum);
    const float inverse = (float)(1.0 / sqrt(sum / (double)a.d + (double)a.eps));
    if constexpr (PIECES > 0) {
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const int k0 = threadIdx.x * 8 + i * kStep;
            if (k0 < end) norm_codes8<T, MX>(a, row, k0, inverse, v[i]);  // whole DPP rows of lanes
        }
    } else {
        AddNorm again = a;
        if (a.r && a.h) again.x = a.h, again.r = nullptr;  // each thread reads back what it wrote
        else again.h = nullptr;
        for (int k0 = threadIdx.x * 8; k0 < end; k0 += kStep) {
            norm_sum8<T>(again, row, k0, v[0]);
            norm_codes8<T, MX>(a, row, k0, inverse, v[0]);
        }
    }
}

template <class T, bool MX>
void add_norm_pieces(const AddNorm &a, hipStream_t s) {
    const dim3 grid(a.m), block(kNormThreads);
    if (a.d <= kNormThreads * 8) hipLaunchKernelGGL((add_norm_kernel<T, MX, 1>), grid, block, 0, s, a);
    else if (a.d <= kNormThreads * 16) hipLaunchKernelGGL((add_norm_kernel<T, MX, 2>), grid, block, 0, s, a);
    else if (a.d <= kNormThreads * 32) hipLaunchKernelGGL((add_norm_kernel<T, MX, 4>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((add_norm_kernel<T, MX, 0>), grid, block, 0, s, a);
}

template <bool MX>
void launch_add_norm(const AddNorm &a, int dtype, hipStream_t s) {
    if (dtype == DZ_F32) add_norm_pieces<float, MX>(a, s);
    else if (dtype == DZ_F16) add_norm_pieces<half_t, MX>(a, s);
    else add_norm_pieces<bf16_t, MX>(a, s);
}

}  // namespace

int32_t add_rmsnorm(dz_ctx *ctx, const void *x, const void *residual, int32_t dtype, size_t rows, size_t d,
                    const float *w, float eps, int32_t zero_centered, void *sum, void *y, uint8_t *q, void *s,
                    bool mx) {
    if (dtype != DZ_F32 && dtype != DZ_F16 && dtype != DZ_BF16)
        return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "unknown dtype");
    if (d == 0 || d > kFp8MostCols) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "invalid activation shape");
    if (!(eps >= 0.0f && eps <= 3.4028235e38f)) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "invalid epsilon");
    if (zero_centered != 0 && zero_centered != 1) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "invalid norm form");
    if (rows && (!x || !w || !q || !s)) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    if (sum && !residual) return ctx_fail(ctx, DZ_INVALID_REQUEST, "a sum without a residual");
    if (rows > kFp8MostRows) return ctx_fail(ctx, DZ_INPUT_TOO_LONG, "input budget exceeded");
    if (((uintptr_t)q & 15) != 0 || (mx && ((uintptr_t)s & 15) != 0))
        return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "codes must be 16-byte aligned");
    if (rows == 0) return DZ_OK;
    const AddNorm a{x, residual, sum, y, w, q, s, (int)rows, (int)d, (int)cdiv(d, 128), eps, zero_centered};
    if (mx) launch_add_norm<true>(a, dtype, ctx_stream(ctx));
    else launch_add_norm<false>(a, dtype, ctx_stream(ctx));
    return ctx_launched(ctx, "add rmsnorm");
}

}  // namespace dz
