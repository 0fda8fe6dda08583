// add_norm.hip -- the residual's addition, the RMS norm, and the normed rows as
// codes with scales for the products on 8-bit and 4-bit floating point weights.
//
//   h = T(f32(x + r)),  i = f32(1 / sqrt(sum h^2 / d + eps)),  y = f32(f32(h i) w)
//
// The sum of squares is held in 64 bits, where each square is exact: its rounding
// (d 2^-53 of it at most) is far below i's own, so that i, and with it every code,
// does not depend on the order of the sum but for one row in some 10^7. Bound by
// memory: x, r and h move once each and the codes once.
#include <algorithm>

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
    double over_d, eps;
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

// Eight values of x and of r, on the way.
template <class T>
struct NormLoad {
    Fp8Raw<T> x, r;
    __device__ __forceinline__ void load(const AddNorm &a, size_t row, int k0) {
        x.load((const T *)a.x + row * a.d, k0, a.d);
        if (a.r) r.load((const T *)a.r + row * a.d, k0, a.d);
    }
    // h = T(x + r) in f32, stored where the caller keeps it
    __device__ __forceinline__ void add(const AddNorm &a, size_t row, int k0, float v[8]) const {
        x.values(v);
        if (!a.r) return;
        float other[8];
        r.values(other);
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = (float)(T)f32_rounded(v[e] + other[e]);
        if (a.h) norm_store8((T *)a.h + row * a.d, k0, a.d, v);
    }
};

// The normed values of eight, y where it is kept, and their codes.
template <class T, bool MX>
__device__ __forceinline__ void norm_codes8(const AddNorm &a, size_t row, int k0, float inverse, float v[8],
                                            const float w[8]) {
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

// What the lane WIDTH (16 or 32) away holds: both sides of a swap of rows, or halves, of two copies.
template <int WIDTH>
__device__ __forceinline__ double norm_swap(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t word[2] = {(uint32_t)b, (uint32_t)(b >> 32)};
    uint32_t other[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint2_t t = __builtin_bit_cast(uint2_t, WIDTH == 16
                                                          ? __builtin_amdgcn_permlane16_swap(word[i], word[i], false, false)
                                                          : __builtin_amdgcn_permlane32_swap(word[i], word[i], false, false));
        other[i] = (threadIdx.x & WIDTH) ? t[0] : t[1];
    }
    return __builtin_bit_cast(double, (uint64_t)other[1] << 32 | other[0]);
}

// The sum over the LANES lanes of a row, in each of them.
template <int LANES>
__device__ __forceinline__ double norm_sum(double v) {
    v += dpp_move_f64<0xB1>(v);   // quad_perm [1,0,3,2]
    v += dpp_move_f64<0x4E>(v);   // quad_perm [2,3,0,1]
    v += dpp_move_f64<0x141>(v);  // row_half_mirror, and not a rotation: every lane adds in the same order
    v += dpp_move_f64<0x140>(v);  // row_mirror
    if constexpr (LANES > 16) {
        v += norm_swap<16>(v);
        v += norm_swap<32>(v);
    }
    if constexpr (LANES > 64) {
        __shared__ double part[kNormThreads / 64];
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
        __syncthreads();
        v = (part[0] + part[1]) + (part[2] + part[3]);
        static_assert(LANES == kNormThreads && kNormThreads == 256, "four waves a row");
    }
    return v;
}

// 1 / sqrt(v) within some 2^-50: the unit's estimate and two steps of Newton's iteration, a third of what a square root
// and a division of 64 bits take. 0 and infinity keep the estimate, which is exact there.
__device__ __forceinline__ double norm_rsqrt(double v) {
    double y = __builtin_amdgcn_rsq(v);
    if (v > 0.0 && v < __builtin_huge_val()) {
        const double half = 0.5 * v;
        y = __builtin_fma(y, __builtin_fma(-half * y, y, 0.5), y);
        y = __builtin_fma(y, __builtin_fma(-half * y, y, 0.5), y);
    }
    return y;
}

// LANES lanes take a row, eight values a lane and piece: PIECES of them stay in
// registers between the sum and the norm, and up to two pieces of w are on the way with
// them; with PIECES = 0, for longer rows, h is read again (x and r where it is not
// kept). In the 4-bit form neighbouring rows are neighbours on one XCD, whose L2 joins
// the 16 bytes that each writes of a chunk (us, 16384 rows of 4096 in bf16 104 against
// 110 with the rows dealt out; in e4m3, whose rows lie apart, 102 against 96). A row a
// workgroup: 1 row of 2560 in bf16 3.6 us, 229 4.2, both a launch and two trips to
// memory; 16384 of 4096 91-95 us, 5.0-5.2 TB/s (f32 158, 5.5), the rate of a copy.
template <class T, bool MX, int LANES, int PIECES>
__global__ __launch_bounds__(kNormThreads) void add_norm_kernel(const AddNorm a) {
    constexpr int ROWS = kNormThreads / LANES, STEP = LANES * 8;
    const size_t block = (size_t)blockIdx.y * gridDim.x + (MX ? xcd_unit(blockIdx.x, gridDim.x) : (int)blockIdx.x);
    const size_t row = block * ROWS + threadIdx.x / LANES;
    if (row >= (size_t)a.m) return;  // whole rows of lanes: all of a workgroup that has a barrier
    const int end = a.kbs * 128, lane = threadIdx.x % LANES;
    double sum = 0.0;
    constexpr int EARLY = PIECES <= 2 ? PIECES : 0;
    float v[PIECES > 0 ? PIECES : 1][8], w[8];
    Fp8Raw<float> early[EARLY > 0 ? EARLY : 1];
    if constexpr (PIECES > 0) {
#pragma unroll
        for (int i = 0; i < EARLY; i++) early[i].load(a.w, lane * 8 + i * STEP, a.d);
        // two pieces' loads are under way together; a store of h, which may lie in x or r, would hold them up
#pragma unroll
        for (int i0 = 0; i0 < PIECES; i0 += 2) {
            NormLoad<T> some[2];
#pragma unroll
            for (int i = i0; i < i0 + 2 && i < PIECES; i++) some[i - i0].load(a, row, lane * 8 + i * STEP);
#pragma unroll
            for (int i = i0; i < i0 + 2 && i < PIECES; i++) some[i - i0].add(a, row, lane * 8 + i * STEP, v[i]);
        }
#pragma unroll
        for (int i = 0; i < PIECES; i++)
#pragma unroll
            for (int e = 0; e < 8; e++) sum += (double)v[i][e] * (double)v[i][e];
    } else {
        for (int k0 = lane * 8; k0 < a.d; k0 += STEP) {
            NormLoad<T> some;
            some.load(a, row, k0);
            some.add(a, row, k0, v[0]);
#pragma unroll
            for (int e = 0; e < 8; e++) sum += (double)v[0][e] * (double)v[0][e];
        }
    }
    sum = norm_sum<LANES>(sum);
    const float inverse = (float)norm_rsqrt(__builtin_fma(sum, a.over_d, a.eps));
    if constexpr (PIECES > 0) {
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const int k0 = lane * 8 + i * STEP;
            if (k0 >= end) break;  // whole DPP rows of lanes
            if (EARLY == 0) early[0].load(a.w, k0, a.d);
            early[EARLY > 0 ? i : 0].values(w);
            norm_codes8<T, MX>(a, row, k0, inverse, v[i], w);
        }
    } else {
        AddNorm again = a;
        if (a.r && a.h) again.x = a.h, again.r = nullptr;  // each lane reads back what it wrote
        else again.h = nullptr;
        for (int k0 = lane * 8; k0 < end; k0 += STEP) {
            NormLoad<T> some;
            some.load(again, row, k0);
            early[0].load(a.w, k0, a.d);
            some.add(again, row, k0, v[0]);
            early[0].values(w);
            norm_codes8<T, MX>(a, row, k0, inverse, v[0], w);
        }
    }
}

template <class T, bool MX, int LANES, int PIECES>
void add_norm_form(const AddNorm &a, hipStream_t s) {
    const unsigned blocks = cdiv(a.m, kNormThreads / LANES), most = 1u << 20;  // a grid has less than 2^32 threads a side
    const dim3 grid(std::min(blocks, most), cdiv(blocks, most));
    hipLaunchKernelGGL((add_norm_kernel<T, MX, LANES, PIECES>), grid, dim3(kNormThreads), 0, s, a);
}

// Short rows share a workgroup (16384 rows of 64 in bf16 4.8 us, a workgroup each 22.8);
// rows up to 2048 have a wave each where there are many. us, wave / workgroup, e4m3:
//   rows            1024        2048        4096        8192        16384
//   1000, bf16      4.4 / 4.4   5.7 / 6.3   8.2 / 9.8   14.2 / 17.4 22.9 / 31.9
//   1000, f32       5.0 / 4.7   7.3 / 6.5   11.9 / 11.6 20.1 / 20.3 36.1 / 36.4
//   1111, bf16      6.5 / 5.2   8.1 / 7.3   12.1 / 12.2 21.3 / 22.2 33.9 / 39.5
//   2000, bf16      6.6 / 5.6   8.9 / 8.1   14.7 / 13.4 25.7 / 25.4 44.4 / 44.3
//   2000, f32       7.7 / 6.8   13.1 / 10.7 20.9 / 19.5 36.5 / 34.7 87.7 / 84.1
// The line suits 16-bit rows; f32 ones past 1024 lose up to a tenth by it. 16384 of 4096
// would be 127 / 102. Lengths that are no multiple of eight end in single values: 1001 rows
// of 1111 in f16 with y kept 5.5, of 1110 5.4, of 1112 5.0, of 1152 4.9; one row 3.4 and 3.0.
template <class T, bool MX>
void add_norm_pieces(const AddNorm &a, hipStream_t s) {
    if (a.d <= 128) return add_norm_form<T, MX, 16, 1>(a, s);
    if (a.d <= 512) return add_norm_form<T, MX, 64, 1>(a, s);
    if (a.m >= 4096 && a.d <= 1024) return add_norm_form<T, MX, 64, 2>(a, s);
    if (a.m >= 4096 && a.d <= 2048) return add_norm_form<T, MX, 64, 4>(a, s);
    if (a.d <= 2048) add_norm_form<T, MX, 256, 1>(a, s);
    else if (a.d <= 4096) add_norm_form<T, MX, 256, 2>(a, s);
    else if (a.d <= 8192) add_norm_form<T, MX, 256, 4>(a, s);
    else if (a.d <= 12288) add_norm_form<T, MX, 256, 6>(a, s);
    else add_norm_form<T, MX, 256, 0>(a, s);
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
    const AddNorm a{x, residual, sum, y, w, q, s, (int)rows, (int)d, (int)cdiv(d, 128), 1.0 / (double)d, (double)eps,
                    zero_centered};
    if (mx) launch_add_norm<true>(a, dtype, ctx_stream(ctx));
    else launch_add_norm<false>(a, dtype, ctx_stream(ctx));
    return ctx_launched(ctx, "add rmsnorm");
}

}  // namespace dz
