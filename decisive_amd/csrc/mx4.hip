// mx4.hip -- products on microscaled 4-bit floating point (mx4.hpp has the form
// and the layout).
//
//   y[i, j] = sum over 32-blocks b of 2^(ex[i, b] + ew[j, b]) sum over k in b of cx[i, k] cw[j, k]
//
// The matrix unit multiplies e2m1 codes, scales them and adds them to f32 sums in
// one instruction: products of codes and the sum over a block are exact in it, and
// its additions of blocks f32's (random codes, scales within 2^10 of each other: 2.7e-8
// off, relative, in the 2-norm), so that f32 outputs need no path of their own.
#include <algorithm>
#include <cmath>

#include "../../include/decisive_rocm.h"
#include "mx4.hpp"
#include "tiles.hpp"

struct dz_mx4_weight {
    int rows = 0, cols = 0, kbs = 0;
    int device = 0;
    uint8_t *codes = nullptr;   // device
    uint8_t *scales = nullptr;  // device, behind the codes in the same allocation
    size_t bytes = 0;
};

namespace dz {

int32_t ctx_fail(dz_ctx *ctx, int32_t code, const std::string &msg);
int32_t ctx_hip_fail(dz_ctx *ctx, hipError_t e, const char *what);
hipStream_t ctx_stream(dz_ctx *ctx);
int *ctx_flag(dz_ctx *ctx);
int ctx_device(dz_ctx *ctx);
int ctx_variant(dz_ctx *ctx, const char *family);
int32_t ctx_workspace(dz_ctx *ctx, size_t bytes, void **out);
int32_t ctx_launched(dz_ctx *ctx, const char *what);
int32_t ctx_flag_value(dz_ctx *ctx, int *value);

namespace {

// ---- weights -------------------------------------------------------------------

// One thread per block of 32 codes (16 bytes of a row), its scale with it;
// consecutive threads take consecutive blocks of a row.
__global__ __launch_bounds__(256) void mx4_retile_kernel(const uint8_t *__restrict__ codes,
                                                         const uint8_t *__restrict__ scales, size_t pieces, int rows,
                                                         int cols, int kbs, uint8_t *__restrict__ dst,
                                                         uint8_t *__restrict__ dst_scales, int *bad) {
    const int row_bytes = (cols + 1) / 2, blocks = (cols + 31) / 32;
    for (size_t id = blockIdx.x * (size_t)256 + threadIdx.x; id < pieces; id += gridDim.x * (size_t)256) {
        const int b = (int)(id % (4 * kbs)), kb = b / 4, g = b % 4;
        const size_t row = id / (4 * kbs);
        uint4_t w = {0, 0, 0, 0};
        uint8_t scale = 0;
        if (row < (size_t)rows && b < blocks) {
            const uint8_t *src = codes + row * row_bytes + 16 * b;
            scale = scales[row * blocks + b];
            if (scale == 255) atomicOr(bad, 1);
            if (32 * b + 32 <= cols) {
                w = *(const uint4_bytes_t *)src;
            } else {
                for (int e = 0; 32 * b + e < cols; e++)
                    w[e / 8] |= (uint32_t)(src[e / 2] >> (4 * (e % 2)) & 15) << (4 * (e % 8));
            }
        }
        *(uint4_t *)(dst + mx4_code_at(row, kb, g, 0, kbs)) = w;
        dst_scales[mx4_scale_at(row, kb, g, kbs)] = scale;
    }
}

// One value a thread, its code and its scale by loads of a byte: 4096 x 4096 46 us, 14336 x 4096 150-158 (1.7 TB/s).
__global__ __launch_bounds__(256) void mx4_dequant_kernel(const uint8_t *__restrict__ codes,
                                                          const uint8_t *__restrict__ scales, int rows, int cols,
                                                          int kbs, float *__restrict__ y) {
    const size_t count = (size_t)rows * cols;
    for (size_t id = blockIdx.x * (size_t)256 + threadIdx.x; id < count; id += gridDim.x * (size_t)256) {
        const size_t row = id / cols;
        const int k = (int)(id % cols), kb = k / 128, g = k / 32 % 4;
        const uint32_t c = codes[mx4_code_at(row, kb, g, 0, kbs) + k % 32 / 2] >> (4 * (k % 2));
        const uint32_t size = c & 7;
        // 0 and 0.5, then 1, 1.5, 2, 3, 4, 6: one mantissa bit under the exponent field
        const float v = size < 2 ? 0.5f * (float)size : word_as_float((size + 252) << 22);
        y[id] = __fmul_rn(c & 8 ? -v : v, mx4_scale_value(scales[mx4_scale_at(row, kb, g, kbs)]));
    }
}

// ---- activations ---------------------------------------------------------------

// A workgroup takes 64 rows of one 128-block, whose scale words it writes side by
// side: 16 lanes a row and eight values a lane, EACH rows a lane. Codes go out as 4-byte
// pieces; four lanes make the 16 bytes of a block. Bound by memory, sizeof(T) + 17/32
// bytes a value: 16384 x 4096 bf16 26 us, 6.5 TB/s; a few rows 2.3 us, a launch's time.
template <class T, int EACH>
__global__ __launch_bounds__(1024 / EACH) void mx4_quantize_kernel(const T *__restrict__ x, int m, int k, int kbs,
                                                                   uint8_t *__restrict__ q, uint8_t *__restrict__ s,
                                                                   int *bad) {
    const int kb = blockIdx.x, piece = threadIdx.x % 16, k0 = kb * 128 + piece * 8;
    const size_t row0 = ((size_t)blockIdx.z * gridDim.y + blockIdx.y) * 64 + threadIdx.x / 16;
    Fp8Raw<T> raw[EACH];
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const size_t row = row0 + i * (64 / EACH);
        raw[i].load(x + (row < (size_t)m ? row : (size_t)m - 1) * k, k0, k);
    }
#pragma unroll
    for (int i = 0; i < EACH; i++) {
        const size_t row = row0 + i * (64 / EACH);
        if (row >= (size_t)m) return;  // whole DPP rows of lanes
        float v[8];
        raw[i].values(v);
        uint32_t scale;
        const uint32_t codes = mx4_quantize8(v, scale);
        *(uint32_t *)(q + mx4_code_at(row, kb, piece / 4, piece % 4, kbs)) = codes;
        if (piece % 4 == 0) {
            s[mx4_scale_at(row, kb, piece / 4, kbs)] = (uint8_t)scale;
            if (bad && scale == 255) atomicOr(bad, 1);
        }
    }
}

// ---- products: the weight streamed over a few rows -----------------------------

// The dots of 16 x 16 rows over 128 k, scaled and added to c: `a` and `b` are a
// lane's 32 codes, sa and sb the words whose byte UA or UB is its block's scale.
template <int UA, int UB>
__device__ __forceinline__ float4_t mx4_mfma(uint4_t a, uint32_t sa, uint4_t b, uint32_t sb, float4_t c) {
    const int8v_t va = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
    const int8v_t vb = {(int)b[0], (int)b[1], (int)b[2], (int)b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(va, vb, c, 4, 4, UA, (int)sa, UB, (int)sb);
}

// A workgroup owns 16 NT weight rows (NT tiles) and up to 16 activation rows. Its
// waves take runs of the k-blocks, four of them at a time, operands straight from
// memory, and their f32 partials are added in wave order, from LDS. The matrix unit's
// operands are swapped (weight first), so a lane holds one activation row and four
// output columns. x comes as codes (ROWS = 0) or, a few rows, as it is: then a wave
// quantizes its own blocks while their weights are on the way, four 128-blocks of a row
// at once, eight values a lane as mx4_quantize_kernel does, and hands the codes to its
// lanes as operands through LDS, which spares a launch. The same bits either way.
// Bound by a launch and one trip to memory, then by the weight's bytes (us, from recorded
// graphs over two weights: K=N=4096, 1 row as it is 3.1, 16 rows of codes 3.4; K=1024,
// N=32000, 16 rows of codes, f32 out 4.4, 4.5 TB/s).
constexpr int kMx4Waves = 8, kMx4Batch = 4;

template <class T, int ROWS, int NT>
__global__ __launch_bounds__(kMx4Waves * 64) void mx4_rows_kernel(const uint8_t *__restrict__ codes,
                                                                  const uint8_t *__restrict__ scales, int n, int kbs,
                                                                  const void *__restrict__ x,
                                                                  const uint8_t *__restrict__ sx, int m, int k,
                                                                  void *__restrict__ y, int dtype) {
    constexpr bool RAW = ROWS > 0;
    __shared__ __align__(16) float part[kMx4Waves][NT * 256];
    __shared__ __align__(16) uint32_t s_codes[RAW ? kMx4Waves : 1][RAW ? ROWS : 1][kMx4Batch * 16];
    __shared__ uint32_t s_scale[RAW ? kMx4Waves : 1][RAW ? ROWS : 1][kMx4Batch * 4];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int g = lane / 16, j = lane % 16;
    const int tiles = (n + 15) / 16, groups = (tiles + NT - 1) / NT, t0 = blockIdx.x % groups * NT;
    const int row0 = blockIdx.x / groups * 16;
    float4_t acc[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) acc[t] = float4_t{0.f, 0.f, 0.f, 0.f};
    const int first = (int)((int64_t)kbs * wave / kMx4Waves), last = (int)((int64_t)kbs * (wave + 1) / kMx4Waves);
    for (int kb0 = first; kb0 < last; kb0 += kMx4Batch) {
        uint4_t w[NT][kMx4Batch], v[kMx4Batch];
        uint32_t sw[NT][kMx4Batch], sv[kMx4Batch];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int tile = min(t0 + t, tiles - 1);
#pragma unroll
            for (int i = 0; i < kMx4Batch; i++) {
                const int kb = min(kb0 + i, last - 1);
                w[t][i] = __builtin_nontemporal_load((const uint4_t *)(codes + ((size_t)tile * kbs + kb) * 1024 + lane * 16));
                sw[t][i] = scales[((size_t)(tile / 4) * kbs + kb) * 256 + lane * 4 + tile % 4];
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // the weight is under way before x is waited for
        if constexpr (RAW) {
            Fp8Raw<T> raw[ROWS];
#pragma unroll
            for (int r = 0; r < ROWS; r++) raw[r].load((const T *)x + (size_t)min(r, m - 1) * k, kb0 * 128 + lane * 8, k);
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                float some[8];
                raw[r].values(some);
                uint32_t scale;
                s_codes[wave][r][lane] = mx4_quantize8(some, scale);
                if (lane % 4 == 0) s_scale[wave][r][lane / 4] = scale;
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            const int r = min(j, m - 1);  // rows past the last one multiply that row again
#pragma unroll
            for (int i = 0; i < kMx4Batch; i++) {
                v[i] = *(const uint4_t *)&s_codes[wave][r][(i * 4 + g) * 4];
                sv[i] = s_scale[wave][r][i * 4 + g];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // read before the next batch is written
        } else {
#pragma unroll
            for (int i = 0; i < kMx4Batch; i++) {
                const int kb = min(kb0 + i, last - 1);
                v[i] = *(const uint4_t *)((const uint8_t *)x + ((size_t)(row0 / 16) * kbs + kb) * 1024 + lane * 16);
                sv[i] = sx[((size_t)(row0 / 64) * kbs + kb) * 256 + lane * 4 + row0 / 16 % 4];
            }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < kMx4Batch; i++) {
            if (kb0 + i >= last) break;
#pragma unroll
            for (int t = 0; t < NT; t++) acc[t] = mx4_mfma<0, 0>(w[t][i], sw[t][i], v[i], sv[i], acc[t]);
        }
    }
#pragma unroll
    for (int t = 0; t < NT; t++) *(float4_t *)&part[wave][(t * 16 + j) * 16 + 4 * g] = acc[t];
    __syncthreads();
    for (int i = threadIdx.x; i < NT * 256; i += kMx4Waves * 64) {
        const int row = row0 + i / 16 % 16, col = (t0 + i / 256) * 16 + i % 16;
        if (row >= m || col >= n) continue;
        float v = part[0][i];
#pragma unroll
        for (int u = 1; u < kMx4Waves; u++) v += part[u][i];
        fp8_store(y, dtype, (size_t)row * n + col, v);
    }
}

template <class T, int ROWS, int NT>
void mx4_rows_form(const dz_mx4_weight *w, const void *x, const uint8_t *sx, int m, void *y, int dtype, hipStream_t s) {
    hipLaunchKernelGGL((mx4_rows_kernel<T, ROWS, NT>), dim3(cdiv(cdiv(w->rows, 16), NT) * cdiv(m, 16)),
                       dim3(kMx4Waves * 64), 0, s, w->codes, w->scales, w->rows, w->kbs, x, sx, m, w->cols, y, dtype);
}

// Four tiles a workgroup past four a compute unit, where a workgroup with one has too little to read (us, one / four:
// 16 rows, K=1024, N=32000 in f32 5.7 / 4.4; K=4096, N=14336 7.7 / 8.2; K=N=4096 3.4 / 5.2).
bool mx4_many_tiles(const dz_mx4_weight *w) { return cdiv(w->rows, 16) > 4u * (unsigned)device_cus(); }

void mx4_rows_launch(const dz_mx4_weight *w, const uint8_t *q, const uint8_t *sx, int m, void *y, int dtype,
                     hipStream_t s) {
    if (mx4_many_tiles(w)) mx4_rows_form<void, 0, 4>(w, q, sx, m, y, dtype, s);
    else mx4_rows_form<void, 0, 1>(w, q, sx, m, y, dtype, s);
}

template <class T>
void mx4_raw_launch(const dz_mx4_weight *w, const void *x, int m, void *y, int dtype, hipStream_t s) {
    if (m == 1) mx4_rows_form<T, 1, 1>(w, x, nullptr, m, y, dtype, s);
    else if (m == 2) mx4_rows_form<T, 2, 1>(w, x, nullptr, m, y, dtype, s);
    else mx4_rows_form<T, 4, 1>(w, x, nullptr, m, y, dtype, s);
}

// ---- products: tiles over many rows ----------------------------------------------

// dma4 with a scalar offset added to every lane's (dma16_at's contract).
__device__ __forceinline__ void dma4_at(uint32_t lds, uint32_t voff, int32x4_t rsrc, uint32_t soff) {
    const int32x4_t r = {__builtin_amdgcn_readfirstlane(rsrc[0]), __builtin_amdgcn_readfirstlane(rsrc[1]),
                         __builtin_amdgcn_readfirstlane(rsrc[2]), 0x00020000};
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(r), "s"(__builtin_amdgcn_readfirstlane(soff))
                 : "memory", "m0");
}

// mx4_mfma with the bytes as values that the compiler knows once loops are unrolled.
template <int UA>
__device__ __forceinline__ float4_t mx4_mfma_b(int ub, uint4_t a, uint32_t sa, uint4_t b, uint32_t sb, float4_t c) {
    if (ub == 0) return mx4_mfma<UA, 0>(a, sa, b, sb, c);
    if (ub == 1) return mx4_mfma<UA, 1>(a, sa, b, sb, c);
    if (ub == 2) return mx4_mfma<UA, 2>(a, sa, b, sb, c);
    return mx4_mfma<UA, 3>(a, sa, b, sb, c);
}
__device__ __forceinline__ float4_t mx4_mfma_ab(int ua, int ub, uint4_t a, uint32_t sa, uint4_t b, uint32_t sb,
                                                float4_t c) {
    if (ua == 0) return mx4_mfma_b<0>(ub, a, sa, b, sb, c);
    if (ua == 1) return mx4_mfma_b<1>(ub, a, sa, b, sb, c);
    if (ua == 2) return mx4_mfma_b<2>(ub, a, sa, b, sb, c);
    return mx4_mfma_b<3>(ub, a, sa, b, sb, c);
}

// Eight consecutive outputs of a 16-bit type at element `at`, `left` of them inside the row.
__device__ __forceinline__ void mx4_store8(void *__restrict__ y, size_t at, uint4_t w, int left) {
    if (left >= 8) {
        *(uint4_any_t *)((uint16_t *)y + at) = w;
    } else {
#pragma unroll
        for (int e = 0; e < 7; e++)
            if (e < left) ((uint16_t *)y)[at + e] = (uint16_t)(w[e / 2] >> (16 * (e % 2)));
    }
}

// Four values rounded once to f16 (dtype 1) or bf16.
__device__ __forceinline__ uint2_t mx4_round4(float4_t v, int dtype) {
    if (dtype == 1) {
        const half2_t a = {(half_t)v[0], (half_t)v[1]}, b = {(half_t)v[2], (half_t)v[3]};
        return uint2_t{half2_as_word(a), half2_as_word(b)};
    }
    const bf16x2_t a = {(bf16_t)v[0], (bf16_t)v[1]}, b = {(bf16_t)v[2], (bf16_t)v[3]};
    return uint2_t{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}

// Block tile BM x BN (activation rows x weight rows). KS groups of WGM x WGN
// waves each take every KS-th 128-block of k; a step is KS blocks, one a group, in
// one of NS LDS stages that buffer_load ... lds fills, chunks and scale words as they
// lie in memory, which is operand order: a lane's 16 bytes are its own, and no two
// lanes' reads meet in a bank. A wave reads the operands of step i + 1 while it
// multiplies step i's, so that its products wait for no read; a stage is free once its
// operands are in registers, a step before it is multiplied, and NS - 1 steps' loads
// are in flight. With KS = 1 a workgroup goes through several tiles, and the loads run
// on into the next one while a tile's outputs are stored. Scales cost nothing: the matrix
// unit adds the exponents. The groups' sums are added in group order, through LDS.
// 16384 rows, K=4096, N=14336, bf16 out, 256 x 256: 455-505 us, 3.8-4.2 PFLOP/s, where
// the unit sustains 7.0 from registers on such operands. Each further 4096 of k takes 370
// us (5.2 PFLOP/s), tiles' ends and 470 MB of outputs the other 120. Bound by power, which
// holds the clock at some 1.85 GHz (zeros instead of random codes take 388), and by the
// loads into LDS (34 KiB a step and compute unit; alone 385 us, 40 B/ns; the products with
// the barriers alone 318); the matrix unit is busy 0.58 of the cycles, LDS has no bank
// conflicts. Four waves of 128 x 128 took 637, 256 x 128 tiles and 32x32x64 instructions
// more than 256 x 256; leaving a tile's stores under way into the next one's steps, the
// same. Shorter products are the latency of their k-steps (1001 rows, K=1111, N=1777 7.1).
template <int BM, int BN, int WGM, int WGN, int KS, int NS>
__global__ __launch_bounds__(WGM *WGN *KS * 64) void mx4_tile_kernel(const uint8_t *__restrict__ codes,
                                                                     const uint8_t *__restrict__ scales, int n, int kbs,
                                                                     const uint8_t *__restrict__ q,
                                                                     const uint8_t *__restrict__ sx, int m,
                                                                     void *__restrict__ y, int dtype, int units) {
    constexpr int WAVES = WGM * WGN, TM = BM / WGM, TN = BN / WGN, MT = TM / 16, NT = TN / 16;
    constexpr int XPW = BM / 16 / WAVES, WPW = BN / 16 / WAVES;            // 1 KiB loads per wave and stage
    constexpr int XP = BM < 64 ? 1 : BM / 64, WP = BN < 64 ? 1 : BN / 64;  // panels of scale words
    constexpr int SPW = (XP + WP + WAVES - 1) / WAVES, PB = XPW + WPW + SPW;
    constexpr int XW = TM < 64 ? 1 : TM / 64, WW = TN < 64 ? 1 : TN / 64;  // scale words of a wave
    constexpr int XB = BM * 64, SB = XB + BN * 64, PART = SB + (XP + WP) * 256, STAGE = KS * PART;
    static_assert(XPW * 16 * WAVES == BM && WPW * 16 * WAVES == BN, "whole loads for each wave");
    static_assert((TM % 64 == 0 || 64 % TM == 0) && (TN % 64 == 0 || 64 % TN == 0), "scale words of whole or one panel");
    static_assert(NS % 2 == 0, "two steps a turn");
    static_assert(NT % 2 == 0, "pairs of column tiles are stored together");
    static_assert((NS - 1) * PB <= 63, "vmcnt range");
    static_assert((KS - 1) * BM * BN * 4 <= NS * STAGE, "the groups' sums fit the stages");
    __shared__ __align__(16) uint8_t lds[NS * STAGE];

    const int wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int group = wave_all / WAVES, wave = wave_all % WAVES;
    const int wm = wave / WGN, wn = wave % WGN, g = lane / 16, j = lane % 16;
    const int tiles_m = (m + BM - 1) / BM, tiles_n = (n + BN - 1) / BN;
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(lds)) + group * PART;

    // the operands change places every step, and the loads are NS steps ahead; steps past the last add nothing
    const int steps = max(NS, (kbs + 2 * KS - 1) / (2 * KS) * 2);

    // A unit of work is a tile.
    struct Unit {
        int row0, col0;
    };
    auto unit_of = [&](int id) {
        int tm, tn;
        xcd_tile(id, units, tiles_m, tiles_n, tm, tn);
        // divisions leave uniform values in vector registers
        return Unit{__builtin_amdgcn_readfirstlane(tm) * BM, __builtin_amdgcn_readfirstlane(tn) * BN};
    };

    // The loads run NS steps ahead of the products: their own unit and step, and what they read of it. Units past the
    // last one, and blocks past k, load nothing (every offset out of range, zeros in LDS).
    int load_id = blockIdx.x, load_step = 0;
    Unit load = unit_of(load_id);
    int32x4_t rx, rw, rs[SPW];
    int panel[SPW];  // this wave's panels of scale words (some load one twice, so that all waits go by count)
    uint32_t soff[SPW];
#pragma unroll
    for (int p = 0; p < SPW; p++) {
        panel[p] = (wave * SPW + p) % (XP + WP);
        soff[p] = (uint32_t)(panel[p] < XP ? panel[p] : panel[p] - XP) * kbs * 256 + lane * 4;
    }
    auto open_unit = [&] {
        const int have_x = min(BM / 16, (m + 15) / 16 - load.row0 / 16), have_w = min(BN / 16, (n + 15) / 16 - load.col0 / 16);
        const int panels_x = min(XP, (m + 63) / 64 - load.row0 / 64), panels_w = min(WP, (n + 63) / 64 - load.col0 / 64);
        rx = buffer_rsrc(q + (size_t)(load.row0 / 16) * kbs * 1024, (uint32_t)(have_x * kbs) * 1024u);
        rw = buffer_rsrc(codes + (size_t)(load.col0 / 16) * kbs * 1024, (uint32_t)(have_w * kbs) * 1024u);
#pragma unroll
        for (int p = 0; p < SPW; p++)
            rs[p] = panel[p] < XP
                        ? buffer_rsrc(sx + (size_t)(load.row0 / 64) * kbs * 256, (uint32_t)(panels_x * kbs) * 256u)
                        : buffer_rsrc(scales + (size_t)(load.col0 / 64) * kbs * 256, (uint32_t)(panels_w * kbs) * 256u);
    };
    open_unit();
    // Load p of a stage's PB.
    auto load_piece = [&](int stage, int p) {
        const int kb = load_step * KS + group;
        const bool live = load_id < units && kb < kbs;
        const uint32_t at = lds0 + stage * STAGE, past = live ? 0u : 0x80000000u, k = live ? (uint32_t)kb : 0u;
        if (p < XPW) {
            const int u = wave * XPW + p;
            dma16_at(at + u * 1024, ((uint32_t)(u * kbs) * 1024u + lane * 16) | past, rx, k * 1024);
        } else if (p < XPW + WPW) {
            const int u = wave * WPW + p - XPW;
            dma16_at(at + XB + u * 1024, ((uint32_t)(u * kbs) * 1024u + lane * 16) | past, rw, k * 1024);
        } else {
            const int u = p - XPW - WPW;
            dma4_at(at + SB + panel[u] * 256, soff[u] | past, rs[u], k * 256);
        }
    };
    // The weight's operands, the scale words and the last XD row tiles of x are held for two steps; a register of the
    // other row tiles takes the next step's operand once its products are under way.
    constexpr int XD = MT >= 4 ? MT / 4 : 1, XH = MT - XD;
    struct Operands {
        uint4_t w[NT], x[XD];
        uint32_t sw[WW], sx[XW];
    };
    uint4_t head[XH > 0 ? XH : 1];
    float4_t acc[NT][MT];
    const uint32_t own = group * PART, x0 = own + wm * TM * 64 + lane * 16, w0 = own + XB + wn * TN * 64 + lane * 16;
    const uint32_t sx0 = own + SB + wm * TM / 64 * 256 + lane * 4, sw0 = own + SB + XP * 256 + wn * TN / 64 * 256 + lane * 4;
    auto read_w = [&](const uint8_t *st, int a, Operands &o) { o.w[a] = *(const uint4_t *)(st + w0 + a * 1024); };
    auto read_x = [&](const uint8_t *st, int b, Operands &o) {
        (b < XH ? head[b < XH ? b : 0] : o.x[b < XH ? 0 : b - XH]) = *(const uint4_t *)(st + x0 + b * 1024);
    };
    auto read_scales = [&](const uint8_t *st, Operands &o) {
#pragma unroll
        for (int i = 0; i < WW; i++) o.sw[i] = *(const uint32_t *)(st + sw0 + i * 256);
#pragma unroll
        for (int i = 0; i < XW; i++) o.sx[i] = *(const uint32_t *)(st + sx0 + i * 256);
    };

#pragma unroll
    for (int i = 0; i < NS; i++) {
#pragma unroll
        for (int p = 0; p < PB; p++) load_piece(i, p);
        load_step++;
    }
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 1) * PB) : "memory");
    Operands two[2];
    read_scales(lds, two[0]);
#pragma unroll
    for (int a = 0; a < NT; a++) read_w(lds, a, two[0]);
#pragma unroll
    for (int b = 0; b < MT; b++) read_x(lds, b, two[0]);
    int stage = 0;
    // where a wave's tiles are part of a panel, its first tile's byte is not the word's first
    int xshift = 0, wshift = 0;
    // The products of a step, the next one's operands read and the loads of the step NS further issued among them, in
    // this order: left to itself the compiler moves the reads to where they are used.
    auto advance = [&](const Operands &now, Operands &next) {
        // This wave's loads of the next step are done once only the later steps' are left (stores among them are
        // waited for too early, never too late), and its reads of this step's stage at lgkmcnt(0); then the barrier
        // covers every wave, and the stage is free.
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 2) * PB) : "memory");
        const int free_stage = stage;
        stage = stage + 1 == NS ? 0 : stage + 1;
        const uint8_t *st = lds + stage * STAGE;
        uint32_t sw[WW], sxw[XW];
#pragma unroll
        for (int i = 0; i < WW; i++) sw[i] = TN < 64 ? now.sw[i] >> wshift : now.sw[i];
#pragma unroll
        for (int i = 0; i < XW; i++) sxw[i] = TM < 64 ? now.sx[i] >> xshift : now.sx[i];
        constexpr int G = MT > 1 ? MT - 1 : 1;  // groups of products with loads and reads after them
#pragma unroll
        for (int b = 0; b < MT; b++) {
#pragma unroll
            for (int a = 0; a < NT; a++)
                acc[a][b] = mx4_mfma_ab(a % 4, b % 4, now.w[a], sw[a / 4], b < XH ? head[b < XH ? b : 0] : now.x[b < XH ? 0 : b - XH],
                                        sxw[b / 4], acc[a][b]);
            __builtin_amdgcn_sched_barrier(0);
            // row tile b's next operand; and, spread over the groups before the last, scales, x's last tiles and w
            if (b < XH) read_x(st, b, next);
            constexpr int READS = 1 + XD + NT;
#pragma unroll
            for (int r = 0; r < READS; r++) {
                if (r * G / READS != b) continue;
                if (r == 0) read_scales(st, next);
                else if (r <= XD) read_x(st, XH + r - 1, next);
                else read_w(st, r - 1 - XD, next);
            }
#pragma unroll
            for (int p = 0; p < PB; p++)
                if (p * G / PB == b) load_piece(free_stage, p);
            __builtin_amdgcn_sched_barrier(0);
        }
        load_step++;
    };

    for (int id = blockIdx.x; id < units; id += gridDim.x) {
        const Unit u = unit_of(id);
        if (TM < 64) xshift = (u.row0 + wm * TM) / 16 % 4 * 8;
        if (TN < 64) wshift = (u.col0 + wn * TN) / 16 % 4 * 8;
#pragma unroll
        for (int a = 0; a < NT; a++)
#pragma unroll
            for (int b = 0; b < MT; b++) acc[a][b] = float4_t{0.f, 0.f, 0.f, 0.f};
        for (int part = 0; part < 2; part++) {  // the last NS steps load the next unit's first
            for (int i = part == 0 ? NS : 0; i < (part == 0 ? steps : NS); i += 2) {
                advance(two[0], two[1]);
                advance(two[1], two[0]);
            }
            if (part == 1) break;
            load_step = 0;
            load_id += gridDim.x;
            if (load_id < units) {
                load = unit_of(load_id);
                open_unit();
            }
        }

        if constexpr (KS > 1) {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // no LDS write in flight
            float4_t *sums = (float4_t *)lds;                            // [groups - 1][waves][tiles][64 lanes]
            __syncthreads();
            if (group > 0) {
#pragma unroll
                for (int a = 0; a < NT; a++)
#pragma unroll
                    for (int b = 0; b < MT; b++)
                        sums[(((group - 1) * WAVES + wave) * NT * MT + a * MT + b) * 64 + lane] = acc[a][b];
            }
            __syncthreads();
            if (group > 0) return;
#pragma unroll
            for (int h = 1; h < KS; h++)
#pragma unroll
                for (int a = 0; a < NT; a++)
#pragma unroll
                    for (int b = 0; b < MT; b++)
                        acc[a][b] += sums[(((h - 1) * WAVES + wave) * NT * MT + a * MT + b) * 64 + lane];
        }
        // A lane holds row j's columns 4 g .. 4 g + 3 of each tile: 16 bytes in f32. Of 16-bit outputs two column
        // tiles change lanes (odd rows of 16 lanes of the one with even rows of the other), so that a lane stores
        // eight columns of one tile, 64 bytes of a row together.
#pragma unroll
        for (int b = 0; b < MT; b++) {
            const int row = u.row0 + wm * TM + b * 16 + j;
            const size_t line = (size_t)row * n;
            if (dtype == 0) {
                if (row >= m) continue;
#pragma unroll
                for (int a = 0; a < NT; a++) {
                    const int col = u.col0 + wn * TN + a * 16 + 4 * g;
                    if (col < n) fp8_store4(y, 0, line + col, acc[a][b], n - col);
                }
            } else {
#pragma unroll
                for (int a = 0; a < NT; a += 2) {
                    const uint2_t v = mx4_round4(acc[a][b], dtype), w = mx4_round4(acc[a + 1][b], dtype);
                    const uint2_t lo = __builtin_bit_cast(uint2_t, __builtin_amdgcn_permlane16_swap(v[0], w[0], false, false));
                    const uint2_t hi = __builtin_bit_cast(uint2_t, __builtin_amdgcn_permlane16_swap(v[1], w[1], false, false));
                    const int col = u.col0 + wn * TN + (a + g % 2) * 16 + g / 2 * 8;
                    if (row < m && col < n) mx4_store8(y, line + col, uint4_t{lo[0], hi[0], lo[1], hi[1]}, n - col);
                }
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // no LDS write in flight when the block ends
}

// With KS = 1 as many workgroups as fit the compute units at once go through the tiles.
template <int BM, int BN, int WGM, int WGN, int KS, int NS>
void mx4_tile_launch(const dz_mx4_weight *w, const uint8_t *q, const uint8_t *sx, int m, void *y, int dtype,
                     hipStream_t s) {
    constexpr int LDS = NS * KS * ((BM + BN) * 64 + ((BM < 64 ? 1 : BM / 64) + (BN < 64 ? 1 : BN / 64)) * 256);
    constexpr int FIT = std::max(1, std::min(160 * 1024 / LDS, 32 / (WGM * WGN * KS)));
    const unsigned units = cdiv(m, BM) * cdiv(w->rows, BN), most = (unsigned)device_cus() * FIT;
    hipLaunchKernelGGL((mx4_tile_kernel<BM, BN, WGM, WGN, KS, NS>), dim3(KS == 1 ? std::min(units, most) : units),
                       dim3(WGM * WGN * KS * 64), 0, s, w->codes, w->scales, w->rows, w->kbs, q, sx, m, y, dtype,
                       (int)units);
}

// Four rows a lane past four workgroups a compute unit (us, one / four: 4096 x 4096 bf16 9.4 / 8.0; 1001 x 4096 3.3 /
// 3.6; 1001 x 1111 f16 3.0 / 5.0).
template <class T>
void mx4_quantize_form(const T *x, int m, int k, uint8_t *q, uint8_t *sx, int *bad, hipStream_t s) {
    const int kbs = (int)cdiv(k, 128);
    const unsigned panels = cdiv(m, 64), most = 32768;  // a grid's y ends at 65535
    const dim3 grid(kbs, std::min(panels, most), cdiv(panels, most));
    if ((size_t)kbs * panels > 4 * (size_t)device_cus())
        hipLaunchKernelGGL((mx4_quantize_kernel<T, 4>), grid, dim3(256), 0, s, x, m, k, kbs, q, sx, bad);
    else
        hipLaunchKernelGGL((mx4_quantize_kernel<T, 1>), grid, dim3(1024), 0, s, x, m, k, kbs, q, sx, bad);
}

void launch_mx4_quantize(const void *x, int dtype, int m, int k, uint8_t *q, uint8_t *sx, int *bad, hipStream_t s) {
    if (dtype == DZ_F32) mx4_quantize_form((const float *)x, m, k, q, sx, bad, s);
    else if (dtype == DZ_F16) mx4_quantize_form((const half_t *)x, m, k, q, sx, bad, s);
    else mx4_quantize_form((const bf16_t *)x, m, k, q, sx, bad, s);
}

// The tiles, in the order of the "mx4" family's variants from kRows on, and the time of
// a grid on each: f + c us a 128-block of k for the first tile of a compute unit, and
// more_f + more_c a block for each further one, halfway between whole rounds of the
// units and their mean (a unit's workgroups overlap). Fitted to 150 shapes drawn at
// random (17 to 4000 rows, K 100 to 9600, N 40 to 14400, every type out), where the
// choice is 0.9% slower than the best of these in the geometric mean and at most 13%.
// Many workgroups a unit hide a short k's latencies, four or two groups of waves on a
// long k spare it, larger tiles load less for each product. Measured (us, rows16 / 32x32
// / 32x32k4 / 64x64 / 64x64k2 / 64x128 / 128x128 / 256x256):
//   57 rows, K=679, N=1096     3.5 / 3.9 / 4.4 / 4.4 / 5.2 / 5.0 / 7.6 / 10
//   95 rows, K=411, N=8289     7.1 / 5.3 / 9.1 / 6.0 / 7.9 / 6.0 / 8.8 / 11
//   85 rows, K=1980, N=2137    4.9 / 5.3 / 5.3 / 6.3 / 6.6 / 7.8 / 9.8 / 17
//   343 rows, K=4096, N=1024   - / 8.7 / 8.4 / 8.3 / 8.1 / 10.0 / 12.6 / 26
//   847 rows, K=1193, N=3394   - / 11.7 / 23.4 / 9.0 / 11.8 / 8.7 / 9.9 / 15
//   586 rows, K=4096, N=14336  - / 70 / 92 / 43 / 55 / 35 / 43 / 38
//   8192 rows, K=N=4096        - / - / 335 / - / 178 / - / 130 / 81
struct Mx4Tile {
    int bm, bn;
    float f, c, more_f, more_c;
    bool persistent;
};
constexpr Mx4Tile kMx4Tiles[] = {
    {16, 16, 3.3f, 0.021f, 0.07f, 0.041f, false}, {32, 32, 3.6f, 0.101f, 0.35f, 0.041f, true},
    {32, 32, 4.3f, 0.064f, 1.4f, 0.047f, false},  {64, 64, 3.9f, 0.141f, 1.1f, 0.103f, true},
    {64, 64, 4.9f, 0.108f, 2.4f, 0.095f, false},  {64, 128, 4.4f, 0.190f, 1.6f, 0.180f, true},
    {128, 128, 7.7f, 0.199f, 7.6f, 0.295f, false}, {256, 256, 13.2f, 0.62f, 0.0f, 1.6f, true}};
constexpr int kRows = 1, kTiles = 8;
constexpr int kMostRows = 160;  // that the rows kernel, which reads the weight again every 16, is measured for

// A grid has less than 2^32 threads: the forms with a workgroup of up to 512 a tile go up to 2^23 tiles.
bool mx4_fits(int variant, int m, int n) {
    const Mx4Tile &t = kMx4Tiles[variant - kRows];
    return t.persistent || (size_t)cdiv(m, t.bm) * cdiv(n, t.bn) < (size_t)1 << 23;
}

int mx4_pick(int variant, int m, int n, int kbs) {
    if (variant) return mx4_fits(variant, m, n) ? variant : kTiles;
    if (m <= 16) return kRows;
    const float cus = (float)device_cus(), k = (float)kbs;
    int best = kRows;
    float least = 1e30f;
    for (int i = m <= kMostRows ? 0 : 1; i < kTiles; i++) {
        const Mx4Tile &t = kMx4Tiles[i];
        const float each = (float)cdiv(m, t.bm) * (float)cdiv(n, t.bn) / cus;
        const float rounds = std::max(1.0f, 0.5f * (each + std::ceil(each)));
        const float us = t.f + t.c * k + (rounds - 1.0f) * (t.more_f + t.more_c * k);
        if (us < least && mx4_fits(kRows + i, m, n)) least = us, best = kRows + i;
    }
    return best;
}

// The product of m > 0 rows of codes.
void launch_mx4_product(const dz_mx4_weight *w, const uint8_t *q, const uint8_t *sx, int m, void *y, int dtype,
                        int variant, hipStream_t s) {
    switch (mx4_pick(variant, m, w->rows, w->kbs)) {
        case kRows: return mx4_rows_launch(w, q, sx, m, y, dtype, s);
        case 2: return mx4_tile_launch<32, 32, 2, 1, 1, 4>(w, q, sx, m, y, dtype, s);
        case 3: return mx4_tile_launch<32, 32, 2, 1, 4, 2>(w, q, sx, m, y, dtype, s);
        case 4: return mx4_tile_launch<64, 64, 2, 2, 1, 4>(w, q, sx, m, y, dtype, s);
        case 5: return mx4_tile_launch<64, 64, 2, 2, 2, 4>(w, q, sx, m, y, dtype, s);
        case 6: return mx4_tile_launch<64, 128, 1, 4, 1, 4>(w, q, sx, m, y, dtype, s);
        case 7: return mx4_tile_launch<128, 128, 2, 2, 2, 4>(w, q, sx, m, y, dtype, s);
        default: return mx4_tile_launch<256, 256, 2, 4, 1, 4>(w, q, sx, m, y, dtype, s);
    }
}

bool mx4_dtype(int32_t d) { return d == DZ_F32 || d == DZ_F16 || d == DZ_BF16; }
size_t whole(size_t n) { return (n + 255) / 256 * 256; }

int32_t mx4_alloc(dz_ctx *ctx, size_t rows, size_t cols, dz_mx4_weight **out) {
    if (rows == 0 || cols == 0 || rows > kMx4MostRows || cols > kMx4MostCols)
        return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "invalid weight shape");
    dz_mx4_weight *w = new (std::nothrow) dz_mx4_weight();
    if (!w) return ctx_fail(ctx, DZ_RESOURCE_LIMIT, "weight allocation");
    w->device = ctx_device(ctx);
    w->rows = (int)rows;
    w->cols = (int)cols;
    w->kbs = (int)((cols + 127) / 128);
    w->bytes = mx4_code_bytes(rows, cols) + mx4_scale_bytes(rows, cols);
    const hipError_t e = hipMalloc(&w->codes, w->bytes);
    w->scales = w->codes + mx4_code_bytes(rows, cols);
    if (e != hipSuccess) {
        delete w;
        return ctx_hip_fail(ctx, e, "weight allocation");
    }
    *out = w;
    return DZ_OK;
}

void mx4_release(dz_mx4_weight *w) {
    if (!w) return;
    hipFree(w->codes);
    delete w;
}

int32_t mx4_weight_ok(dz_ctx *ctx, const dz_mx4_weight *w) {
    if (!w) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    if (w->device != ctx_device(ctx)) return ctx_fail(ctx, DZ_INVALID_REQUEST, "the weight lives on another device");
    return DZ_OK;
}

int32_t mx4_codes_ok(dz_ctx *ctx, const uint8_t *q, const uint8_t *s) {
    if (((uintptr_t)q & 15) != 0 || ((uintptr_t)s & 15) != 0)
        return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "codes and scales must be 16-byte aligned");
    return DZ_OK;
}

// A handle once its contents are checked (the flag that the kernels just enqueued may set).
int32_t mx4_finish(dz_ctx *ctx, dz_mx4_weight *w, const char *complaint, dz_mx4_weight **out) {
    int value = 0;
    int32_t rc = ctx_flag_value(ctx, &value);
    if (!rc && value) rc = ctx_fail(ctx, DZ_INVALID_CHECKPOINT, complaint);
    if (rc) {
        mx4_release(w);
        return rc;
    }
    *out = w;
    return DZ_OK;
}

}  // namespace

int32_t mx4_weight_create(dz_ctx *ctx, const uint8_t *codes, const uint8_t *scales, size_t rows, size_t cols,
                          dz_mx4_weight **out) {
    if (!out) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    *out = nullptr;
    if (!codes || !scales) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    dz_mx4_weight *w = nullptr;
    if (int32_t rc = mx4_alloc(ctx, rows, cols, &w)) return rc;
    hipStream_t s = ctx_stream(ctx);
    launch_fill_i32(ctx_flag(ctx), 0, 1, s);
    const size_t pieces = (rows + 15) / 16 * 16 * w->kbs * 4;
    hipLaunchKernelGGL(mx4_retile_kernel, dim3((unsigned)std::min((pieces + 255) / 256, (size_t)1 << 20)), dim3(256), 0,
                       s, codes, scales, pieces, w->rows, w->cols, w->kbs, w->codes, w->scales, ctx_flag(ctx));
    return mx4_finish(ctx, w, "invalid 4-bit floating point weight", out);
}

int32_t mx4_weight_quantize(dz_ctx *ctx, const void *values, int32_t dtype, size_t rows, size_t cols,
                            dz_mx4_weight **out) {
    if (!out) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    *out = nullptr;
    if (!values) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    if (!mx4_dtype(dtype)) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "unknown dtype");
    dz_mx4_weight *w = nullptr;
    if (int32_t rc = mx4_alloc(ctx, rows, cols, &w)) return rc;
    hipStream_t s = ctx_stream(ctx);
    launch_fill_i32(ctx_flag(ctx), 0, 1, s);
    launch_mx4_quantize(values, dtype, w->rows, w->cols, w->codes, w->scales, ctx_flag(ctx), s);
    return mx4_finish(ctx, w, "non-finite weight", out);
}

void mx4_weight_free(dz_mx4_weight *w) { mx4_release(w); }

int32_t mx4_weight_info(const dz_mx4_weight *w, size_t *rows, size_t *cols, size_t *device_bytes) {
    if (!w) return DZ_INVALID_REQUEST;
    if (rows) *rows = (size_t)w->rows;
    if (cols) *cols = (size_t)w->cols;
    if (device_bytes) *device_bytes = w->bytes;
    return DZ_OK;
}

int32_t mx4_dequant(dz_ctx *ctx, const dz_mx4_weight *w, float *y) {
    if (int32_t rc = mx4_weight_ok(ctx, w)) return rc;
    if (!y) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    const size_t blocks = ((size_t)w->rows * w->cols + 255) / 256;
    hipLaunchKernelGGL(mx4_dequant_kernel, dim3((unsigned)std::min(blocks, (size_t)1 << 20)), dim3(256), 0,
                       ctx_stream(ctx), w->codes, w->scales, w->rows, w->cols, w->kbs, y);
    return ctx_launched(ctx, "mx4 dequant");
}

int32_t mx4_bytes(size_t m, size_t k, size_t *codes, size_t *scales) {
    if (k == 0 || k > kMx4MostCols || m > kMx4MostRows) return DZ_INVALID_PARAMETERS;
    if (codes) *codes = mx4_code_bytes(m, k);
    if (scales) *scales = mx4_scale_bytes(m, k);
    return DZ_OK;
}

int32_t mx4_quantize(dz_ctx *ctx, const void *x, int32_t dtype, size_t m, size_t k, uint8_t *q, uint8_t *s) {
    if (!mx4_dtype(dtype)) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "unknown dtype");
    if (k == 0 || k > kMx4MostCols) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "invalid activation shape");
    if (m && (!x || !q || !s)) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    if (m > kMx4MostRows) return ctx_fail(ctx, DZ_INPUT_TOO_LONG, "input budget exceeded");
    if (int32_t rc = mx4_codes_ok(ctx, q, s)) return rc;
    if (m == 0) return DZ_OK;
    launch_mx4_quantize(x, dtype, (int)m, (int)k, q, s, nullptr, ctx_stream(ctx));
    return ctx_launched(ctx, "mx4 quantize");
}

int32_t mx4_linear_q4(dz_ctx *ctx, const dz_mx4_weight *w, const uint8_t *q, const uint8_t *s, size_t m, void *y,
                      int32_t y_dtype) {
    if (int32_t rc = mx4_weight_ok(ctx, w)) return rc;
    if (m && (!q || !s || !y)) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    if (!mx4_dtype(y_dtype)) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "unknown dtype");
    if (m > kMx4MostRows) return ctx_fail(ctx, DZ_INPUT_TOO_LONG, "input budget exceeded");
    if (int32_t rc = mx4_codes_ok(ctx, q, s)) return rc;
    if (m == 0) return DZ_OK;
    launch_mx4_product(w, q, s, (int)m, y, y_dtype, ctx_variant(ctx, "mx4"), ctx_stream(ctx));
    return ctx_launched(ctx, "mx4 linear");
}

int32_t mx4_linear(dz_ctx *ctx, const dz_mx4_weight *w, const void *x, int32_t x_dtype, size_t m, void *y,
                   int32_t y_dtype) {
    if (int32_t rc = mx4_weight_ok(ctx, w)) return rc;
    if (m && (!x || !y)) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    if (!mx4_dtype(x_dtype) || !mx4_dtype(y_dtype)) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "unknown dtype");
    if (m > kMx4MostRows) return ctx_fail(ctx, DZ_INPUT_TOO_LONG, "input budget exceeded");
    if (m == 0) return DZ_OK;
    const size_t codes = whole(mx4_code_bytes(m, w->cols)), scales = whole(mx4_scale_bytes(m, w->cols));
    void *work = nullptr;
    const int variant = ctx_variant(ctx, "mx4");
    // Up to four rows as they are, one launch less. us, one launch / two, bf16 x (f32 where it differs), two weights in turn:
    //   K x N          1 row       2           3                     4
    //   1024 x 1024    2.7 / 4.1   2.9 / 4.2   3.4 / 4.2             3.4 / 4.2
    //   4096 x 4096    2.8 / 5.4   3.0 / 5.5   3.5 / 5.5             3.5 / 5.5
    //   2560 x 9216    4.7 / 7.0   5.1 / 7.0   5.9 / 7.1 (8.8)       6.0 / 7.1 (9.0)
    //   9216 x 2560    5.1 / 8.6   5.9 / 8.7   7.0 / 8.7             7.1 / 8.7
    //   4096 x 14336   6.8 / 10.9  7.6 / 11.0  8.3 / 10.9 (10.2)     8.4 / 11.0 (10.5)
    //   1024 x 16384   4.9 / 5.4   5.8 / 5.3   7.3 / 5.4 (8.1)       7.4 / 5.4 (8.0)
    // Every workgroup quantizes all of x, so it loses where many of them share a short k (the last line from two rows on),
    // and on wide weights, whose form of four tiles a workgroup is built for codes only: 1024 x 32000 8.1 / 7.0, 4 rows
    // 14.1 / 6.9; only 4096 x 32000 would gain (12.5 / 18.4, 4 rows of bf16 17.7 / 18.6).
    if (variant == 0 && m <= 4 && !mx4_many_tiles(w)) {
        hipStream_t s = ctx_stream(ctx);
        if (x_dtype == DZ_F32) mx4_raw_launch<float>(w, x, (int)m, y, y_dtype, s);
        else if (x_dtype == DZ_F16) mx4_raw_launch<half_t>(w, x, (int)m, y, y_dtype, s);
        else mx4_raw_launch<bf16_t>(w, x, (int)m, y, y_dtype, s);
        return ctx_launched(ctx, "mx4 linear");
    }
    if (int32_t rc = ctx_workspace(ctx, codes + scales, &work)) return rc;
    uint8_t *q = (uint8_t *)work, *sx = q + codes;
    launch_mx4_quantize(x, x_dtype, (int)m, w->cols, q, sx, nullptr, ctx_stream(ctx));
    launch_mx4_product(w, q, sx, (int)m, y, y_dtype, variant, ctx_stream(ctx));
    return ctx_launched(ctx, "mx4 linear");
}

}  // namespace dz
