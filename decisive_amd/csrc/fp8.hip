// fp8.hip -- products on 8-bit floating point weights with a scale for each
// 128 x 128 block (fp8.hpp has the form and the layout).
//
//   y[i, j] = sum over 128-blocks b of sx[i, b] sw[j / 128, b] dot_b(i, j)
//
// dot_b is the dot of 128 codes. The blocks are folded in f32, in order of b:
// acc = fma(dot_b, sx * sw, acc).
#include <algorithm>
#include <type_traits>

#include "../../include/decisive_rocm.h"
#include "fp8.hpp"
#include "tiles.hpp"

struct dz_fp8_weight {
    dz::Fp8Weight w;
    int device = 0;
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

// One thread per 16-byte piece of the native layout; consecutive threads take
// consecutive pieces of a row, so that whole lines are read.
__global__ __launch_bounds__(256) void fp8_retile_kernel(const uint8_t *__restrict__ codes, size_t pieces, int rows,
                                                         int cols, int np, int kbs, uint8_t *__restrict__ dst,
                                                         size_t matrix_bytes, size_t tile_bytes, size_t kb_bytes,
                                                         int *bad) {
    for (size_t id = blockIdx.x * (size_t)256 + threadIdx.x; id < pieces; id += gridDim.x * (size_t)256) {
        const int piece = (int)(id % 8), kb = (int)(id / 8 % kbs);
        const size_t line = id / 8 / kbs;
        const int n = (int)(line % np), h = piece / 4, g = piece % 4, k0 = kb * 128 + 16 * piece;
        const size_t matrix = line / np;
        const uint8_t *src = codes + (matrix * rows + n) * cols + k0;
        uint32_t w[4] = {0, 0, 0, 0};
        if (n < rows && k0 + 16 <= cols) {
            const uint4_t v = *(const uint4_bytes_t *)src;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = v[e];
        } else if (n < rows) {
            for (int e = 0; e < 16 && k0 + e < cols; e++) w[e / 4] |= (uint32_t)src[e] << (8 * (e % 4));
        }
        bool nan = false;  // a byte whose low seven bits are all set
#pragma unroll
        for (int e = 0; e < 4; e++) nan |= (((w[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
        if (nan) atomicOr(bad, 1);
        *(uint4_t *)(dst + matrix * matrix_bytes + (size_t)(n / 16) * tile_bytes + (size_t)kb * kb_bytes + h * 1024 +
                     (g * 16 + n % 16) * 16) = uint4_t{w[0], w[1], w[2], w[3]};
    }
}

__global__ __launch_bounds__(256) void fp8_scales_kernel(const float *__restrict__ src, float *__restrict__ dst,
                                                         size_t n, int *bad) {
    const size_t id = blockIdx.x * (size_t)256 + threadIdx.x;
    if (id >= n) return;
    const float v = src[id];
    if (!(v >= 0.0f && v <= 3.4028235e38f)) atomicOr(bad, 1);
    dst[id] = v;
}

// One block of threads per 128 x 128 block of values: its scale
// max(max|v| / 448, 2^-126) and its codes, as fp8_quantize8 makes them.
template <class T>
__global__ __launch_bounds__(256) void fp8_quantize_weight_kernel(const T *__restrict__ values, int rows, int cols,
                                                                  int np, int kbs, uint8_t *__restrict__ codes,
                                                                  float *__restrict__ scales, int *bad) {
    const int kb = blockIdx.x % kbs, nb = blockIdx.x / kbs;
    __shared__ uint32_t part[4];
    uint32_t most = 0;
    for (int i = threadIdx.x; i < 128 * 128; i += 256) {
        const int n = nb * 128 + i / 128, k = kb * 128 + i % 128;
        if (n >= rows || k >= cols) continue;
        const uint32_t b = __builtin_bit_cast(uint32_t, (float)values[(size_t)n * cols + k]) & 0x7fffffffu;
        most = most > b ? most : b;
    }
    for (int o = 32; o; o >>= 1) {
        const uint32_t other = (uint32_t)__shfl_xor((int)most, o);
        most = most > other ? most : other;
    }
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = most;
    __syncthreads();
    for (int i = 0; i < 4; i++) most = most > part[i] ? most : part[i];
    if (most >= 0x7f800000u) {
        if (threadIdx.x == 0) atomicOr(bad, 1);
        return;
    }
    const float s = fmaxf(__fdiv_rn(word_as_float(most), 448.0f), 1.17549435e-38f);
    if (threadIdx.x == 0) scales[(size_t)nb * kbs + kb] = s;
    for (int i = threadIdx.x; i < 128 * 8; i += 256) {
        const int n = nb * 128 + i / 8, piece = i % 8, k0 = kb * 128 + 16 * piece;
        if (n >= np) continue;
        uint32_t w[4];
        for (int e = 0; e < 16; e += 4) {
            float q[4];
            for (int f = 0; f < 4; f++)
                q[f] = n < rows && k0 + e + f < cols ? __fdiv_rn((float)values[(size_t)n * cols + k0 + e + f], s) : 0.0f;
            int p = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
            w[e / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], p, true);
        }
        *(uint4_t *)(codes + ((size_t)(n / 16) * kbs + kb) * 2048 + piece / 4 * 1024 + (piece % 4 * 16 + n % 16) * 16) =
            uint4_t{w[0], w[1], w[2], w[3]};
    }
}

__global__ __launch_bounds__(256) void fp8_dequant_kernel(const uint8_t *__restrict__ codes,
                                                          const float *__restrict__ scales, int rows, int cols,
                                                          int kbs, float *__restrict__ y) {
    for (size_t id = blockIdx.x * (size_t)256 + threadIdx.x; id < (size_t)rows * cols; id += gridDim.x * (size_t)256) {
        const int n = (int)(id / cols), k = (int)(id % cols), kb = k / 128, kk = k % 128;
        const uint8_t c = codes[((size_t)(n / 16) * kbs + kb) * 2048 + kk / 64 * 1024 + (kk / 16 % 4 * 16 + n % 16) * 16 +
                                kk % 16];
        const half2_t v = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((uint32_t)c, 1.0f, false);
        y[id] = __fmul_rn((float)v[0], scales[(size_t)(n / 128) * kbs + kb]);
    }
}

// ---- activations ---------------------------------------------------------------

// Codes [m x 128 kbs] and scales [kbs x m] of the rows of x. 16 lanes take a
// block of 128 values; a workgroup takes the same block of 16 rows, so that it
// writes their scales side by side, and its neighbours go on along the rows (down the
// rows instead: 8192 x 4096 bf16 20.1 us). Bound by memory, (sizeof(T) + 1) bytes a
// value: 8192 x 4096 bf16 16.2 us, 6.2 TB/s; a few rows 1.8 us, a launch's time.
template <class T>
__global__ __launch_bounds__(256) void fp8_quantize_kernel(const T *__restrict__ x, int m, int k, int kbs,
                                                           uint8_t *__restrict__ q, float *__restrict__ sx) {
    const int kb = blockIdx.x, k0 = kb * 128 + threadIdx.x % 16 * 8;
    const int row = (blockIdx.z * gridDim.y + blockIdx.y) * 16 + threadIdx.x / 16;
    float v[8];
    const bool live = row < m;  // whole DPP rows of lanes
    fp8_load8(x + (size_t)(live ? row : 0) * k, k0, k, v);
    uint2_t codes;
    const float s = fp8_quantize8(v, codes);
    if (!live) return;
    *(uint2_t *)(q + ((size_t)row * kbs + kb) * 128 + threadIdx.x % 16 * 8) = codes;
    if (threadIdx.x % 16 == 0) sx[(size_t)kb * m + row] = s;
}

// ---- products: the weight streamed over a few rows -----------------------------

// A workgroup owns 16 weight rows and 16 MB activation rows. Its 8 waves take
// the k-blocks in turn (block b on wave b % 8), operands straight from memory,
// and their f32 partials are added in wave order, from LDS. The matrix unit's
// operands are swapped (weight first), so a lane holds one activation row and
// four output columns. Bound by the weight's bytes: 16 rows, K=4096, N=14336 13.9 us,
// 4.2 TB/s; K=1024, N=32000 in f32 8.7 us, 4.0 TB/s; smaller ones by one trip to memory
// and the launch (K=N=4096 5.5 us).
constexpr int kRowsWaves = 8;

template <int MB, bool WIDE, bool AHEAD>
__global__ __launch_bounds__(kRowsWaves * 64) void fp8_rows_kernel(const uint8_t *__restrict__ codes,
                                                                   const float *__restrict__ scales, int n, int kbs,
                                                                   const uint8_t *__restrict__ q,
                                                                   const float *__restrict__ sx, int m,
                                                                   void *__restrict__ y, int dtype) {
    __shared__ __align__(16) float part[kRowsWaves][MB * 256];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int g = lane / 16, j = lane % 16;
    const int tiles = (n + 15) / 16, t = blockIdx.x % tiles, row0 = blockIdx.x / tiles * 16 * MB;
    const uint8_t *wbase = codes + (size_t)t * kbs * 2048 + lane * 16;
    const float *swrow = scales + (size_t)(t / 8) * kbs;
    float4_t acc[MB];
#pragma unroll
    for (int b = 0; b < MB; b++) acc[b] = float4_t{0.f, 0.f, 0.f, 0.f};
    struct Block {
        uint4_t w[2], x[MB][2];
        float sw, sx[MB];
    };
    auto load = [&](int kb, Block &o) {
        o.w[0] = __builtin_nontemporal_load((const uint4_t *)(wbase + (size_t)kb * 2048));
        o.w[1] = __builtin_nontemporal_load((const uint4_t *)(wbase + (size_t)kb * 2048 + 1024));
        o.sw = swrow[kb];
#pragma unroll
        for (int b = 0; b < MB; b++) {
            const int row = row0 + 16 * b + j;
            o.x[b][0] = o.x[b][1] = uint4_t{0, 0, 0, 0};
            o.sx[b] = 0.0f;
            if (row < m) {
                const uint8_t *xr = q + ((size_t)row * kbs + kb) * 128 + 16 * g;
                o.x[b][0] = *(const uint4_t *)xr;
                o.x[b][1] = *(const uint4_t *)(xr + 64);
                o.sx[b] = sx[(size_t)kb * m + row];
            }
        }
    };
    auto add = [&](const Block &now) {
#pragma unroll
        for (int b = 0; b < MB; b++) {
            const float4_t d = WIDE ? fp8_mfma_wide(fp8_widen(now.w[0], now.w[1]), fp8_widen(now.x[b][0], now.x[b][1]))
                                    : fp8_mfma(now.w[0], now.w[1], now.x[b][0], now.x[b][1]);
            const float s = now.sx[b] * now.sw;
#pragma unroll
            for (int e = 0; e < 4; e++) acc[b][e] = __builtin_fmaf(d[e], s, acc[b][e]);
        }
    };
    if constexpr (AHEAD) {
        Block two[2];
        auto step = [&](int kb, const Block &now, Block &next) {
            if (kb + kRowsWaves < kbs) load(kb + kRowsWaves, next);
            __builtin_amdgcn_sched_barrier(0);
            add(now);
        };
        if (wave < kbs) load(wave, two[0]);
        for (int kb = wave; kb < kbs; kb += 2 * kRowsWaves) {
            step(kb, two[0], two[1]);
            if (kb + kRowsWaves < kbs) step(kb + kRowsWaves, two[1], two[0]);
        }
    } else {
        for (int kb = wave; kb < kbs; kb += kRowsWaves) {
            Block one;
            load(kb, one);
            add(one);
        }
    }
#pragma unroll
    for (int b = 0; b < MB; b++) *(float4_t *)&part[wave][(b * 16 + j) * 16 + 4 * g] = acc[b];
    __syncthreads();
    for (int i = threadIdx.x; i < MB * 256; i += kRowsWaves * 64) {
        const int row = row0 + i / 16, col = t * 16 + i % 16;
        if (row >= m || col >= n) continue;
        float v = part[0][i];
#pragma unroll
        for (int w = 1; w < kRowsWaves; w++) v += part[w][i];
        fp8_store(y, dtype, (size_t)row * n + col, v);
    }
}

// The same for one row straight from x, sparing the launch that quantizes it:
// each workgroup makes the codes it needs, a wave those of its own k-blocks, four
// at a time and while their weights are on the way, 16 lanes a block as
// fp8_quantize_kernel does, and hands them to its lanes as operands through LDS.
// The same bits as fp8_rows_kernel on fp8_quantize_kernel's codes.
template <class T, bool WIDE>
__global__ __launch_bounds__(kRowsWaves * 64) void fp8_one_kernel(const uint8_t *__restrict__ codes,
                                                                  const float *__restrict__ scales, int n, int kbs,
                                                                  const T *__restrict__ x, int k,
                                                                  void *__restrict__ y, int dtype) {
    constexpr int NB = 4;  // k-blocks of a batch, one for each 16 lanes
    __shared__ __align__(16) uint8_t s_codes[kRowsWaves][NB * 128];
    __shared__ float s_scale[kRowsWaves][NB];
    __shared__ float part[kRowsWaves][16];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int g = lane / 16, j = lane % 16, t = blockIdx.x;
    const uint8_t *wbase = codes + (size_t)t * kbs * 2048 + lane * 16;
    const float *swrow = scales + (size_t)(t / 8) * kbs;
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int b0 = wave; b0 < kbs; b0 += kRowsWaves * NB) {
        uint4_t w[NB][2];
        float sw[NB];
#pragma unroll
        for (int i = 0; i < NB; i++) {
            const int kb = min(b0 + i * kRowsWaves, kbs - 1);
            w[i][0] = __builtin_nontemporal_load((const uint4_t *)(wbase + (size_t)kb * 2048));
            w[i][1] = __builtin_nontemporal_load((const uint4_t *)(wbase + (size_t)kb * 2048 + 1024));
            sw[i] = swrow[kb];
        }
        float v[8];
        const int mine = b0 + g * kRowsWaves;
        fp8_load8(x, mine < kbs ? mine * 128 + j * 8 : k, k, v);
        uint2_t c;
        const float scale = fp8_quantize8(v, c);
        *(uint2_t *)&s_codes[wave][g * 128 + j * 8] = c;
        if (j == 0) s_scale[wave][g] = scale;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < NB; i++) {
            if (b0 + i * kRowsWaves >= kbs) break;
            uint4_t x0 = {0, 0, 0, 0}, x1 = {0, 0, 0, 0};
            float s = 0.0f;
            if (j == 0) {
                x0 = *(const uint4_t *)&s_codes[wave][i * 128 + 16 * g];
                x1 = *(const uint4_t *)&s_codes[wave][i * 128 + 16 * g + 64];
                s = s_scale[wave][i] * sw[i];
            }
            const float4_t d = WIDE ? fp8_mfma_wide(fp8_widen(w[i][0], w[i][1]), fp8_widen(x0, x1))
                                    : fp8_mfma(w[i][0], w[i][1], x0, x1);
#pragma unroll
            for (int e = 0; e < 4; e++) acc[e] = __builtin_fmaf(d[e], s, acc[e]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // read before the next batch is written
    }
    if (j == 0)
#pragma unroll
        for (int e = 0; e < 4; e++) part[wave][4 * g + e] = acc[e];
    __syncthreads();
    const int i = threadIdx.x, col = t * 16 + i;
    if (i >= 16 || col >= n) return;
    float sum = part[0][i];
#pragma unroll
    for (int u = 1; u < kRowsWaves; u++) sum += part[u][i];
    fp8_store(y, dtype, col, sum);
}

// From three blocks a wave on, its loads run one block ahead (us, without / with:
// 4 rows, K=9216, N=2560 8.2 / 7.2; 32 rows 13.1 / 11.2; 32 rows, K=N=4096 7.5 / 7.0;
// below that the registers cost more waves than it gives: 20 rows, K=1024, N=32000,
// f32 10.6 / 13.7).
template <int MB, bool WIDE>
void fp8_rows_form(const Fp8Weight &w, const uint8_t *q, const float *sx, int m, void *y, int dtype, hipStream_t s) {
    const dim3 grid(cdiv(w.rows, 16) * cdiv(m, 16 * MB)), block(kRowsWaves * 64);
    if (w.kbs > 3 * kRowsWaves)
        hipLaunchKernelGGL((fp8_rows_kernel<MB, WIDE, true>), grid, block, 0, s, w.codes, w.scales, w.rows, w.kbs, q, sx,
                           m, y, dtype);
    else
        hipLaunchKernelGGL((fp8_rows_kernel<MB, WIDE, false>), grid, block, 0, s, w.codes, w.scales, w.rows, w.kbs, q,
                           sx, m, y, dtype);
}

template <int MB>
void fp8_rows_launch(const Fp8Weight &w, const uint8_t *q, const float *sx, int m, void *y, int dtype, hipStream_t s) {
    if (dtype == DZ_F32) fp8_rows_form<MB, true>(w, q, sx, m, y, dtype, s);
    else fp8_rows_form<MB, false>(w, q, sx, m, y, dtype, s);
}

// ---- products: tiles over many rows ----------------------------------------------

// Block tile BM x BN (activation rows x weight rows). KS groups of WGM x WGN
// waves each take every KS-th 128-block of k; a step is KS blocks, one a group,
// in one of NS LDS stages that buffer_load ... lds fills. The weight's chunks
// land as they are, in operand order; activation rows of 128 bytes are
// swizzled, chunk c of row r in slot c ^ (r / 2 % 8), so that 16 lanes reading 16
// rows meet distinct banks. NS - 1 steps' loads are in flight or in use. Each
// block's dots come from a zero accumulator and are folded by sx * sw with one fma
// per output, in the shadow of the next MFMAs. The groups' sums are added in group
// order, through LDS. Where k is cut, workgroup b / tiles takes `per` of its blocks
// and writes their sums as f32 for fp8_join_kernel.
//
// 256x256 (8192 rows, K=N=4096): 127 to 140 us by the card, at 127 2.16 PFLOP/s of the
// 3.39 that MFMAs and fold alone reach from registers; 82 us of it are those, 78 the
// loads into LDS, 94 loads and LDS reads, which the two waves of a SIMD hide in part.
// Small tiles are bound by their loads, about 60 bytes a nanosecond into each unit.
template <int BM, int BN, int WGM, int WGN, int KS, int NS, bool WIDE>
__global__ __launch_bounds__(WGM *WGN *KS * 64) void fp8_tile_kernel(const uint8_t *__restrict__ codes,
                                                                     const float *__restrict__ scales, int n, int kbs,
                                                                     const uint8_t *__restrict__ q,
                                                                     const float *__restrict__ sx, int m,
                                                                     void *__restrict__ y, int dtype, int tiles,
                                                                     int per) {
    constexpr int WAVES = WGM * WGN, TM = BM / WGM, TN = BN / WGN, MT = TM / 16, NT = TN / 16;
    constexpr int XPW = BM / 8 / WAVES, WPW = BN / 8 / WAVES;  // 1 KiB loads per wave and stage
    constexpr int PB = XPW + WPW + 1;                          // and the row scales
    constexpr int XB = BM * 128, PART = XB + BN * 128 + (BM < 64 ? 64 : BM) * 4, STAGE = KS * PART;
    static_assert(XPW * 8 * WAVES == BM && WPW * 8 * WAVES == BN, "whole loads for each wave");
    static_assert(WPW == 1 || WPW % 2 == 0, "column tiles and halves known at compile time");
    static_assert(TN <= 128 && 128 % TN == 0, "one column block a wave");
    static_assert((NS - 2) * PB <= 63, "vmcnt range");
    static_assert((KS - 1) * BM * BN * 4 <= NS * STAGE, "the groups' sums fit the stages");
    __shared__ __align__(16) uint8_t lds[NS * STAGE];

    const int wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int group = wave_all / WAVES, wave = wave_all % WAVES;
    const int wm = wave / WGN, wn = wave % WGN, g = lane / 16, j = lane % 16;
    const int tiles_m = (m + BM - 1) / BM, tiles_n = (n + BN - 1) / BN;
    int tm, tn;
    const int split = blockIdx.x / tiles, first = split * per, last = min(kbs, first + per);  // its blocks of k
    xcd_tile(blockIdx.x - split * tiles, tiles, tiles_m, tiles_n, tm, tn);
    const int row0 = tm * BM, col0 = tn * BN, rows = min(BM, m - row0);
    const int kp = kbs * 128, tile0 = col0 / 16, tvalid = min(BN / 16, (n + 15) / 16 - tile0);
    const int32x4_t rx = buffer_rsrc(q + (size_t)row0 * kp, (uint32_t)(rows * kp));
    const int32x4_t rw = buffer_rsrc(codes + (size_t)tile0 * kbs * 2048, (uint32_t)(tvalid * kbs) * 2048u);
    // load p of this wave fills rows 8 (wave XPW + p) + lane / 8, slot lane % 8
    uint32_t xoff[XPW], woff[WPW];
#pragma unroll
    for (int p = 0; p < XPW; p++) {
        const int r = (wave * XPW + p) * 8 + lane / 8;
        xoff[p] = (uint32_t)r * kp + (lane % 8 ^ (r / 2 % 8)) * 16;
    }
#pragma unroll
    for (int p = 0; p < WPW; p++) {
        const int u = wave * WPW + p;
        woff[p] = (uint32_t)(u / 2) * kbs * 2048 + u % 2 * 1024 + lane * 16;
    }
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(lds)) + group * PART;
    // a wave's columns lie in one block of 128
    const float *sw = scales + (size_t)min((col0 + wn * TN) / 128, (n - 1) / 128) * kbs;

    // Blocks past the last one load nothing (every offset out of range, zeros in LDS), so that all waits go by count.
    auto load_stage = [&](int stage, int step) {
        const int kb = first + step * KS + group;
        const bool live = kb < last;
        const uint32_t at = lds0 + stage * STAGE, past = live ? 0u : 0x80000000u;
#pragma unroll
        for (int p = 0; p < XPW; p++)
            dma16_at(at + (wave * XPW + p) * 1024, xoff[p] | past, rx, live ? (uint32_t)kb * 128 : 0u);
#pragma unroll
        for (int p = 0; p < WPW; p++)
            dma16_at(at + XB + (wave * WPW + p) * 1024, woff[p] | past, rw, live ? (uint32_t)kb * 2048 : 0u);
        // every wave loads 64 of the row scales
        const int part = wave % (BM < 64 ? 1 : BM / 64);
        const int32x4_t rs = buffer_rsrc(sx + (live ? (size_t)kb * m + row0 : 0), live ? (uint32_t)rows * 4 : 0u);
        dma4(__builtin_amdgcn_readfirstlane(at + XB + BN * 128 + part * 256), (uint32_t)(part * 64 + lane) * 4,
             int32x4_t{__builtin_amdgcn_readfirstlane(rs[0]), __builtin_amdgcn_readfirstlane(rs[1]),
                       __builtin_amdgcn_readfirstlane(rs[2]), 0x00020000});
    };

    float4_t acc[NT][MT];
#pragma unroll
    for (int a = 0; a < NT; a++)
#pragma unroll
        for (int b = 0; b < MT; b++) acc[a][b] = float4_t{0.f, 0.f, 0.f, 0.f};
    const uint32_t sl = (j >> 1) & 7, own = group * PART;
    const uint32_t x0 = own + (wm * TM + j) * 128 + (g ^ sl) * 16, x1 = own + (wm * TM + j) * 128 + ((4 + g) ^ sl) * 16;
    const uint32_t w0 = own + XB + wn * TN * 128 + lane * 16, s0 = own + XB + BN * 128 + (wm * TM + j) * 4;
    auto compute = [&](int stage, float scale) {
        const uint8_t *st = lds + stage * STAGE;
        uint4_t w[NT][2], x[2][2];
        float s[MT];
#pragma unroll
        for (int a = 0; a < NT; a++) {
            w[a][0] = *(const uint4_t *)(st + w0 + a * 2048);
            w[a][1] = *(const uint4_t *)(st + w0 + a * 2048 + 1024);
        }
        x[0][0] = *(const uint4_t *)(st + x0);
        x[0][1] = *(const uint4_t *)(st + x1);
#pragma unroll
        for (int b = 0; b < MT; b++) s[b] = *(const float *)(st + s0 + b * 64);
#pragma unroll
        for (int b = 0; b < MT; b++) s[b] *= scale;
        Fp8Wide ww[WIDE ? NT : 1];
        if constexpr (WIDE) {
#pragma unroll
            for (int a = 0; a < NT; a++) ww[a] = fp8_widen(w[a][0], w[a][1]);
        }
        float4_t d[2][NT];
#pragma unroll
        for (int b = 0; b <= MT; b++) {
            if (b + 1 < MT) {
                x[(b + 1) & 1][0] = *(const uint4_t *)(st + x0 + (b + 1) * 2048);
                x[(b + 1) & 1][1] = *(const uint4_t *)(st + x1 + (b + 1) * 2048);
            }
            Fp8Wide xw;
            if constexpr (WIDE) xw = fp8_widen(x[b & 1][0], x[b & 1][1]);
#pragma unroll
            for (int a = 0; a < NT; a++) {
                if (b < MT)
                    d[b & 1][a] = WIDE ? fp8_mfma_wide(ww[WIDE ? a : 0], xw)
                                       : fp8_mfma(w[a][0], w[a][1], x[b & 1][0], x[b & 1][1]);
                if (b > 0) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        acc[a][b - 1][e] = __builtin_fmaf(d[(b - 1) & 1][a][e], s[b - 1], acc[a][b - 1][e]);
                }
            }
        }
    };

    const int steps = (last - first + KS - 1) / KS;
#pragma unroll
    for (int p = 0; p < NS - 1; p++) load_stage(p, p);
    float scale = sw[min(first + group, last - 1)];
    int stage = 0;
    for (int i = 0; i < steps; i++) {
        // This wave's loads of step i are done once only the later steps' are left, and its reads of the stage that the
        // next loads overwrite at lgkmcnt(0); then the barrier covers every wave.
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 2) * PB) : "memory");
        load_stage(stage == 0 ? NS - 1 : stage - 1, i + NS - 1);  // the stage that the step before read
        const float next = sw[min(first + (i + 1) * KS + group, last - 1)];
        compute(stage, scale);
        scale = next;
        stage = stage + 1 == NS ? 0 : stage + 1;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // no LDS write in flight once the block goes on

    if constexpr (KS > 1) {
        float4_t *sums = (float4_t *)lds;  // [groups - 1][waves][tiles][64 lanes]
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
                for (int b = 0; b < MT; b++) acc[a][b] += sums[(((h - 1) * WAVES + wave) * NT * MT + a * MT + b) * 64 + lane];
    }
#pragma unroll
    for (int b = 0; b < MT; b++) {
        const int row = row0 + wm * TM + b * 16 + j;
        if (row >= m) continue;
#pragma unroll
        for (int a = 0; a < NT; a++) {
            const int col = col0 + wn * TN + a * 16 + 4 * g;
            if (col < n) fp8_store4(y, dtype, ((size_t)split * m + row) * n + col, acc[a][b], n - col);
        }
    }
}

// y from the sums of `splits` runs of blocks, [splits][count] f32, added in
// their order; four loads of a thread are under way together.
__global__ __launch_bounds__(256) void fp8_join_kernel(const float *__restrict__ part, int splits, size_t count,
                                                       void *__restrict__ y, int dtype) {
    const size_t at = (blockIdx.x * (size_t)256 + threadIdx.x) * 4;
    if (at >= count) return;
    const int left = (int)min(count - at, (size_t)4);
    float4_t v = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < splits; i0 += 4) {
        float4_t p[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float *from = part + min(i0 + i, splits - 1) * count + at;
            if (left == 4) p[i] = *(const float4_any_t *)from;
            else p[i] = float4_t{from[0], left > 1 ? from[1] : 0.0f, left > 2 ? from[2] : 0.0f, 0.0f};
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i0 + i < splits) v += p[i];
    }
    fp8_store4(y, dtype, at, v, left);
}

// What a product needs beside its operands: how its tile cuts k (`splits` runs of
// blocks), and where the runs' sums go.
struct Fp8Split {
    int splits = 1;
    float *part = nullptr;  // [splits][m][n]
};

template <int BM, int BN, int WGM, int WGN, int KS, int NS, bool WIDE>
void fp8_tile_form(const Fp8Weight &w, const uint8_t *q, const float *sx, int m, void *y, int dtype, Fp8Split cut,
                   hipStream_t s) {
    const unsigned tiles = cdiv(m, BM) * cdiv(w.rows, BN);
    const int per = (int)cdiv(w.kbs, cut.splits), splits = (int)cdiv(w.kbs, per);
    hipLaunchKernelGGL((fp8_tile_kernel<BM, BN, WGM, WGN, KS, NS, WIDE>), dim3(tiles * splits),
                       dim3(WGM * WGN * KS * 64), 0, s, w.codes, w.scales, w.rows, w.kbs, q, sx, m,
                       splits > 1 ? cut.part : y, splits > 1 ? (int)DZ_F32 : dtype, (int)tiles, per);
    if (splits > 1) {
        const size_t count = (size_t)m * w.rows;
        hipLaunchKernelGGL(fp8_join_kernel, dim3(cdiv(count, 1024)), dim3(256), 0, s, cut.part, splits, count, y, dtype);
    }
}

template <int BM, int BN, int WGM, int WGN, int KS, int NS>
void fp8_tile_launch(const Fp8Weight &w, const uint8_t *q, const float *sx, int m, void *y, int dtype, Fp8Split cut,
                     hipStream_t s) {
    if (dtype == DZ_F32) fp8_tile_form<BM, BN, WGM, WGN, KS, NS, true>(w, q, sx, m, y, dtype, cut, s);
    else fp8_tile_form<BM, BN, WGM, WGN, KS, NS, false>(w, q, sx, m, y, dtype, cut, s);
}

void launch_fp8_quantize(const void *x, int dtype, int m, int k, uint8_t *q, float *sx, hipStream_t s) {
    const int kbs = (int)cdiv(k, 128);
    const unsigned rows = cdiv(m, 16), most = 32768;  // a grid's y ends at 65535
    const dim3 grid(kbs, std::min(rows, most), cdiv(rows, most));
    if (dtype == DZ_F32)
        hipLaunchKernelGGL(fp8_quantize_kernel<float>, grid, dim3(256), 0, s, (const float *)x, m, k, kbs, q, sx);
    else if (dtype == DZ_F16)
        hipLaunchKernelGGL(fp8_quantize_kernel<half_t>, grid, dim3(256), 0, s, (const half_t *)x, m, k, kbs, q, sx);
    else
        hipLaunchKernelGGL(fp8_quantize_kernel<bf16_t>, grid, dim3(256), 0, s, (const bf16_t *)x, m, k, kbs, q, sx);
}

// The tiles, in the order of the "fp8" family's variants from kTile0 on. A grid
// takes rounds of the chip (`resident` blocks a compute unit), each about f + blocks
// of k * c us, and the least sum is taken. f covers a block's first loads and its
// stores; c, the time of one 128-block, is measured with 8-bit and with f32-accurate
// dots; `share` is what c grows by where two blocks share a unit. A smaller tile
// walks k faster and loads more for it; a wave's larger part of a tile reads and, for
// f32, converts less for each MFMA (64x64k2's waves have 32x64, 64x64's 32x32), and
// needs deeper k to fill. Measured (us, 32x32k4 / 64x32k4 / 64x64k4 / 64x64 / 64x64k2 /
// 128x128 / 256x128, f16 or bf16 out; long sums cut as below):
//   64 rows, K=N=4096         8.0 / 9.8 / 11.4 / 10.2 / 11.4 / 14.6 / 15.9
//   128 rows, K=N=4096        11.9 / 8.5 / 10.9 / 12.4 / 12.0 / 15.5 / 18.2
//   40 rows, K=2560, N=9216   15.0 / 13.4 / 11.4 / 10.3 / 12.3 / 15.0 / 15.6
//   366 rows, K=4096, N=2560  22.3 / 15.0 / 11.6 / 14.1 / 15.4 / 18.5 / 21.7
//   308 rows, K=1024, N=4096  15.4 / 11.5 / 10.5 / 7.0 / 6.9 / 9.7 / 13.6
//   512 rows, K=4096, N=2560  27.8 / 21.8 / 20.4 / 17.7 / 15.0 / 18.8 / 22.1
//   600 rows, K=N=4096        53.8 / 35.6 / 31.2 / 28.4 / 25.8 / 23.2 / 29.4
//   1024 rows, K=2560, N=8192 131 / 84 / 62 / 45 / 41.6 / 34.6 / 29.2
//   229 rows, K=9216, N=2560  29.0 / 26.4 / 20.8 / 18.2 / 16.1 / 19.2 / 22.0; f32 out
//                             37.8 / 34.6 / 26.0 / 24.0 / 21.8 / 22.8 / 27.1
// 256x256: 8192 rows, K=N=4096 127 against 151 on 256x128; 4096 rows, K=1024 25.3, 28.8.
// Over 120 shapes drawn at random (33 to 3000 rows, K 100 to 9600, N 40 to 14400, every
// type out) the choice is 0.7% slower than the best tile in the geometric mean, within
// 3% on 112 of them and at most 21% (1506 rows, K=583, N=11248, f32 out 49.6 / 41.0).
struct Fp8Tile {
    int bm, bn, resident;
    float f, c, wide_c, share;
};
constexpr Fp8Tile kFp8Tiles[] = {
    {32, 32, 1, 3.0f, 0.13f, 0.165f, 1.0f},   {64, 32, 1, 3.2f, 0.166f, 0.22f, 1.0f},
    {64, 64, 1, 3.6f, 0.25f, 0.335f, 1.0f},   {64, 64, 2, 2.7f, 0.36f, 0.53f, 1.45f},
    {64, 64, 2, 3.8f, 0.40f, 0.63f, 1.0f},    {128, 128, 1, 5.0f, 0.57f, 0.95f, 1.0f},
    {256, 128, 1, 7.5f, 1.05f, 1.75f, 1.0f},  {256, 256, 1, 8.0f, 1.72f, 1e9f, 1.0f}};
constexpr int kRowsVariants = 2, kTile0 = 1 + kRowsVariants, kTiles = 8;
constexpr int kMostSplits = 16;

struct Fp8Pick {
    int variant, splits;
};

// A forced variant keeps its tile. Where a tile leaves units idle, k is cut into
// runs of blocks that fill one round; their sums go through memory and another
// launch, 2.5 us, 0.12 us a run (that kernel reads them in order) and some time a
// value. Measured (us, whole / cut, the best tile of each): 229 rows, K=9216, N=2560,
// f32 out 26.0 (64x64k4) / 21.8 (64x64k2, 3 runs), bf16 20.8 / 16.1; 128 rows, K=9000,
// N=500, f32 13.2 / 8.3 (32x32k4, 4 runs); 60 rows, K=9600, N=300 10.9 / 7.3 (8 runs).
// Not worth it for 100 rows, K=4096, N=1024 (6.3 / 7.1).
Fp8Pick fp8_pick(int variant, int m, int n, int kbs, bool wide) {
    if (variant == 0 && m <= 32) variant = m <= 16 ? 1 : 2;
    if (variant && variant < kTile0) return {variant, 1};
    if (wide && variant == kTile0 + kTiles - 1) variant--;
    const size_t cus = (size_t)device_cus();
    Fp8Pick best{variant, 1};
    float least = 1e30f;
    for (int i = 0; i < kTiles; i++) {
        if (variant && variant != kTile0 + i) continue;
        const Fp8Tile &t = kFp8Tiles[i];
        const size_t tiles = (size_t)cdiv(m, t.bm) * cdiv(n, t.bn), round = cus * t.resident;
        for (int splits = 1; splits <= kMostSplits && splits <= kbs; splits++) {
            const size_t blocks = tiles * splits;
            if (splits > 1 && blocks > round) break;
            const float c = (float)cdiv(kbs, splits) * (wide ? t.wide_c : t.c);
            const size_t full = blocks / round, rest = blocks % round;
            float us = (float)full * (t.f + t.share * c);
            if (rest) us += t.f + (rest > cus ? t.share : full && t.resident > 1 ? 0.67f * t.share : 1.0f) * c;
            if (splits > 1) us += 2.5f + (float)splits * (0.12f + (float)m * (float)n * 1.2e-6f);
            if (us < least) least = us, best = {kTile0 + i, splits};
        }
    }
    return best;
}

// f32 values that a product of m rows needs for its runs' sums.
size_t fp8_parts(const Fp8Weight &w, size_t m, int dtype, int variant) {
    const int splits = fp8_pick(variant, (int)m, w.rows, w.kbs, dtype == DZ_F32).splits;
    return splits > 1 ? splits * m * w.rows : 0;
}

// The product of m > 0 rows of codes. Few rows stream the weight (up to 32 rows:
// K=N=4096 7.0 us against 8.0 on 32x32 tiles, and N many times K far less).
void launch_fp8_product(const Fp8Weight &w, const uint8_t *q, const float *sx, int m, void *y, int dtype,
                        int variant, float *part, hipStream_t s) {
    const Fp8Pick pick = fp8_pick(variant, m, w.rows, w.kbs, dtype == DZ_F32);
    const Fp8Split cut{pick.splits, part};
    switch (pick.variant) {
        case 1: return fp8_rows_launch<1>(w, q, sx, m, y, dtype, s);
        case 2: return fp8_rows_launch<2>(w, q, sx, m, y, dtype, s);
        case 3: return fp8_tile_launch<32, 32, 2, 1, 4, 4>(w, q, sx, m, y, dtype, cut, s);
        case 4: return fp8_tile_launch<64, 32, 2, 1, 4, 3>(w, q, sx, m, y, dtype, cut, s);
        case 5: return fp8_tile_launch<64, 64, 2, 2, 4, 2>(w, q, sx, m, y, dtype, cut, s);
        case 6: return fp8_tile_launch<64, 64, 2, 2, 1, 4>(w, q, sx, m, y, dtype, cut, s);
        case 7: return fp8_tile_launch<64, 64, 2, 1, 2, 2>(w, q, sx, m, y, dtype, cut, s);
        case 8: return fp8_tile_launch<128, 128, 2, 2, 2, 2>(w, q, sx, m, y, dtype, cut, s);
        case 9: return fp8_tile_launch<256, 128, 4, 2, 1, 3>(w, q, sx, m, y, dtype, cut, s);
        default: break;
    }
    // its f32-accurate form would not fit the registers: fp8_pick takes 256x128 instead
    fp8_tile_form<256, 256, 2, 4, 1, 2, false>(w, q, sx, m, y, dtype, cut, s);
}

// One row quantized by the product's own kernel, in each of its workgroups: up
// to four of them a compute unit (us, against two launches: K=N=1024 3.7 / 4.4;
// K=N=4096 4.6 / 7.0 (5.0 on another card); K=4096, N=14336 11.7 / 13.5; K=1024, N=32000 13.9 / 9.0). Two
// rows so measured 6.1 / 7.0 at K=N=4096, but 5.1 / 4.5 at 1024 and 12.0 / 8.3 at K=2560,
// N=9216.
bool fp8_one(const Fp8Weight &w, size_t m) { return m == 1 && cdiv(w.rows, 16) <= 4u * (unsigned)device_cus(); }

template <class T>
void launch_fp8_one(const Fp8Weight &w, const T *x, void *y, int dtype, hipStream_t s) {
    const dim3 grid(cdiv(w.rows, 16)), block(kRowsWaves * 64);
    if (dtype == DZ_F32)
        hipLaunchKernelGGL((fp8_one_kernel<T, true>), grid, block, 0, s, w.codes, w.scales, w.rows, w.kbs, x, w.cols,
                           y, dtype);
    else
        hipLaunchKernelGGL((fp8_one_kernel<T, false>), grid, block, 0, s, w.codes, w.scales, w.rows, w.kbs, x, w.cols,
                           y, dtype);
}

bool fp8_dtype(int32_t d) { return d == DZ_F32 || d == DZ_F16 || d == DZ_BF16; }

int32_t fp8_alloc(dz_ctx *ctx, size_t rows, size_t cols, dz_fp8_weight **out) {
    if (rows == 0 || cols == 0 || rows > kFp8MostRows || cols > kFp8MostCols)
        return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "invalid weight shape");
    dz_fp8_weight *h = new (std::nothrow) dz_fp8_weight();
    if (!h) return ctx_fail(ctx, DZ_RESOURCE_LIMIT, "weight allocation");
    h->device = ctx_device(ctx);
    Fp8Weight &w = h->w;
    w.rows = (int)rows;
    w.cols = (int)cols;
    w.np = (int)((rows + 15) / 16 * 16);
    w.kbs = (int)((cols + 127) / 128);
    const hipError_t e = hipMalloc(&w.codes, w.code_bytes() + w.scale_bytes());
    w.scales = (float *)(w.codes + w.code_bytes());
    if (e != hipSuccess) {
        delete h;
        return ctx_hip_fail(ctx, e, "weight allocation");
    }
    *out = h;
    return DZ_OK;
}

void fp8_release(dz_fp8_weight *h) {
    if (!h) return;
    hipFree(h->w.codes);
    delete h;
}

int32_t fp8_weight_ok(dz_ctx *ctx, const dz_fp8_weight *w) {
    if (!w) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    if (w->device != ctx_device(ctx)) return ctx_fail(ctx, DZ_INVALID_REQUEST, "the weight lives on another device");
    return DZ_OK;
}

}  // namespace

void launch_fp8_retile(const uint8_t *codes, int count, int rows, int cols, uint8_t *dst, size_t matrix_bytes,
                       size_t tile_bytes, size_t kb_bytes, int *bad, hipStream_t s) {
    const int np = (rows + 15) / 16 * 16, kbs = (cols + 127) / 128;
    const size_t pieces = (size_t)count * np * kbs * 8;
    hipLaunchKernelGGL(fp8_retile_kernel, dim3((unsigned)std::min((pieces + 255) / 256, (size_t)1 << 20)), dim3(256), 0,
                       s, codes, pieces, rows, cols, np, kbs, dst, matrix_bytes, tile_bytes, kb_bytes, bad);
}

void launch_fp8_scales(const float *src, float *dst, size_t n, int *bad, hipStream_t s) {
    hipLaunchKernelGGL(fp8_scales_kernel, dim3(cdiv(n, 256)), dim3(256), 0, s, src, dst, n, bad);
}

int32_t fp8_weight_create(dz_ctx *ctx, const uint8_t *codes, const float *scales, size_t rows, size_t cols,
                          dz_fp8_weight **out) {
    if (!out) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    *out = nullptr;
    if (!codes || !scales) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    dz_fp8_weight *h = nullptr;
    int32_t rc = fp8_alloc(ctx, rows, cols, &h);
    if (rc) return rc;
    int *bad = ctx_flag(ctx), value = 0;
    hipStream_t s = ctx_stream(ctx);
    launch_fill_i32(bad, 0, 1, s);
    launch_fp8_retile(codes, 1, h->w.rows, h->w.cols, h->w.codes, 0, (size_t)h->w.kbs * 2048, 2048, bad, s);
    launch_fp8_scales(scales, h->w.scales, h->w.scale_bytes() / sizeof(float), bad, s);
    rc = ctx_flag_value(ctx, &value);
    if (!rc && value) rc = ctx_fail(ctx, DZ_INVALID_CHECKPOINT, "invalid 8-bit floating point weight");
    if (rc) {
        fp8_release(h);
        return rc;
    }
    *out = h;
    return DZ_OK;
}

int32_t fp8_weight_quantize(dz_ctx *ctx, const void *values, int32_t dtype, size_t rows, size_t cols,
                            dz_fp8_weight **out) {
    if (!out) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    *out = nullptr;
    if (!values) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    if (!fp8_dtype(dtype)) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "unknown dtype");
    dz_fp8_weight *h = nullptr;
    int32_t rc = fp8_alloc(ctx, rows, cols, &h);
    if (rc) return rc;
    int *bad = ctx_flag(ctx), value = 0;
    hipStream_t s = ctx_stream(ctx);
    launch_fill_i32(bad, 0, 1, s);
    const Fp8Weight &w = h->w;
    const dim3 grid((unsigned)w.kbs * cdiv(w.rows, 128));
    if (dtype == DZ_F32)
        hipLaunchKernelGGL(fp8_quantize_weight_kernel<float>, grid, dim3(256), 0, s, (const float *)values, w.rows,
                           w.cols, w.np, w.kbs, w.codes, w.scales, bad);
    else if (dtype == DZ_F16)
        hipLaunchKernelGGL(fp8_quantize_weight_kernel<half_t>, grid, dim3(256), 0, s, (const half_t *)values, w.rows,
                           w.cols, w.np, w.kbs, w.codes, w.scales, bad);
    else
        hipLaunchKernelGGL(fp8_quantize_weight_kernel<bf16_t>, grid, dim3(256), 0, s, (const bf16_t *)values, w.rows,
                           w.cols, w.np, w.kbs, w.codes, w.scales, bad);
    rc = ctx_flag_value(ctx, &value);
    if (!rc && value) rc = ctx_fail(ctx, DZ_INVALID_CHECKPOINT, "non-finite weight");
    if (rc) {
        fp8_release(h);
        return rc;
    }
    *out = h;
    return DZ_OK;
}

void fp8_weight_free(dz_fp8_weight *w) { fp8_release(w); }

int32_t fp8_weight_info(const dz_fp8_weight *w, size_t *rows, size_t *cols, size_t *device_bytes) {
    if (!w) return DZ_INVALID_REQUEST;
    if (rows) *rows = (size_t)w->w.rows;
    if (cols) *cols = (size_t)w->w.cols;
    if (device_bytes) *device_bytes = w->w.code_bytes() + w->w.scale_bytes();
    return DZ_OK;
}

int32_t fp8_dequant(dz_ctx *ctx, const dz_fp8_weight *w, float *y) {
    if (int32_t rc = fp8_weight_ok(ctx, w)) return rc;
    if (!y) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    const size_t blocks = ((size_t)w->w.rows * w->w.cols + 255) / 256;
    hipLaunchKernelGGL(fp8_dequant_kernel, dim3((unsigned)std::min(blocks, (size_t)1 << 20)), dim3(256), 0,
                       ctx_stream(ctx), w->w.codes, w->w.scales, w->w.rows, w->w.cols, w->w.kbs, y);
    return ctx_launched(ctx, "fp8 dequant");
}

int32_t fp8_quantize(dz_ctx *ctx, const void *x, int32_t dtype, size_t m, size_t k, uint8_t *q, float *s) {
    if (!fp8_dtype(dtype)) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "unknown dtype");
    if (k == 0 || k > kFp8MostCols) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "invalid activation shape");
    if (m && (!x || !q || !s)) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    if (m > kFp8MostRows) return ctx_fail(ctx, DZ_INPUT_TOO_LONG, "input budget exceeded");
    if (((uintptr_t)q & 15) != 0) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "codes must be 16-byte aligned");
    if (m == 0) return DZ_OK;
    launch_fp8_quantize(x, dtype, (int)m, (int)k, q, s, ctx_stream(ctx));
    return ctx_launched(ctx, "fp8 quantize");
}

int32_t fp8_linear_q8(dz_ctx *ctx, const dz_fp8_weight *w, const uint8_t *q, const float *s, size_t m, void *y,
                      int32_t y_dtype) {
    if (int32_t rc = fp8_weight_ok(ctx, w)) return rc;
    if (m && (!q || !s || !y)) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    if (!fp8_dtype(y_dtype)) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "unknown dtype");
    if (m > kFp8MostRows) return ctx_fail(ctx, DZ_INPUT_TOO_LONG, "input budget exceeded");
    if (((uintptr_t)q & 15) != 0) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "codes must be 16-byte aligned");
    if (m == 0) return DZ_OK;
    const int variant = ctx_variant(ctx, "fp8");
    const size_t parts = fp8_parts(w->w, m, y_dtype, variant);
    void *work = nullptr;
    if (parts)
        if (int32_t rc = ctx_workspace(ctx, parts * sizeof(float), &work)) return rc;
    launch_fp8_product(w->w, q, s, (int)m, y, y_dtype, variant, (float *)work, ctx_stream(ctx));
    return ctx_launched(ctx, "fp8 linear");
}

int32_t fp8_linear(dz_ctx *ctx, const dz_fp8_weight *w, const void *x, int32_t x_dtype, size_t m, void *y,
                   int32_t y_dtype) {
    if (int32_t rc = fp8_weight_ok(ctx, w)) return rc;
    if (m && (!x || !y)) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    if (!fp8_dtype(x_dtype) || !fp8_dtype(y_dtype)) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "unknown dtype");
    if (m > kFp8MostRows) return ctx_fail(ctx, DZ_INPUT_TOO_LONG, "input budget exceeded");
    if (m == 0) return DZ_OK;
    const int variant = ctx_variant(ctx, "fp8");
    if (fp8_one(w->w, m) && variant == 0) {
        hipStream_t s = ctx_stream(ctx);
        if (x_dtype == DZ_F32) launch_fp8_one(w->w, (const float *)x, y, y_dtype, s);
        else if (x_dtype == DZ_F16) launch_fp8_one(w->w, (const half_t *)x, y, y_dtype, s);
        else launch_fp8_one(w->w, (const bf16_t *)x, y, y_dtype, s);
        return ctx_launched(ctx, "fp8 linear");
    }
    const size_t codes = (m * (size_t)w->w.kbs * 128 + 255) / 256 * 256;
    const size_t scales = (m * (size_t)w->w.kbs * sizeof(float) + 255) / 256 * 256;
    void *work = nullptr;
    if (int32_t rc = ctx_workspace(ctx, codes + scales + fp8_parts(w->w, m, y_dtype, variant) * sizeof(float), &work))
        return rc;
    uint8_t *q = (uint8_t *)work;
    float *sx = (float *)(q + codes), *part = (float *)(q + codes + scales);
    launch_fp8_quantize(x, x_dtype, (int)m, w->w.cols, q, sx, ctx_stream(ctx));
    launch_fp8_product(w->w, q, sx, (int)m, y, y_dtype, variant, part, ctx_stream(ctx));
    return ctx_launched(ctx, "fp8 linear");
}

}  // namespace dz
