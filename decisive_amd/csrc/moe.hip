// moe.hip -- a mixture-of-experts layer for a few tokens on 8-bit floating
// point weights (fp8.hpp has their form), activations kept as they come.
//
//   l = x router^T, p = softmax(l), E(x) = the top_k experts of largest l
//   y = sum over e in E(x) of c_e down_e (silu(gate_e x) * up_e x)
//
// c_e is p_e, or p_e / (sum of the chosen p). A few tokens read far more
// weight than they multiply (2 operations a byte and row), so the layer is
// bound by the bytes of the experts that are chosen, each read once:
//   1 moe_logits_kernel   logits, and x as bf16 terms
//   2 moe_gate_up_kernel  finds each token's experts; per (chosen expert, 16
//                         columns of ff): h = silu(gate) * up of its rows; or
//     moe_top_kernel      the experts of each token, then
//     moe_wide_kernel     h, 128 columns of ff a workgroup
//   3 moe_down_kernel     per 16 columns of the output: every chosen expert's down
//                         product, times the rows' shares, summed; or
//     moe_wide_kernel     each slot's down product, 256 columns a workgroup, then
//     moe_combine_kernel  the shares' sum
// The first of each are for few rows, where launches and trips to memory count
// (launch_experts has the rule).
// A token's i-th expert is slot = token * top_k + i, and h has a row for each
// slot. Each workgroup finds the rows of its experts from the slots' experts,
// expert by expert and in order of tokens; no order depends on timing.
// The products run on the bf16 matrix unit: e4m3 is exact in bf16, and an
// activation is a sum of bf16 terms: x is one term (bf16), two (f16, exactly)
// or three (f32, exactly down to bf16's smallest step, 2^-133); h, which never leaves the layer, is two terms (16
// bits of it: 2^-16 off at most, against the 2^-9 or 2^-12 of the result's own
// rounding) or three for f32. Sums are f32.
#include <algorithm>
#include <new>

#include "../../include/decisive_rocm.h"
#include "fp8.hpp"
#include "tiles.hpp"

struct dz_moe {
    dz_moe_config cfg{};
    int device = 0;
    int kbd = 0, kbf = 0;           // 128-blocks of hidden and ff
    uint8_t *gate_up = nullptr;     // [experts][ff/16][kbd][gate, up] chunks of 2 KiB
    uint8_t *down = nullptr;        // [experts][hidden/16][kbf] chunks
    float *gate_scales = nullptr;   // [experts][ff/128][kbd]
    float *up_scales = nullptr;
    float *down_scales = nullptr;   // [experts][hidden/128][kbf]
    float *router = nullptr;        // [experts][128 kbd], zero past hidden
    uint8_t *memory = nullptr;      // all of these
    size_t bytes = 0;
};

namespace dz {

int32_t ctx_fail(dz_ctx *ctx, int32_t code, const std::string &msg);
int32_t ctx_hip_fail(dz_ctx *ctx, hipError_t e, const char *what);
hipStream_t ctx_stream(dz_ctx *ctx);
int *ctx_flag(dz_ctx *ctx);
int ctx_device(dz_ctx *ctx);
int32_t ctx_workspace(dz_ctx *ctx, size_t bytes, void **out);
int32_t ctx_launched(dz_ctx *ctx, const char *what);
int32_t ctx_flag_value(dz_ctx *ctx, int *value);

namespace {

constexpr int kMostExperts = 512, kMostTop = 16, kMostWidth = 65536;
constexpr int kRouteTokens = 4;  // tokens a workgroup of the logits kernel takes together
constexpr int kFewTokens = 16;   // tokens that moe_gate_up_kernel takes
constexpr int kFewSlots = 16;    // moe_down_kernel takes fewer

// What the kernels leave for the ones after, in the workspace.
struct MoePlan {
    float *logits;  // [tokens][experts]
    int *ids;       // [slots] experts
    float *shares;  // [slots]
    bf16_t *x;      // [terms][tokens][128 kbd]
    bf16_t *h;      // [terms][slots][128 kbf]
    float *p;       // [slots][128 kbd] the experts' outputs, for moe_combine_kernel
};

// v as TERMS bf16 values that add up to it: each term the leading 8 bits of
// what is left (cut, so that nothing overflows), the last one rounded.
template <int TERMS>
__device__ __forceinline__ void moe_split(float v, bf16_t out[TERMS]) {
#pragma unroll
    for (int i = 0; i + 1 < TERMS; i++) {
        const float head = word_as_float(__builtin_bit_cast(uint32_t, v) & 0xffff0000u);
        out[i] = (bf16_t)head;
        v -= head;
    }
    out[TERMS - 1] = (bf16_t)v;
}

// Maximum over the wave, in every lane (wave_max_dpp's pattern).
__device__ __forceinline__ uint32_t moe_wave_max(uint32_t v) {
    v = dpp_max_u32<0xB1>(v);
    v = dpp_max_u32<0x4E>(v);
    v = dpp_max_u32<0x124>(v);
    v = dpp_max_u32<0x128>(v);
    uint32_t a = v, b = v;
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
    v = a > b ? a : b;
    a = v;
    b = v;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
    return a > b ? a : b;
}

// A logit's order as an unsigned number above 0 (0 marks an expert that is taken or absent).
__device__ __forceinline__ uint32_t moe_key(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v == 0.0f ? 0.0f : v);
    return b & 0x80000000u ? (b == 0xffffffffu ? 1u : ~b) : b | 0x80000000u;
}

// The experts of one token by one wave: top times the largest logit, equal
// ones by the lower index (lane l holds experts PER l .. + PER - 1, so the first
// lane with the largest has the lowest). Lane i < top is left with the i-th.
template <int PER>
__device__ __forceinline__ void moe_top(const float *__restrict__ logits, int experts, int top, int renormalize,
                                        int &expert, float &share) {
    const int lane = threadIdx.x % 64;
    constexpr float kLeast = -3.4028235e38f;
    float l[PER], most = kLeast;
    uint32_t key[PER];
    bool fine = true;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const bool here = lane * PER + i < experts;
        l[i] = here ? logits[lane * PER + i] : kLeast;
        key[i] = here ? moe_key(l[i]) : 0u;
        if (!(fabsf(l[i]) <= 3.4028235e38f)) fine = false;
        most = fmaxf(most, l[i]);
    }
    fine = __all(fine);
    most = wave_max_dpp(most);
    float p[PER], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        p[i] = lane * PER + i < experts ? expf(l[i] - most) : 0.0f;
        sum += p[i];
    }
    float picked = 0.0f;
    expert = 0;
    share = 0.0f;
    for (int s = 0; s < top; s++) {
        uint32_t best = 0;
        int at = 0;
        float mine = 0.0f;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (key[i] > best) best = key[i], at = i, mine = p[i];
        const uint32_t largest = moe_wave_max(best);
        const int owner = __ffsll((unsigned long long)__ballot(best == largest)) - 1;
        const float c = word_as_float((uint32_t)__builtin_amdgcn_readlane(__builtin_bit_cast(int, mine), owner));
        const int e = owner * PER + __builtin_amdgcn_readlane(at, owner);
        picked += c;
        if (lane == s) expert = e, share = c;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (lane == owner && i == at) key[i] = 0;
    }
    const float whole = renormalize ? picked : wave_sum_dpp(sum);
    share = fine ? share / whole : __builtin_nanf("");
}

// The same for up to 128 experts by counting, for each of a lane's experts (l
// and l + 64), the larger logits: 64 or 128 comparisons that wait for nothing,
// where each of moe_top's rounds is a chain of some 40 instructions. Counts that
// are a permutation say that no two logits are equal; else moe_top decides.
struct MoeTopShared {
    uint32_t key[128];
    int expert[kMostTop];
    float p[kMostTop];
};
__device__ __forceinline__ void moe_top_any(const float *__restrict__ logits, int experts, int top, int renormalize,
                                            MoeTopShared &own, int &expert, float &share) {
    if (experts > 256) return moe_top<8>(logits, experts, top, renormalize, expert, share);
    if (experts > 128) return moe_top<4>(logits, experts, top, renormalize, expert, share);
    const int lane = threadIdx.x % 64;
    constexpr float kLeast = -3.4028235e38f;
    float l[2], p[2];
    uint32_t key[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const bool here = lane + 64 * i < experts;
        l[i] = here ? logits[lane + 64 * i] : kLeast;
        key[i] = here ? moe_key(l[i]) : 0u;
        own.key[lane + 64 * i] = key[i];
    }
    const bool fine = __all(fabsf(l[0]) <= 3.4028235e38f && fabsf(l[1]) <= 3.4028235e38f);
    const float most = wave_max_dpp(fmaxf(l[0], l[1]));
#pragma unroll
    for (int i = 0; i < 2; i++) p[i] = lane + 64 * i < experts ? expf(l[i] - most) : 0.0f;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    int rank[2] = {0, 0};
    for (int e0 = 0; e0 < experts; e0 += 16) {
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const uint4_t other = *(const uint4_t *)&own.key[e0 + e];
#pragma unroll
            for (int c = 0; c < 4; c++) {
                rank[0] += other[c] > key[0];
                rank[1] += other[c] > key[1];
            }
        }
    }
    const int ranks = (lane < experts ? rank[0] : 0) + (lane + 64 < experts ? rank[1] : 0);
    const float sum = wave_sum_dpp((float)ranks);  // at most 127 * 64: exact
    if (sum != (float)(experts * (experts - 1) / 2)) {
        if (experts > 64) moe_top<2>(logits, experts, top, renormalize, expert, share);
        else moe_top<1>(logits, experts, top, renormalize, expert, share);
        return;
    }
    float part = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; i++)
        if (lane + 64 * i < experts) {
            if (rank[i] < top) {
                own.expert[rank[i]] = lane + 64 * i;
                own.p[rank[i]] = p[i];
            }
            if (!renormalize || rank[i] < top) part += p[i];
        }
    const float whole = wave_sum_dpp(part);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    expert = lane < top ? own.expert[lane] : 0;
    share = fine ? (lane < top ? own.p[lane] : 0.0f) / whole : __builtin_nanf("");
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // before the wave's next token writes it
}

// A workgroup takes one expert and four tokens: its waves share hidden, f32
// throughout. Workgroups also write their share of x's bf16 terms. A launch and a
// trip to memory: 64 experts of 2560, one token 2.2 us; 32 of 4096, 64 tokens in f32 7.1.
template <class T, int TERMS>
__global__ __launch_bounds__(256) void moe_logits_kernel(const T *__restrict__ x, const float *__restrict__ router,
                                                         int tokens, int experts, int d, int kbd,
                                                         MoePlan plan) {
    __shared__ float part[4][kRouteTokens];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int dp = kbd * 128, e = blockIdx.x, first = blockIdx.y * kRouteTokens;
    const int mine = min(kRouteTokens, tokens - first);
    const float *r = router + (size_t)e * dp;
    float acc[kRouteTokens] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
    for (int k0 = threadIdx.x * 8; k0 < d; k0 += 2048) {
        const float4_t r0 = *(const float4_t *)(r + k0), r1 = *(const float4_t *)(r + k0 + 4);
#pragma unroll
        for (int i = 0; i < kRouteTokens; i++) {
            if (i >= mine) break;
            float v[8];
            fp8_load8(x + (size_t)(first + i) * d, k0, d, v);
#pragma unroll
            for (int c = 0; c < 4; c++) {
                acc[i] = __builtin_fmaf(r0[c], v[c], acc[i]);
                acc[i] = __builtin_fmaf(r1[c], v[4 + c], acc[i]);
            }
        }
    }
    for (int i = 0; i < mine; i++) {
        const float l = wave_sum_dpp(acc[i]);
        if (lane == 0) part[wave][i] = l;
    }
    __syncthreads();
    if (threadIdx.x < mine)
        plan.logits[(size_t)(first + threadIdx.x) * experts + e] =
            (part[0][threadIdx.x] + part[1][threadIdx.x]) + (part[2][threadIdx.x] + part[3][threadIdx.x]);
    if (!plan.x) return;
    const int units = dp / 8 * mine;
    for (int u = blockIdx.x * 256 + threadIdx.x; u < units; u += gridDim.x * 256) {
        const int i = u / (dp / 8), k0 = u % (dp / 8) * 8;
        float v[8];
        fp8_load8(x + (size_t)(first + i) * d, k0, d, v);
        bf16x8_t out[TERMS];
#pragma unroll
        for (int c = 0; c < 8; c++) {
            bf16_t t[TERMS];
            moe_split<TERMS>(v[c], t);
#pragma unroll
            for (int s = 0; s < TERMS; s++) out[s][c] = t[s];
        }
#pragma unroll
        for (int s = 0; s < TERMS; s++) *(bf16x8_t *)(plan.x + ((size_t)s * tokens + first + i) * dp + k0) = out[s];
    }
}

// One wave per token; a chain of dependent steps, 4.6 us for 64 tokens and 32 experts.
__global__ __launch_bounds__(64) void moe_top_kernel(const float *__restrict__ logits, int experts, int top,
                                                     int renormalize, int *__restrict__ ids,
                                                     float *__restrict__ shares) {
    __shared__ __align__(16) MoeTopShared shared;
    int e;
    float c;
    moe_top_any(logits + (size_t)blockIdx.x * experts, experts, top, renormalize, shared, e, c);
    if ((int)threadIdx.x < top) {
        ids[blockIdx.x * top + threadIdx.x] = e;
        shares[blockIdx.x * top + threadIdx.x] = c;
    }
}

// Eight codes (two words) as bf16, exactly.
__device__ __forceinline__ bf16x8_t moe_to_bf16(uint32_t lo, uint32_t hi) {
    const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
struct MoeWide {
    bf16x8_t h[4];
};
__device__ __forceinline__ MoeWide moe_widen(uint4_t lo, uint4_t hi) {
    return {{moe_to_bf16(lo[0], lo[1]), moe_to_bf16(lo[2], lo[3]), moe_to_bf16(hi[0], hi[1]),
             moe_to_bf16(hi[2], hi[3])}};
}

// The operands of one row's 128-block at p (this lane's 16 g already added): 8 values each.
__device__ __forceinline__ MoeWide moe_rows(const bf16_t *p, bool live) {
    MoeWide v;
#pragma unroll
    for (int s = 0; s < 4; s++) {
        v.h[s] = bf16x8_t{};
        if (live) v.h[s] = *(const bf16x8_t *)(p + s / 2 * 64 + s % 2 * 8);
    }
    return v;
}

__device__ __forceinline__ float4_t moe_dot(const MoeWide &w, const MoeWide &x, float4_t d) {
#pragma unroll
    for (int s = 0; s < 4; s++) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.h[s], x.h[s], d, 0, 0, 0);
    return d;
}

constexpr int kGateWaves = 8;

// Where a wave keeps columns 4 p .. 4 p + 3 of row r of a 16-column tile in LDS:
// the pieces of four rows change places, so that 16 rows' vectors meet distinct
// banks (13 tokens, 3 of 24 experts of 1000x700: a layer 26.8 us without, 26.3 with).
__device__ __forceinline__ int moe_part_at(int r, int p) { return r * 16 + (p ^ (r >> 2 & 3)) * 4; }

// One workgroup: tiles of 16 columns of ff (blockIdx.x, + gridDim.x, ...) of one
// chosen expert, gate and up, for its rows (16 at most). The waves share hidden
// (block b on wave b % 8); their partials are added in wave order. Codes are
// loaded a block ahead, across tiles too. Columns past ff, up to a whole 128-block, are written as
// zero. With fewer slots than experts blockIdx.y is the first slot that chose an
// expert, else the expert. One token, 8 of 64 experts of 2560x1024 in bf16: 11.4 us for
// 42 MB, 3.7 TB/s, some 4 us of it the launch, the choice and the sum over the waves;
// 8 tokens, 2 of 16 of 1024x512 6.8 us, nearly all of it those.
template <int XT, int HT>
__global__ __launch_bounds__(kGateWaves * 64) void moe_gate_up_kernel(
    const uint8_t *__restrict__ codes, const float *__restrict__ gs, const float *__restrict__ us, int tokens,
    int experts, int top, int renormalize, int ff, int kbd, int kbf, MoePlan plan) {
    __shared__ __align__(16) float part[kGateWaves][2][256];
    __shared__ __align__(16) MoeTopShared s_top[kGateWaves];
    __shared__ int s_ids[kFewTokens * kMostTop], s_slot[kFewTokens];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int g = lane / 16, j = lane % 16, tiles = (ff + 15) / 16, slots = tokens * top;
    const bool writes = blockIdx.x == 0 && blockIdx.y == 0;
    for (int i = wave; i < tokens; i += kGateWaves) {
        int e;
        float c;
        moe_top_any(plan.logits + (size_t)i * experts, experts, top, renormalize, s_top[wave], e, c);
        if (lane < top) {
            s_ids[i * top + lane] = e;
            if (writes) plan.ids[i * top + lane] = e, plan.shares[i * top + lane] = c;
        }
    }
    __syncthreads();
    const bool by_slot = slots <= experts;
    const int expert = __builtin_amdgcn_readfirstlane(by_slot ? s_ids[blockIdx.y] : (int)blockIdx.y);
    int rows = 0;
    for (int s0 = 0; s0 < slots; s0 += 64) {
        const int s = s0 + lane;
        const bool hit = s < slots && s_ids[s] == expert;
        const unsigned long long hits = __ballot(hit);
        if (by_slot && hits && rows == 0 && s0 + __ffsll(hits) - 1 != (int)blockIdx.y) return;  // an earlier slot has it
        if (hit) s_slot[rows + __popcll(hits & ((1ull << lane) - 1))] = s;  // every wave writes the same
        rows += __popcll(hits);
    }
    if (rows == 0) return;
    __syncthreads();
    const size_t hp = (size_t)kbf * 128;
    const uint8_t *w = codes + (size_t)expert * tiles * kbd * 4096 + lane * 16;
    const size_t srow = (size_t)expert * ((ff + 127) / 128) * kbd;
    // x is loaded ahead too where it is one term; two or three terms wait for
    // the L2 instead of taking the registers of other waves
    constexpr bool kAhead = XT == 1;
    const bool live = j < rows;
    const bf16_t *xr = plan.x + (size_t)(live ? s_slot[j] / top : 0) * kbd * 128 + 16 * g;
    struct Block {
        uint4_t w[2][2];
        float s[2];
        MoeWide x[kAhead ? XT : 1];
    };
    auto x_of = [&](int kb, int i) {
        return moe_rows(xr + (size_t)i * tokens * kbd * 128 + kb * 128, live);
    };
    auto load = [&](int t, int kb, Block &b) {
        const uint8_t *p = w + ((size_t)t * kbd + kb) * 4096;
#pragma unroll
        for (int o = 0; o < 2; o++)
#pragma unroll
            for (int h = 0; h < 2; h++)
                b.w[o][h] = __builtin_nontemporal_load((const uint4_t *)(p + o * 2048 + h * 1024));
        b.s[0] = gs[srow + (size_t)(t / 8) * kbd + kb];
        b.s[1] = us[srow + (size_t)(t / 8) * kbd + kb];
        if constexpr (kAhead) b.x[0] = x_of(kb, 0);
    };
    float4_t acc[2];
    auto step = [&](int t, int kb, Block &now, Block &next) {
        MoeWide x[XT];
        if constexpr (kAhead) {
            x[0] = now.x[0];
        } else {
#pragma unroll
            for (int i = 0; i < XT; i++) x[i] = x_of(kb, i);
        }
        if (kb + kGateWaves < kbd) load(t, kb + kGateWaves, next);
        else if (t + (int)gridDim.x < tiles) load(t + gridDim.x, wave, next);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int o = 0; o < 2; o++) {
            const MoeWide m = moe_widen(now.w[o][0], now.w[o][1]);
            float4_t d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < XT; i++) d = moe_dot(m, x[i], d);
#pragma unroll
            for (int e = 0; e < 4; e++) acc[o][e] = __builtin_fmaf(d[e], now.s[o], acc[o][e]);
        }
    };
    Block b[2];
    if (wave < kbd && (int)blockIdx.x < tiles) load(blockIdx.x, wave, b[0]);
    for (int t = blockIdx.x; t < kbf * 8; t += gridDim.x) {
        acc[0] = acc[1] = float4_t{0.f, 0.f, 0.f, 0.f};
        if (wave < kbd && t < tiles) {
            for (int kb = wave; kb < kbd; kb += 2 * kGateWaves) {
                step(t, kb, b[0], b[1]);
                if (kb + kGateWaves < kbd) step(t, kb + kGateWaves, b[1], b[0]);
                else b[0] = b[1];  // the next tile's first block
            }
        }
        __syncthreads();
        *(float4_t *)&part[wave][0][moe_part_at(j, g)] = acc[0];
        *(float4_t *)&part[wave][1][moe_part_at(j, g)] = acc[1];
        __syncthreads();
        const int i = threadIdx.x, r = i / 16;
        if (i < 256 && r < rows) {
            const int at = moe_part_at(r, i / 4 % 4) + i % 4;
            float gate = part[0][0][at], up = part[0][1][at];
#pragma unroll
            for (int v = 1; v < kGateWaves; v++) gate += part[v][0][at], up += part[v][1][at];
            bf16_t out[HT];
            moe_split<HT>(t < tiles ? gate / (1.0f + expf(-gate)) * up : 0.0f, out);
#pragma unroll
            for (int s = 0; s < HT; s++) plan.h[((size_t)s * slots + s_slot[r]) * hp + t * 16 + i % 16] = out[s];
        }
    }
}

// One workgroup: 16 columns of y, for fewer than kFewSlots slots. Units (chosen
// expert, 128-block of ff) in order, an equal run of them to each wave; a wave
// adds its rows, times their shares, into its own copy of the 16 columns in LDS,
// and the copies are added in wave order. Every wave first sorts the slots by
// expert for itself, comparing each with all: no barrier, and one trip to memory. One
// token, 8 experts of 2560x1024: 8.6 us for 21 MB (2.4 TB/s): 160 workgroups, the
// slots, h and the codes one after another.
template <int HT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void moe_down_kernel(const uint8_t *__restrict__ codes,
                                                              const float *__restrict__ ds, int tokens, int top, int d,
                                                              int kbf, MoePlan plan, void *__restrict__ y, int dtype) {
    constexpr int THREADS = WAVES * 64, kStage = 16 * HT * 256;  // one unit of 16 rows
    static_assert(kFewTokens <= 16 && kFewSlots <= 16, "an expert's rows fit a tile");
    __shared__ __align__(16) uint8_t lds[WAVES * kStage];
    __shared__ __align__(16) float sums[WAVES * kFewTokens * 16];  // [waves][tokens][16]
    __shared__ __align__(16) int s_ids[WAVES][16];
    __shared__ int s_slot[WAVES][16], s_first[WAVES][16], s_expert[WAVES][16];  // slots by expert; per expert
    __shared__ float s_share[WAVES][16];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int g = lane / 16, j = lane % 16, t = blockIdx.x, tiles = (d + 15) / 16, slots = tokens * top;
    const size_t hp = (size_t)kbf * 128;
    float *mine = sums + (size_t)wave * tokens * 16;
    const int my_expert = lane < slots ? plan.ids[lane] : kMostExperts;
    const float my_share = lane < slots ? plan.shares[lane] : 0.0f;
    for (int i = lane; i < tokens * 4; i += 64) ((float4_t *)mine)[i] = float4_t{0.f, 0.f, 0.f, 0.f};
    if (lane < 16) s_ids[wave][lane] = my_expert;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    int ids[16], rank = 0, before = 0, rows_of = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        ids[i] = s_ids[wave][i];
        rank += ids[i] < my_expert || (ids[i] == my_expert && i < lane);
        before += ids[i] == my_expert && i < lane;
        rows_of += ids[i] == my_expert;
    }
    const bool leads = lane < slots && before == 0;  // its expert's first slot
    const unsigned long long leaders = __ballot(leads);
    int group = 0;
#pragma unroll
    for (int i = 0; i < 16; i++) group += (leaders >> i & 1) && ids[i] < my_expert;
    if (lane < slots) {
        s_slot[wave][rank] = lane;
        s_share[wave][rank] = my_share;
    }
    if (leads) {
        s_first[wave][group] = rank << 8 | rows_of;
        s_expert[wave][group] = my_expert;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int units = __popcll(leaders) * kbf;
    const int u0 = (int)((int64_t)units * wave / WAVES), u1 = (int)((int64_t)units * (wave + 1) / WAVES);
    // A run of units of one expert at a time. h of a batch of units goes through
    // this wave's part of LDS: whole rows of it, loaded without registers and all
    // at once, while the operands in memory order would leave most lanes of a load
    // idle where an expert has a row or two. Codes of up to four units together.
    uint8_t *stage = lds + wave * kStage;
    const uint32_t stage0 = __builtin_amdgcn_readfirstlane(lds_address(stage));
    const int32x4_t rh = buffer_rsrc(plan.h, (uint32_t)((size_t)HT * slots * hp * 2));
    for (int u = u0; u < u1;) {
        const int a = u / kbf, k0 = u - a * kbf, k1 = min(kbf, k0 + u1 - u);
        u += k1 - k0;
        const int expert = __builtin_amdgcn_readfirstlane(s_expert[wave][a]);
        const int group = __builtin_amdgcn_readfirstlane(s_first[wave][a]), first = group >> 8, rows = group & 255;
        const uint8_t *w = codes + ((size_t)expert * tiles + t) * kbf * 2048 + lane * 16;
        const float *sw = ds + ((size_t)expert * ((d + 127) / 128) + t / 8) * kbf;
        // the batch: the most units, a power of two, whose rows fit the stage
        int log_nb = 0;
        while (log_nb < 4 && (rows * HT * 256 << (log_nb + 1)) <= kStage && (1 << log_nb) < k1 - k0) log_nb++;
        const int nb = 1 << log_nb, pieces = rows * HT << (log_nb + 4);
        float4_t acc = {0.f, 0.f, 0.f, 0.f};
        for (int kb0 = k0; kb0 < k1; kb0 += nb) {
            // piece p: row and term p / (16 nb), 16 bytes p % (16 nb) of the batch's columns
            for (int p0 = 0; p0 < pieces; p0 += 64) {
                const int p = p0 + lane, rt = p >> (log_nb + 4), r = rt / HT, i = rt - r * HT;
                const uint32_t at = p < pieces
                                        ? (uint32_t)(((size_t)i * slots + s_slot[wave][first + r]) * hp * 2 + kb0 * 256 +
                                                     (p & ((16 << log_nb) - 1)) * 16)
                                        : 0x80000000u;
                dma16_at(stage0 + p0 * 16, at, rh, 0u);
            }
            const int kend = min(k1, kb0 + nb);
            for (int k = kb0; k < kend; k += 4) {
                uint4_t wb[4][2];
                float s[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int kb = min(k + i, kend - 1);
                    wb[i][0] = __builtin_nontemporal_load((const uint4_t *)(w + (size_t)kb * 2048));
                    wb[i][1] = __builtin_nontemporal_load((const uint4_t *)(w + (size_t)kb * 2048 + 1024));
                    s[i] = sw[kb];
                }
                if (k == kb0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    if (k + i >= kend) break;
                    const MoeWide m = moe_widen(wb[i][0], wb[i][1]);
                    float4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int o = 0; o < HT; o++) {
                        const uint8_t *at = stage + (((j * HT + o) << log_nb) + k + i - kb0) * 256 + 32 * g;
                        MoeWide x;
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            x.h[q] = bf16x8_t{};
                            if (j < rows) x.h[q] = *(const bf16x8_t *)(at + q / 2 * 128 + q % 2 * 16);
                        }
                        v = moe_dot(m, x, v);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[e] = __builtin_fmaf(v[e], s[i], acc[e]);
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the next batch lands
        }
        if (j < rows) {  // the run's rows into this wave's sums
            float4_t *at = (float4_t *)(mine + s_slot[wave][first + j] / top * 16 + 4 * g);
            const float share = s_share[wave][first + j];
            float4_t v = *at;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = __builtin_fmaf(acc[e], share, v[e]);
            *at = v;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * 16; i += THREADS) {
        const int col = t * 16 + i % 16;
        if (col >= d) continue;
        float v = sums[i];
        for (int w = 1; w < WAVES; w++) v += sums[(size_t)w * tokens * 16 + i];
        fp8_store(y, dtype, (size_t)(i / 16) * d + col, v);
    }
}

// ---- more tokens ------------------------------------------------------------------

// The rows of an expert against its weight where tokens are many enough that
// most experts have several rows: eight waves side by side, two 16-column tiles
// each (GATE: gate and up of one tile of ff, and h = silu(gate) * up; else two
// tiles of the output, f32 rows by slot that moe_combine_kernel sums). A step is
// a 128-block of the width: a wave's own 4 KiB of codes and the block's rows,
// which all waves share, through NS LDS stages by buffer_load ... lds. Loaded by
// each wave for itself instead, the rows cost more than the weight (x of eight
// rows in f32 is three times a tile's codes). A row's 256 bytes of a term are 16
// pieces, piece p of row r in slot p ^ (r & 15), so that 16 rows' reads meet
// distinct banks. 16 MC rows at a time; more read the weight again. Bound by the
// codes' bytes: 64 tokens, 4 of 32 experts of 4096x1536 in f32 89 us for gate and up
// (403 MB, 4.5 TB/s) and 43 for down (201 MB, 4.6 TB/s).
template <int MC, int XT, int HT, bool GATE, int NS>
__global__ __launch_bounds__(512) void moe_wide_kernel(const uint8_t *__restrict__ codes,
                                                       const float *__restrict__ s0, const float *__restrict__ s1,
                                                       int tokens, int experts, int top, int n, int kbs, int out_width,
                                                       const bf16_t *__restrict__ in, MoePlan plan) {
    constexpr int WAVES = 8, RT = XT * 16 * MC, LOADS = RT / 4, XPW = (LOADS + WAVES - 1) / WAVES, PB = 4 + XPW;
    constexpr int XB = WAVES * 4096, STAGE = XB + RT * 256;
    static_assert((NS - 2) * PB <= 63, "vmcnt range");
    __shared__ __align__(16) uint8_t lds[NS * STAGE];
    __shared__ int s_slot[DZ_MOE_MAX_TOKENS];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int g = lane / 16, j = lane % 16, slots = tokens * top, tiles = (n + 15) / 16;
    const bool by_slot = slots <= experts;
    const int expert = __builtin_amdgcn_readfirstlane(by_slot ? plan.ids[blockIdx.y] : (int)blockIdx.y);
    int rows = 0;
    for (int b = 0; b < slots; b += 64) {
        const int s = b + lane;
        const bool hit = s < slots && plan.ids[s] == expert;
        const unsigned long long hits = __ballot(hit);
        if (by_slot && hits && rows == 0 && b + __ffsll(hits) - 1 != (int)blockIdx.y) return;  // an earlier slot has it
        if (hit) s_slot[rows + __popcll(hits & ((1ull << lane) - 1))] = s;  // every wave writes the same
        rows += __popcll(hits);
    }
    if (rows == 0) return;
    __syncthreads();

    // this wave's tiles: one of gate and up, or two; past the last one zeros are loaded
    const int t0 = GATE ? blockIdx.x * WAVES + wave : (blockIdx.x * WAVES + wave) * 2;
    const size_t matrix = (size_t)tiles * kbs * (GATE ? 4096 : 2048);
    const uint8_t *wbase = codes + (size_t)expert * matrix + (size_t)t0 * kbs * (GATE ? 4096 : 2048);
    const int have = max(0, min(GATE ? 1 : 2, tiles - t0));
    const int32x4_t rw = buffer_rsrc(have ? wbase : codes, (uint32_t)have * kbs * (GATE ? 4096u : 2048u));
    uint32_t woff[4];
#pragma unroll
    for (int p = 0; p < 4; p++)
        woff[p] = GATE ? (uint32_t)(p * 1024 + lane * 16) : (uint32_t)(p / 2 * kbs * 2048 + p % 2 * 1024 + lane * 16);
    const int blocks = (n + 127) / 128;
    const float *sw[2];
#pragma unroll
    for (int o = 0; o < 2; o++)
        sw[o] = (GATE && o ? s1 : s0) + ((size_t)expert * blocks + min((GATE ? t0 : t0 + o) / 8, blocks - 1)) * kbs;
    const int in_rows = GATE ? tokens : slots, width = kbs * 128;
    const int32x4_t rx = buffer_rsrc(in, (uint32_t)((size_t)XT * in_rows * width * 2));
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(lds));

    for (int r0 = 0; r0 < rows; r0 += 16 * MC) {
        const int chunks = min(MC, (rows - r0 + 15) / 16);
        // load p of this wave: four (term, row)s, 16 lanes each
        uint32_t xoff[XPW];
        int xload[XPW];
#pragma unroll
        for (int p = 0; p < XPW; p++) {
            xload[p] = (wave * XPW + p) % LOADS;
            const int rt = xload[p] * 4 + lane / 16, i = rt / (16 * MC), r = rt % (16 * MC);
            const int from = r0 + r < rows ? (GATE ? s_slot[r0 + r] / top : s_slot[r0 + r]) : -1;
            xoff[p] = from < 0 ? 0x80000000u
                               : (uint32_t)(((size_t)i * in_rows + from) * width * 2 + ((lane % 16) ^ (r & 15)) * 16);
        }
        // past the last block nothing is loaded (every offset out of range), so that all waits go by count
        auto load_stage = [&](int stage, int kb) {
            const bool live = kb < kbs;
            const uint32_t at = lds0 + stage * STAGE, past = live ? 0u : 0x80000000u;
#pragma unroll
            for (int p = 0; p < XPW; p++)
                dma16_at(at + XB + xload[p] * 1024, xoff[p] | past, rx, live ? (uint32_t)kb * 256 : 0u);
#pragma unroll
            for (int p = 0; p < 4; p++)
                dma16_at(at + wave * 4096 + p * 1024, woff[p] | past, rw,
                         live && have ? (uint32_t)kb * (GATE ? 4096u : 2048u) : 0u);
        };
        float4_t acc[MC][2];
#pragma unroll
        for (int c = 0; c < MC; c++) acc[c][0] = acc[c][1] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int p = 0; p < NS - 1; p++) load_stage(p, p);
        float sc[2] = {sw[0][0], sw[1][0]};
        int stage = 0;
        for (int kb = 0; kb < kbs; kb++) {
            // lgkmcnt: this wave's reads of the stage that the next loads overwrite are done too
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NS - 2) * PB) : "memory");
            load_stage(stage == 0 ? NS - 1 : stage - 1, kb + NS - 1);  // the stage that the step before read
            const int after = min(kb + 1, kbs - 1);
            const float next[2] = {sw[0][after], sw[1][after]};
            const uint8_t *st = lds + stage * STAGE, *ws = st + wave * 4096 + lane * 16;
            MoeWide m[2];
#pragma unroll
            for (int o = 0; o < 2; o++)
                m[o] = moe_widen(*(const uint4_t *)(ws + o * 2048), *(const uint4_t *)(ws + o * 2048 + 1024));
#pragma unroll
            for (int c = 0; c < MC; c++) {
                if (c >= chunks) break;
                float4_t d[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int i = 0; i < XT; i++) {
                    const uint8_t *row = st + XB + ((i * MC + c) * 16 + j) * 256;
                    MoeWide x;
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        x.h[q] = *(const bf16x8_t *)(row + ((q / 2 * 8 + 2 * g + q % 2) ^ j) * 16);
                    d[0] = moe_dot(m[0], x, d[0]);
                    d[1] = moe_dot(m[1], x, d[1]);
                }
#pragma unroll
                for (int o = 0; o < 2; o++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[c][o][e] = __builtin_fmaf(d[o][e], sc[o], acc[c][o][e]);
            }
            sc[0] = next[0];
            sc[1] = next[1];
            stage = stage + 1 == NS ? 0 : stage + 1;
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");  // no LDS write in flight, every stage read
#pragma unroll
        for (int c = 0; c < MC; c++) {
            const int r = r0 + 16 * c + j;
            if (r >= rows) break;
            const size_t slot = s_slot[r];
            if constexpr (GATE) {
                bf16_t out[4][HT];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float gate = acc[c][0][e];
                    moe_split<HT>(gate / (1.0f + expf(-gate)) * acc[c][1][e], out[e]);
                }
#pragma unroll
                for (int i = 0; i < HT; i++) {
                    const bf16x2_t lo = {out[0][i], out[1][i]}, hi = {out[2][i], out[3][i]};
                    *(uint2_t *)(plan.h + ((size_t)i * slots + slot) * out_width + t0 * 16 + 4 * g) =
                        uint2_t{__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi)};
                }
            } else {
#pragma unroll
                for (int o = 0; o < 2; o++)
                    if (o < have) *(float4_t *)(plan.p + slot * out_width + (t0 + o) * 16 + 4 * g) = acc[c][o];
            }
        }
    }
}

// y of a token: its slots' rows times their shares, in order, four loaded together
// (2.1 us, a launch's time; 64 tokens of 4 x 4096 4.4).
__global__ __launch_bounds__(64) void moe_combine_kernel(MoePlan plan, int top, int d, int width, void *__restrict__ y,
                                                         int dtype) {
    const int t = blockIdx.y, c = (blockIdx.x * 64 + threadIdx.x) * 4;
    if (c >= d) return;
    const float *p = plan.p + (size_t)t * top * width + c, *shares = plan.shares + t * top;
    float4_t v = {0.f, 0.f, 0.f, 0.f};
    for (int i0 = 0; i0 < top; i0 += 4) {
        float4_t row[4];
        float share[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int at = min(i0 + i, top - 1);
            row[i] = *(const float4_t *)(p + (size_t)at * width);
            share[i] = shares[at];
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i0 + i < top)
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = __builtin_fmaf(row[i][e], share[i], v[e]);
    }
    fp8_store4(y, dtype, (size_t)t * d + c, v, d - c);
}

template <class T>
__global__ __launch_bounds__(256) void moe_router_kernel(const T *__restrict__ src, int experts, int d, int dp,
                                                         float *__restrict__ dst, int *bad) {
    for (size_t id = blockIdx.x * (size_t)256 + threadIdx.x; id < (size_t)experts * dp; id += gridDim.x * (size_t)256) {
        const int e = (int)(id / dp), k = (int)(id % dp);
        const float v = k < d ? (float)src[(size_t)e * d + k] : 0.0f;
        if (!(fabsf(v) <= 3.4028235e38f)) atomicOr(bad, 1);
        dst[id] = v;
    }
}

size_t aligned(size_t n) { return (n + 255) / 256 * 256; }

int terms_of_x(int dtype) { return dtype == DZ_BF16 ? 1 : dtype == DZ_F16 ? 2 : 3; }
int terms_of_h(int dtype) { return dtype == DZ_F32 ? 3 : 2; }

bool moe_wide_gate(const dz_moe *e, int tokens, int x_terms) {
    const size_t grid = (size_t)e->kbf * std::min(tokens * e->cfg.top_k, e->cfg.experts);
    return tokens > kFewTokens || (x_terms == 3 && grid >= 2 * (size_t)device_cus());
}
bool moe_wide_down(const dz_moe *e, int tokens) { return tokens * e->cfg.top_k >= kFewSlots; }

// The workspace of a call: its size, and with `work` the plan's pointers into it.
size_t moe_plan(const dz_moe *e, size_t tokens, int dtype, bool forward, uint8_t *work, MoePlan *plan) {
    const size_t rows = tokens * e->cfg.top_k;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t p = at;
        at += aligned(bytes);
        return work ? work + p : nullptr;
    };
    MoePlan p{};
    p.logits = (float *)take(tokens * e->cfg.experts * sizeof(float));
    if (forward) {
        p.ids = (int *)take(rows * sizeof(int));
        p.shares = (float *)take(rows * sizeof(float));
        p.x = (bf16_t *)take(tokens * terms_of_x(dtype) * e->kbd * 256);
        p.h = (bf16_t *)take(rows * terms_of_h(dtype) * e->kbf * 256);
        if (moe_wide_down(e, (int)tokens)) p.p = (float *)take(rows * e->kbd * 512);
    }
    if (plan) *plan = p;
    return at;
}

void launch_logits(const dz_moe *e, const void *x, int dtype, int tokens, const MoePlan &plan, hipStream_t s) {
    const dz_moe_config &c = e->cfg;
    const dim3 grid(c.experts, cdiv(tokens, kRouteTokens));
    if (dtype == DZ_F32)
        hipLaunchKernelGGL((moe_logits_kernel<float, 3>), grid, dim3(256), 0, s, (const float *)x, e->router, tokens,
                           c.experts, c.hidden, e->kbd, plan);
    else if (dtype == DZ_F16)
        hipLaunchKernelGGL((moe_logits_kernel<half_t, 2>), grid, dim3(256), 0, s, (const half_t *)x, e->router, tokens,
                           c.experts, c.hidden, e->kbd, plan);
    else
        hipLaunchKernelGGL((moe_logits_kernel<bf16_t, 1>), grid, dim3(256), 0, s, (const bf16_t *)x, e->router, tokens,
                           c.experts, c.hidden, e->kbd, plan);
}

void launch_top(const dz_moe *e, int tokens, const MoePlan &plan, int *ids, float *shares, hipStream_t s) {
    hipLaunchKernelGGL(moe_top_kernel, dim3(tokens), dim3(64), 0, s, plan.logits, e->cfg.experts, e->cfg.top_k,
                       e->cfg.renormalize, ids, shares);
}

template <int MC, int XT, int HT, int NS>
void launch_wide_gate(const dz_moe *e, int tokens, const MoePlan &plan, hipStream_t s) {
    const dz_moe_config &c = e->cfg;
    hipLaunchKernelGGL((moe_wide_kernel<MC, XT, HT, true, NS>), dim3(e->kbf, std::min(tokens * c.top_k, c.experts)),
                       dim3(512), 0, s, e->gate_up, e->gate_scales, e->up_scales, tokens, c.experts, c.top_k, c.ff,
                       e->kbd, e->kbf * 128, plan.x, plan);
}

template <int MC, int HT, int NS>
void launch_wide_down(const dz_moe *e, int dtype, int tokens, const MoePlan &plan, void *y, hipStream_t s) {
    const dz_moe_config &c = e->cfg;
    const int width = e->kbd * 128;
    hipLaunchKernelGGL((moe_wide_kernel<MC, HT, HT, false, NS>),
                       dim3(cdiv(c.hidden, 256), std::min(tokens * c.top_k, c.experts)), dim3(512), 0, s, e->down,
                       e->down_scales, nullptr, tokens, c.experts, c.top_k, c.hidden, e->kbf, width, plan.h, plan);
    hipLaunchKernelGGL(moe_combine_kernel, dim3(cdiv(c.hidden, 256), tokens), dim3(64), 0, s, plan, c.top_k, c.hidden,
                       width, y, dtype);
}

// Which kernels. Measured (us; few / wide, the choice's and the sum's kernels not counted):
//  gate and up, 8 of 64 experts of 2560x1024 in bf16: 1 token 11.6 / 16.4, 4 28.4 /
//    27.1, 16 56 / 53; 2 of 16 of 1024x512 in f16, 8 tokens 7.6 / 10.2; 8 of 128 of
//    2048x768 in f32, 16 tokens 90 / 61: the wide kernel past 16 tokens, where it
//    needs a launch for the choice anyway, and for f32 on grids of two workgroups a
//    compute unit, since few's waves load three terms of x for themselves;
//  down: the same, 1 token 9.4 / 8.8 + 2.5 for the sum, 8 tokens 9.9 / 6.0 + 2.5,
//    3 of 24 of 1000x700 in bf16, 13 tokens 18.4 / 7.8 + 2.5: the wide kernel from 16 slots on.
//  32 rows of an expert at a time (MC = 2) where experts have more than 12 on average,
//    since past 16 rows the 16-row form reads their weight again (us a layer, 16 / 32
//    rows at a time): 4 of 32 of 4096x1536, 8 rows on average bf16 135.6 / 137.0, f32
//    145.2 / 159.3; 12 rows 169.4 / 144.0, 187.0 / 166.9; 16 rows 189.7 / 149.1, 208.4 /
//    169.5. 2 of 8 of the same, 10 rows 52.3 / 51.6, f32 62.3 / 71.5; 14 rows 76.0 / 58.5,
//    103.4 / 76.7; 32 rows 110.4 / 87.9, 150.2 / 119.4. Below the line the larger stages
//    leave fewer of them (f32 keeps two of three), above it a reading is saved.
// Stages of the wide kernel are 32 KiB of codes and 4 KiB a term of the rows,
// twice that for 32 rows at a time: as many as fit a compute unit's 160 KiB.
template <int XT, int HT>
void launch_experts(const dz_moe *e, int dtype, int tokens, const MoePlan &plan, void *y, hipStream_t s) {
    const dz_moe_config &c = e->cfg;
    const int slots = tokens * c.top_k, entries = std::min(slots, c.experts);
    const unsigned tiles = e->kbf * 8, cus = (unsigned)device_cus();
    const bool many = slots > 12 * c.experts;  // rows an expert, on average
    if (moe_wide_gate(e, tokens, XT)) {
        launch_top(e, tokens, plan, plan.ids, plan.shares, s);
        if (many) launch_wide_gate<2, XT, HT, XT == 3 ? 2 : 3>(e, tokens, plan, s);
        else launch_wide_gate<1, XT, HT, XT == 1 ? 4 : 3>(e, tokens, plan, s);
    } else {
        // two workgroups a compute unit fit; each goes through its share of the tiles
        const unsigned share = std::max(1u, 2u * cus / entries);
        hipLaunchKernelGGL((moe_gate_up_kernel<XT, HT>), dim3(std::min(tiles, share), entries), dim3(kGateWaves * 64),
                           0, s, e->gate_up, e->gate_scales, e->up_scales, tokens, c.experts, c.top_k, c.renormalize,
                           c.ff, e->kbd, e->kbf, plan);
    }
    if (moe_wide_down(e, tokens)) {
        if (many) launch_wide_down<2, HT, HT == 3 ? 2 : 3>(e, dtype, tokens, plan, y, s);
        else launch_wide_down<1, HT, 3>(e, dtype, tokens, plan, y, s);
    } else {
        constexpr int WAVES = HT == 3 ? 8 : 16;  // a unit's rows of each wave fit LDS
        hipLaunchKernelGGL((moe_down_kernel<HT, WAVES>), dim3(cdiv(c.hidden, 16)), dim3(WAVES * 64), 0, s, e->down,
                           e->down_scales, tokens, c.top_k, c.hidden, e->kbf, plan, y, dtype);
    }
}

void moe_release(dz_moe *e) {
    if (!e) return;
    hipFree(e->memory);
    delete e;
}

bool moe_dtype(int32_t d) { return d == DZ_F32 || d == DZ_F16 || d == DZ_BF16; }

int32_t moe_call_ok(dz_ctx *ctx, const dz_moe *e, const void *x, int32_t dtype, size_t tokens, const void *out) {
    if (!e || (tokens && (!x || !out))) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    if (e->device != ctx_device(ctx)) return ctx_fail(ctx, DZ_INVALID_REQUEST, "the layer lives on another device");
    if (!moe_dtype(dtype)) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "unknown dtype");
    if (tokens > DZ_MOE_MAX_TOKENS) return ctx_fail(ctx, DZ_INPUT_TOO_LONG, "input budget exceeded");
    return DZ_OK;
}

}  // namespace

int32_t moe_create(dz_ctx *ctx, const dz_moe_config *cfg, const void *router, int32_t router_dtype,
                   const uint8_t *gate, const float *gate_scales, const uint8_t *up, const float *up_scales,
                   const uint8_t *down, const float *down_scales, dz_moe **out) {
    if (!out) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    *out = nullptr;
    if (!cfg || !router || !gate || !gate_scales || !up || !up_scales || !down || !down_scales)
        return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    if (!moe_dtype(router_dtype)) return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "unknown dtype");
    if (cfg->experts < 1 || cfg->experts > kMostExperts || cfg->top_k < 1 || cfg->top_k > kMostTop ||
        cfg->top_k > cfg->experts || cfg->hidden < 1 || cfg->hidden > kMostWidth || cfg->ff < 1 ||
        cfg->ff > kMostWidth || (cfg->renormalize != 0 && cfg->renormalize != 1))
        return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "invalid mixture-of-experts shape");
    dz_moe *e = new (std::nothrow) dz_moe();
    if (!e) return ctx_fail(ctx, DZ_RESOURCE_LIMIT, "layer allocation");
    e->cfg = *cfg;
    e->device = ctx_device(ctx);
    const int E = cfg->experts, d = cfg->hidden, ff = cfg->ff;
    e->kbd = (d + 127) / 128;
    e->kbf = (ff + 127) / 128;
    const size_t ftiles = (ff + 15) / 16, dtiles = (d + 15) / 16, blocks = (size_t)e->kbd * e->kbf;
    // one allocation, each part at a multiple of 256 bytes
    struct {
        void **p;
        size_t bytes;
    } parts[] = {{(void **)&e->gate_up, E * ftiles * e->kbd * 4096},
                 {(void **)&e->down, E * dtiles * e->kbf * 2048},
                 {(void **)&e->gate_scales, E * blocks * sizeof(float)},
                 {(void **)&e->up_scales, E * blocks * sizeof(float)},
                 {(void **)&e->down_scales, E * blocks * sizeof(float)},
                 {(void **)&e->router, (size_t)E * e->kbd * 128 * sizeof(float)}};
    for (auto &part : parts) e->bytes += aligned(part.bytes);
    const hipError_t err = hipMalloc(&e->memory, e->bytes);
    if (err != hipSuccess) {
        delete e;
        return ctx_hip_fail(ctx, err, "layer allocation");
    }
    size_t at = 0;
    for (auto &part : parts) {
        *part.p = e->memory + at;
        at += aligned(part.bytes);
    }
    int *bad = ctx_flag(ctx), value = 0;
    hipStream_t s = ctx_stream(ctx);
    launch_fill_i32(bad, 0, 1, s);
    const size_t gu = ftiles * e->kbd * 4096, dn = dtiles * e->kbf * 2048;
    launch_fp8_retile(gate, E, ff, d, e->gate_up, gu, (size_t)e->kbd * 4096, 4096, bad, s);
    launch_fp8_retile(up, E, ff, d, e->gate_up + 2048, gu, (size_t)e->kbd * 4096, 4096, bad, s);
    launch_fp8_retile(down, E, d, ff, e->down, dn, (size_t)e->kbf * 2048, 2048, bad, s);
    launch_fp8_scales(gate_scales, e->gate_scales, E * blocks, bad, s);
    launch_fp8_scales(up_scales, e->up_scales, E * blocks, bad, s);
    launch_fp8_scales(down_scales, e->down_scales, E * blocks, bad, s);
    const int dp = e->kbd * 128;
    const dim3 grid((unsigned)std::min(((size_t)E * dp + 255) / 256, (size_t)1 << 20));
    if (router_dtype == DZ_F32)
        hipLaunchKernelGGL(moe_router_kernel<float>, grid, dim3(256), 0, s, (const float *)router, E, d, dp, e->router,
                           bad);
    else if (router_dtype == DZ_F16)
        hipLaunchKernelGGL(moe_router_kernel<half_t>, grid, dim3(256), 0, s, (const half_t *)router, E, d, dp, e->router,
                           bad);
    else
        hipLaunchKernelGGL(moe_router_kernel<bf16_t>, grid, dim3(256), 0, s, (const bf16_t *)router, E, d, dp, e->router,
                           bad);
    int32_t rc = ctx_flag_value(ctx, &value);
    if (!rc && value) rc = ctx_fail(ctx, DZ_INVALID_CHECKPOINT, "invalid mixture-of-experts weight");
    if (rc) {
        moe_release(e);
        return rc;
    }
    *out = e;
    return DZ_OK;
}

void moe_free(dz_moe *e) { moe_release(e); }

int32_t moe_info(const dz_moe *e, dz_moe_config *cfg, size_t *device_bytes) {
    if (!e) return DZ_INVALID_REQUEST;
    if (cfg) *cfg = e->cfg;
    if (device_bytes) *device_bytes = e->bytes;
    return DZ_OK;
}

int32_t moe_route(dz_ctx *ctx, const dz_moe *e, const void *x, int32_t dtype, size_t tokens, int32_t *ids,
                  float *shares) {
    if (int32_t rc = moe_call_ok(ctx, e, x, dtype, tokens, ids)) return rc;
    if (tokens && !shares) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    if (tokens == 0) return DZ_OK;
    void *work = nullptr;
    if (int32_t rc = ctx_workspace(ctx, moe_plan(e, tokens, dtype, false, nullptr, nullptr), &work)) return rc;
    MoePlan plan;
    moe_plan(e, tokens, dtype, false, (uint8_t *)work, &plan);
    launch_logits(e, x, dtype, (int)tokens, plan, ctx_stream(ctx));
    launch_top(e, (int)tokens, plan, ids, shares, ctx_stream(ctx));
    return ctx_launched(ctx, "mixture of experts route");
}

int32_t moe_forward(dz_ctx *ctx, const dz_moe *e, const void *x, int32_t dtype, size_t tokens, void *y) {
    if (int32_t rc = moe_call_ok(ctx, e, x, dtype, tokens, y)) return rc;
    if (tokens == 0) return DZ_OK;
    void *work = nullptr;
    if (int32_t rc = ctx_workspace(ctx, moe_plan(e, tokens, dtype, true, nullptr, nullptr), &work)) return rc;
    MoePlan plan;
    moe_plan(e, tokens, dtype, true, (uint8_t *)work, &plan);
    hipStream_t s = ctx_stream(ctx);
    const int t = (int)tokens;
    launch_logits(e, x, dtype, t, plan, s);
    if (dtype == DZ_F32) launch_experts<3, 3>(e, dtype, t, plan, y, s);
    else if (dtype == DZ_F16) launch_experts<2, 2>(e, dtype, t, plan, y, s);
    else launch_experts<1, 2>(e, dtype, t, plan, y, s);
    return ctx_launched(ctx, "mixture of experts");
}

}  // namespace dz
