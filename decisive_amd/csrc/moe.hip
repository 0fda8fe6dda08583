// moe.hip -- a mixture-of-experts layer for a few tokens on 8-bit floating
// point weights (fp8.hpp has their form), activations kept as they come.
//
//   l = x router^T, p = softmax(l), E(x) = the top_k experts of largest l
//   y = sum over e in E(x) of c_e down_e (silu(gate_e x) * up_e x)
//
// c_e is p_e, or p_e / (sum of the chosen p). A few tokens read far more
// weight than they multiply (2 operations a byte and row), so the layer is
// bound by the bytes of the experts that are chosen, each read once:
//   1 moe_route_kernel    logits; its last workgroup picks the experts and lists
//                         each expert's rows (token and share), ordered by expert then token
//   2 moe_gate_up_kernel  per (chosen expert, 16 columns of ff): h = silu(gate) * up of its rows
//   3 moe_down_kernel     per 16 columns of the output: every chosen expert's down
//                         product, times the rows' shares, summed
// The products run on the bf16 matrix unit: e4m3 is exact in bf16, and an
// activation is a sum of bf16 terms: x is one term (bf16), two (f16, exactly)
// or three (f32, exactly); h, which never leaves the layer, is two terms (16
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
    size_t bytes = 0;
};

namespace dz {

int32_t ctx_fail(dz_ctx *ctx, int32_t code, const std::string &msg);
int32_t ctx_hip_fail(dz_ctx *ctx, hipError_t e, const char *what);
hipStream_t ctx_stream(dz_ctx *ctx);
int *ctx_flag(dz_ctx *ctx);
int *ctx_ticket(dz_ctx *ctx);
int ctx_device(dz_ctx *ctx);
int32_t ctx_workspace(dz_ctx *ctx, size_t bytes, void **out);
int32_t ctx_launched(dz_ctx *ctx, const char *what);
int32_t ctx_flag_value(dz_ctx *ctx, int *value);

namespace {

constexpr int kMostExperts = 512, kMostTop = 16, kMostWidth = 65536;
constexpr int kRouteThreads = 512, kRouteTokens = 4;

// What the first kernel leaves for the other two, in the workspace.
struct MoePlan {
    float *logits;     // [tokens][experts]
    int *active;       // [0] how many experts are chosen, then per chosen expert {expert, first row, rows}
    int *token;        // [rows] the row's token
    float *share;      // [rows] c of the row
    bf16_t *x;         // [terms][tokens][128 kbd]
    bf16_t *h;         // [terms][rows][128 kbf]
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

__device__ __forceinline__ uint32_t moe_wave_max(uint32_t v) {
    v = dpp_max_u32<0xB1>(v);
    v = dpp_max_u32<0x4E>(v);
    v = dpp_max_u32<0x124>(v);
    v = dpp_max_u32<0x128>(v);
    for (int o = 16; o < 64; o *= 2) {
        const uint32_t other = (uint32_t)__shfl_xor((int)v, o);
        v = v > other ? v : other;
    }
    return v;
}

// A logit's order as an unsigned number above 0 (0 marks an expert that is taken or absent).
__device__ __forceinline__ uint32_t moe_key(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v == 0.0f ? 0.0f : v);
    return b & 0x80000000u ? (b == 0xffffffffu ? 1u : ~b) : b | 0x80000000u;
}

// A wave takes one expert and four tokens: its router row against theirs, f32
// throughout. Workgroups also write their share of x's bf16 terms. The last
// workgroup to finish (a ticket that it sets back to 0) picks the experts:
// per token a wave finds the largest logit top_k times, equal ones by the lower
// index; lists come from bit masks of tokens per expert, so their order never
// depends on which wave came first.
template <class T, int TERMS>
__global__ __launch_bounds__(kRouteThreads) void moe_route_kernel(
    const T *__restrict__ x, const float *__restrict__ router, int tokens, int experts, int top, int d, int kbd,
    int renormalize, int vec, MoePlan plan, int *ticket, int *ids_out, float *shares_out) {
    constexpr int WAVES = kRouteThreads / 64;
    __shared__ uint32_t mask[kMostExperts][4];
    __shared__ uint32_t scan[kMostExperts];
    __shared__ int last;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int dp = kbd * 128;
    const int e = blockIdx.x * WAVES + wave, first = blockIdx.y * kRouteTokens;
    const int mine = min(kRouteTokens, tokens - first);
    if (e < experts) {
        const float *r = router + (size_t)e * dp;
        float acc[kRouteTokens] = {0.f, 0.f, 0.f, 0.f};
        for (int k0 = lane * 8; k0 < d; k0 += 512) {
            const float4_t r0 = *(const float4_t *)(r + k0), r1 = *(const float4_t *)(r + k0 + 4);
#pragma unroll
            for (int i = 0; i < kRouteTokens; i++) {
                if (i >= mine) break;
                float v[8];
                fp8_load8(x + (size_t)(first + i) * d, k0, d, vec, v);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    acc[i] = __builtin_fmaf(r0[c], v[c], acc[i]);
                    acc[i] = __builtin_fmaf(r1[c], v[4 + c], acc[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kRouteTokens; i++) {
            const float l = wave_sum_dpp(acc[i]);
            if (lane == 0 && i < mine)
                __hip_atomic_store(plan.logits + (size_t)(first + i) * experts + e, l, __ATOMIC_RELAXED,
                                   __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    if (plan.x) {
        const int units = dp / 8 * mine;
        for (int u = blockIdx.x * kRouteThreads + threadIdx.x; u < units; u += gridDim.x * kRouteThreads) {
            const int i = u / (dp / 8), k0 = u % (dp / 8) * 8;
            float v[8];
            fp8_load8(x + (size_t)(first + i) * d, k0, d, vec, v);
            bf16x8_t out[TERMS];
#pragma unroll
            for (int c = 0; c < 8; c++) {
                bf16_t t[TERMS];
                moe_split<TERMS>(v[c], t);
#pragma unroll
                for (int s = 0; s < TERMS; s++) out[s][c] = t[s];
            }
#pragma unroll
            for (int s = 0; s < TERMS; s++)
                *(bf16x8_t *)(plan.x + ((size_t)s * tokens + first + i) * dp + k0) = out[s];
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "agent");
    __syncthreads();
    if (threadIdx.x == 0) {
        const int all = gridDim.x * gridDim.y;
        last = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == all - 1;
        if (last) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    for (int i = threadIdx.x; i < kMostExperts * 4; i += kRouteThreads) (&mask[0][0])[i] = 0;
    __syncthreads();
    if (!last) return;

    // the experts of each token: lane l holds experts per * l .. + per - 1
    const int per = (experts + 63) / 64;
    __shared__ int pick_e[128][kMostTop];
    __shared__ float pick_c[128][kMostTop];
    for (int t = wave; t < tokens; t += WAVES) {
        float l[kMostExperts / 64];
        uint32_t key[kMostExperts / 64];
        bool fine = true;
        float most = -3.4028235e38f;
#pragma unroll
        for (int i = 0; i < kMostExperts / 64; i++) {
            const int ex = lane * per + i;
            const bool here = i < per && ex < experts;
            l[i] = here ? __hip_atomic_load(plan.logits + (size_t)t * experts + ex, __ATOMIC_RELAXED,
                                            __HIP_MEMORY_SCOPE_AGENT)
                        : -3.4028235e38f;
            key[i] = here ? moe_key(l[i]) : 0u;
            if (here && !(fabsf(l[i]) <= 3.4028235e38f)) fine = false;
            most = fmaxf(most, l[i]);
        }
        fine = __all(fine);
        most = wave_max_dpp(most);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < kMostExperts / 64; i++)
            if (i < per && lane * per + i < experts) sum += expf(l[i] - most);
        sum = wave_sum_dpp(sum);
        float picked = 0.0f;
        for (int s = 0; s < top; s++) {
            uint32_t best = 0;
            int at = 0;
#pragma unroll
            for (int i = 0; i < kMostExperts / 64; i++)
                if (key[i] > best) best = key[i], at = i;
            const uint32_t top_key = moe_wave_max(best);
            const int owner = __ffsll((unsigned long long)__ballot(best == top_key)) - 1;
            float p = 0.0f;
            if (lane == owner) {
#pragma unroll
                for (int i = 0; i < kMostExperts / 64; i++)
                    if (i == at) {
                        p = expf(l[i] - most);
                        key[i] = 0;
                    }
                pick_e[t][s] = lane * per + at;
                pick_c[t][s] = p;
            }
            picked += __shfl(p, owner);
        }
        const float whole = renormalize ? picked : sum;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the owners' picks, read by other lanes
        if (lane < top) {
            const float c = fine ? pick_c[t][lane] / whole : __builtin_nanf("");
            const int ex = pick_e[t][lane];
            pick_c[t][lane] = c;
            atomicOr(&mask[ex][t / 32], 1u << (t % 32));
            if (ids_out) ids_out[t * top + lane] = ex;
            if (shares_out) shares_out[t * top + lane] = c;
        }
    }
    if (!plan.active) return;
    __syncthreads();
    // scan[e]: (chosen experts << 16 | rows) up to and with e
    static_assert(kMostExperts == kRouteThreads, "an expert a thread");
    const int ex = threadIdx.x;
    const int rows = __popc(mask[ex][0]) + __popc(mask[ex][1]) + __popc(mask[ex][2]) + __popc(mask[ex][3]);
    const uint32_t own = rows ? 0x10000u + (uint32_t)rows : 0u;
    uint32_t v = own;
    scan[ex] = v;
    __syncthreads();
    for (int o = 1; o < kMostExperts; o *= 2) {
        const uint32_t add = ex >= o ? scan[ex - o] : 0u;
        __syncthreads();
        v += add;
        scan[ex] = v;
        __syncthreads();
    }
    if (rows) {
        int *entry = plan.active + 1 + 3 * ((v - own) >> 16);
        entry[0] = ex;
        entry[1] = (int)((v - own) & 0xffffu);
        entry[2] = rows;
    }
    if (ex == kMostExperts - 1) plan.active[0] = (int)(v >> 16);
    for (int u = threadIdx.x; u < tokens * top; u += kRouteThreads) {
        const int t = u / top, s = u % top, pe = pick_e[t][s];
        int at = pe ? (int)(scan[pe - 1] & 0xffffu) : 0;
        for (int w = 0; w < t / 32; w++) at += __popc(mask[pe][w]);
        at += __popc(mask[pe][t / 32] & ((1u << (t % 32)) - 1u));
        plan.token[at] = t;
        plan.share[at] = pick_c[t][s];
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

constexpr int kGateWaves = 8, kDownWaves = 16;

// One workgroup: 16 columns of ff of one chosen expert, gate and up, for all
// its rows (16 MC at most). The waves split hidden (block b on wave b % 8), so
// that a wave's loads are few and all in flight; their partials are added in
// wave order. Columns past ff, up to a whole 128-block, are written as zero.
template <int MC, int XT, int HT>
__global__ __launch_bounds__(kGateWaves * 64) void moe_gate_up_kernel(const uint8_t *__restrict__ codes,
                                                                      const float *__restrict__ gs,
                                                                      const float *__restrict__ us, int tokens, int ff,
                                                                      int kbd, int kbf, int all_rows, MoePlan plan) {
    __shared__ __align__(16) float part[kGateWaves][2][256];
    const int a = blockIdx.y;
    if (a >= plan.active[0]) return;
    const int expert = plan.active[1 + 3 * a], base = plan.active[2 + 3 * a], rows = plan.active[3 + 3 * a];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int g = lane / 16, j = lane % 16, t = blockIdx.x, tiles = (ff + 15) / 16;
    const size_t hp = (size_t)kbf * 128;
    const int chunks = (rows + 15) / 16;
    if (t >= tiles) {
        for (int i = threadIdx.x; i < rows * 16; i += kGateWaves * 64)
#pragma unroll
            for (int s = 0; s < HT; s++)
                plan.h[((size_t)s * all_rows + base + i / 16) * hp + t * 16 + i % 16] = (bf16_t)0.0f;
        return;
    }
    const uint8_t *w = codes + (((size_t)expert * tiles + t) * kbd) * 4096 + lane * 16;
    const size_t srow = ((size_t)expert * ((ff + 127) / 128) + t / 8) * kbd;
    bool live[MC];
    const bf16_t *xr[MC];
#pragma unroll
    for (int c = 0; c < MC; c++) {
        const int r = 16 * c + j;
        live[c] = r < rows;
        xr[c] = plan.x + (size_t)(live[c] ? plan.token[base + r] : 0) * kbd * 128 + 16 * g;
    }
    float4_t acc[MC][2];
#pragma unroll
    for (int c = 0; c < MC; c++) acc[c][0] = acc[c][1] = float4_t{0.f, 0.f, 0.f, 0.f};
    for (int kb = wave; kb < kbd; kb += kGateWaves) {
        const uint8_t *p = w + (size_t)kb * 4096;
        MoeWide m[2];
#pragma unroll
        for (int o = 0; o < 2; o++)
            m[o] = moe_widen(__builtin_nontemporal_load((const uint4_t *)(p + o * 2048)),
                             __builtin_nontemporal_load((const uint4_t *)(p + o * 2048 + 1024)));
        const float sg = gs[srow + kb], su = us[srow + kb];
#pragma unroll
        for (int c = 0; c < MC; c++) {
            if (c >= chunks) break;
            float4_t d[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int s = 0; s < XT; s++) {
                const MoeWide x = moe_rows(xr[c] + (size_t)s * tokens * kbd * 128 + kb * 128, live[c]);
                d[0] = moe_dot(m[0], x, d[0]);
                d[1] = moe_dot(m[1], x, d[1]);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                acc[c][0][e] = __builtin_fmaf(d[0][e], sg, acc[c][0][e]);
                acc[c][1][e] = __builtin_fmaf(d[1][e], su, acc[c][1][e]);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < MC; c++) {
        if (c >= chunks) break;
        if (c) __syncthreads();
        *(float4_t *)&part[wave][0][j * 16 + 4 * g] = acc[c][0];
        *(float4_t *)&part[wave][1][j * 16 + 4 * g] = acc[c][1];
        __syncthreads();
        const int i = threadIdx.x;
        if (i < 256 && 16 * c + i / 16 < rows) {
            float gate = part[0][0][i], up = part[0][1][i];
#pragma unroll
            for (int v = 1; v < kGateWaves; v++) gate += part[v][0][i], up += part[v][1][i];
            bf16_t out[HT];
            moe_split<HT>(gate / (1.0f + expf(-gate)) * up, out);
#pragma unroll
            for (int s = 0; s < HT; s++)
                plan.h[((size_t)s * all_rows + base + 16 * c + i / 16) * hp + t * 16 + i % 16] = out[s];
        }
    }
}

// One workgroup: 16 columns of y. Units (chosen expert, 128-block of ff) in
// order, an equal run of them to each wave; a wave adds its experts' rows,
// times their shares, into its own copy of the 16 columns in LDS, and the
// copies are added in wave order.
template <int MC, int HT>
__global__ __launch_bounds__(kDownWaves * 64) void moe_down_kernel(const uint8_t *__restrict__ codes,
                                                                   const float *__restrict__ ds, int tokens, int d,
                                                                   int kbf, int all_rows, MoePlan plan,
                                                                   void *__restrict__ y, int dtype) {
    __shared__ __align__(16) float sums[kDownWaves * MC * 256];  // [waves][tokens][16]
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int g = lane / 16, j = lane % 16, t = blockIdx.x, tiles = (d + 15) / 16;
    const size_t hp = (size_t)kbf * 128;
    float *mine = sums + (size_t)wave * tokens * 16;
    for (int i = lane; i < tokens * 4; i += 64) ((float4_t *)mine)[i] = float4_t{0.f, 0.f, 0.f, 0.f};
    const int units = plan.active[0] * kbf;
    const int u0 = (int)((int64_t)units * wave / kDownWaves), u1 = (int)((int64_t)units * (wave + 1) / kDownWaves);
    for (int u = u0; u < u1;) {
        const int a = u / kbf, end = min(u1, (a + 1) * kbf);
        const int expert = plan.active[1 + 3 * a], base = plan.active[2 + 3 * a], rows = plan.active[3 + 3 * a];
        const int chunks = (rows + 15) / 16;
        const uint8_t *w = codes + ((size_t)expert * tiles + t) * kbf * 2048 + lane * 16;
        const float *sw = ds + ((size_t)expert * ((d + 127) / 128) + t / 8) * kbf;
        float4_t acc[MC];
#pragma unroll
        for (int c = 0; c < MC; c++) acc[c] = float4_t{0.f, 0.f, 0.f, 0.f};
        for (; u < end; u++) {
            const int kb = u - a * kbf;
            const MoeWide m = moe_widen(__builtin_nontemporal_load((const uint4_t *)(w + (size_t)kb * 2048)),
                                        __builtin_nontemporal_load((const uint4_t *)(w + (size_t)kb * 2048 + 1024)));
            const float s = sw[kb];
#pragma unroll
            for (int c = 0; c < MC; c++) {
                if (c >= chunks) break;
                const int r = 16 * c + j;
                float4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < HT; i++)
                    v = moe_dot(m, moe_rows(plan.h + ((size_t)i * all_rows + base + r) * hp + kb * 128 + 16 * g, r < rows), v);
#pragma unroll
                for (int e = 0; e < 4; e++) acc[c][e] = __builtin_fmaf(v[e], s, acc[c][e]);
            }
        }
#pragma unroll
        for (int c = 0; c < MC; c++) {
            const int r = 16 * c + j;
            if (c >= chunks || r >= rows) break;
            float4_t *at = (float4_t *)(mine + plan.token[base + r] * 16 + 4 * g);
            const float share = plan.share[base + r];
            float4_t v = *at;
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = __builtin_fmaf(acc[c][e], share, v[e]);
            *at = v;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * 16; i += kDownWaves * 64) {
        const int col = t * 16 + i % 16;
        if (col >= d) continue;
        float v = sums[i];
        for (int w = 1; w < kDownWaves; w++) v += sums[(size_t)w * tokens * 16 + i];
        fp8_store(y, dtype, (size_t)(i / 16) * d + col, v);
    }
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
        p.active = (int *)take((1 + 3 * (size_t)e->cfg.experts) * sizeof(int));
        p.token = (int *)take(rows * sizeof(int));
        p.share = (float *)take(rows * sizeof(float));
        p.x = (bf16_t *)take(tokens * terms_of_x(dtype) * e->kbd * 256);
        p.h = (bf16_t *)take(rows * terms_of_h(dtype) * e->kbf * 256);
    }
    if (plan) *plan = p;
    return at;
}

void launch_route(const dz_moe *e, const void *x, int dtype, int tokens, const MoePlan &plan, int *ticket, int *ids,
                  float *shares, hipStream_t s) {
    const dz_moe_config &c = e->cfg;
    const dim3 grid(cdiv(c.experts, kRouteThreads / 64), cdiv(tokens, kRouteTokens));
    const int vec = c.hidden % 8 == 0 && ((uintptr_t)x & 15) == 0;
    if (dtype == DZ_F32)
        hipLaunchKernelGGL((moe_route_kernel<float, 3>), grid, dim3(kRouteThreads), 0, s, (const float *)x, e->router,
                           tokens, c.experts, c.top_k, c.hidden, e->kbd, c.renormalize, vec, plan, ticket, ids, shares);
    else if (dtype == DZ_F16)
        hipLaunchKernelGGL((moe_route_kernel<half_t, 2>), grid, dim3(kRouteThreads), 0, s, (const half_t *)x, e->router,
                           tokens, c.experts, c.top_k, c.hidden, e->kbd, c.renormalize, vec, plan, ticket, ids, shares);
    else
        hipLaunchKernelGGL((moe_route_kernel<bf16_t, 1>), grid, dim3(kRouteThreads), 0, s, (const bf16_t *)x, e->router,
                           tokens, c.experts, c.top_k, c.hidden, e->kbd, c.renormalize, vec, plan, ticket, ids, shares);
}

template <int MC, int XT, int HT>
void launch_experts(const dz_moe *e, int dtype, int tokens, const MoePlan &plan, void *y, hipStream_t s) {
    const dz_moe_config &c = e->cfg;
    const int rows = tokens * c.top_k;
    hipLaunchKernelGGL((moe_gate_up_kernel<MC, XT, HT>), dim3(e->kbf * 8, std::min(rows, c.experts)),
                       dim3(kGateWaves * 64), 0, s, e->gate_up, e->gate_scales, e->up_scales, tokens, c.ff, e->kbd,
                       e->kbf, rows, plan);
    hipLaunchKernelGGL((moe_down_kernel<MC, HT>), dim3(cdiv(c.hidden, 16)), dim3(kDownWaves * 64), 0, s, e->down,
                       e->down_scales, tokens, c.hidden, e->kbf, rows, plan, y, dtype);
}

template <int MC>
void launch_experts_dtype(const dz_moe *e, int dtype, int tokens, const MoePlan &plan, void *y, hipStream_t s) {
    if (dtype == DZ_F32) return launch_experts<MC, 3, 3>(e, dtype, tokens, plan, y, s);
    if (dtype == DZ_F16) return launch_experts<MC, 2, 2>(e, dtype, tokens, plan, y, s);
    return launch_experts<MC, 1, 2>(e, dtype, tokens, plan, y, s);
}

void moe_release(dz_moe *e) {
    if (!e) return;
    for (void *p : {(void *)e->gate_up, (void *)e->down, (void *)e->gate_scales, (void *)e->up_scales,
                    (void *)e->down_scales, (void *)e->router})
        if (p) hipFree(p);
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
    struct {
        void **p;
        size_t bytes;
    } parts[] = {{(void **)&e->gate_up, E * ftiles * e->kbd * 4096},
                 {(void **)&e->down, E * dtiles * e->kbf * 2048},
                 {(void **)&e->gate_scales, E * blocks * sizeof(float)},
                 {(void **)&e->up_scales, E * blocks * sizeof(float)},
                 {(void **)&e->down_scales, E * blocks * sizeof(float)},
                 {(void **)&e->router, (size_t)E * e->kbd * 128 * sizeof(float)}};
    for (auto &part : parts) {
        const hipError_t err = hipMalloc(part.p, part.bytes);
        if (err != hipSuccess) {
            *part.p = nullptr;
            moe_release(e);
            return ctx_hip_fail(ctx, err, "layer allocation");
        }
        e->bytes += part.bytes;
    }
    int *bad = ctx_flag(ctx), value = 0;
    hipStream_t s = ctx_stream(ctx);
    launch_fill_i32(bad, 0, 1, s);
    for (int i = 0; i < E; i++) {
        const size_t src = (size_t)i * ff * d;
        uint8_t *gu = e->gate_up + (size_t)i * ftiles * e->kbd * 4096;
        launch_fp8_retile(gate + src, ff, d, gu, (size_t)e->kbd * 4096, 4096, bad, s);
        launch_fp8_retile(up + src, ff, d, gu + 2048, (size_t)e->kbd * 4096, 4096, bad, s);
        launch_fp8_retile(down + src, d, ff, e->down + (size_t)i * dtiles * e->kbf * 2048, (size_t)e->kbf * 2048, 2048,
                          bad, s);
    }
    launch_fp8_scales(gate_scales, e->gate_scales, E * blocks, bad, s);
    launch_fp8_scales(up_scales, e->up_scales, E * blocks, bad, s);
    launch_fp8_scales(down_scales, e->down_scales, E * blocks, bad, s);
    const int dp = e->kbd * 128;
    const dim3 grid(std::min(cdiv((size_t)E * dp, 256), 1u << 20));
    if (router_dtype == DZ_F32)
        hipLaunchKernelGGL(moe_router_kernel<float>, grid, dim3(256), 0, s, (const float *)router, E, d, dp, e->router, bad);
    else if (router_dtype == DZ_F16)
        hipLaunchKernelGGL(moe_router_kernel<half_t>, grid, dim3(256), 0, s, (const half_t *)router, E, d, dp, e->router, bad);
    else
        hipLaunchKernelGGL(moe_router_kernel<bf16_t>, grid, dim3(256), 0, s, (const bf16_t *)router, E, d, dp, e->router, bad);
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
    launch_route(e, x, dtype, (int)tokens, plan, ctx_ticket(ctx), ids, shares, ctx_stream(ctx));
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
    launch_route(e, x, dtype, (int)tokens, plan, ctx_ticket(ctx), nullptr, nullptr, s);
    const int t = (int)tokens;
    if (t <= 16) launch_experts_dtype<1>(e, dtype, t, plan, y, s);
    else if (t <= 32) launch_experts_dtype<2>(e, dtype, t, plan, y, s);
    else if (t <= 64) launch_experts_dtype<4>(e, dtype, t, plan, y, s);
    else launch_experts_dtype<8>(e, dtype, t, plan, y, s);
    return ctx_launched(ctx, "mixture of experts");
}

}  // namespace dz
