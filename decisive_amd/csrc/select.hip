// select.hip -- the choice of a token's experts from its logits (the rule is
// dz_moe_select's in the header).
//
// Scores that lie next to each other are no rarity among many tokens: two f32
// evaluations of one rule disagree on some token's order in 10^4. The choice is
// made in 64 bits, where they do not.
#include "../../include/decisive_rocm.h"
#include "fp8.hpp"

namespace dz {

int32_t ctx_fail(dz_ctx *ctx, int32_t code, const std::string &msg);
hipStream_t ctx_stream(dz_ctx *ctx);
int32_t ctx_launched(dz_ctx *ctx, const char *what);

namespace {

constexpr int kMostExperts = 512, kMostTop = 16, kMostGroups = 64;
constexpr double kNothing = -__builtin_huge_val();

__device__ __forceinline__ double select_wave_max(double v) {
    for (int o = 32; o; o >>= 1) v = fmax(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ double select_wave_sum(double v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// One wave a token; lane l holds the experts PER l .. PER l + PER - 1, so that the
// first lane with the largest score has the lowest index.
template <class T, int PER>
__global__ __launch_bounds__(64) void select_kernel(const T *__restrict__ logits, const float *__restrict__ bias,
                                                    dz_moe_selection rule, int *__restrict__ ids,
                                                    float *__restrict__ shares) {
    const int lane = threadIdx.x, experts = rule.experts, top = rule.top_k;
    const size_t token = blockIdx.x;
    double s[PER], c[PER], most = kNothing;
    bool wrong = false;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = lane * PER + i;
        s[i] = e < experts ? (double)(float)logits[token * experts + e] : kNothing;
        wrong |= !(s[i] < __builtin_huge_val());
        most = fmax(most, s[i]);
    }
    if (rule.sigmoid) {
#pragma unroll
        for (int i = 0; i < PER; i++) c[i] = s[i], s[i] = 1.0 / (1.0 + exp(-s[i]));
    } else {
        most = select_wave_max(most);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            c[i] = s[i];
            s[i] = s[i] > kNothing ? exp(s[i] - most) : 0.0;
            sum += s[i];
        }
        sum = select_wave_sum(sum);
#pragma unroll
        for (int i = 0; i < PER; i++) s[i] = sum > 0.0 ? s[i] / sum : 0.0;
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = lane * PER + i;
        if (c[i] > kNothing) c[i] = bias ? s[i] + (double)bias[e] : s[i];
        wrong |= !(c[i] < __builtin_huge_val());
    }
    wrong = __any(wrong);

    // an expert may be chosen once, and only in a group that stays
    uint32_t open = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) open |= (uint32_t)(lane * PER + i < experts) << i;
    if (rule.top_groups < rule.groups) {
        const int width = experts / rule.groups;
        double score = kNothing;  // lane g: group g's
        for (int g = 0; g < rule.groups; g++) {
            double first = kNothing, second = kNothing;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int e = lane * PER + i;
                if (e < g * width || e >= (g + 1) * width) continue;
                second = fmax(second, fmin(first, c[i]));
                first = fmax(first, c[i]);
            }
            for (int o = 32; o; o >>= 1) {
                const double f = __shfl_xor(first, o), t = __shfl_xor(second, o);
                second = fmax(fmax(second, t), fmin(first, f));
                first = fmax(first, f);
            }
            if (lane == g) score = rule.group_best == 2 && second > kNothing ? first + second : first;
        }
        int rank = 0;
        for (int g = 0; g < rule.groups; g++) {
            const double other = __shfl(score, g);
            rank += other > score || (other == score && g < lane);
        }
        const unsigned long long stays = __ballot(lane < rule.groups && rank < rule.top_groups);
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int e = lane * PER + i;
            if (e < experts && !(stays >> (e / width) & 1)) open &= ~(1u << i);
        }
    }

    int expert = 0;
    double share = 0.0, whole = 0.0;
    for (int k = 0; k < top; k++) {
        double best = kNothing, mine = 0.0;
        int at = -1;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if ((open >> i & 1) && (at < 0 || c[i] > best)) best = c[i], mine = s[i], at = i;
        const double largest = select_wave_max(best);
        const unsigned long long owners = __ballot(at >= 0 && best == largest);
        const int owner = owners ? __ffsll(owners) - 1 : 0;
        const double value = __shfl(mine, owner);
        const int e = owner * PER + __shfl(at, owner);
        if (lane == owner) open &= ~(1u << at);
        whole += value;
        if (lane == k) expert = e, share = value;
    }
    if (lane >= top) return;
    if (wrong) expert = lane;
    if (rule.renormalize) share = whole > 0.0 ? share / whole : 0.0;
    ids[token * top + lane] = expert;
    shares[token * top + lane] = wrong ? __builtin_nanf("") : (float)(share * (double)rule.scale);
}

template <class T>
void launch_select(const dz_moe_selection &rule, const T *logits, const float *bias, size_t tokens, int *ids,
                   float *shares, hipStream_t s) {
    const dim3 grid((unsigned)tokens), block(64);
    if (rule.experts <= 64) hipLaunchKernelGGL((select_kernel<T, 1>), grid, block, 0, s, logits, bias, rule, ids, shares);
    else if (rule.experts <= 128) hipLaunchKernelGGL((select_kernel<T, 2>), grid, block, 0, s, logits, bias, rule, ids, shares);
    else if (rule.experts <= 256) hipLaunchKernelGGL((select_kernel<T, 4>), grid, block, 0, s, logits, bias, rule, ids, shares);
    else hipLaunchKernelGGL((select_kernel<T, 8>), grid, block, 0, s, logits, bias, rule, ids, shares);
}

bool flag(int32_t v) { return v == 0 || v == 1; }

}  // namespace

int32_t moe_select(dz_ctx *ctx, const dz_moe_selection *rule, const void *logits, int32_t dtype, size_t tokens,
                   const float *bias, int32_t *ids, float *shares) {
    if (!rule || (tokens && (!logits || !ids || !shares))) return ctx_fail(ctx, DZ_INVALID_REQUEST, "null pointer");
    if (dtype != DZ_F32 && dtype != DZ_F16 && dtype != DZ_BF16)
        return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "unknown dtype");
    const dz_moe_selection &r = *rule;
    if (r.experts < 1 || r.experts > kMostExperts || r.groups < 1 || r.groups > kMostGroups ||
        r.experts % r.groups != 0 || r.top_groups < 1 || r.top_groups > r.groups || r.top_k < 1 ||
        r.top_k > kMostTop || r.top_k > r.experts / r.groups * r.top_groups || r.group_best < 1 || r.group_best > 2 ||
        !flag(r.sigmoid) || !flag(r.renormalize) || !(r.scale >= -3.4028235e38f && r.scale <= 3.4028235e38f))
        return ctx_fail(ctx, DZ_INVALID_PARAMETERS, "invalid choice of experts");
    if (tokens > kFp8MostRows) return ctx_fail(ctx, DZ_INPUT_TOO_LONG, "input budget exceeded");
    if (tokens == 0) return DZ_OK;
    hipStream_t s = ctx_stream(ctx);
    if (dtype == DZ_F32) launch_select(r, (const float *)logits, bias, tokens, ids, shares, s);
    else if (dtype == DZ_F16) launch_select(r, (const half_t *)logits, bias, tokens, ids, shares, s);
    else launch_select(r, (const bf16_t *)logits, bias, tokens, ids, shares, s);
    return ctx_launched(ctx, "choice of experts");
}

}  // namespace dz
