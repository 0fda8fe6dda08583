// select.hip -- the choice of a token's experts from its logits (the rule is
// dz_moe_select's in the header).
//
// Scores that lie next to each other are no rarity among many tokens: two f32
// evaluations of one rule disagree on some token's order in 10^4. The choice is
// therefore the one that 64 bits make, but few experts need them:
//  - without a bias the scores order as their logits do, which are exact, but where 64
//    bits cannot tell scores of different logits apart: those that are 0 count as one
//    logit, and a row with others (a sigmoid's logit above 16 or just above those, a
//    softmax's 700 to 746 below the largest or any where that is past 2^22, one so near 0
//    that its neighbours in f32 lie within 2^-50 of it) is chosen by scores;
//  - with one, f32 scores (6 2^-24 off at most) leave the experts that may be among the
//    largest, some 11 of 256 for eight of them, and 64 bits order those;
//  - groups are ranked in f32, and again in 64 bits only where one that stays lies
//    within 2^-18 (of the largest summand, where that is above 1) of one that does not.
// What those tests do not cover (masked experts that have to be chosen, more candidates
// than kMostCandidates) goes through 64 bits expert by expert.
//
// A token takes 16 lanes, a DPP row, and lane j the experts j, j + 16, ..., so that the
// groups that stay are spread over the lanes. The k-th largest of the lanes' largest
// scores is below the k-th largest of all: candidates are at or above it.
//
// Bound by the vector unit's issue, some 1300 instructions a wave of four tokens with
// their 64-bit ones, and by the chain of one wave (us, 256 experts, f32, eight by biased
// sigmoids in 4 of 8 groups: 16384 tokens 16.8, of which groups 4.4 and the bias 1.0 (its
// 64-bit scores); 8 of 64 8.4, 16 of 512 27.8; the logits' bytes alone would take 3.4). A
// few tokens are a launch and that chain: 8.9, without groups and bias 5.5, of 64 4.1.
// Where 64 bits choose all of a row the values decide the time (16384 tokens; one): plain
// softmax 11.7; 5.5, of equal logits, of masks that leave fewer than eight or of logits
// past 2^22 24-25; 13-14. Unbiased sigmoids in groups 15.5; 7.6, with a logit above 16 in
// each row 38; 18. Biased sigmoids in groups 18; 9.0, with biases near 1000 26; 15.
#include "../../include/decisive_rocm.h"
#include "fp8.hpp"
#include "tiles.hpp"

namespace dz {

int32_t ctx_fail(dz_ctx *ctx, int32_t code, const std::string &msg);
hipStream_t ctx_stream(dz_ctx *ctx);
int32_t ctx_launched(dz_ctx *ctx, const char *what);

namespace {

constexpr int kMostExperts = 512, kMostTop = 16, kMostGroups = 64, kMostCandidates = 32, kSelectWaves = 4;
constexpr float kMasked = -__builtin_huge_valf();

// Over the 16 lanes of a row, in every lane and in one order for all of them (rotations would give each lane a sum of
// its own, and equal logits unequal scores): quads by xor 1 and xor 2, their halves and the row by mirroring.
#define DZ_ROW_REDUCE(name, type, move, combine)        \
    __device__ __forceinline__ type name(type v) {      \
        type o = move<0xB1>(v);                         \
        v = combine;                                    \
        o = move<0x4E>(v);                              \
        v = combine;                                    \
        o = move<0x141>(v);                             \
        v = combine;                                    \
        o = move<0x140>(v);                             \
        return combine;                                 \
    }
template <int CTRL>
__device__ __forceinline__ int dpp_move_i32(int v) {
    return __builtin_amdgcn_mov_dpp(v, CTRL, 0xF, 0xF, true);
}
DZ_ROW_REDUCE(row_max_f32, float, dpp_move_f32, fmaxf(v, o))
DZ_ROW_REDUCE(row_max_f64, double, dpp_move_f64, fmax(v, o))
DZ_ROW_REDUCE(row_sum_f64, double, dpp_move_f64, v + o)
DZ_ROW_REDUCE(row_sum_i32, int, dpp_move_i32, v + o)
DZ_ROW_REDUCE(row_min_i32, int, dpp_move_i32, v < o ? v : o)
#undef DZ_ROW_REDUCE
// Of a row's other lanes those whose `of` is at least v: all rotations of the row from O on.
template <int O>
__device__ __forceinline__ int row_not_below(float of, float v) {
    if constexpr (O == 16) return 0;
    else return (dpp_move_f32<0x120 + O>(of) >= v) + row_not_below<O + 1>(of, v);
}

// What a row's scores come from.
struct Scores {
    float most;   // the largest logit
    double sum;   // of exp(logit - most), or 1 where only ratios count
    bool sigmoid;

    __device__ __forceinline__ double of(float l) const {
        if (sigmoid) return 1.0 / (1.0 + exp(-(double)l));
        return l > kMasked ? exp((double)l - (double)most) / sum : 0.0;
    }
    // The same in f32, 6 u off at most, u = 2^-24: the exponent x log2 e, off by 2.3 |x| u (l - most, the product, the
    // constant), costs 2.3 |x| e^-|x| u < 0.9 u (a sigmoid less); the unit's 2^x and 1 / x 2 u each of a value up to 1, the
    // sum in f32, its quotient and the product with it u each: a softmax 0.9 + 2 + 3, a sigmoid 0.3 + 0.5 + 1 + 2.
    // Measured over 2^28 logits each: 1.5 u and 1.8 u.
    __device__ __forceinline__ float near(float l, float over_sum) const {
        constexpr float kLog2e = 1.44269504f;
        if (sigmoid) return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-l * kLog2e));
        return __builtin_amdgcn_exp2f((l - most) * kLog2e) * over_sum;  // 0 for a masked logit
    }
};

// A row's choice one expert after the other, in 64 bits: lane i < top is left with the
// i-th. `logits` of the row in LDS; bias may be null; bit i of `open`: expert 16 i + j
// may be chosen.
template <int PER>
__device__ __attribute__((noinline)) int select_wide(const float *logits, const float *__restrict__ bias, uint32_t open,
                                                     int top, Scores scores) {
    const int j = threadIdx.x % 16;
    double c[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        c[i] = (double)logits[16 * i + j];
        if ((open >> i & 1) && c[i] > (double)kMasked)
            c[i] = scores.of(logits[16 * i + j]) + (bias ? (double)bias[16 * i + j] : 0.0);
    }
    int mine = 0;
    for (int k = 0; k < top; k++) {
        double best = 0.0;
        int at = kMostExperts;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const bool better = (open >> i & 1) && (at == kMostExperts || c[i] > best);
            best = better ? c[i] : best;
            at = better ? 16 * i + j : at;
        }
        best = at == kMostExperts ? (double)kMasked : best;
        const double largest = row_max_f64(best);
        const int e = row_min_i32(best == largest ? at : kMostExperts) % kMostExperts;
        if (e % 16 == j) open &= ~(1u << (e / 16));
        if (j == k) mine = e;
    }
    return mine;
}

// Which groups stay, as bits, from the values of their experts (`value`, of type V): a group ranks by its largest one
// or by `score` of its two largest added. Also the least rank that stays, the largest that does not, and the largest
// size of a lane's summands, which may cancel. 16 / groups lanes take a group, or a lane several groups.
template <class V, class F, class G>
__device__ __forceinline__ uint64_t select_groups(const dz_moe_selection &rule, V *ranks, F value, G score,
                                                  V &least_kept, V &most_left, V &summand) {
    const int j = threadIdx.x % 16, width = rule.experts / rule.groups;
    const V nothing = -(V)__builtin_huge_val();
    summand = 0;
    int parts = 1;
    while (parts * 2 * rule.groups <= 16) parts *= 2;
    for (int g = j / parts; g < rule.groups; g += 16 / parts) {
        V first = nothing, second = nothing;
#pragma unroll 4
        for (int e = g * width + j % parts; e < (g + 1) * width; e += parts) {
            const V v = value(e);
            second = max(second, min(first, v));
            first = max(first, v);
        }
        for (int o = 1; o < parts; o *= 2) {
            const V f = __shfl_xor(first, o, 16), s = __shfl_xor(second, o, 16);
            second = max(max(second, s), min(first, f));
            first = max(first, f);
        }
        if (rule.group_best == 2 && first > nothing) {
            const V other = second > nothing ? score(second) : (V)0;
            first = score(first);
            summand = max(summand, max(first, -other));  // the lower one is the larger if it is below 0
            first += other;
        }
        if (j % parts == 0) ranks[g] = first;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    uint64_t stays = 0;
    least_kept = -nothing;
    most_left = nothing;
    for (int g = j; g < (rule.groups + 15) / 16 * 16; g += 16) {
        const V mine = ranks[g < rule.groups ? g : 0];
        int above = 0;
#pragma unroll 4
        for (int o = 0; o < rule.groups; o++) {
            const V other = ranks[o];
            above += other > mine || (other == mine && o < g);
        }
        const bool kept = g < rule.groups && above < rule.top_groups;
        if (kept) least_kept = min(least_kept, mine);
        else if (g < rule.groups) most_left = max(most_left, mine);
        stays |= (__ballot(kept) >> (threadIdx.x % 64 / 16 * 16) & 0xffff) << (g - j);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // read before the ranks are written again
    return stays;
}

// Where LDS keeps expert e, so that lanes that walk groups of 32 meet distinct banks.
__device__ __forceinline__ int select_at(int e) { return e + e / 32; }

template <class T, int PER, bool BIASED>
__global__ __launch_bounds__(kSelectWaves * 64) void select_kernel(const T *__restrict__ logits,
                                                                   const float *__restrict__ bias,
                                                                   dz_moe_selection rule, int tokens,
                                                                   int *__restrict__ ids, float *__restrict__ shares) {
    // A row's part of LDS: sixteen of 256 experts fit four times, so that 16384 tokens are under way at once.
    struct Row {
        union {
            double wide_rank[kMostGroups];               // where the f32 ranks are too near each other
            float key[PER * 16 + (PER * 16 + 31) / 32];  // for the groups
        };
        float logit[PER * 16];
        union {
            float rank[kMostGroups];
            struct {
                union {
                    double value[kMostCandidates];  // what candidates are ordered by
                    double share[kMostTop];         // the chosen ones' scores, once they are ordered
                };
                int expert[kMostCandidates];
            };
        };
    };
    __shared__ Row s_row[kSelectWaves * 4];
    const int row = threadIdx.x / 16, j = threadIdx.x % 16, experts = rule.experts, top = rule.top_k;
    const int token = blockIdx.x * (kSelectWaves * 4) + row;
    const T *from = logits + (size_t)min(token, tokens - 1) * experts;  // rows past the last one choose for it again
    Row &at_row = s_row[row];
    float *own = at_row.logit, *keys = at_row.key;

    float key[PER], most = kMasked;
    int wrong = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) key[i] = 16 * i + j < experts ? (float)from[16 * i + j] : kMasked;
#pragma unroll
    for (int i = 0; i < PER; i++) {
        wrong |= !(key[i] < __builtin_huge_valf());
        most = fmaxf(most, key[i]);
        own[16 * i + j] = key[i];
    }
    Scores scores{row_max_f32(most), 1.0, rule.sigmoid != 0};
    float over_sum = 1.0f;
    if (!rule.sigmoid && (BIASED || !rule.renormalize)) {
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < PER; i++) sum += key[i] > kMasked ? exp((double)key[i] - (double)scores.most) : 0.0;
        sum = row_sum_f64(sum);
        scores.sum = sum > 0.0 ? sum : 1.0;
        over_sum = 1.0f / (float)scores.sum;
    }
    if constexpr (BIASED) {
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const float b = 16 * i + j < experts ? bias[16 * i + j] : 0.0f;
            wrong |= key[i] > kMasked && !(b < __builtin_huge_valf());
            key[i] = key[i] > kMasked ? scores.near(key[i], over_sum) + b : kMasked;
        }
    }
    wrong = row_sum_i32(wrong);
    bool odd = false;  // scores of different logits may be equal
    if constexpr (!BIASED) {
        // below 2^22 `zero` is rounded by 2^-2 at most and lies under 745.14, where 64 bits make exp 0; from 2^25 on it does
        // not always
        odd = !rule.sigmoid && !(fabsf(scores.most) < 0x1p22f);
        const float zero = rule.sigmoid ? -709.79f : scores.most - 746.0f;  // at and below it a score is 0
        // up to `low` some are: exp passes 64 bits' range at 709.7827, short of a sigmoid's `zero`
        const float high = rule.sigmoid ? 16.0f : __builtin_huge_valf(), low = rule.sigmoid ? -709.0f : scores.most - 700.0f;
        // neighbours lie 2^-24 of their size apart, and exp's argument is rounded by 2^-53 of the largest logit's
        const float tiny = 0x1p-26f * fmaxf(1.0f, fabsf(scores.most));
        float least = __builtin_huge_valf();
        uint32_t nearest = ~0u;  // of the keys' sizes as bits, 0 the last of all
#pragma unroll
        for (int i = 0; i < PER; i++) {
            least = fminf(least, 16 * i + j < experts ? key[i] : least);
            const uint32_t size = (__builtin_bit_cast(uint32_t, key[i]) << 1) - 1;
            nearest = size < nearest ? size : nearest;
        }
        const bool look = least < low || nearest < __builtin_bit_cast(uint32_t, tiny) << 1;
        if (scores.most > high || row_sum_i32(look)) {  // masks, logits far apart, above 16 or next to 0
            int odds = 0;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const bool here = key[i] > kMasked;
                odds |= here && (key[i] > high || (key[i] > zero && key[i] < low) ||
                                 (fabsf(key[i]) < tiny && key[i] != 0.0f));
                key[i] = here ? fmaxf(key[i], zero) : kMasked;
            }
            odd |= row_sum_i32(odds) != 0;
        }
    }
    // Of values up to 1; of larger ones, S, their share. A key is 6 u and its sum's rounding, u S, off (u = 2^-24), two
    // keys 14 u S where 64 u S are allowed.
    const float tol = BIASED ? 0x1p-18f : 0.0f;

    uint32_t open = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) open |= (uint32_t)(16 * i + j < experts) << i;
    if (rule.top_groups < rule.groups) {
#pragma unroll
        for (int i = 0; i < PER; i++) keys[select_at(16 * i + j)] = key[i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        float kept, left, summand;
        uint64_t stays = select_groups<float>(
            rule, at_row.rank, [&](int e) { return keys[select_at(e)]; },
            [&](float v) { return BIASED ? v : scores.near(v, over_sum); }, kept, left, summand);
        if (BIASED || odd || rule.group_best == 2) {
            kept = -row_max_f32(-kept);
            left = row_max_f32(left);
            summand = fmaxf(1.0f, BIASED ? row_max_f32(summand) : 1.0f);
            // two keys added are 14 u S and 2 u S for the addition off, two such ranks 32 u S: half of what is allowed
            if (odd || !(kept - left > 0x1p-18f * fmaxf(summand, fabsf(kept)))) {
                double wide_kept, wide_left, wide_summand;
                stays = select_groups<double>(
                    rule, at_row.wide_rank,
                    [&](int e) {
                        const float l = own[e];
                        return l > kMasked ? scores.of(l) + (BIASED ? (double)bias[e] : 0.0) : (double)kMasked;
                    },
                    [&](double v) { return v; }, wide_kept, wide_left, wide_summand);
            }
        }
        const int width = experts / rule.groups;
        if (width % 16 == 0) {  // a group is whole steps of 16 experts, the same for all lanes
            int g = 0, at = 0;
#pragma unroll
            for (int i = 0; i < PER; i++) {
                if (!((uint32_t)stays & 1u << g)) key[i] = kMasked, open &= ~(1u << i);  // 32 groups at most
                at += 16;
                if (at == width) at = 0, g++;
            }
        } else {
            int g = j / width, at = j - g * width;  // of expert 16 i + j
#pragma unroll
            for (int i = 0; i < PER; i++) {
                if (!(stays >> (g & 63) & 1)) key[i] = kMasked, open &= ~(1u << i);
                at += 16;
                while (at >= width) at -= width, g++;
            }
        }
    }

    // the lanes' largest keys, and the top-th largest of them
    float mine = kMasked;
#pragma unroll
    for (int i = 0; i < PER; i++) mine = fmaxf(mine, key[i]);
    float line;
    if (top <= 8) {
        line = row_max_f32(1 + row_not_below<1>(mine, mine) >= top ? mine : kMasked);
    } else {  // the lanes' two largest: one of each would let too many pass
        float first = kMasked, next = kMasked;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            next = fmaxf(next, fminf(first, key[i]));
            first = fmaxf(first, key[i]);
        }
        const int of_mine = 1 + (next >= mine) + row_not_below<1>(mine, mine) + row_not_below<1>(next, mine);
        const int of_next = 2 + row_not_below<1>(mine, next) + row_not_below<1>(next, next);
        line = row_max_f32(of_mine >= top ? mine : of_next >= top ? next : kMasked);
    }
    const float least = line - tol * fmaxf(1.0f, fabsf(line));
    int count = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) count += key[i] >= least;  // a line of nothing counts all, and is not sure
    const int total = row_sum_i32(count);
    const bool sure = !odd && line > kMasked && total <= kMostCandidates;
    int expert = 0;
    if (wrong) {
        expert = j;
    } else if (sure) {
        int slot = count;  // the candidates of the lanes before this one
#pragma unroll
        for (int o = 1; o < 16; o *= 2) {
            const int before = __shfl_up(slot, o, 16);
            slot += j >= o ? before : 0;
        }
        slot -= count;
#pragma unroll
        for (int i = 0; i < PER; i++)
            if (key[i] >= least) {
                at_row.expert[slot] = 16 * i + j;
                if (!BIASED) at_row.value[slot] = (double)key[i];
                slot++;
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        // each candidate's place by counting those before it
        int place[2], named[2];
        double share_of[2];
        if constexpr (BIASED) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int c = j + 16 * h;
                if (c >= total) continue;
                const int e = at_row.expert[c];
                share_of[h] = scores.of(own[e]);
                at_row.value[c] = share_of[h] + (double)bias[e];
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int c = j + 16 * h;
            place[h] = kMostTop;
            named[h] = 0;
            if (c >= total) continue;
            const double v = at_row.value[c];
            const int e = at_row.expert[c];
            int before = 0;
            for (int o0 = 0; o0 < total; o0 += 4) {
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int o = (o0 + u) % kMostCandidates;
                    const double other = at_row.value[o];
                    before += o0 + u < total && (other > v || (other == v && at_row.expert[o] < e));
                }
            }
            place[h] = before;
            named[h] = e;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // read before the places are written
#pragma unroll
        for (int h = 0; h < 2; h++)
            if (place[h] < top) {
                at_row.expert[place[h]] = named[h];
                if (BIASED) at_row.share[place[h]] = share_of[h];
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        expert = at_row.expert[j];
    } else {
        expert = select_wide<PER>(own, BIASED ? bias : nullptr, open, top, scores);
    }

    double share = 0.0;
    if (j < top && !wrong) share = BIASED && sure ? at_row.share[j] : scores.of(own[expert]);
    if (rule.renormalize) {
        const double whole = row_sum_f64(share);
        share = whole > 0.0 ? share / whole : 0.0;
    }
    if (j >= top || token >= tokens) return;
    ids[(size_t)token * top + j] = expert;
    shares[(size_t)token * top + j] = wrong ? __builtin_nanf("") : (float)(share * (double)rule.scale);
}

template <class T, int PER>
void launch_select_form(const dz_moe_selection &rule, const T *logits, const float *bias, int tokens, int *ids,
                        float *shares, hipStream_t s) {
    const dim3 grid(cdiv(tokens, kSelectWaves * 4)), block(kSelectWaves * 64);
    if (bias) hipLaunchKernelGGL((select_kernel<T, PER, true>), grid, block, 0, s, logits, bias, rule, tokens, ids, shares);
    else hipLaunchKernelGGL((select_kernel<T, PER, false>), grid, block, 0, s, logits, bias, rule, tokens, ids, shares);
}

template <class T>
void launch_select(const dz_moe_selection &rule, const T *logits, const float *bias, int tokens, int *ids,
                   float *shares, hipStream_t s) {
    if (rule.experts <= 64) launch_select_form<T, 4>(rule, logits, bias, tokens, ids, shares, s);
    else if (rule.experts <= 128) launch_select_form<T, 8>(rule, logits, bias, tokens, ids, shares, s);
    else if (rule.experts <= 256) launch_select_form<T, 16>(rule, logits, bias, tokens, ids, shares, s);
    else launch_select_form<T, 32>(rule, logits, bias, tokens, ids, shares, s);
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
    const int n = (int)tokens;
    if (dtype == DZ_F32) launch_select(r, (const float *)logits, bias, n, ids, shares, s);
    else if (dtype == DZ_F16) launch_select(r, (const half_t *)logits, bias, n, ids, shares, s);
    else launch_select(r, (const bf16_t *)logits, bias, n, ids, shares, s);
    return ctx_launched(ctx, "choice of experts");
}

}  // namespace dz
