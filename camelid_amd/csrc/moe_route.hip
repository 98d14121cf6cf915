// Choice of experts with everything that routers vary: softmax or sigmoid scores, a bias that only selects (load balance), experts in
// groups of which a few are kept, top-k, weights of the chosen renormalised and scaled.
//
//   score[e]  softmax over all experts, or 1 / (1 + exp(-logit))
//   key[e]    score[e] + bias[e]; without a bias the logit itself, which orders the same and does not round
//   group     its worth is the sum of its group_top (1 or 2) best keys (without a bias, of two: of the scores); the best groups_kept stay
//   chosen    the k best keys of the groups that stay, in order; ties go to the lower index everywhere
//   weight    score / sum of the chosen scores (renormalise), times weight_scale
//
// An expert whose logit is NaN or -inf, or whose key is, takes no part; a token left with fewer than k experts has id -1 and weight 0 in the slots behind
// them (the expert lane drops such slots).  +inf counts as the largest finite logit.
//
// One wave per token, lane l holding the NE neighbouring experts from l * NE: the lowest lane of a ballot is the lowest index.
#include <type_traits>

#include "typed_rows.hpp"

#pragma clang fp contract(off)

namespace cml {

struct RouteArgs {
    const void *logits;
    const float *bias;
    int32_t *idx;
    float *weight;
    int64_t stride, n_tokens;
    int n_experts, n_groups, groups_kept, group_top, k;
    int group_size;
    int group_lanes;        // lanes that hold a group, or 0: no power of two up to 16
    uint32_t size_inverse;  // ceil(2^20 / group_size): e / group_size = e * size_inverse >> 20 for e < 1024
    int renormalise;
    float weight_scale;
};

constexpr int kOut = INT32_MIN;  // key of an expert that takes no part: below every ordered float

template <class T, bool SIGMOID, int NE>
__global__ __launch_bounds__(256) void moe_route_scored_kernel(RouteArgs a) {
    typedef typename T::Bits Bits;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    if (t >= a.n_tokens) return;  // (a wave's work is its own: no barriers)
    const Bits *lg = static_cast<const Bits *>(a.logits) + t * a.stride;
    float score[NE];
    int key[NE];
    bool in[NE];
    float most = -3.4028235e38f;
#pragma unroll
    for (int j = 0; j < NE; j++) {
        const int e = lane * NE + j;
        float v = e < a.n_experts ? load_value<T>(lg + e) : -INFINITY;
        in[j] = v > -INFINITY;  // (false for NaN)
        v = fminf(v, 3.4028235e38f);
        score[j] = v;
        if (in[j]) most = fmaxf(most, v);
    }
    float total = 1.0f;
    if constexpr (!SIGMOID) most = from_total_key(wave_allmax_i32(total_key(most)));
    float logit[NE];
#pragma unroll
    for (int j = 0; j < NE; j++) {
        logit[j] = score[j];
        if constexpr (SIGMOID) score[j] = in[j] ? 1.0f / (1.0f + expf(-logit[j])) : 0.0f;
        else score[j] = in[j] ? expf(logit[j] - most) : 0.0f;
    }
    if constexpr (!SIGMOID) {
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < NE; j++) sum = sum + score[j];
        total = wave_allsum(sum);
        if (total > 0.0f)
#pragma unroll
            for (int j = 0; j < NE; j++) score[j] = score[j] / total;
    }
    float value[NE];
#pragma unroll
    for (int j = 0; j < NE; j++) {
        const int e = lane * NE + j;
        value[j] = a.bias && in[j] ? score[j] + a.bias[e] : logit[j];
        in[j] = in[j] && value[j] > -INFINITY;
        key[j] = in[j] ? total_key(value[j] + 0.0f) : kOut;  // (-0 is 0)
    }
    if (a.n_groups > 1) {
        // A group's worth.  Its two best keys: without a bias and for two, of the scores, which order as the logits do.
        int rated[NE], worth = kOut;
#pragma unroll
        for (int j = 0; j < NE; j++) rated[j] = in[j] ? (a.bias || a.group_top == 1 ? key[j] : total_key(score[j])) : kOut;
        const auto both = [&](int first, int second) __attribute__((always_inline)) {
            if (first == kOut) return kOut;
            if (a.group_top == 1 || second == kOut) return first;
            return total_key(from_total_key(first) + from_total_key(second) + 0.0f);
        };
        unsigned long long kept = 0;
        if (a.group_lanes > 0) {
            // A group is 1, 2, 4, 8 or 16 whole lanes: two best per lane, then of pairs of lanes, of fours, ...
            int first = kOut, second = kOut;
#pragma unroll
            for (int j = 0; j < NE; j++) {
                second = max(second, min(first, rated[j]));
                first = max(first, rated[j]);
            }
            auto meet = [&](auto ctrl) __attribute__((always_inline)) {
                constexpr int kCtrl = decltype(ctrl)::value;
                const int f = __builtin_amdgcn_update_dpp(0, first, kCtrl, 0xf, 0xf, false), s = __builtin_amdgcn_update_dpp(0, second, kCtrl, 0xf, 0xf, false);
                second = max(min(first, f), max(second, s));
                first = max(first, f);
            };
            if (a.group_lanes >= 2) meet(std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
            if (a.group_lanes >= 4) meet(std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
            if (a.group_lanes >= 8) meet(std::integral_constant<int, 0x141>{});  // row_half_mirror: the other quad
            if (a.group_lanes >= 16) meet(std::integral_constant<int, 0x140>{}); // row_mirror: the other eight
            worth = both(first, second);
            // it stays if fewer than groups_kept are ahead of it
            const int mine = lane / a.group_lanes;
            int ahead = 0;
            for (int g = 0; g < a.n_groups; g++) {
                const int theirs = __builtin_amdgcn_readlane(worth, g * a.group_lanes);
                ahead += (theirs > worth) | ((theirs == worth) & (g < mine));
            }
            if (ahead >= a.groups_kept)
#pragma unroll
                for (int j = 0; j < NE; j++) key[j] = kOut;
        } else {
            // any size: the groups one after the other, each lane's experts of that group against the wave
            for (int g = 0; g < a.n_groups; g++) {
                int best[2] = {kOut, kOut}, taken = -1;
#pragma unroll 1
                for (int s = 0; s < a.group_top; s++) {
                    int most = kOut, at = -1;
#pragma unroll
                    for (int j = NE - 1; j >= 0; j--) {
                        const int e = lane * NE + j;
                        if (static_cast<int>(e * a.size_inverse >> 20) == g && e != taken && rated[j] >= most) {
                            most = rated[j];
                            at = e;
                        }
                    }
                    const int m = wave_allmax_i32(most);
                    if (m == kOut) break;
                    taken = __builtin_amdgcn_readlane(at, __builtin_ctzll(__builtin_amdgcn_ballot_w64(most == m)));
                    best[s] = m;
                }
                if (lane == g) worth = both(best[0], best[1]);
            }
            for (int s = 0; s < a.groups_kept; s++) {
                const int m = wave_allmax_i32(worth);
                if (m == kOut) break;
                const int g = __builtin_ctzll(__builtin_amdgcn_ballot_w64(worth == m));
                kept |= 1ull << g;
                if (lane == g) worth = kOut;
            }
#pragma unroll
            for (int j = 0; j < NE; j++)
                if (!(kept >> ((lane * NE + j) * a.size_inverse >> 20 & 63) & 1)) key[j] = kOut;
        }
    }
    int chosen = -1;  // lane s: slot s
    for (int s = 0; s < a.k; s++) {
        int best = key[NE - 1], at = NE - 1;
#pragma unroll
        for (int j = NE - 2; j >= 0; j--) {
            at = key[j] >= best ? j : at;
            best = max(best, key[j]);
        }
        const int m = wave_allmax_i32(best);
        if (m == kOut) break;
        const int e = __builtin_amdgcn_readlane(lane * NE + at, __builtin_ctzll(__builtin_amdgcn_ballot_w64(best == m)));
#pragma unroll
        for (int j = 0; j < NE; j++) key[j] = e == lane * NE + j ? kOut : key[j];
        chosen = lane == s ? e : chosen;
    }
    // the chosen experts' scores, from the lanes that hold them
    float w = 0.0f;
#pragma unroll
    for (int j = 0; j < NE; j++) {
        const float theirs = __shfl(score[j], (chosen < 0 ? 0 : chosen) / NE);
        w = chosen >= 0 && chosen % NE == j ? theirs : w;
    }
    if (a.renormalise) {
        const float sum = wave_allsum(w);
        const int live = __builtin_popcountll(__builtin_amdgcn_ballot_w64(chosen >= 0));
        w = sum > 0.0f ? w / sum : chosen >= 0 ? 1.0f / static_cast<float>(live) : 0.0f;  // (all chosen scores 0: alike)
    }
    if (lane < a.k) {
        a.idx[t * a.k + lane] = chosen;
        a.weight[t * a.k + lane] = w * a.weight_scale;
    }
}

template <class T, bool SIGMOID, int NE>
static int launch_route_lanes(RouteArgs a, hipStream_t st) {
    const int lanes = a.group_size % NE == 0 ? a.group_size / NE : 0;
    a.group_lanes = lanes <= 16 && (lanes & (lanes - 1)) == 0 ? lanes : 0;
    hipLaunchKernelGGL((moe_route_scored_kernel<T, SIGMOID, NE>), dim3(static_cast<unsigned>((a.n_tokens + 3) / 4)), dim3(256), 0, st, a);
    CML_HIP_TRY(hipGetLastError());
    return CML_OK;
}
template <class T, bool SIGMOID>
static int launch_route(const RouteArgs &a, hipStream_t st) {
    if (a.n_experts <= 64) return launch_route_lanes<T, SIGMOID, 1>(a, st);
    if (a.n_experts <= 128) return launch_route_lanes<T, SIGMOID, 2>(a, st);
    if (a.n_experts <= 256) return launch_route_lanes<T, SIGMOID, 4>(a, st);
    if (a.n_experts <= 512) return launch_route_lanes<T, SIGMOID, 8>(a, st);
    return launch_route_lanes<T, SIGMOID, 16>(a, st);
}

int launch_moe_route_scored(int score, int dtype, const void *logits, int64_t stride, const float *bias, int64_t n_tokens, int n_experts, int n_groups, int groups_kept, int group_top, int k,
                            int renormalise, float weight_scale, int32_t *idx, float *weight, hipStream_t st) {
    const int size = n_experts / n_groups;
    const RouteArgs a{logits, bias, idx, weight, stride, n_tokens, n_experts, n_groups, groups_kept, group_top, k, size, 0, ((1u << 20) + size - 1) / size, renormalise, weight_scale};
    CML_COUNT_LAUNCH("moe.route.scored");
    return with_type(dtype, [&](auto t) { return score == CML_ROUTE_SIGMOID ? launch_route<decltype(t), true>(a, st) : launch_route<decltype(t), false>(a, st); });
}

}  // namespace cml
